"""The operators of a step of many requests: their latent caches in pages, the
attention that reads them, and what is told of the tokens they come to.

A key of the compressed cache is a latent row (the value too) and a rope row.
A batch is a list of sequences, each with the pages that hold its keys, its
length, and its newest rows, which are its last keys.  A case is a dict of plain
values; `kind` names the operator:

  append   norm of the new latent rows, rotation by position of the new rope rows
           and of the queries, and their place in the pages (mlk_latent_append);
           what 4 bits hold is read back by mlk_latent_gather
  gather   cached rows as values (mlk_latent_gather)
  attend   each row's attention over its sequence's keys (mlk_latent_attend)
  logprobs log probability of a given token, entropy and the most likely tokens
           (mlk_token_logprobs)

`type` is the type of rows, queries and results: f32 or bf16; `cache` that of the
latent values in the pages: bf16, or fp4 (e2m1 codes, a power of two for each 32).
"""
import torch

own = False

LATENT, ROPE, HEADS, NOPE, VOCAB, THETA, EPS = 512, 64, 16, 128, 163840, 50000.0, 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP, LEAST, HUGE = 32, -100, 2.0 ** 127  # of an fp4 scale
WORKSPACE = 64 << 20
MOST_BYTES, MOST_FLOPS = 310e6, 80e9


def listed():
    def batch(name, kind, type, cache, seqs, shortest, longest, new=1, page=64, heads=HEADS):
        return dict(name=name, kind=kind, type=type, cache=cache, seqs=seqs, shortest=shortest,
                    longest=longest, new=new, page=page, heads=heads, latent=LATENT, rope=ROPE)

    return [
        # one decoded token of one request: the smallest call
        batch("append_f32_1", "append", "f32", "bf16", 1, 1000, 1000),
        # chunks of 8 prompts, 4095 new rows in all, that go to 4 bits
        batch("append_fp4_4095", "append", "bf16", "fp4", 8, 512, 4096, new=910),
        # a request's prefix read back for an attention on expanded heads
        batch("gather_fp4_8192", "gather", "bf16", "fp4", 1, 8192, 8192),
        # ragged prefixes of several requests
        batch("gather_f32_ragged", "gather", "f32", "bf16", 13, 0, 3001, page=16),
        # one request's next token
        batch("attend_bf16_1", "attend", "bf16", "bf16", 1, 4096, 4096),
        # a serving batch, the cache held in 4 bits
        batch("attend_fp4_64", "attend", "bf16", "fp4", 64, 4096, 8192),
        # a smaller one of mixed lengths beside f32 projections
        batch("attend_f32_fp4_17", "attend", "f32", "fp4", 17, 1, 4099, page=16),
        # long contexts
        batch("attend_bf16_16x16384", "attend", "bf16", "bf16", 16, 16000, 16384, page=128),
        # chunks of prompts behind what is cached of them
        batch("attend_chunk", "attend", "bf16", "bf16", 4, 3000, 4096, new=128),
        # one decoded token and its alternatives
        dict(name="logprobs_f32_1", kind="logprobs", type="f32", rows=1, vocab=VOCAB, top=5),
        # a prompt's tokens scored
        dict(name="logprobs_bf16_512", kind="logprobs", type="bf16", rows=512, vocab=VOCAB, top=0),
        # a decode batch with as many alternatives as servers give, odd vocabulary
        dict(name="logprobs_f32_61", kind="logprobs", type="f32", rows=61, vocab=50021, top=20),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _draw(rng):
    kind = rng.choice(["append", "append", "gather", "attend", "attend", "attend", "attend",
                       "logprobs", "logprobs"])
    case = dict(kind=kind, type=rng.choice(["f32", "bf16"]))
    if kind == "logprobs":
        return dict(case, rows=_log_int(rng, 1, 512), vocab=rng.choice([VOCAB, _log_int(rng, 100, 200000)]),
                    top=rng.choice([0, 1, 5, rng.randint(2, 20), 20]))
    latent, rope = rng.choice([(LATENT, ROPE)] * 5 + [(64, 16), (128, 32), (256, 64)])
    longest = _log_int(rng, 1, 16384)
    shortest = rng.choice([longest, rng.randint(0, longest), min(longest, 1)])
    new = 1 if rng.random() < 0.6 else _log_int(rng, 2, 300)
    return dict(case, cache=rng.choice(["bf16", "fp4"]), seqs=_log_int(rng, 1, 128), shortest=shortest,
                longest=longest, new=new, page=rng.choice([1, 16, 64, 64, 128, rng.randint(2, 200)]),
                heads=rng.choice([HEADS, HEADS, HEADS, rng.randint(1, 40), 128]), latent=latent,
                rope=rope)


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS:
            continue
        if case["kind"] != "attend" or _plain_size(case) < 1e9:
            return case


def _plain_size(case):
    """Values of the scores and of the keys that the plain form spreads out."""
    return case["seqs"] * case["longest"] * (case["new"] * case["heads"] + case["latent"])


# ---- inputs -------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _pairs(case):
    """(length, new rows) of each sequence; a length below the new rows leaves some of
    them without a key."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lengths = [hi if n == 1 else lo + (hi - lo) * k // (n - 1) for k in range(n)]
    if case["kind"] == "gather":
        return [(v, v) for v in lengths]
    return [(v, 1 + (case["new"] - 1) * (1 + k * 5 % n) // n) for k, v in enumerate(lengths)]


def _row_bytes(case):
    latent = 2 * case["latent"] if case["cache"] == "bf16" else case["latent"] // 2 + 16
    return latent + 2 * case["rope"]


def _keys(g, rows, case):
    """Rows of which a few columns are far above the rest."""
    loud = 1.0 + 4.0 * (torch.rand(case["latent"] + case["rope"], generator=g, device="cuda") < 0.02)
    return _normal(g, rows, case["latent"] + case["rope"]) * loud


def prepare(case, seed):
    g, kind, t = _generator(seed), case["kind"], TYPES[case["type"]]
    s = dict(case, t=t, workspace=torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda"))
    if kind == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        x = 2.5 * _normal(g, rows, vocab) + 4.0 * (torch.rand(vocab, generator=g, device="cuda") < 1e-3)
        # some tokens are not allowed
        x.masked_fill_(torch.rand(vocab, generator=g, device="cuda") < 0.01, -torch.inf)
        s["x"] = x.to(t)
        # the token is one of the likely ones, or any
        likely = (s["x"] + _normal(g, rows, 1)).argmax(1)
        other = torch.randint(vocab, (rows,), generator=g, device="cuda")
        any_ = torch.rand(rows, generator=g, device="cuda") < 0.3
        s["tokens"] = torch.where(any_, other, likely).int()
        s["logprob"] = torch.empty(rows, device="cuda")
        s["entropy"] = torch.empty(rows, device="cuda")
        s["ids"] = torch.empty(rows, top, dtype=torch.int32, device="cuda")
        s["top_logprob"] = torch.empty(rows, top, device="cuda")
        return s
    page, seqs, width = case["page"], case["seqs"], case["latent"] + case["rope"]
    order = torch.randperm(seqs, generator=g, device="cuda").tolist()
    pairs = _pairs(case)
    pairs = [pairs[k] for k in order]
    pages_of = [-(-length // page) for length, _ in pairs]
    pages = sum(pages_of) + 2
    places = torch.randperm(pages, generator=g, device="cuda").int()
    tables = torch.full((seqs, max(pages_of) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for k, count in enumerate(pages_of):
        tables[k, :count] = places[at:at + count]
        at += count
    starts = [0]
    for _, new in pairs:
        starts.append(starts[-1] + new)
    rows = starts[-1]
    s.update(pages=pages, tables=tables, rows=rows, most=max(new for _, new in pairs),
             lengths=torch.tensor([v for v, _ in pairs], dtype=torch.int32, device="cuda"),
             starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    pool = _keys(g, pages * page, case)
    s["pool"] = _encode(pool, case).reshape(pages, page, -1)
    if kind == "gather":
        s["out"] = torch.empty(rows, width, dtype=t, device="cuda")
    elif kind == "attend":
        # some heads look at few keys
        sharp = torch.where(torch.rand(case["heads"], 1, generator=g, device="cuda") < 0.2, 3.0, 0.7)
        s["q"] = (_normal(g, rows, case["heads"], width) * sharp).to(t)
        s["out"] = torch.empty(rows, case["heads"], case["latent"], dtype=t, device="cuda")
    else:
        heads = case["heads"]
        s["norm"] = 1.0 + 0.1 * _normal(g, case["latent"])
        s["freq"] = THETA ** (-torch.arange(0, case["rope"], 2, device="cuda").float() / case["rope"])
        # a row of the projection: every head's query, then the latent and the rope row
        s["both"] = (2.0 * _normal(g, rows, heads * (NOPE + case["rope"]) + width)).to(t)
        s["q"] = torch.zeros(rows, heads, width, dtype=t, device="cuda")
        s["back"] = torch.empty(rows, width, dtype=t, device="cuda")
    return s


# ---- rows of the pages ----------------------------------------------------------


def _power(e):
    """2^e, e whole numbers."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(v, case):
    """Rows of values as the pages hold them: bf16, or the bytes of codes, of scales and
    of the rope row."""
    if case["cache"] == "bf16":
        return v.to(torch.bfloat16)
    latent = case["latent"]
    x = v[:, :latent].double().reshape(v.shape[0], -1, GROUP)
    amax = x.abs().amax(-1)
    share, power = torch.frexp(amax)  # amax = share * 2^power, share in [0.5, 1)
    e = torch.where(share <= 0.75, power - 3, power - 2)
    e = torch.where(amax == 0, LEAST, e).clamp(LEAST, 125)
    bad = ~(amax < HUGE)
    a = x.abs() / _power(e)[..., None]
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) +
            (a > 5.0) + 8 * (x < 0)).reshape(v.shape[0], -1, 2)
    field = torch.zeros(v.shape[0], 16, dtype=torch.uint8, device=v.device)
    field[:, _scale_places(latent, v.device)] = torch.where(bad, 255, e + 127).to(torch.uint8)
    rope = v[:, latent:].to(torch.bfloat16).contiguous().view(torch.uint8)
    return torch.cat([(code[..., 0] + 16 * code[..., 1]).to(torch.uint8), field, rope], 1)


def _scale_places(latent, device):
    b = torch.arange(latent // GROUP, device=device)
    return 4 * (b % 4) + b // 4


MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _decode(rows, case):
    """f32 values of rows of the pages."""
    if case["cache"] == "bf16":
        return rows.float()
    latent = case["latent"]
    table = torch.tensor(MAGNITUDES + [-m for m in MAGNITUDES], device=rows.device)
    codes = rows[:, :latent // 2].int()
    v = table[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(rows.shape[0], -1, GROUP)
    e = rows[:, latent // 2:latent // 2 + 16].long()[:, _scale_places(latent, rows.device)]
    scale = torch.where(e == 255, torch.nan, _power(e - 127).float())
    rope = rows[:, latent // 2 + 16:].contiguous().view(torch.bfloat16).float()
    return torch.cat([(v * scale[..., None]).reshape(rows.shape[0], -1), rope], 1)


def _rows_of(s):
    """Of each row of the batch its sequence and its key's position (below 0: none)."""
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), r, right=True)
    return seq, s["lengths"][seq].long() - s["starts"][seq + 1].long() + r


def _slots(s, seq, position):
    """Places of keys in the pages, one after the other."""
    page = s["page"]
    return s["tables"][seq, position // page].long() * page + position % page


# ---- one pass -----------------------------------------------------------------


def _rotated(v, position, freq):
    """Pairs of neighbours in `v` [rows, ..., rope] turned by their position's angles:
    first halves of the results, then second ones."""
    angle = position.double()[:, None] * freq.double()
    angle = angle.reshape(angle.shape[0], *[1] * (v.dim() - 2), -1)
    a, b = v[..., 0::2].double(), v[..., 1::2].double()
    cos, sin = torch.cos(angle), torch.sin(angle)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _split_rows(s):
    """Queries [rows, heads, NOPE + rope], latent rows and rope rows of the projections."""
    heads, head = s["heads"], NOPE + s["rope"]
    q = s["both"][:, :heads * head].reshape(-1, heads, head)
    kv = s["both"][:, heads * head:]
    return q, kv[:, :s["latent"]], kv[:, s["latent"]:]


def _plain_append(s):
    query, c, k = _split_rows(s)
    seq, position = _rows_of(s)
    c = c.double()
    v = c / torch.sqrt(c.square().mean(-1, keepdim=True) + EPS) * s["norm"].double()
    rows = _encode(torch.cat([v, _rotated(k, position, s["freq"])], 1), s)
    held = position >= 0
    turned = _rotated(query[..., NOPE:], position, s["freq"]).to(s["t"])
    s["q"][held, :, s["latent"]:] = turned[held]
    slots = _slots(s, seq[held], position[held])
    pool = s["pool"].flatten(0, 1)
    pool[slots] = rows[held]
    if s["cache"] == "bf16":
        return {"q": s["q"], "pool": s["pool"]}
    return {"q": s["q"], "rows": _plain_gather(s)}


def _plain_gather(s):
    seq, position = _rows_of(s)
    held = position >= 0
    slots = _slots(s, seq, position.clamp(min=0)).clamp(min=0)
    rows = _decode(s["pool"].flatten(0, 1)[slots], s)
    return torch.where(held[:, None], rows, 0.0).to(s["t"])


def _plain_attend(s):
    seqs, heads, latent, most = s["seqs"], s["heads"], s["latent"], s["most"]
    longest = max(s["longest"], 1)
    key = torch.arange(longest, device="cuda")
    length = s["lengths"].long()
    held = key < length[:, None]
    sequence = torch.arange(seqs, device="cuda")[:, None].expand_as(held)
    k = torch.zeros(seqs, longest, latent + s["rope"], device="cuda")
    k[held] = _decode(s["pool"].flatten(0, 1)[_slots(s, sequence[held], key.expand_as(held)[held])], s)
    # every sequence's rows side by side, padded to the most
    row = s["starts"][:-1, None].long() + torch.arange(most, device="cuda")
    valid = row < s["starts"][1:, None]
    q = s["q"][row.clamp(max=s["rows"] - 1)].float().reshape(seqs, most * heads, -1)
    score = torch.bmm(q, k.transpose(1, 2).contiguous()) * _scale(s)
    last = length[:, None] - s["starts"][1:, None].long() + row
    seen = key <= last.repeat_interleave(heads, 1)[..., None]
    score = score.masked_fill(~seen, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p, k[..., :latent].contiguous()) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(seqs, most, heads, latent)[valid].to(s["t"])}


def _scale(case):
    return (NOPE + case["rope"]) ** -0.5


def _plain_logprobs(s):
    x, top = s["x"].float(), s["top"]
    rows, vocab = x.shape
    largest = x.amax(-1, keepdim=True)
    d = x - largest
    e = torch.exp(d)
    total = e.double().sum(-1)
    mean = torch.where(e > 0, e * d, 0.0).double().sum(-1) / total
    rest = largest[:, 0].double() + torch.log(total)
    # f32 bits in the order of their values, then the lower index first
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -2 ** 31 - bits, bits) * 2 ** 32 - torch.arange(vocab, device="cuda")
    ids = key.topk(top, dim=1, largest=True, sorted=True).indices if top else s["ids"].long()
    return {"logprob": (x.gather(1, s["tokens"].long()[:, None])[:, 0].double() - rest).float(),
            "entropy": (torch.log(total) - mean).float(), "ids": ids.int(),
            "top_logprob": (x.gather(1, ids).double() - rest[:, None]).float()}


def _plain(s):
    kind = s["kind"]
    if kind == "append":
        return _plain_append(s)
    if kind == "gather":
        return {"rows": _plain_gather(s)}
    return _plain_attend(s) if kind == "attend" else _plain_logprobs(s)


def _batch(s):
    from floyd_amd import native
    return native.LatentBatch(native.MLK_BF16 if s["cache"] == "bf16" else native.MLK_FP4,
                              s["pool"].data_ptr(), s["latent"], s["rope"], s["pages"], s["page"],
                              s["seqs"], s["tables"].data_ptr(), s["tables"].shape[1],
                              s["lengths"].data_ptr(), s["starts"].data_ptr())


def _framework(s):
    from floyd_amd import native
    kind, t = s["kind"], native.MLK_F32 if s["type"] == "f32" else native.MLK_BF16
    work_at, work_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    if kind == "logprobs":
        native.token_logprobs(t, s["x"].data_ptr(), s["rows"], s["vocab"], s["tokens"].data_ptr(),
                              s["logprob"].data_ptr(), work_at, work_bytes,
                              entropy=s["entropy"].data_ptr(), top=s["top"],
                              top_ids=s["ids"].data_ptr(), top_logprobs=s["top_logprob"].data_ptr())
        return {"logprob": s["logprob"], "entropy": s["entropy"], "ids": s["ids"],
                "top_logprob": s["top_logprob"]}
    batch = _batch(s)
    if kind == "attend":
        native.latent_attend(batch, t, s["q"].data_ptr(), s["out"].data_ptr(), s["rows"], s["heads"],
                             _scale(s), work_at, work_bytes)
        return {"out": s["out"]}
    if kind == "gather":
        native.latent_gather(batch, t, s["out"].data_ptr(), s["rows"])
        return {"rows": s["out"]}
    head = NOPE + s["rope"]
    at, stride = s["both"].data_ptr(), s["both"].shape[1]
    native.latent_append(batch, t, at + s["heads"] * head * s["t"].itemsize, s["rows"],
                         s["norm"].data_ptr(), s["freq"].data_ptr(), eps=EPS, stride=stride, query=at,
                         query_stride=stride, heads=s["heads"], head_width=head, q=s["q"].data_ptr())
    if s["cache"] == "bf16":
        return {"q": s["q"], "pool": s["pool"]}
    native.latent_gather(batch, t, s["back"].data_ptr(), s["rows"])
    return {"q": s["q"], "rows": s["back"]}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": rows * (vocab * size + 12 + 8 * top), "flops": 5 * rows * vocab}
    pairs, width, row = _pairs(case), case["latent"] + case["rope"], _row_bytes(case)
    held = [(length, min(length, new)) for length, new in pairs]
    rows, there = sum(new for _, new in pairs), sum(new for _, new in held)
    tables = 4 * sum(-(-length // case["page"]) for length, _ in pairs) + 8 * case["seqs"] + 4
    if kind == "gather":
        return {"bytes": there * row + rows * width * size + tables, "flops": there * width}
    if kind == "append":
        queries = 2 * there * case["heads"] * case["rope"] * size
        back = there * row + rows * width * size if case["cache"] == "fp4" else 0
        return {"bytes": there * (width * size + row) + queries + back + tables + 4 * case["latent"],
                "flops": there * (6 * case["latent"] + 3 * (case["heads"] + 1) * case["rope"])}
    # keys that a sequence's rows see, in all
    seen = sum(there * length - there * (there - 1) // 2 for length, there in held)
    heads, latent = case["heads"], case["latent"]
    return {"bytes": sum(length for length, _ in pairs) * row + tables +
            rows * heads * (width + latent) * size,
            "flops": 2 * seen * heads * (width + latent)}


# ---- the same in 64 bits --------------------------------------------------------


def _values(s):
    """f64 [pages * page, latent + rope]: what the pages stand for."""
    rows, latent = s["pool"].flatten(0, 1), s["latent"]
    if s["cache"] == "bf16":
        return rows.double()
    out = torch.empty(rows.shape[0], latent + s["rope"], dtype=torch.float64, device=rows.device)
    levels = torch.tensor(MAGNITUDES, dtype=torch.float64, device=rows.device)
    for half in (0, 1):
        code = (rows[:, :latent // 2] >> (4 * half)) % 16
        out[:, half:latent:2] = levels[(code % 8).long()] * torch.where(code >= 8, -1.0, 1.0)
    for b in range(latent // GROUP):
        e = rows[:, latent // 2 + 4 * (b % 4) + b // 4].double() - 127.0
        out[:, b * GROUP:(b + 1) * GROUP] *= torch.exp2(e)[:, None]
    out[:, latent:] = rows[:, latent // 2 + 16:].contiguous().view(torch.bfloat16).double()
    return out


def _fp4_exact(v):
    """The values that 4 bits keep of v [rows, latent]."""
    out = torch.empty_like(v)
    for b in range(v.shape[1] // GROUP):
        part = v[:, b * GROUP:(b + 1) * GROUP]
        amax = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -200) / 6.0))
        e = torch.where(amax > 6.0 * torch.exp2(e), e + 1, e)
        e = torch.where(amax <= 6.0 * torch.exp2(e - 1), e - 1, e).clamp(min=LEAST)
        a = part.abs() * torch.exp2(-e)
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        out[:, b * GROUP:(b + 1) * GROUP] = torch.round(a / step) * step * torch.sign(part) * torch.exp2(e)
    return out


def _turn(v, position, freq):
    out = torch.empty_like(v)
    half = v.shape[-1] // 2
    for i in range(half):
        angle = position.double() * freq[i].double()
        angle = angle.reshape(-1, *[1] * (v.dim() - 2))
        x = torch.complex(v[..., 2 * i], v[..., 2 * i + 1]) * torch.polar(torch.ones_like(angle), angle)
        out[..., i], out[..., half + i] = x.real, x.imag
    return out


def _each_row(s):
    """(row, sequence, position) of every row of the batch."""
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for k, length in enumerate(lengths):
        for r in range(starts[k], starts[k + 1]):
            yield r, k, length - starts[k + 1] + r


def _exact_append(s):
    latent, heads = s["latent"], s["heads"]
    rows = s["both"].double()
    head = NOPE + s["rope"]
    c, k = rows[:, heads * head:heads * head + latent], rows[:, heads * head + latent:]
    query = torch.stack([rows[:, h * head + NOPE:(h + 1) * head] for h in range(heads)], 1)
    v = c * torch.rsqrt((c * c).sum(1, keepdim=True) / latent + EPS) * s["norm"].double()
    which, seq, position = (torch.tensor(t, device="cuda") for t in zip(*_each_row(s)))
    there = torch.nonzero(position >= 0)[:, 0]
    q = s["q"].double()
    q[there, :, latent:] = _turn(query[there], position[there], s["freq"])
    turned = _turn(k, position, s["freq"])
    if s["cache"] == "fp4":  # the rope row is held in bf16
        new = torch.cat([_fp4_exact(v), turned.to(torch.bfloat16).double()], 1)
        new[position < 0] = 0.0
        return {"q": q, "rows": new}
    new = torch.cat([v, turned], 1)
    pool = s["pool"].double()
    at = position[there]
    pool[s["tables"][seq[there], at // s["page"]].long(), at % s["page"]] = new[there]
    return {"q": q, "pool": pool}


def _sequence(s, values, k, length):
    """The first `length` keys of sequence k."""
    at = torch.arange(length, device="cuda")
    return values[s["tables"][k][at // s["page"]].long() * s["page"] + at % s["page"]]


def _exact_gather(s):
    values, starts = _values(s), s["starts"].tolist()
    out = torch.zeros(s["rows"], s["latent"] + s["rope"], dtype=torch.float64, device="cuda")
    for k, length in enumerate(s["lengths"].tolist()):
        there = min(length, starts[k + 1] - starts[k])
        out[starts[k + 1] - there:starts[k + 1]] = _sequence(s, values, k, length)[length - there:]
    return {"rows": out}


def _exact_attend(s):
    values, starts, latent = _values(s), s["starts"].tolist(), s["latent"]
    out = torch.zeros(s["rows"], s["heads"], latent, dtype=torch.float64, device="cuda")
    for k, length in enumerate(s["lengths"].tolist()):
        keys = _sequence(s, values, k, length)
        new = starts[k + 1] - starts[k]
        for r in range(starts[k], starts[k + 1]):
            seen = length - new + r - starts[k] + 1
            if seen > 0:
                p = torch.softmax(s["q"][r].double() @ keys[:seen].T * _scale(s), -1)
                out[r] = p @ keys[:seen, :latent]
    return {"out": out}


def _exact_logprobs(s):
    logprob, entropy, ids, tops = [], [], [], []
    for r in range(s["rows"]):
        lp = torch.log_softmax(s["x"][r].double(), 0)
        logprob.append(lp[s["tokens"][r].long()])
        entropy.append(-torch.xlogy(lp.exp(), lp.exp()).sum())
        first = torch.sort(s["x"][r].double(), descending=True, stable=True).indices[:s["top"]]
        ids.append(first.int())
        tops.append(lp[first])
    return {"logprob": torch.stack(logprob), "entropy": torch.stack(entropy), "ids": torch.stack(ids),
            "top_logprob": torch.stack(tops)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "gather": _exact_gather, "attend": _exact_attend,
            "logprobs": _exact_logprobs}[case["kind"]](s)
