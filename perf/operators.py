"""The fp8 operators: from the residual stream to quantised rows, and the
products of fp8 rows with fp8 matrices, dense and per expert.

Values are held as e4m3 codes with one f32 scale per block: 1 x 128 columns for
activations, 128 x 128 for weights.  A case is a dict of plain values; `kind`
names the operator:

  norm     residual addition, RMSNorm, quantised rows (mlk_rmsnorm_fp8)
  pack     rows (block 1) or a matrix (block 128) quantised (mlk_quantize_fp8)
  swiglu   silu(gate) * up, quantised rows (mlk_swiglu_fp8)
  mm       rows times one matrix (mlk_matmul_fp8)
  grouped  rows sorted by expert, or gathered into that order, times each
           expert's matrix (mlk_matmul_fp8_grouped)

`type` is the type of the values that are not fp8: f32 or bf16.
"""
import torch

own = False

HIDDEN, DENSE, INTER, EXPERTS, TOP_K, SHARED = 2048, 11264, 1408, 64, 6, 2816
EPS, BLOCK, TOP = 1e-5, 128, 448.0
TINY = 2.0 ** -126  # the smallest scale, that of a block of zeros
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# (out, in) of the configuration's matrices, gate and up as one
SHAPES = [(576, HIDDEN), (HIDDEN, HIDDEN), (2 * DENSE, HIDDEN), (HIDDEN, DENSE),
          (2 * SHARED, HIDDEN), (HIDDEN, SHARED), (2 * INTER, HIDDEN), (HIDDEN, INTER)]
MOST_MACS, MOST_WEIGHTS, MOST_VALUES = 4096 * 2 * DENSE * HIDDEN, 64 * HIDDEN * 2 * INTER, 1 << 25


def listed():
    return [
        # one decoded token between attention and its FFN: the smallest call
        dict(name="norm_f32_1", kind="norm", type="f32", rows=1, cols=HIDDEN, resid=True),
        # a prompt of 4096 tokens, residual stream in bf16
        dict(name="norm_bf16_4096", kind="norm", type="bf16", rows=4096, cols=HIDDEN, resid=True),
        # a checkpoint's bf16 matrix packed while it is loaded
        dict(name="pack_2048x11264", kind="pack", type="bf16", rows=HIDDEN, cols=DENSE, block=128),
        # attention's output rows of a long prompt before o_proj
        dict(name="pack_rows_777", kind="pack", type="f32", rows=777, cols=HIDDEN, block=1),
        # a decode batch of 5 streams inside the dense FFN
        dict(name="swiglu_f32_5", kind="swiglu", type="f32", rows=5, width=DENSE),
        # the routed experts of a 2048-token prompt
        dict(name="swiglu_bf16_12288", kind="swiglu", type="bf16", rows=2048 * TOP_K, width=INTER),
        # one token through gate and up of the dense FFN
        dict(name="mm_f32_1", kind="mm", type="f32", rows=1, out=2 * DENSE, inp=HIDDEN, resid=False),
        # 61 streams through its down projection, onto the residual stream
        dict(name="mm_bf16_61", kind="mm", type="bf16", rows=61, out=HIDDEN, inp=DENSE, resid=True),
        # a matrix whose sides are no multiple of anything
        dict(name="mm_ragged_333", kind="mm", type="f32", rows=333, out=1001, inp=1999, resid=False),
        # a 4096-token prompt through gate and up of the dense FFN
        dict(name="mm_bf16_4096", kind="mm", type="bf16", rows=4096, out=2 * DENSE, inp=HIDDEN,
             resid=False),
        # 8 streams through their experts' gate and up, gathered
        dict(name="grouped_f32_8", kind="grouped", type="f32", tokens=8, experts=EXPERTS,
             top_k=TOP_K, out=2 * INTER, inp=HIDDEN, gather=True, spare=0),
        # a 2048-token prompt through its experts' down projections, in a buffer
        # with room for more
        dict(name="grouped_bf16_2048", kind="grouped", type="bf16", tokens=2048, experts=EXPERTS,
             top_k=TOP_K, out=HIDDEN, inp=INTER, gather=False, spare=37),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "pack", "swiglu", "mm", "mm", "mm", "grouped", "grouped", "grouped"])
    case = dict(kind=kind, type=rng.choice(["f32", "bf16"]))
    odd = rng.random() < 0.4  # other models' widths, most of them no multiple of a tile
    if kind in ("norm", "pack", "swiglu"):
        cols = _log_int(rng, 64, 16384) if odd else rng.choice([512, INTER, HIDDEN, SHARED, DENSE])
        rows = _log_int(rng, 1, min(16384, MOST_VALUES // cols))
        if kind == "swiglu":
            return dict(case, rows=rows, width=cols)
        if kind == "norm":
            return dict(case, rows=rows, cols=cols, resid=rng.random() < 0.7)
        return dict(case, rows=rows, cols=cols, block=rng.choice([1, 128]))
    out, inp = rng.choice(SHAPES)
    if odd:
        out, inp = _log_int(rng, 60, 12000), _log_int(rng, 60, 12000)
    if kind == "mm":
        most = min(4096, MOST_MACS // (out * inp))
        return dict(case, rows=_log_int(rng, 1, most), out=out, inp=inp, resid=rng.random() < 0.4)
    experts = max(2, min(_log_int(rng, 4, 160), MOST_WEIGHTS // (out * inp)))
    top_k = min(experts, rng.choice([1, 2, 4, 6, 8]))
    most = min(2048, MOST_MACS // (out * inp * top_k))
    return dict(case, tokens=_log_int(rng, 1, most), experts=experts, top_k=top_k, out=out,
                inp=inp, gather=rng.random() < 0.5, spare=rng.choice([0, 0, 1, 100]))


# ---- inputs -------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _stream(g, rows, cols):
    """Rows as a residual stream holds them: a few columns far above the rest."""
    loud = 1.0 + 30.0 * (torch.rand(cols, generator=g, device="cuda") < 0.004)
    return _normal(g, rows, cols) * loud


def _blocks(count):
    return (count + BLOCK - 1) // BLOCK


def _quantize(y, block):
    """f32 [..., rows, cols] as e4m3 codes and the f32 scales of its blocks."""
    *lead, rows, cols = y.shape
    full = torch.nn.functional.pad(y, (0, -cols % BLOCK, 0, -rows % block))
    tiles = full.reshape(*lead, -1, block, _blocks(cols), BLOCK)
    scale = (tiles.abs().amax((-3, -1)) / TOP).clamp(min=TINY)
    codes = (tiles * (1.0 / scale)[..., None, :, None]).reshape(full.shape)
    return codes[..., :rows, :cols].to(torch.float8_e4m3fn).contiguous(), scale


def _rows_fp8(g, rows, cols):
    return _quantize(_stream(g, rows, cols), 1)


def prepare(case, seed):
    g, kind, t = _generator(seed), case["kind"], TYPES[case["type"]]
    s = dict(case, t=t)
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        s.update(x=_normal(g, rows, cols).to(t), norm=1.0 + 0.1 * _normal(g, cols),
                 resid=_stream(g, rows, cols).to(t) if case["resid"] else None,
                 sum=torch.empty(rows, cols, dtype=t, device="cuda"))
    elif kind == "pack":
        rows, cols = case["rows"], case["cols"]
        weights = case["block"] == BLOCK
        s.update(x=(0.02 * _normal(g, rows, cols) if weights else _normal(g, rows, cols)).to(t))
    elif kind == "swiglu":
        rows, cols = case["rows"], case["width"]
        s.update(x=(2.0 * _normal(g, rows, 2 * cols)).to(t))
    if kind in ("norm", "pack", "swiglu"):
        scale_rows = rows if case.get("block", 1) == 1 else _blocks(rows)
        s.update(q=torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda"),
                 scale=torch.empty(scale_rows, _blocks(cols), device="cuda"))
        return s
    out, inp = case["out"], case["inp"]
    if kind == "mm":
        s["x"], s["xs"] = _rows_fp8(g, case["rows"], inp)
        s["w"], s["ws"] = _quantize(0.02 * _normal(g, out, inp), BLOCK)
        s["resid"] = _stream(g, case["rows"], out).to(t) if case["resid"] else None
        s["y"] = torch.empty(case["rows"], out, dtype=t, device="cuda")
        return s
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    entries = tokens * top_k
    # some experts are asked for more often than others
    liked = _normal(g, tokens, experts) + 0.7 * _normal(g, experts)
    ids = liked.topk(top_k, dim=1).indices.flatten()
    counts = torch.bincount(ids, minlength=experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    s.update(offsets=offsets, most=int(counts.max()), entries=entries + case["spare"], row_ids=None)
    if case["gather"]:
        s["row_ids"] = torch.zeros(s["entries"], dtype=torch.int32, device="cuda")
        s["row_ids"][:entries] = ids.sort(stable=True).indices // top_k
    s["x"], s["xs"] = _rows_fp8(g, tokens if case["gather"] else s["entries"], inp)
    s["w"], s["ws"] = _quantize(0.02 * _normal(g, experts, out, inp), BLOCK)
    s["y"] = torch.zeros(s["entries"], out, dtype=t, device="cuda")
    return s


# ---- one pass -----------------------------------------------------------------


def _values(codes, scale, block):
    """The f32 values of codes [..., rows, cols]."""
    wide = scale.repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]
    if block > 1:
        wide = wide.repeat_interleave(block, -2)[..., :codes.shape[-2], :]
    return codes.float() * wide


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        h = s["x"].float() if s["resid"] is None else s["x"].float() + s["resid"].float()
        h = h.to(s["t"])
        v = h.float()
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s["norm"]
        q, scale = _quantize(v, 1)
        return {"sum": h, "q": q, "scale": scale}
    if kind == "pack":
        q, scale = _quantize(s["x"].float(), s["block"])
        return {"q": q, "scale": scale}
    if kind == "swiglu":
        g, u = s["x"].float().chunk(2, dim=-1)
        q, scale = _quantize(g / (1.0 + torch.exp(-g)) * u, 1)
        return {"q": q, "scale": scale}
    x = _values(s["x"], s["xs"], 1)
    if kind == "mm":
        y = x @ _values(s["w"], s["ws"], BLOCK).T
        return (y if s["resid"] is None else y + s["resid"].float()).to(s["t"])
    # every expert's rows side by side, padded to the longest
    at = torch.arange(s["most"], device="cuda")
    pos = s["offsets"][:-1, None].long() + at
    valid = pos < s["offsets"][1:, None]
    held = pos.clamp(max=s["entries"] - 1)
    x = x[held if s["row_ids"] is None else s["row_ids"][held].long()] * valid[..., None]
    y = torch.bmm(x, _values(s["w"], s["ws"], BLOCK).transpose(1, 2).contiguous())
    out = torch.zeros(s["entries"] + 1, y.shape[-1], device="cuda")
    out.index_copy_(0, torch.where(valid, pos, s["entries"]).flatten(), y.flatten(0, 1))
    return out[:-1].to(s["t"])


def _framework(s):
    from floyd_amd import native
    kind, t = s["kind"], native.MLK_F32 if s["type"] == "f32" else native.MLK_BF16

    def p(name):
        return None if s[name] is None else s[name].data_ptr()

    if kind == "norm":
        native.rmsnorm_fp8(t, p("x"), p("norm"), s["rows"], s["cols"], p("q"), p("scale"),
                           resid=p("resid"), total=p("sum"), eps=EPS)
        return {"sum": s["sum"], "q": s["q"], "scale": s["scale"]}
    if kind == "pack":
        native.quantize_fp8(t, p("x"), s["rows"], s["cols"], s["block"], p("q"), p("scale"))
        return {"q": s["q"], "scale": s["scale"]}
    if kind == "swiglu":
        native.swiglu_fp8(t, p("x"), s["rows"], s["width"], p("q"), p("scale"))
        return {"q": s["q"], "scale": s["scale"]}
    if kind == "mm":
        native.matmul_fp8(t, p("w"), p("ws"), p("x"), p("xs"), p("y"), s["out"], s["inp"],
                          s["rows"], resid=p("resid"))
        return s["y"]
    native.matmul_fp8_grouped(t, p("w"), p("ws"), p("x"), p("xs"), p("y"), s["out"], s["inp"],
                              s["experts"], p("offsets"), s["entries"], row_ids=p("row_ids"),
                              x_rows=s["x"].shape[0])
    return s["y"]


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind in ("norm", "pack", "swiglu"):
        rows, cols = case["rows"], case.get("cols") or case["width"]
        scales = (rows if case.get("block", 1) == 1 else _blocks(rows)) * _blocks(cols)
        tensors = {"pack": 1, "swiglu": 2}.get(kind) or (3 if case["resid"] else 2)
        return {"bytes": rows * cols * (size * tensors + 1) + 4 * scales +
                (4 * cols if kind == "norm" else 0),
                "flops": rows * cols * {"pack": 2, "swiglu": 8, "norm": 7}[kind]}
    out, inp = case["out"], case["inp"]
    matrix = out * inp + 4 * _blocks(out) * _blocks(inp)
    row = inp + 4 * _blocks(inp)
    if kind == "mm":
        return {"bytes": matrix + case["rows"] * (row + out * size * (2 if case["resid"] else 1)),
                "flops": 2 * case["rows"] * out * inp}
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    used = experts * (1.0 - (1.0 - top_k / experts) ** tokens)
    entries = tokens * top_k
    return {"bytes": used * matrix + (tokens if case["gather"] else entries) * row +
            entries * (out * size + (4 if case["gather"] else 0)) + 4 * (experts + 1),
            "flops": 2 * entries * out * inp}


# ---- the same in 64 bits --------------------------------------------------------


def _e4m3(v):
    """The nearest e4m3 value, ties to the even one: 3 fraction bits from 2^-6 on,
    steps of 2^-9 below."""
    power = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    # log2 may round up to the next whole number just below a power of two
    power = torch.where(torch.exp2(power) > v.abs(), (power - 1.0).clamp(min=-6.0), power)
    step = torch.exp2(power - 3.0)
    return torch.round(v / step) * step


def _pack_exact(v, block):
    rows, cols = v.shape
    up, across = -(-rows // block), _blocks(cols)
    codes = torch.empty_like(v)
    scale = torch.empty(up, across, dtype=torch.float64, device=v.device)
    for b in range(across):
        part = v[:, b * BLOCK:(b + 1) * BLOCK]
        top = torch.zeros(up * block, dtype=torch.float64, device=v.device)
        top[:rows] = part.abs().amax(1)
        scale[:, b] = torch.clamp(top.reshape(up, block).amax(1) / TOP, min=TINY)
        codes[:, b * BLOCK:(b + 1) * BLOCK] = _e4m3(
            part / scale[:, b].repeat_interleave(block)[:rows, None])
    return codes, scale


def _product_exact(x, xs, w, ws):
    """Rows of codes times a matrix of codes: each block of 128 columns' sum, scaled."""
    y = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    tall = torch.arange(w.shape[0], device=x.device) // BLOCK
    for b in range(xs.shape[1]):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        part = x[:, at].double() @ w[:, at].double().T
        y += part * xs[:, b].double()[:, None] * ws[tall, b].double()[None, :]
    return y


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h = s["x"].double()
        if s["resid"] is not None:
            h = h + s["resid"].double()
        v = h.to(s["t"]).double()  # the norm is that of the sum as it is stored
        v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS) * s["norm"].double()
        q, scale = _pack_exact(v, 1)
        return {"sum": h, "q": q, "scale": scale}
    if kind in ("pack", "swiglu"):
        v = s["x"].double()
        if kind == "swiglu":
            g, u = v[:, :case["width"]], v[:, case["width"]:]
            v = g * torch.sigmoid(g) * u
        q, scale = _pack_exact(v, case.get("block", 1))
        return {"q": q, "scale": scale}
    if kind == "mm":
        y = _product_exact(s["x"], s["xs"], s["w"], s["ws"])
        return y if s["resid"] is None else y + s["resid"].double()
    y = torch.zeros(s["entries"], case["out"], dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e in range(case["experts"]):
        rows = torch.arange(ends[e], ends[e + 1], device="cuda")
        if rows.numel():
            at = rows if s["row_ids"] is None else s["row_ids"][rows].long()
            y[rows] = _product_exact(s["x"][at], s["xs"][at], s["w"][e], s["ws"][e])
    return y
