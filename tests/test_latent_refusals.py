"""Calls that the latent cache and log probability entry points refuse before they touch
the GPU."""
import ctypes

import numpy as np
import pytest

import latent_util as L
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, MLK_FP4, MLK_Q8, NativeError

P = 1 << 20  # stands for an address; the refusals below never look at it
SPACE = 1 << 26
BATCH = dict(cache_type=MLK_BF16, data=P, latent=512, rope=64, pages=4, page_size=16, seqs=2, tables=P,
             table_width=3, lengths=P, row_starts=P)


def split(more):
    batch = {k: more.pop(k) for k in list(more) if k in BATCH}
    return native.LatentBatch(**{**BATCH, **batch})


def append(dtype=MLK_F32, kv=P, rows=4, norm_w=P, inv_freq=P, **more):
    native.latent_append(split(more), dtype, kv, rows, norm_w, inv_freq, **more)


def gather(dtype=MLK_F32, out=P, rows=4, **more):
    native.latent_gather(split(more), dtype, out, rows)


def attend(dtype=MLK_F32, q=P, out=P, rows=4, heads=16, scale=0.1, workspace=P, space=SPACE, **more):
    native.latent_attend(split(more), dtype, q, out, rows, heads, scale, workspace, space)


def logprobs(dtype=MLK_F32, logits=P, rows=4, vocab=100000, tokens=P, out=P, workspace=P, space=SPACE,
             **more):
    native.token_logprobs(dtype, logits, rows, vocab, tokens, out, workspace, space, **more)


TURN = dict(query=P, heads=2, head_width=64, q=P)


@pytest.mark.parametrize("call", [append, gather, attend])
@pytest.mark.parametrize("bad,says", [
    (dict(dtype=MLK_Q8), "type must be MLK_F32"),
    (dict(dtype=MLK_FP4), "type must be MLK_F32"),
    (dict(cache_type=MLK_F32), "batch's type"),
    (dict(cache_type=9), "batch's type"),
    (dict(latent=0), "latent"), (dict(latent=576), "latent"), (dict(latent=96), "latent"),
    (dict(latent=-64), "latent"), (dict(rope=0), "rope"), (dict(rope=24), "rope"), (dict(rope=80), "rope"),
    (dict(pages=0), "pages"), (dict(page_size=0), "page_size"), (dict(page_size=-1), "page_size"),
    (dict(table_width=0), "table_width"), (dict(seqs=-1), "seqs"),
    (dict(rows=-1), "rows"),
    (dict(rows=1, row_starts=None), "needs a row"),
    (dict(data=None), "data is null"), (dict(data=P + 8), "data is not aligned"),
    (dict(tables=None), "tables is null"), (dict(tables=P + 2), "tables is not aligned"),
    (dict(lengths=None), "lengths is null"), (dict(lengths=P + 1), "lengths is not aligned"),
    (dict(row_starts=P + 2), "row_starts is not aligned"),
])
def test_batches_refused(call, bad, says):
    with pytest.raises(NativeError, match=says):
        call(**bad)


@pytest.mark.parametrize("call,bad,says", [
    (append, dict(kv=None), "kv is null"),
    (append, dict(kv=P + 2), "kv is not aligned"),
    (append, dict(dtype=MLK_BF16, kv=P + 1), "kv is not aligned"),
    (append, dict(stride=575), "kv_stride"),
    (append, dict(rows=1 << 24), "rows must be below"), (gather, dict(rows=(1 << 26) - 3), "rows must be at most"),
    (logprobs, dict(rows=1 << 24, vocab=1, space=0), "too many rows"),
    (logprobs, dict(rows=1 << 19, vocab=1 << 22, space=1 << 62), "too many rows"),
    (append, dict(norm_w=P + 2), "norm_w is not aligned"),
    (append, dict(inv_freq=None), "inv_freq is null"),
    (append, dict(inv_freq=P + 3), "inv_freq is not aligned"),
    (append, dict(eps=-1e-6), "eps"), (append, dict(eps=float("nan")), "eps"),
    (append, dict(eps=float("inf")), "eps"),
    (append, dict(TURN, heads=0), "heads"), (append, dict(TURN, heads=1025), "heads"),
    (append, dict(TURN, head_width=63), "head_width"),
    (append, dict(TURN, query_stride=127), "query_stride"),
    (append, dict(TURN, q=None), "q is null"), (append, dict(TURN, q=P + 2), "q is not aligned"),
    (append, dict(TURN, query=P + 1), "query is not aligned"),
    (gather, dict(out=None), "out is null"), (gather, dict(out=P + 2), "out is not aligned"),
    (attend, dict(q=None), "q is null"), (attend, dict(q=P + 2), "q is not aligned"),
    (attend, dict(out=None), "out is null"), (attend, dict(out=P + 1), "out is not aligned"),
    (attend, dict(heads=0), "heads"), (attend, dict(heads=1025), "heads"),
    (attend, dict(rows=(1 << 31) - 1, heads=2), "rows . heads"),
    (attend, dict(scale=float("inf")), "scale"), (attend, dict(scale=float("nan")), "scale"),
    (attend, dict(workspace=None), "workspace is null"),
    (attend, dict(workspace=P + 8), "workspace is not aligned"),
    (attend, dict(space=1000), "workspace needs"),
    (logprobs, dict(dtype=MLK_Q8), "type"),
    (logprobs, dict(rows=-1), "rows"), (logprobs, dict(vocab=0), "vocab"),
    (logprobs, dict(vocab=(1 << 22) + 1), "vocab"),
    (logprobs, dict(stride=99999), "stride"),
    (logprobs, dict(top=-1), "top"), (logprobs, dict(top=33), "top"), (logprobs, dict(vocab=4, top=5), "top"),
    (logprobs, dict(logits=None), "logits is null"), (logprobs, dict(logits=P + 2), "logits is not aligned"),
    (logprobs, dict(tokens=None), "tokens is null"), (logprobs, dict(out=None), "logprobs is null"),
    (logprobs, dict(entropy=P + 2), "entropy is not aligned"),
    (logprobs, dict(top=2, top_logprobs=P), "top_ids is null"),
    (logprobs, dict(top=2, top_ids=P), "top_logprobs is null"),
    (logprobs, dict(space=0), "workspace needs"),
    (logprobs, dict(workspace=None), "workspace is null"),
])
def test_refused(call, bad, says):
    with pytest.raises(NativeError, match=says):
        call(**bad)


@pytest.mark.parametrize("call", [append, gather, attend])
@pytest.mark.parametrize("seqs", [(1 << 30) + 1, (1 << 31) - 1])
def test_more_sequences_than_are_counted(call, seqs):
    with pytest.raises(NativeError, match="seqs must be at most"):
        call(seqs=seqs)
    with pytest.raises(NativeError, match="no HIP device|not device memory"):
        call(seqs=1 << 30)


@pytest.mark.parametrize("scale", [2.0 ** 127, -2.0 ** 127, 2.0 ** 127.8, float("-inf")])
def test_scales_that_log2_e_takes_past_f32(scale):
    with pytest.raises(NativeError, match="scale"):
        attend(scale=scale)
    with pytest.raises(NativeError, match="no HIP device|not device memory"):
        attend(scale=np.nextafter(np.float32(2.0 ** 127), np.float32(0)))


def test_null_batch():
    lib = native.load()
    assert lib.mlk_latent_gather(None, MLK_F32, 1, P) == -1 and "batch is null" in native.last_error()


@pytest.mark.parametrize("call,empty", [
    (append, dict(rows=0, kv=None, inv_freq=None)), (append, dict(seqs=0, kv=None)),
    (gather, dict(rows=0, out=None)), (gather, dict(seqs=0, out=None)),
    (attend, dict(rows=0, q=None, out=None, workspace=None, space=0)),
    (attend, dict(seqs=0, q=None, out=None, workspace=None, space=0)),
    (logprobs, dict(rows=0, logits=None, tokens=None, out=None, workspace=None, space=0)),
])
def test_nothing_to_do(call, empty):
    call(**empty)


@pytest.mark.parametrize("call", [append, gather, attend, logprobs])
def test_without_a_device(call):
    """A full call reports the missing GPU, or the address that is none of its memory."""
    with pytest.raises(NativeError, match="no HIP device|not device memory"):
        call()


def test_row_bytes():
    assert native.latent_row_bytes(MLK_BF16, 512, 64) == 1152
    assert native.latent_row_bytes(MLK_FP4, 512, 64) == 400
    assert native.latent_row_bytes(MLK_FP4, 64, 16) == 80
    for cache_type, latent, rope in ((MLK_F32, 512, 64), (MLK_FP4, 500, 64), (MLK_BF16, 512, 8)):
        with pytest.raises(NativeError):
            native.latent_row_bytes(cache_type, latent, rope)


def test_workspaces():
    assert 0 < native.latent_attend_workspace() < SPACE
    assert native.token_logprobs_workspace(0, 100, 0) == 0
    assert native.token_logprobs_workspace(4, (1 << 22) + 1, 0) == 0
    assert 0 < native.token_logprobs_workspace(4, 163840, 20) < 1 << 20


def test_logprobs_workspace_serves_smaller_calls():
    """It never falls as rows, vocabulary or top grow, and no call of at most as many of each asks
    for more."""
    size = native.token_logprobs_workspace
    vocabs = [1, 300, 2048, 2049, 8192, 8193, 16385, 50021, 131072, 163840, 262144, 1 << 20, 2 << 20, 1 << 22]
    for top in (0, 20):
        for vocab in vocabs:
            sizes = [size(rows, vocab, top) for rows in range(1, 700)]
            assert sizes == sorted(sizes), vocab
        for rows in (1, 2, 3, 12, 13, 36, 37, 60, 255, 256, 600):
            sizes = [size(rows, vocab, top) for vocab in vocabs + list(range(1900, 100000, 700))]
            assert sizes[:len(vocabs)] == sorted(sizes[:len(vocabs)]), rows
            assert sizes[len(vocabs):] == sorted(sizes[len(vocabs):]), rows
    for rows, vocab, top in ((13, 163840, 20), (64, 50021, 20), (300, 8200, 32), (300, 8192, 5), (1, 1 << 22, 32)):
        space = size(rows, vocab, top)
        assert size(rows, vocab, top - 1) <= space
        for fewer in {1, 2, 12, 36, 255, 256, rows - 1, rows} & set(range(1, rows + 1)):
            for less in {vocab, vocab // 2 + 1, min(vocab, 8193), min(vocab, 2049), min(vocab, 40)}:
                for some in (0, top):
                    with pytest.raises(NativeError, match="no HIP device|not device memory"):
                        logprobs(rows=fewer, vocab=less, top=some, top_ids=P, top_logprobs=P, space=space)


@pytest.mark.gpu
def test_host_memory_is_refused(device):
    d = native.DeviceBuffer(1 << 20)
    x = np.zeros(4096, np.float32)
    real = dict(data=d, tables=d, lengths=d, row_starts=d)
    with pytest.raises(NativeError, match="kv is not device memory"):
        append(**real, kv=x.ctypes.data, norm_w=d, inv_freq=d)
    with pytest.raises(NativeError, match="tables is not device memory"):
        gather(**dict(real, tables=x.ctypes.data), out=d)
    buf = ctypes.create_string_buffer(4096 + 16)
    with pytest.raises(NativeError, match="workspace is not device memory"):
        attend(**real, q=d, out=d, workspace=ctypes.addressof(buf) + -ctypes.addressof(buf) % 16)
    with pytest.raises(NativeError, match="logits is not device memory"):
        logprobs(logits=x.ctypes.data, vocab=1000, tokens=d, out=d, workspace=d)


def test_codec_of_the_oracle():
    """Every code's value has that code; ties go to the even one; scales at their borders."""
    assert list(L.fp4_nearest(L.MAGNITUDES)) == list(range(8))
    mid = (L.MAGNITUDES[:-1] + L.MAGNITUDES[1:]) / 2
    assert list(L.fp4_nearest(mid)) == [0, 2, 2, 4, 4, 6, 6]
    rng = np.random.default_rng(1)
    for k in range(50):
        v = rng.standard_normal(80) * 2.0 ** rng.integers(-60, 60)
        for cache_type in (MLK_BF16, MLK_FP4):
            raw = L.encode_row(v, cache_type, 64)
            back = L.decode_row(raw, cache_type, 64)
            assert np.array_equal(L.decode_row(L.encode_row(back, cache_type, 64), cache_type, 64), back)
    row = np.zeros(80)
    row[0], row[32] = 6.0, np.nextafter(6.0, 7.0)
    raw = L.encode_row(row, MLK_FP4, 64)
    assert raw[32 + 0] == 127 and raw[32 + 4] == 128
