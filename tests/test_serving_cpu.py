"""What the adapters, the normalized append and the log probabilities refuse, before
any launch."""
import ctypes
import math

import pytest

from evo_hip import native as N
from test_paged_cpu import A, B, C, BAD_BATCHES, BAD_CACHES, batch, cache


def append_normed(c=None, b=None, dtype=N.DTYPE_F32, projected=C, row_stride=512, heads=4, split=0,
                  query_scale=A, key_scale=A, stride=0, eps=1e-6, inside=1, inv_freq=A, rotary=64,
                  interleaved=0, scale=1.0, query=B, query_stride=256):
    N.call("evo_hip_paged_append_normed", ctypes.byref(c or cache()), ctypes.byref(b or batch()),
           dtype, projected, row_stride, heads, split, query_scale, key_scale, stride, eps, inside,
           inv_freq, rotary, interleaved, scale, query, query_stride, None)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_normed_cache_refused(bad):
    c = cache()
    for name, value in bad.items():
        setattr(c, name, value)
    with pytest.raises(N.OpError, match="invalid_argument"):
        append_normed(c=c)


@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_normed_batch_refused(bad):
    b = batch()
    for name, value in bad.items():
        setattr(b, name, value)
    with pytest.raises(N.OpError, match="invalid_argument"):
        append_normed(b=b)


@pytest.mark.parametrize("bad", [
    dict(dtype=N.DTYPE_SPLIT), dict(projected=None), dict(projected=C + 2), dict(row_stride=511),
    dict(heads=0), dict(heads=3), dict(split=1), dict(inv_freq=None), dict(rotary=63),
    dict(rotary=66), dict(scale=0.0), dict(query=None), dict(query=B + 8), dict(query_stride=252),
    dict(query_scale=A + 4), dict(key_scale=A + 8), dict(stride=63), dict(stride=66),
    dict(stride=60), dict(stride=1 << 40), dict(eps=0.0), dict(eps=-1e-6), dict(eps=1.5),
    dict(eps=math.nan), dict(eps=math.inf)])
def test_normed_append_refused(bad):
    with pytest.raises(N.OpError, match="paged_append"):
        append_normed(**bad)


def test_normed_launch_beyond_32_bit_threads_refused():
    with pytest.raises(N.OpError, match="grid too large"):
        append_normed(b=batch(tokens=1 << 24, max_tokens=4))


def logprobs(dtype=N.DTYPE_F32, logits=A, rows=3, vocab=512, stride=512, tokens=B, logprob=C,
             rank=C, entropy=C, top=4, top_tokens=C, top_logprobs=C, workspace=None, size=0):
    N.call("evo_hip_token_logprobs", dtype, logits, rows, vocab, stride, tokens, logprob, rank,
           entropy, top, top_tokens, top_logprobs, workspace, size, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=N.DTYPE_SPLIT), dict(dtype=99), dict(logits=None), dict(logits=A + 2),
    dict(logits=A + 1, dtype=N.DTYPE_BF16), dict(rows=0), dict(rows=(1 << 20) + 1), dict(vocab=0),
    dict(vocab=(1 << 20) + 1, stride=1 << 21), dict(stride=511), dict(tokens=None),
    dict(tokens=None, rank=None), dict(top=65), dict(top=9, vocab=8), dict(top_tokens=None),
    dict(top_logprobs=None), dict(logprob=None, rank=None, entropy=None, top=0)])
def test_logprobs_refused(bad):
    with pytest.raises(N.OpError, match="token_logprobs"):
        logprobs(**bad)


def test_logprobs_workspace_refused():
    need = N.call("evo_hip_token_logprobs_workspace_bytes", 3, 5000, 4)
    assert need > 0 and N.call("evo_hip_token_logprobs_workspace_bytes", 3, 2048, 4) == 0
    for workspace, size in ((None, need), (C, need - 1), (C + 8, need)):
        with pytest.raises(N.OpError, match="workspace"):
            logprobs(vocab=5000, stride=5000, workspace=workspace, size=size)


def test_logprobs_launch_beyond_32_bit_threads_refused():
    with pytest.raises(N.OpError, match="grid too large"):
        logprobs(rows=1 << 20, vocab=1 << 20, stride=1 << 20, top=0, workspace=A, size=1 << 62)


def adapters(pool=None, adapter=A, x_hi=B, x_lo=C, x_stride=64, rows=5, residual=None, out=A,
             out_stride=40, workspace=B, size=1 << 40):
    fields = dict(adapters=3, rank=16, in_width=64, out_width=40, down=A, up=B)
    struct = N.Adapters(**fields)
    for name, value in (pool or {}).items():
        setattr(struct, name, value)
    N.call("evo_hip_adapter_linear", ctypes.byref(struct), adapter, x_hi, x_lo, x_stride, rows,
           residual, out, out_stride, workspace, size, None)


@pytest.mark.parametrize("bad", [
    dict(struct_size=8), dict(adapters=0), dict(adapters=8193), dict(rank=0), dict(rank=12),
    dict(rank=136), dict(in_width=0), dict(in_width=60), dict(in_width=1 << 25), dict(out_width=0),
    dict(out_width=1 << 25), dict(down=None), dict(up=None), dict(down=A + 8), dict(up=A + 2),
    dict(down_stride=16 * 64 - 8), dict(down_stride=16 * 64 + 4), dict(up_stride=16),
    dict(up_stride=1 << 41)])
def test_adapter_pool_refused(bad):
    with pytest.raises(N.OpError, match="invalid_argument"):
        adapters(pool=bad)
    fields = dict(adapters=3, rank=16, in_width=64, out_width=40, down=A, up=B)
    struct = N.Adapters(**fields)
    assert N.call("evo_hip_adapter_linear_workspace_bytes", ctypes.byref(struct), 5) > 0
    for name, value in bad.items():
        setattr(struct, name, value)
    assert N.call("evo_hip_adapter_linear_workspace_bytes", ctypes.byref(struct), 5) == 0


@pytest.mark.parametrize("bad", [
    dict(adapter=None), dict(adapter=A + 2), dict(x_hi=None), dict(x_hi=B + 8), dict(x_lo=C + 2),
    dict(x_stride=56), dict(x_stride=68), dict(rows=0), dict(rows=(1 << 20) + 1), dict(out=None),
    dict(out=A + 2), dict(residual=A + 1), dict(out_stride=39), dict(workspace=None),
    dict(workspace=B + 8), dict(size=100)])
def test_adapter_call_refused(bad):
    with pytest.raises(N.OpError, match="invalid_argument"):
        adapters(**bad)


def test_null_pool_refused():
    with pytest.raises(N.OpError, match="null"):
        N.call("evo_hip_adapter_linear", None, A, B, C, 64, 5, None, A, 40, B, 1 << 40, None)
    assert N.call("evo_hip_adapter_linear_workspace_bytes", None, 5) == 0


@pytest.mark.parametrize("bad", [
    dict(stride=(1 << 40) + 1), dict(tokens=B + 2), dict(logprob=C + 1), dict(rank=C + 2),
    dict(entropy=C + 3), dict(top_tokens=C + 2), dict(top_logprobs=C + 2)])
def test_logprobs_strides_and_alignment_refused(bad):
    with pytest.raises(N.OpError, match="token_logprobs"):
        logprobs(**bad)


@pytest.mark.parametrize("name", ["scales", "ranks", "error"])
def test_misaligned_adapter_arrays_refused(name):
    with pytest.raises(N.OpError, match="4-byte aligned"):
        adapters(pool={name: A + 2})
