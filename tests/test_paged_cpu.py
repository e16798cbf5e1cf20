"""The batched serving operators without a GPU: what their entry points refuse
before any launch, and the index rules that keep a kernel inside its tensors
whatever the device arrays hold."""
import ctypes
import os

import numpy as np
import pytest

from evo_hip import native as N

TESTLIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evo.cpp_amd",
                       "lib", "libevo_hip_testing.so")
A, B, C = 1 << 20, 1 << 21, 1 << 22  # addresses that no refused call follows


def cache(**change):
    fields = dict(dtype=N.DTYPE_BF16, key_pages=A, value_pages=B, pages=8, page_size=16,
                  kv_heads=2, head_dim=64)
    return N.PagedCache(**{**fields, **change})


def batch(**change):
    fields = dict(sequences=2, tokens=6, max_tokens=4, max_length=40, token_start=A, lengths=A,
                  page_table=A, table_stride=4)
    return N.PagedBatch(**{**fields, **change})


def append(c=None, b=None, dtype=N.DTYPE_F32, projected=C, row_stride=512, heads=4, split=0,
           inv_freq=A, rotary=64, interleaved=0, scale=1.0, query=B, query_stride=256):
    N.call("evo_hip_paged_append", ctypes.byref(c or cache()), ctypes.byref(b or batch()), dtype,
           projected, row_stride, heads, split, inv_freq, rotary, interleaved, scale, query,
           query_stride, None)


def attend(c=None, b=None, query=C, query_stride=256, heads=4, scale=0.125, out=B, out_stride=256,
           workspace=A, workspace_bytes=1 << 40):
    N.call("evo_hip_paged_attention", ctypes.byref(c or cache()), ctypes.byref(b or batch()),
           query, query_stride, heads, scale, out, out_stride, workspace, workspace_bytes, None)


BAD_CACHES = [dict(struct_size=8), dict(dtype=N.DTYPE_F32), dict(dtype=7), dict(key_pages=None),
              dict(value_pages=None), dict(key_pages=A + 2), dict(value_pages=A + 8),
              dict(pages=0), dict(pages=1 << 31), dict(page_size=0), dict(page_size=8),
              dict(page_size=48), dict(page_size=65536), dict(kv_heads=0), dict(kv_heads=65537),
              dict(head_dim=16), dict(head_dim=96), dict(head_dim=256),
              dict(page_stride=4096, head_stride=1024, token_stride=60),
              dict(page_stride=4096, head_stride=1024, token_stride=56),
              dict(page_stride=4100, head_stride=1024, token_stride=64),
              dict(page_stride=4096, head_stride=1024, token_stride=(1 << 24) + 8),
              dict(page_stride=2 ** 62, head_stride=1024, token_stride=64)]
BAD_BATCHES = [dict(struct_size=0), dict(sequences=0), dict(sequences=(1 << 20) + 1),
               dict(tokens=0), dict(tokens=(1 << 24) + 1), dict(max_tokens=0), dict(max_tokens=7),
               dict(max_length=0), dict(max_length=65), dict(max_length=1 << 31),
               dict(token_start=None), dict(lengths=None), dict(page_table=None),
               dict(shared_length=16), dict(shared_length=8, shared_table=A),
               dict(shared_length=48, shared_table=A)]


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("bad", BAD_CACHES)
def test_cache_refused(call, bad):
    c = cache()
    for name, value in bad.items():
        setattr(c, name, value)
    with pytest.raises(N.OpError, match="invalid_argument"):
        call(c=c)


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_batch_refused(call, bad):
    b = batch()
    for name, value in bad.items():
        setattr(b, name, value)
    with pytest.raises(N.OpError, match="invalid_argument"):
        call(b=b)


@pytest.mark.parametrize("bad", [
    dict(dtype=N.DTYPE_SPLIT), dict(dtype=99), dict(projected=None), dict(projected=C + 2),
    dict(projected=C + 1, dtype=N.DTYPE_BF16), dict(row_stride=511), dict(heads=0), dict(heads=3),
    dict(split=1), dict(inv_freq=None), dict(rotary=63), dict(rotary=66), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(query=None),
    dict(query=B + 8), dict(query_stride=255), dict(query_stride=252), dict(query_stride=248)])
def test_append_refused(bad):
    with pytest.raises(N.OpError, match="paged_append"):
        append(**bad)


@pytest.mark.parametrize("bad", [
    dict(query=None), dict(out=None), dict(query=C + 2), dict(out=C + 8), dict(query_stride=248),
    dict(out_stride=250), dict(heads=0), dict(heads=3), dict(heads=131072), dict(scale=0.0),
    dict(scale=float("nan")), dict(scale=float("inf"))])
def test_attention_refused(bad):
    with pytest.raises(N.OpError, match="paged_attention"):
        attend(**bad)


def test_in_place_with_another_stride_refused():
    """A row's output would lie on another row's query."""
    with pytest.raises(N.OpError, match="in place"):
        attend(query=B, out=B, query_stride=256, out_stride=264)


def test_launches_beyond_32_bit_threads_refused():
    """Rows that a launch could not count."""
    with pytest.raises(N.OpError, match="grid too large"):
        append(b=batch(tokens=1 << 24, max_tokens=4))
    with pytest.raises(N.OpError, match="too many rows|grid too large"):
        attend(b=batch(tokens=1 << 24, max_tokens=1 << 24), heads=256, query_stride=256 * 64,
               out_stride=256 * 64)
    with pytest.raises(N.OpError, match="grid too large"):
        attend(b=batch(sequences=1 << 20, tokens=1 << 20, max_tokens=1, max_length=1 << 16,
                       table_stride=1 << 12), c=cache(kv_heads=32), heads=32, query_stride=2048,
               out_stride=2048)


def test_rows_up_to_the_end_of_their_tile_refused():
    """2^31 - 128 rows of one key/value head: the end of the last tile is counted too."""
    with pytest.raises(N.OpError, match="too many rows"):
        attend(c=cache(kv_heads=1, head_dim=32),
               b=batch(tokens=(1 << 24) - 1, max_tokens=(1 << 24) - 1, max_length=40), heads=128,
               query_stride=128 * 32, out_stride=128 * 32)


def test_attention_workspace_refused():
    """A call whose keys are split needs all of its workspace."""
    b = batch(max_length=60, shared_length=32, shared_table=A)
    need = N.call("evo_hip_paged_attention_workspace_bytes", ctypes.byref(cache()),
                  ctypes.byref(b), 4)
    assert need > 0
    for workspace, size in ((None, need), (A, need - 1), (A + 4, need)):
        with pytest.raises(N.OpError, match="workspace"):
            attend(b=b, workspace=workspace, workspace_bytes=size)


@pytest.mark.parametrize("seed", range(4))
def test_attention_workspace_bound(seed):
    """Of any batch: whole slots of all rows, and two phases of at most 136 MB, or of
    one slot where that is more."""
    rng = np.random.default_rng(seed)
    for _ in range(500):
        def size(high, low=1):
            return int(np.exp(rng.uniform(np.log(low), np.log(high))))
        dim, page = int(rng.choice([32, 64, 128])), 16 << rng.integers(0, 8)
        kv_heads = size(64)
        heads = kv_heads * int(rng.choice([1, 2, 3, 4, 7, 8, 16, 32]))
        max_tokens, sequences = size(16384), size(2000)
        tokens = max(max_tokens, min(max_tokens * sequences, size(65536)))
        shared = page * (size(1 << 20) // page) if rng.random() < 0.5 else 0
        length = shared + max(max_tokens, size(1 << 21))
        c = cache(head_dim=dim, page_size=page, kv_heads=kv_heads, pages=1 << 20)
        b = batch(sequences=sequences, tokens=tokens, max_tokens=max_tokens, max_length=length,
                  table_stride=length // page + 1, shared_length=shared,
                  shared_table=A if shared else None)
        need = N.call("evo_hip_paged_attention_workspace_bytes", ctypes.byref(c),
                      ctypes.byref(b), heads)
        slot = tokens * heads * (dim + 2) * 4
        slots, rest = divmod(need, slot)
        assert rest == 0 and slots != 1 and slots <= 256 and (not shared or slots >= 2)
        assert need <= 2 * max(136e6, slot)


def test_workspace_query_of_refused_structs_is_zero():
    query = "evo_hip_paged_attention_workspace_bytes"
    assert N.call(query, ctypes.byref(cache(page_size=3)), ctypes.byref(batch()), 4) == 0
    assert N.call(query, ctypes.byref(cache()), ctypes.byref(batch(tokens=0)), 4) == 0
    assert N.call(query, ctypes.byref(cache()), ctypes.byref(batch()), 3) == 0
    assert N.call(query, None, None, 4) == 0


@pytest.mark.parametrize("bad", [
    dict(dtype=N.DTYPE_SPLIT), dict(logits=None), dict(logits=A + 2), dict(rows=0),
    dict(rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 20) + 1, stride=1 << 21),
    dict(stride=511), dict(uniform=None), dict(tokens=None)])
def test_sample_refused(bad):
    v = {**dict(dtype=N.DTYPE_F32, logits=A, rows=3, vocab=512, stride=512, uniform=A, tokens=B),
         **bad}
    with pytest.raises(N.OpError, match="sample"):
        N.call("evo_hip_sample", v["dtype"], v["logits"], v["rows"], v["vocab"], v["stride"], None,
               None, None, None, v["uniform"], v["tokens"], None, 0, None)


def test_sample_workspace_refused():
    need = N.call("evo_hip_sample_workspace_bytes", 4, 100000)
    assert need > 0
    assert N.call("evo_hip_sample_workspace_bytes", 4, 512) == 0
    for workspace, size in ((C, need - 1), (C + 8, need)):
        with pytest.raises(N.OpError, match="workspace"):
            N.call("evo_hip_sample", N.DTYPE_F32, A, 4, 100000, 100000, None, None, None, None, A,
                   B, workspace, size, None)


# ------------------------------------------------------------ index rules
@pytest.fixture(scope="module")
def rules():
    return ctypes.CDLL(TESTLIB)


def ints(values):
    return np.asarray(values, np.int32).ctypes.data_as(ctypes.POINTER(ctypes.c_int32))


LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("start,end,length,shared,valid", [
    (0, 3, 3, 0, True), (0, 3, 40, 0, True), (2, 6, 17, 0, True), (6, 6, 0, 0, True),
    (0, 3, 2, 0, True), (0, 3, 0, 0, True),            # more rows than positions: padding
    (0, 5, 9, 0, False),                               # above max_tokens
    (0, 3, 41, 0, False), (0, 3, -1, 0, False), (0, 3, LOW, 0, False),
    (-1, 2, 5, 0, False), (4, 3, 5, 0, False), (4, 7, 5, 0, False), (LOW, HIGH, 5, 0, False),
    (HIGH, LOW, 5, 0, False), (LOW, LOW, 5, 0, False), (HIGH, HIGH, 5, 0, False),
    (0, 3, 35, 32, True), (0, 3, 34, 32, False), (0, 3, 0, 32, True), (3, 3, 5, 32, True)])
def test_sequence_rows(rules, start, end, length, shared, valid):
    rows = (ctypes.c_int * 3)()
    sizes = ints([1, 6, 4, 40, shared])
    assert rules.evo_test_paged_rows(sizes, ints([start, end]), ints([length]), 0, rows) == valid
    if valid:
        assert list(rows) == [start, end - start, length]


@pytest.mark.parametrize("starts", [
    [0, 3, 3, 4, 9], [0, 0, 0, 0, 9], [2, 2, 5, 5, 5], [0, 9, 9, 9, 9], [0, 1],
    [5, 1, 8, 0, 9], [HIGH, LOW, HIGH, LOW, HIGH], [LOW, LOW, HIGH, HIGH, HIGH], [0, -5, 20, 3, 7]])
def test_sequence_of_row(rules, starts):
    """The owner of a row, and only a true one where the array is no ascending one."""
    n = len(starts) - 1
    sizes, lengths = ints([n, 9, 9, 40, 0]), ints([9] * n)
    ascending = sorted(starts) == starts
    for token in range(-1, 11):
        found = rules.evo_test_paged_sequence(sizes, ints(starts), lengths, token)
        owners = [s for s in range(n) if starts[s] <= token < starts[s + 1]]
        assert found in owners or found == -1
        if ascending:
            assert found == (owners[0] if owners else -1)


@pytest.mark.parametrize("entry,page", [(0, 0), (7, 7), (8, -1), (-1, -1), (LOW, -1), (HIGH, -1)])
def test_page_of_table(rules, entry, page):
    assert rules.evo_test_paged_page(ints([3, entry]), 1, 8) == page


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scale_beyond_its_binary_form_refused(scale):
    """A finite scale whose multiple by log2(e) is infinite: every weight would be NaN."""
    with pytest.raises(N.OpError, match="scale"):
        attend(scale=scale)
