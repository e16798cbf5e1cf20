"""Appending to a paged cache with the rotation, and the attention that reads it,
against their definitions in 64 bits: ragged batches, grouped heads, shared
prefixes, padding, pages that end inside a tile, and device arrays that hold
nonsense."""
import ctypes

import pytest
import torch

from evo_hip import native as N
from paged_util import (CODES, DEVICE, KINDS, Paged, attend, check_attention, exact_attention,
                        exact_rotation, half_step)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- append
def append(p, projected, inv_freq, rotary, interleaved=False, scale=1.0, split=False, query=None,
           stream=None, **change):
    if query is None:
        query = torch.full((p.tokens, p.heads * p.dim), 77.0, dtype=p.kind, device=p.device)
    stream = torch.cuda.current_stream(p.device) if stream is None else stream
    N.call("evo_hip_paged_append", p.cache(), p.batch(**change), CODES[projected.dtype],
           projected.data_ptr(), projected.stride(0), p.heads, int(split),
           inv_freq.data_ptr() if rotary else None, rotary, int(interleaved), scale,
           query.data_ptr(), query.stride(0), stream.cuda_stream)
    return query


def frequencies(rotary, device=DEVICE):
    return 10000.0 ** (-torch.arange(0, max(rotary, 2), 2, device=device) / max(rotary, 2))


def within(got, expected, far, kind):
    u = half_step(kind)
    room = far * (1 + u) + expected.abs() * u + torch.finfo(kind).smallest_normal * u * 2
    excess = (got.double() - expected).abs() - room
    assert excess.max() <= 0, f"{excess.max()} beyond the bound"


def check_append(p, projected, rotary, interleaved=False, scale=1.0, split=False):
    """Every slot of the pools is looked at: those not appended to keep their bits."""
    before = p.keys.clone(), p.values.clone()
    inv_freq = frequencies(rotary)
    query = append(p, projected, inv_freq, rotary, interleaved, scale, split)
    heads, kv, dim = p.heads, p.kv_heads, p.dim
    x = projected[:, :(heads + 2 * kv) * dim].double()
    if split:
        x = x.view(-1, heads, 3, dim)
        q, k, v = x[:, :, 0], x[:, :, 1], x[:, :, 2]
    else:
        x = x.view(-1, heads + 2 * kv, dim)
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    rows = list(p.rows())
    owned = [r for r in rows if r[2] >= 0]
    padding = [r for r, _, position in rows if position < 0]
    if owned:
        at = torch.tensor([r for r, _, _ in owned], device=DEVICE)
        position = torch.tensor([position for _, _, position in owned], device=DEVICE)
        page = torch.tensor([p.page_of(s, q) for _, s, q in owned], device=DEVICE)
        slot = position % p.page
        for got, source in ((query.view(-1, heads, dim)[at], q[at]),
                            (p.keys[page, :, slot], k[at])):
            expected, far = exact_rotation(source, position, inv_freq, rotary, interleaved, scale)
            within(got, expected, far, p.kind)
        assert torch.equal(p.values[page, :, slot], v[at].to(p.kind))
        for pool, old in zip((p.keys, p.values), before):
            old[page, :, slot] = pool[page, :, slot]
    for pool, old in zip((p.keys, p.values), before):
        assert torch.equal(pool.isnan(), old.isnan())
        assert torch.equal(pool.nan_to_num(), old.nan_to_num())
    assert (query[padding] == 0).all()
    assert (query[len(rows):] == 77.0).all()
    assert p.error.item() == 0


@pytest.mark.parametrize("dim,rotary,interleaved", [
    (128, 128, False), (128, 128, True), (128, 32, False), (128, 32, True), (64, 64, False),
    (64, 24, False), (64, 24, True), (64, 2, False), (64, 2, True), (32, 32, False),
    (32, 32, True), (32, 8, False), (128, 120, False), (128, 118, True), (64, 0, False)])
@pytest.mark.parametrize("source,kind", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"),
                                         ("f32", "f16")])
def test_append_rotations(dim, rotary, interleaved, source, kind):
    p = Paged([(5, 21), (1, 1), (0, 30), (3, 16), (17, 49)], dim=dim, kind=kind, seed=rotary)
    projected = p.normal(p.tokens, (p.heads + 2 * p.kv_heads) * dim, kind=KINDS[source])
    check_append(p, projected, rotary, interleaved, scale=4.0)


@pytest.mark.parametrize("heads,kv_heads,page,layout,split", [
    (32, 32, 64, "dense", True), (32, 8, 16, "token", False), (15, 15, 128, "dense", True),
    (7, 1, 32, "token", False), (1, 1, 16, "dense", True), (28, 4, 16, "dense", False)])
def test_append_heads_and_strides(heads, kv_heads, page, layout, split):
    p = Paged([(1, 1000), (40, 40), (2, 17)], heads=heads, kv_heads=kv_heads, dim=128, page=page,
              layout=layout, seed=heads)
    projected = p.normal(p.tokens, (heads + 2 * kv_heads) * 128, kind=torch.float32)
    check_append(p, projected, 128, split=split, scale=16.0)


@pytest.mark.parametrize("offset,extra", [(0, 8), (1, 0), (1, 3), (4, 4)])
@pytest.mark.parametrize("source", ["f32", "bf16"])
def test_append_from_unaligned_rows(offset, extra, source):
    """Rows inside a larger tensor that start anywhere."""
    p = Paged([(9, 30), (2, 2)], dim=64)
    width = (p.heads + 2 * p.kv_heads) * 64 + extra
    whole = p.normal(p.tokens * width + offset, kind=KINDS[source])
    check_append(p, whole[offset:].view(p.tokens, width), 48)


def test_append_many_rows():
    """Enough rows for a block each, with padding and rows behind the last sequence."""
    p = Paged([(700, 700), (0, 0), (300, 4000), (20, 12), (3, 0)], heads=8, kv_heads=2, dim=64,
              page=32, trailing=5)
    check_append(p, p.normal(p.tokens, 12 * 64, kind=torch.float32), 64)


@pytest.mark.parametrize("position", [2 ** 20 - 1, 2 ** 24 + 1, 2 ** 29 - 1])
def test_append_far_position(position):
    """The angle of a position beyond 2^24 keeps its fraction of a turn. (A length on the
    device whose earlier pages the table does not hold.)"""
    p = Paged([(1, 1)], dim=64, page=32768)
    index = position >> 15
    table = p.ints([[-1] * index + [p.pages - 1]])
    p.lengths.fill_(position + 1)
    projected = p.normal(1, 8 * 64, kind=torch.float32)
    inv_freq = frequencies(64)
    query = append(p, projected, inv_freq, 64, max_length=position + 1,
                   page_table=table.data_ptr(), table_stride=index + 1)
    expected, far = exact_rotation(projected.view(1, 8, 64)[:, :6],
                                   torch.tensor([position], device=DEVICE), inv_freq, 64, False,
                                   1.0)
    within(query.view(1, 4, 64), expected[:, :4], far[:, :4], p.kind)
    within(p.keys[p.pages - 1, :, position % 32768][None], expected[:, 4:], far[:, 4:], p.kind)
    assert p.error.item() == 0


def test_append_nonfinite_values_stay_apart():
    """An infinity or NaN reaches its own pair, no neighbour that does not turn with it."""
    p = Paged([(1, 3)], dim=64)
    projected = p.normal(1, 8 * 64, kind=torch.float32)
    projected[0, 5], projected[0, 40] = float("inf"), float("nan")
    for interleaved, rotary, touched in ((False, 24, {5, 17, 40}), (True, 10, {4, 5, 40}),
                                         (False, 32, {5, 21, 40}), (True, 4, {5, 40})):
        query = append(p, projected, frequencies(rotary), rotary, interleaved)
        bad = (~torch.isfinite(query[0, :64].float())).nonzero()[:, 0].tolist()
        assert set(bad) == touched


# -------------------------------------------------------------- attention
RAGGED = [(1, 1), (1, 16), (1, 17), (1, 300), (1, 31), (1, 1025)]


def run(p, std=1.5, scale=None, **change):
    query = p.normal(p.tokens, p.heads * p.dim, std=std)
    scale = p.dim ** -0.5 if scale is None else scale
    out = attend(p, query, scale, **change)
    check_attention(p, query, scale, out)
    assert p.error.item() == 0


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (32, 8), (7, 1), (28, 4), (48, 3), (1, 1)])
@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("f16", 128), ("bf16", 64), ("f16", 32)])
def test_attention_single_tokens(heads, kv_heads, kind, dim):
    run(Paged(RAGGED, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind, seed=heads))


@pytest.mark.parametrize("page,layout", [(16, "dense"), (32, "token"), (64, "dense"),
                                         (256, "token"), (1024, "dense")])
def test_attention_pages_and_strides(page, layout):
    run(Paged([(1, 700), (3, 50), (1, 1), (64, 64), (33, 1000)], page=page, layout=layout, dim=128,
              heads=8, kv_heads=2))


@pytest.mark.parametrize("sequences", [
    [(1, 1)], [(2, 2)], [(15, 15)], [(16, 16)], [(17, 33)], [(100, 100)], [(129, 513)],
    [(64, 64), (65, 65), (63, 63)], [(0, 5), (300, 300), (0, 0), (1, 900)], [(513, 2000)]])
@pytest.mark.parametrize("heads,kv_heads,kind,dim", [(3, 3, "bf16", 128), (8, 2, "f16", 64),
                                                     (5, 1, "bf16", 32)])
def test_attention_prompts(sequences, heads, kv_heads, kind, dim):
    run(Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind, trailing=3))


@pytest.mark.parametrize("shared,sequences", [
    (16, [(1, 17), (1, 40)]), (64, [(1, 65)]), (512, [(1, 513 + 7 * i) for i in range(40)]),
    (1600, [(1, 1601), (5, 1700), (0, 1600), (0, 0), (1, 2300)]),
    (128, [(33, 161), (1, 129), (20, 400)]), (2048, [(70, 2118), (70, 2200)])])
@pytest.mark.parametrize("heads,kv_heads,kind,dim", [(4, 4, "bf16", 128), (8, 2, "f16", 64),
                                                     (7, 1, "bf16", 32)])
def test_attention_shared_prefix(shared, sequences, heads, kv_heads, kind, dim):
    run(Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind, shared=shared,
              trailing=2))


@pytest.mark.parametrize("sequences,shared,heads,kv_heads", [
    ([(1, 40000)], 0, 2, 1), ([(2, 20001), (1, 3)], 0, 3, 1), ([(1, 33000), (2, 40000)], 32768, 2, 2),
    ([(40, 30000)], 0, 1, 1), ([(1, 16400)] * 9, 16384, 4, 4)])
def test_attention_many_chunks(sequences, shared, heads, kv_heads):
    """Rows of more chunks than a wave has lanes, and both ways of joining them."""
    run(Paged(sequences, heads=heads, kv_heads=kv_heads, dim=64, page=128, shared=shared))


@pytest.mark.parametrize("shared", [0, 64])
def test_attention_many_sequences(shared):
    """More sequences than a wave looks at together, single tokens among prompts."""
    counts = [1 + (37 * i) % 5 if i % 7 else 30 + i for i in range(150)]
    sequences = [(n, shared + n + (13 * i) % 50) for i, n in enumerate(counts)]
    run(Paged(sequences, heads=4, kv_heads=2, dim=64, shared=shared, trailing=1))
    run(Paged([(1, shared + 1 + (29 * i) % 90) for i in range(300)], heads=4, kv_heads=2, dim=32,
              shared=shared))


def test_shared_prefix_matches_own_pages():
    """The same batch with the prefix's pages in every table row: the same rows, within
    the bounds of both."""
    shared = 320
    p = Paged([(1, 321), (4, 400), (2, 322)], shared=shared, dim=128, heads=8, kv_heads=2)
    query = p.normal(p.tokens, 8 * 128)
    apart = attend(p, query, 0.09)
    check_attention(p, query, 0.09, apart)
    p.table[:, :shared // p.page] = p.shared_table
    whole = attend(p, query, 0.09, shared_length=0, shared_table=None)
    check_attention(p, query, 0.09, whole)


@pytest.mark.parametrize("heads,kv_heads,n,length,kind,dim", [
    (4, 4, 7, 7, "bf16", 128), (4, 4, 9, 300, "f16", 128), (8, 2, 4, 40, "bf16", 64),
    (2, 1, 8, 70, "f16", 32), (4, 4, 100, 100, "bf16", 128), (8, 2, 90, 700, "f16", 128),
    (7, 1, 40, 41, "bf16", 64), (4, 2, 70, 130, "f16", 32)])
@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_nonfinite_values_reach_only_rows_that_see_them(heads, kv_heads, n, length, kind, dim,
                                                        what):
    """A value and then a key of a later row: the rows before it keep their bits, the
    others get it where the definition puts it."""
    p = Paged([(n, length), (3, 20)], heads=heads, kv_heads=kv_heads, dim=dim, kind=kind)
    query = p.normal(p.tokens, heads * dim)
    clean = attend(p, query, dim ** -0.5).view(-1, heads, dim)
    for position in (length - n + 1, length - 2, length - 1):
        row, kv, d = position - (length - n), kv_heads - 1, dim - 3
        mine = slice(kv * (heads // kv_heads), heads)
        at = p.page_of(0, position), kv, position % p.page, d
        kept = p.values[at].clone()
        p.values[at] = what
        out = attend(p, query, dim ** -0.5).view(-1, heads, dim)
        p.values[at] = kept
        touched = out[row:n, mine]
        assert torch.equal(out[:row], clean[:row]) and torch.equal(out[n:], clean[n:])
        got = touched[..., d].float()
        assert got.isnan().all() if what != what else (got == what).all()
        p.values[at] = 0.0
        expected, far = exact_attention(p, query, dim ** -0.5)
        p.values[at] = kept
        rest = [e for e in range(dim) if e != d]
        assert ((touched[..., rest].double() - expected[row:n, mine][..., rest]).abs() <=
                far[row:n, mine][..., rest]).all()
        kept = p.keys[at].clone()
        p.keys[at] = float("nan")
        out = attend(p, query, dim ** -0.5).view(-1, heads, dim)
        p.keys[at] = kept
        assert torch.equal(out[:row], clean[:row]) and torch.equal(out[n:], clean[n:])
        assert out[row:n, mine].isnan().all()


@pytest.mark.parametrize("heads,kv_heads,n,length,kind,dim", [
    (2, 1, 40, 6000, "bf16", 64), (4, 4, 3, 5000, "f16", 128), (1, 1, 150, 9000, "bf16", 32)])
@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_nonfinite_values_in_rows_of_many_chunks(heads, kv_heads, n, length, kind, dim, what):
    test_nonfinite_values_reach_only_rows_that_see_them(heads, kv_heads, n, length, kind, dim,
                                                        what)


def test_attention_rows_without_keys_are_zero():
    p = Paged([(3, 0), (5, 2), (1, 1), (40, 7), (0, 0)], dim=64, trailing=4)
    run(p)
    q = p.normal(p.tokens, p.heads * p.dim)
    out = attend(p, q, 0.125)
    assert (out[:3] == 0).all() and (out[3:6] == 0).all() and (out[9:42] == 0).all()


def test_shared_prefix_beside_an_empty_sequence():
    p = Paged([(2, 0), (1, 70), (3, 0)], shared=64, dim=64, trailing=1)
    run(p)


def test_attention_sharp_and_flat_scores():
    """Scores hundreds apart (one key takes all), and all equal."""
    run(Paged([(1, 500), (20, 300)], dim=64), std=60.0)
    p = Paged([(1, 500), (20, 300)], dim=64)
    run(p, std=0.0)


def test_attention_in_place_and_with_strides():
    p = Paged([(1, 90), (7, 30), (1, 16)], dim=64)
    wide = p.normal(p.tokens, p.heads * 64 + 40)
    query = wide[:, 8:8 + p.heads * 64]
    kept = query.clone()
    rest = wide.clone()
    attend(p, query, 0.125, out=query)
    check_attention(p, kept, 0.125, query.contiguous())
    rest[:, 8:8 + p.heads * 64] = query
    assert torch.equal(rest, wide)


def test_attention_long_cache():
    """Offsets beyond 2^31 elements, in the pages and in the table."""
    page, dim = 32768, 128
    p = Paged([(1, 20)], heads=1, kv_heads=1, dim=dim, page=page, spare=0)
    pages = 2 ** 32 // (page * dim) + 2  # 4.3e9 elements, 8.6 GB each
    small_keys, small_values = p.keys, p.values
    p.keys, p.values = (torch.empty(pages, 1, page, dim, dtype=p.kind, device=DEVICE)
                        for _ in range(2))
    p.keys[pages - 1, :, :20], p.values[pages - 1, :, :20] = small_keys[0, :, :20], \
        small_values[0, :, :20]
    p.pages, p.rows_of = pages, [[pages - 1]]
    p.table = p.ints([[pages - 1]])
    run(p)
    projected = p.normal(1, 3 * dim, kind=torch.float32)
    append(p, projected, frequencies(dim), 0)
    assert torch.equal(p.values[pages - 1, 0, 19], projected[0, 2 * dim:].to(p.kind))


# ------------------------------------------------- arrays that hold nonsense
def test_bad_pages_are_masked_and_reported():
    p = Paged([(1, 100), (1, 40), (6, 60)], dim=64)
    query = p.normal(p.tokens, p.heads * 64)
    for entry in (-1, p.pages, 2 ** 31 - 1, -2 ** 31):
        p.error.zero_()
        p.table[0, 2] = entry
        out = attend(p, query, 0.125)
        assert p.error.item() == N.PAGED_BAD_PAGE
        # Sequence 0 without positions 32 .. 47.
        q = query[0].view(p.heads, 64).double()
        at = [i for i in range(100) if not 32 <= i < 48]
        page = torch.tensor([p.page_of(0, i) for i in at], device=DEVICE)
        k, v = (pool[page, :, torch.tensor(at, device=DEVICE) % 16].double()
                .repeat_interleave(2, 1) for pool in (p.keys, p.values))
        w = torch.softmax(torch.einsum("hd,khd->hk", q, k) * 0.125, 1)
        expected = torch.einsum("hk,khd->hd", w, v)
        size = torch.einsum("hk,khd->hd", w, v.abs())
        u = half_step(p.kind)
        assert ((out[0].view(p.heads, 64).double() - expected).abs() <=
                size * (2.1 * u + 1e-4) + expected.abs() * u).all()
    everything = p.table.clone()
    p.table.fill_(-5)
    assert (attend(p, query, 0.125) == 0).all()  # nothing is left to see
    before = p.keys.clone().nan_to_num()
    p.error.zero_()
    append(p, p.normal(p.tokens, 8 * 64, kind=torch.float32), frequencies(64), 64)
    assert p.error.item() == N.PAGED_BAD_PAGE
    assert torch.equal(p.keys.nan_to_num(), before)
    p.table.copy_(everything)


@pytest.mark.parametrize("shared", [0, 32])
def test_bad_sequences_are_left_out_and_reported(shared):
    """Each kind of broken entry in one of three sequences: the others are served, its own
    rows and everything else stay as they were."""
    good = [(2, shared + 30), (3, shared + 50), (1, shared + 20)]
    broken = [("lengths", 1, -3), ("lengths", 1, 10 ** 6), ("lengths", 1, 2 ** 31 - 1),
              ("start", 3, 99), ("start", 3, 2)]
    if shared:
        broken.append(("lengths", 1, shared + 2))
    for name, at, value in broken:
        p = Paged(good, dim=64, shared=shared)
        query = p.normal(p.tokens, p.heads * 64)
        whole = attend(p, query, 0.125)
        getattr(p, name)[at] = value
        out = attend(p, query, 0.125)
        assert p.error.item() == N.PAGED_BAD_SEQUENCE
        rows = slice(2, 5) if name == "lengths" else slice(5, 6)
        served = torch.ones(p.tokens, dtype=torch.bool)
        served[rows] = False
        assert (out[rows] == 77.0).all()
        assert torch.equal(out[served], whole[served])
        before = p.keys.clone().nan_to_num()
        p.error.zero_()
        q = append(p, p.normal(p.tokens, 8 * 64, kind=torch.float32), frequencies(64), 64)
        assert (q[rows] == 77.0).all()
        changed = (p.keys.nan_to_num() != before).any(-1).any(1)
        assert changed.sum() == served.sum()


# ----------------------------------------------- streams, graphs, a run of them
def test_another_stream_and_two_at_once():
    p = [Paged([(1, 900), (9, 200)], dim=128, seed=i) for i in range(2)]
    query = [x.normal(x.tokens, x.heads * 128) for x in p]
    alone = [attend(x, q, 0.1) for x, q in zip(p, query)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(q) for q in query]
    for _ in range(4):
        for x, q, o, s in zip(p, query, outs, streams):
            with torch.cuda.stream(s):
                attend(x, q, 0.1, out=o, stream=s)
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        assert torch.equal(o, a)


def test_captured_step_follows_the_lengths():
    """A decode step (append, attention, sampling) in one graph: replays with longer
    lengths, eager work and synchronisation between them, each equal to the eager step."""
    p = Paged([(1, 200), (1, 90), (1, 33)], dim=64, shared=0)
    start = [180, 70, 20]
    vocab, width = 512, 8 * 64
    inv_freq = frequencies(64)
    projected = p.normal(3, width, kind=torch.float32)
    head = p.normal(vocab, p.heads * 64, std=0.3)
    uniform = torch.rand(3, generator=p.gen, device=DEVICE)
    need = N.call("evo_hip_paged_attention_workspace_bytes", p.cache(), p.batch(), p.heads)
    workspace = torch.zeros(max(16, need), dtype=torch.uint8, device=DEVICE)
    query = torch.zeros(3, p.heads * 64, dtype=p.kind, device=DEVICE)
    out, tokens = torch.zeros_like(query), torch.zeros(3, dtype=torch.int32, device=DEVICE)
    logits = torch.zeros(3, vocab, dtype=p.kind, device=DEVICE)

    def step(stream):
        append(p, projected, inv_freq, 64, query=query, stream=stream)
        attend(p, query, 0.125, out=out, stream=stream, workspace=workspace)
        torch.matmul(out, head.T, out=logits)
        N.call("evo_hip_sample", CODES[p.kind], logits.data_ptr(), 3, vocab, vocab, None, None,
               None, None, uniform.data_ptr(), tokens.data_ptr(), None, 0, stream.cuda_stream)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        p.lengths.copy_(p.ints(start))
        step(stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(stream)
    for i in range(1, 14):
        p.lengths.copy_(p.ints([n + i for n in start]))
        projected.copy_(p.normal(3, width, kind=torch.float32))
        keys, values = p.keys.clone(), p.values.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in (query, out, tokens, p.keys.nan_to_num(),
                                        p.values.nan_to_num())]
        p.keys.copy_(keys)
        p.values.copy_(values)
        step(torch.cuda.current_stream())
        torch.cuda.synchronize()
        for a, b in zip(replayed, (query, out, tokens, p.keys.nan_to_num(),
                                   p.values.nan_to_num())):
            assert torch.equal(a, b)
    assert p.error.item() == 0


def test_decode_step_by_step_matches_the_prompt():
    """A prompt appended and attended at once, and token by token, with the library's own
    product in front: the same keys bit for bit, outputs within both bounds."""
    tokens, width, dim = 70, 256, 64
    whole = Paged([(tokens, tokens)], dim=dim, heads=4, kv_heads=4, seed=3)
    x = whole.normal(tokens, width, kind=torch.bfloat16)
    w = whole.normal(12 * dim, width, std=width ** -0.5, kind=torch.bfloat16)
    projected = torch.empty(tokens, 12 * dim, device=DEVICE)
    N.call("evo_hip_linear", x.data_ptr(), None, w.data_ptr(), None, None, tokens, 12 * dim, width,
           projected.data_ptr(), torch.cuda.current_stream().cuda_stream)
    inv_freq = frequencies(dim)
    query = append(whole, projected, inv_freq, dim)
    at_once = attend(whole, query, 0.125)
    check_attention(whole, query, 0.125, at_once)
    steps = Paged([(1, tokens)], dim=dim, heads=4, kv_heads=4, seed=4)
    for i in range(tokens):
        steps.lengths.fill_(i + 1)
        q = append(steps, projected[i:i + 1], inv_freq, dim)
        assert torch.equal(q, query[i:i + 1])
        one = attend(steps, q, 0.125)
        steps.sequences = [(1, i + 1)]
        check_attention(steps, q, 0.125, one)
        steps.sequences = [(1, tokens)]
    for a, b in ((whole.keys, steps.keys), (whole.values, steps.values)):
        for i in range(tokens):
            assert torch.equal(a[whole.page_of(0, i), :, i % 16], b[steps.page_of(0, i), :, i % 16])
