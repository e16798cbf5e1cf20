"""Paged attention at the ends of its numeric range: scores far beyond 2^24."""
import math

import pytest
import torch

from paged_util import DEVICE, Paged, attend, exact_attention, half_step

pytestmark = pytest.mark.gpu

# Batches of 16-row and of 128-row blocks, of one chunk and of several, and behind a prefix.
BATCHES = [([(1, 700), (2, 90)], 0, 4, 2), ([(1, 9000)], 0, 2, 1), ([(40, 300), (7, 50)], 0, 4, 2),
           ([(150, 3000)], 0, 1, 1), ([(1, 100), (1, 90)], 64, 4, 4),
           ([(20, 1200), (1, 600)], 512, 4, 1)]


def whole_numbers(p, *shape):
    return torch.randint(-3, 4, shape, generator=p.gen, device=DEVICE).float()


@pytest.mark.parametrize("sequences,shared,heads,kv_heads", BATCHES)
@pytest.mark.parametrize("kind,dim,power", [("bf16", 64, 4), ("bf16", 64, 8), ("bf16", 128, 11),
                                            ("bf16", 64, 14), ("bf16", 32, 30), ("f16", 64, 4),
                                            ("f16", 64, 8), ("f16", 128, 9)])
@pytest.mark.parametrize("sign", [1, -1])
def test_far_scores(sequences, shared, heads, kv_heads, kind, dim, power, sign):
    """Scores of 2^17 to 2^70 (FP16: 2^25 to 2^35) and all of one sign, exact in F32: products of whole numbers
    times 2^(2 power), 4096 of them in the first element and at most 9 in each other one. Two
    scores are equal or at least 2^(2 power) * scale apart, 22, and the keys are copies of
    six, so that the largest score is met in many steps and chunks. Equal weights are exact
    in 16 bits, the others are below 2^-32, 2^-18 for all 9000 keys at most. A row is off by
    them, by its F32 sums (a lane adds less than 2^10 values, the rest is a tree: below
    2^-13 of the values' size) and by one rounding of the output."""
    p = Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind, shared=shared)
    few, query = whole_numbers(p, 6, kv_heads, dim), whole_numbers(p, p.tokens, heads, dim)
    few[..., 0], query[..., 0] = 64.0 * sign, 64.0
    none = p.keys.isnan()
    which = torch.randint(0, 6, (p.pages, p.page), generator=p.gen, device=DEVICE)
    p.keys.copy_((few * 2.0 ** power)[which].transpose(1, 2).to(p.kind))
    p.keys.masked_fill_(none, math.nan)
    query = (query * 2.0 ** power).view(p.tokens, heads * dim).to(p.kind)
    scale = dim ** -0.5 * (256 if kind == "f16" else 1)
    out = attend(p, query, scale).view(p.tokens, heads, dim).double()
    expected, _ = exact_attention(p, query, scale)
    room = p.values.nan_to_num().abs().max().double() * 2.0 ** -12 + \
        expected.abs() * half_step(p.kind)
    assert torch.isfinite(out).all()
    assert ((out - expected).abs() <= room).all()


@pytest.mark.parametrize("sequences,shared,heads,kv_heads", BATCHES)
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_around_a_thousand(sequences, shared, heads, kv_heads, sign):
    """Largest scores of a row on both sides of 1024 in units of ln 2 (1012 and 1044, 71 more
    or less), exact in F32, and a softmax over many keys: 128-row blocks form a weight in
    another way beyond it. Its exponent is off by one rounding at 1115 (2^-14), where chunks
    of both ways meet by twice that: below 2^-13 of a weight, and as much in the sum. The weights' rounding counts twice, as the rounded ones are summed."""
    dim = 32
    p = Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, shared=shared)
    query = whole_numbers(p, p.tokens, heads, dim)
    none = p.keys.isnan()
    keys = whole_numbers(p, *p.keys.shape)
    keys[..., 0], query[..., 0] = 64.0 * sign, 62.0 if sign > 0 else 64.0
    p.keys.copy_(keys.to(p.kind))
    p.keys.masked_fill_(none, math.nan)
    query = query.view(p.tokens, heads * dim).to(p.kind)
    scale = dim ** -0.5
    out = attend(p, query, scale).view(p.tokens, heads, dim).double()
    expected, _ = exact_attention(p, query, scale)
    values, p.values = p.values, p.values.abs()
    size, _ = exact_attention(p, query, scale)  # sum of p |v|
    p.values = values
    u = half_step(p.kind)
    room = size * (2 * u * (1 + 4 * u) + 2.0 ** -12) + expected.abs() * u
    assert ((out - expected).abs() <= room * (1 + u)).all()


@pytest.mark.parametrize("heads,kv_heads,n,length,kind,dim", [
    (2, 2, 12, 300, "bf16", 64), (8, 2, 4, 900, "f16", 128), (4, 4, 100, 500, "bf16", 128),
    (8, 2, 40, 700, "f16", 64), (2, 1, 40, 5000, "bf16", 32), (1, 1, 10, 5000, "f16", 64)])
def test_large_later_key_leaves_earlier_rows(heads, kv_heads, n, length, kind, dim):
    """A key that one row and those after it see gets far larger scores than any other:
    the rows before it keep their bits, and another sequence's."""
    p = Paged([(n, length), (3, 20)], heads=heads, kv_heads=kv_heads, dim=dim, kind=kind)
    query = p.normal(p.tokens, heads * dim, std=1.5)
    clean = attend(p, query, dim ** -0.5)
    for position in (length - 1, length - 2, length - n // 2):
        row = position - (length - n)
        at = p.page_of(0, position), slice(None), position % p.page
        kept = p.keys[at].clone()
        own = query[row:n].view(n - row, kv_heads, heads // kv_heads, dim).float().sum((0, 2))
        p.keys[at] = (own * (60.0 / own.norm(dim=-1, keepdim=True))).to(p.kind)
        out = attend(p, query, dim ** -0.5)
        p.keys[at] = kept
        assert torch.equal(out[:row], clean[:row]) and torch.equal(out[n:], clean[n:])
        assert not torch.equal(out[row:n], clean[row:n])


@pytest.mark.parametrize("sequences,shared,heads,kv_heads", [
    ([(1, 330), (1, 400), (1, 321)], 320, 2, 2), ([(2, 900)] * 3, 640, 4, 2),
    ([(30, 400), (25, 500), (9, 900)], 320, 4, 4), ([(1, 2100)] * 150, 2048, 4, 2)])
@pytest.mark.parametrize("kind,dim", [("bf16", 64), ("f16", 128)])
def test_other_sequences_queries_leave_a_row(sequences, shared, heads, kv_heads, kind, dim):
    """Behind a shared prefix rows of all sequences share a block: one sequence's queries
    ten times as large change no bit of another's rows."""
    p = Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind, shared=shared)
    query = p.normal(p.tokens, heads * dim, std=1.5)
    clean = attend(p, query, dim ** -0.5)
    n, other = sequences[0][0], query.clone()
    other[n:n + sequences[1][0]] *= 10.0
    out = attend(p, other, dim ** -0.5)
    rest = torch.ones(p.tokens, dtype=torch.bool)
    rest[n:n + sequences[1][0]] = False
    assert torch.equal(out[rest], clean[rest])
    assert not torch.equal(out[~rest], clean[~rest])


@pytest.mark.parametrize("step", [13.5, 15.5, 20, 23.5, 26, 28.5])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("rows,length,heads,shared", [
    (1, 16000, 1, 0), (40, 16000, 1, 0), (1, 300, 4, 0), (100, 400, 2, 0), (2, 4200, 2, 4096),
    (70, 4300, 2, 4096)])
def test_many_small_fp16_weights(step, first, rows, length, heads, shared):
    """One key takes 2^step times the weight of every other, and its values are small: the
    others, down to 2^-28.5, make the row. Scores are exact: (step, 0, ..) times ln 2. The
    bound counts the weights' rounding twice, as the rounded ones are summed: relative, or
    for each key half the spacing of FP16's smallest values, 2^-25, where the largest weight
    is 2^9 and more; F32 sums, below 2^-14; the output's rounding."""
    dim = 64
    p = Paged([(rows, length)], heads=heads, kv_heads=1, dim=dim, kind="f16", shared=shared)
    query = torch.zeros(rows, heads, dim, device=DEVICE)
    query[..., 0] = 1.0
    query = query.view(rows, heads * dim).to(p.kind)
    none = p.keys.isnan()
    p.keys.zero_()
    # (Every row sees both places.)
    place = 0 if first else length - rows
    at = p.page_of(0, place), slice(None), place % p.page
    p.keys[at + (0,)] = float(step)
    p.keys.masked_fill_(none, math.nan)
    p.values.copy_((p.values.abs() + 0.5) * 512.0)
    p.values[at] = 2.0 ** -10
    scale = math.log(2.0)
    out = attend(p, query, scale).view(rows, heads, dim).double()
    expected, _ = exact_attention(p, query, scale)
    u, most = half_step(p.kind), p.values.nan_to_num().double().abs().max()
    room = expected * (2 * u * (1 + 4 * u) + 2.0 ** -14 + u) + 2 * length * 2.0 ** -34 * most
    assert ((out - expected).abs() <= room + torch.finfo(p.kind).smallest_normal * u * 2).all()


@pytest.mark.parametrize("n,length,heads,kv_heads", [(3, 200, 4, 2), (40, 300, 2, 2), (1, 3000, 1, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_scores_of_minus_infinity(n, length, heads, kv_heads, kind):
    """Keys whose scores are -infinity have no weight; rows that see no other are zero."""
    p = Paged([(n, length)], heads=heads, kv_heads=kv_heads, dim=64, kind=kind)
    query = p.normal(n, heads, 64)
    query[..., 0] = 1.0
    query = query.view(n, -1).contiguous()
    first = length - n + 1  # The first row sees only what lies before this position.
    for position in range(length):
        if position < first - 1 or position % 3 == 0:
            p.keys[p.page_of(0, position), :, position % p.page, 0] = -math.inf
    out = attend(p, query, 0.125)
    everything = p.keys.clone()
    p.keys[..., 0].masked_fill_(~p.keys[..., 0].isnan(), -math.inf)
    assert (attend(p, query, 0.125) == 0).all()
    p.keys.copy_(everything)
    seen = [i for i in range(length) if not (i < first - 1 or i % 3 == 0)]
    rows = query.view(n, heads, 64).double()
    if not seen:
        assert (out == 0).all()
        return
    at = torch.tensor(seen, device=DEVICE)
    pages = torch.tensor([p.page_of(0, i) for i in seen], device=DEVICE)
    k, v = (pool[pages, :, at % p.page].double().repeat_interleave(heads // kv_heads, 1)
            for pool in (p.keys, p.values))
    for row in range(n):
        mine = at <= length - n + row
        if not mine.any():
            assert (out[row] == 0).all()
            continue
        w = torch.softmax(torch.einsum("hd,khd->hk", rows[row], k[mine]) * 0.125, 1)
        expected, size = (torch.einsum("hk,khd->hd", w, x[mine]) for x in (v, v.abs()))
        u = half_step(p.kind)
        # (Scores: sums of 64 products of size 64 at most in all, 72 roundings, felt twice.)
        room = size * (2 * u * (1 + 4 * u) + 2 * 72 * 64 * 2.0 ** -24) + expected.abs() * u
        assert ((out[row].view(heads, 64).double() - expected).abs() <= room * (1 + u) + 1e-6).all()


@pytest.mark.parametrize("sequences,shared,heads,kv_heads", BATCHES)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("what", [1000.0, 1e30, math.inf, math.nan])
def test_one_rows_query_leaves_the_others(sequences, shared, heads, kv_heads, kind, what):
    """A row of far larger scores, of infinite ones, or of NaN, in a block of others."""
    p = Paged(sequences, heads=heads, kv_heads=kv_heads, dim=64, kind=kind, shared=shared)
    query = p.normal(p.tokens, heads * 64, std=1.5)
    clean = attend(p, query, 0.125)
    row = p.tokens // 2
    other = query.clone()
    other[row] = (query[row].float() * what).to(p.kind)
    out = attend(p, other, 0.125)
    rest = torch.arange(p.tokens) != row
    assert torch.equal(out[rest], clean[rest])
    assert not torch.equal(out[row], clean[row])


@pytest.mark.parametrize("n,length,heads,kv_heads,dim", [
    (10, 300, 2, 2, 64), (40, 300, 2, 2, 64), (100, 900, 4, 2, 128), (70, 5000, 1, 1, 32)])
def test_leading_key_of_far_scores_with_an_infinite_value(n, length, heads, kv_heads, dim):
    """Scores near 2^34 that are not exact in F32, and a key that leads every row which sees
    it by 2^30 and more: these rows are its values, one of them infinite."""
    p = Paged([(n, length), (3, 20)], heads=heads, kv_heads=kv_heads, dim=dim)
    query = p.normal(p.tokens, heads, dim, std=2e4)
    query[..., 0] = 2.0 ** 17
    query = query.view(p.tokens, -1)
    none = p.keys.isnan()
    p.keys.copy_(p.keys.float() * 2e4).masked_fill_(none, math.nan)
    position = length - n + 1
    at = p.page_of(0, position), slice(None), position % p.page
    p.keys[at + (0,)] = 2.0 ** 19
    p.values[at + (dim - 3,)] = math.inf
    out = attend(p, query, dim ** -0.5).view(p.tokens, kv_heads, heads // kv_heads, dim)
    expected = p.values[at][None, :, None].expand_as(out[1:n])
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[n:]).all()
    assert torch.equal(out[1:n], expected)
