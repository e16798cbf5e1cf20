"""The paged append of query and key heads that are normalized first, against its
definition in 64 bits: head layouts, both places of eps, scales of each head, values
whose squares leave F32, and heads of zeros."""
import math

import pytest
import torch

from evo_hip import native as N
from paged_util import CODES, DEVICE, KINDS, Paged, half_step
from test_gpu_paged import append, frequencies, within

pytestmark = pytest.mark.gpu


def append_normed(p, projected, query_scale, key_scale, eps, inside, rotary, interleaved=False,
                  scale=1.0, split=False, per_head=False, query=None, stream=None, **change):
    if query is None:
        query = torch.full((p.tokens, p.heads * p.dim), 77.0, dtype=p.kind, device=p.device)
    stream = torch.cuda.current_stream(p.device) if stream is None else stream
    inv_freq = frequencies(rotary)
    N.call("evo_hip_paged_append_normed", p.cache(), p.batch(**change), CODES[projected.dtype],
           projected.data_ptr(), projected.stride(0), p.heads, int(split),
           None if query_scale is None else query_scale.data_ptr(),
           None if key_scale is None else key_scale.data_ptr(),
           query_scale.stride(0) if per_head else 0, eps, int(inside),
           inv_freq.data_ptr() if rotary else None, rotary, int(interleaved), scale,
           query.data_ptr(), query.stride(0), stream.cuda_stream)
    inv_freq.record_stream(stream)
    return query


def exact_heads(x, weight, eps, inside, position, rotary, interleaved, scale):
    """Heads [rows, heads, dim] normalized and rotated in 64 bits, and the bound of a
    kernel's F32 forms before its rounding: 16 + 3 roundings of the sum of squares, halved
    by the root, five of root, sum, inverse and products, rounded up to 20 half steps of
    the normalized value; the rotation as paged_util.exact_rotation counts it."""
    eps = float(torch.tensor(eps, dtype=torch.float32))
    z = x.double()
    mean = z.square().mean(-1, keepdim=True)
    z = z / ((mean + eps).sqrt() if inside else mean.sqrt() + eps) * weight.double()
    y, far = z.clone(), z.abs() * 20 * 2.0 ** -24
    inv_freq = frequencies(rotary)
    half = rotary // 2
    for i in range(half):
        low, high = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        angle = (position.double() / scale * inv_freq[i].double())[:, None]
        a, b = z[..., low], z[..., high]
        y[..., low], y[..., high] = (a * angle.cos() - b * angle.sin(),
                                     b * angle.cos() + a * angle.sin())
        far[..., low] = far[..., high] = (a.abs() + b.abs()) * 26 * 2.0 ** -24
    return y, far


def check(p, projected, eps=1e-6, inside=True, rotary=64, interleaved=False, scale=1.0,
          split=False, per_head=False, scales=True):
    """Every slot of the pools is looked at: those not appended to keep their bits."""
    heads, kv, dim = p.heads, p.kv_heads, p.dim
    before = p.keys.clone(), p.values.clone()
    wq, wk = ((1 + p.normal(n, dim, std=0.3, kind=torch.float32)) if scales else
              torch.ones(n, dim, device=DEVICE)
              for n in ((heads, kv) if per_head else (1, 1)))
    query = append_normed(p, projected, wq if scales else None, wk if scales else None, eps,
                          inside, rotary, interleaved, scale, split, per_head)
    x = projected[:, :(heads + 2 * kv) * dim]
    if split:
        x = x.reshape(-1, heads, 3, dim)
        q, k, v = x[:, :, 0], x[:, :, 1], x[:, :, 2]
    else:
        x = x.reshape(-1, heads + 2 * kv, dim)
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    rows = list(p.rows())
    owned = [r for r in rows if r[2] >= 0]
    padding = [r for r, _, position in rows if position < 0]
    at = torch.tensor([r for r, _, _ in owned], device=DEVICE)
    position = torch.tensor([position for _, _, position in owned], device=DEVICE)
    page = torch.tensor([p.page_of(s, q) for _, s, q in owned], device=DEVICE)
    slot = position % p.page
    for got, source, weight in ((query.view(-1, heads, dim)[at], q[at], wq),
                                (p.keys[page, :, slot], k[at], wk)):
        expected, far = exact_heads(source, weight, eps, inside, position, rotary, interleaved,
                                    scale)
        within(got, expected, far, p.kind)
    assert torch.equal(p.values[page, :, slot], v[at].to(p.kind))
    for pool, old in zip((p.keys, p.values), before):
        old[page, :, slot] = pool[page, :, slot]
        assert torch.equal(pool.isnan(), old.isnan())
        assert torch.equal(pool.nan_to_num(), old.nan_to_num())
    assert (query[padding] == 0).all()
    assert (query[len(rows):] == 77.0).all()
    assert p.error.item() == 0


@pytest.mark.parametrize("dim,rotary,interleaved", [
    (128, 128, False), (128, 128, True), (128, 32, False), (128, 32, True), (64, 64, False),
    (64, 24, False), (64, 24, True), (64, 2, False), (32, 32, False), (32, 32, True),
    (32, 8, False), (128, 118, True), (64, 0, False)])
@pytest.mark.parametrize("source,kind", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"),
                                         ("f32", "f16")])
def test_rotations(dim, rotary, interleaved, source, kind):
    p = Paged([(5, 21), (1, 1), (0, 30), (3, 16), (17, 49), (4, 2)], dim=dim, kind=kind,
              seed=rotary, trailing=2)
    projected = p.normal(p.tokens, (p.heads + 2 * p.kv_heads) * dim, kind=KINDS[source])
    check(p, projected, rotary=rotary, interleaved=interleaved, scale=4.0, inside=rotary % 3 == 0)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("heads,kv_heads,page,layout,split", [
    (32, 32, 64, "dense", True), (32, 8, 16, "token", False), (15, 15, 128, "dense", True),
    (7, 1, 32, "token", False), (1, 1, 16, "dense", True), (28, 4, 16, "dense", False)])
def test_heads_and_strides(heads, kv_heads, page, layout, split, per_head):
    p = Paged([(1, 1000), (40, 40), (2, 17)], heads=heads, kv_heads=kv_heads, dim=128, page=page,
              layout=layout, seed=heads)
    projected = p.normal(p.tokens, (heads + 2 * kv_heads) * 128, kind=torch.float32)
    check(p, projected, rotary=128, split=split, scale=16.0, per_head=per_head)


@pytest.mark.parametrize("offset,extra", [(1, 3), (4, 4)])
@pytest.mark.parametrize("source", ["f32", "bf16"])
def test_unaligned_rows(offset, extra, source):
    p = Paged([(9, 30), (2, 2)], dim=64)
    width = (p.heads + 2 * p.kv_heads) * 64 + extra
    whole = p.normal(p.tokens * width + offset, kind=KINDS[source])
    check(p, whole[offset:].view(p.tokens, width), rotary=48)


def test_many_rows():
    p = Paged([(700, 700), (0, 0), (300, 4000), (20, 12), (3, 0)], heads=8, kv_heads=2, dim=64,
              page=32, trailing=5)
    check(p, p.normal(p.tokens, 12 * 64, kind=torch.float32), inside=False)


@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("power", [-140, -100, -60, -48, 0, 45, 61, 100, 126])
def test_sizes_of_heads(power, inside):
    """Heads of any size that F32 holds, with an eps that counts among small ones."""
    p = Paged([(6, 9)], dim=64, seed=power)
    x = p.normal(p.tokens, 8 * 64, kind=torch.float32).clamp(-1.9, 1.9)
    # (Beside the powers of the test, one head of zeros and one of a lone element.)
    x = torch.ldexp(x.double(), torch.tensor(power, device=DEVICE)).float()
    x[:, :64] = 0.0
    x[:, 64:128] = 0.0
    x[:, 70] = 2.0 ** power
    x[:, 6 * 64:] = 1.0  # values
    check(p, x, eps=1e-6 if power % 3 else 2.0 ** -100, inside=inside, rotary=32)


def test_without_scales_and_zero_heads():
    p = Paged([(3, 3)], dim=128)
    x = p.normal(3, 8 * 128, kind=torch.float32)
    x[1] = 0.0
    check(p, x, rotary=128, scales=False, inside=False)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("inside", [False, True])
def test_infinities_stay_in_their_head(bad, inside):
    """A head that holds one becomes what the formula gives; the others keep their bits."""
    p = Paged([(4, 4)], dim=64)
    x = p.normal(4, 8 * 64, kind=torch.float32)
    weight = torch.ones(1, 64, device=DEVICE)
    clean = append_normed(p, x, weight, weight, 1e-6, inside, 0).clone()
    y = x.clone()
    y[2, 64 + 5] = bad
    spoilt = append_normed(p, y, weight, weight, 1e-6, inside, 0)
    same = torch.ones(4, 4 * 64, dtype=torch.bool, device=DEVICE)
    same[2, 64:128] = False
    assert torch.equal(clean[same], spoilt[same])
    head = spoilt[2, 64:128].float()
    assert head[5].isnan()
    rest = torch.cat([head[:5], head[6:]])
    assert rest.isnan().all() if math.isnan(bad) else (rest == 0).all()


def test_same_rows_as_norm_and_append():
    """The library's own row norm of a head, then the append without norms: both within
    their roundings of each other."""
    dim = 128
    p = Paged([(20, 31)], heads=2, kv_heads=2, dim=dim, kind="f16")
    x = p.normal(20, 6 * dim, kind=torch.float32)
    weight = 1 + p.normal(1, dim, std=0.2, kind=torch.float32)
    query = append_normed(p, x, weight, weight, 1e-5, False, dim)
    keys = p.keys.clone()
    rows = x.view(20 * 6, dim)
    normed = torch.empty_like(rows)
    N.call("evo_hip_rms_norm", rows.data_ptr(), rows.shape[0], dim, weight.data_ptr(), 1e-5,
           normed.data_ptr(), None, None, torch.cuda.current_stream().cuda_stream)
    normed = torch.cat([normed.view(20, 6, dim)[:, :4], x.view(20, 6, dim)[:, 4:]], 1)
    apart = append(p, normed.view(20, 6 * dim), frequencies(dim), dim)
    # Both round values of at most 12 once; a border between two roundings is a step.
    u = half_step(p.kind)
    for a, b in ((query, apart), (keys, p.keys)):
        a, b = a.double().nan_to_num(), b.double().nan_to_num()
        assert ((a - b).abs() <= 2 * u * b.abs() + 64 * 2.0 ** -24 * 12).all()


@pytest.mark.parametrize("what", ["page", "sequence"])
def test_bad_tables(what):
    """A page outside the pool takes nothing, a bad sequence nothing at all."""
    p = Paged([(2, 20), (2, 5)], dim=64)
    x = p.normal(4, 8 * 64, kind=torch.float32)
    weight = torch.ones(1, 64, device=DEVICE)
    before = p.keys.clone().nan_to_num()
    if what == "page":
        p.table[0] = 1 << 30
    else:
        p.lengths[0] = -4
    query = append_normed(p, x, weight, weight, 1e-6, True, 64)
    assert p.error.item() == (N.PAGED_BAD_PAGE if what == "page" else N.PAGED_BAD_SEQUENCE)
    changed = (p.keys.nan_to_num() != before).any(-1).any(1).nonzero().tolist()
    assert sorted(changed) == sorted([p.page_of(1, q), q % 16] for q in (3, 4))
    if what == "sequence":
        assert (query[:2] == 77.0).all()
    else:
        assert (query != 77.0).any(1).all()
