"""Low-rank adapters of many requests beside a shared product, against their definition
in 64 bits."""
import math
import random

import pytest
import torch

from evo_hip import native as N
from adapter_util import Pool, adapt, check, exact
from paged_util import DEVICE

pytestmark = pytest.mark.gpu


def picks(rows, adapters, seed=0, runs=False):
    rng = random.Random(seed)
    if not runs:
        return [rng.randint(-1, adapters - 1) for _ in range(rows)]
    ids = []
    while len(ids) < rows:
        ids += [rng.randint(-1, adapters - 1)] * rng.randint(1, max(1, rows // 3))
    return ids[:rows]


def run(pool, ids, planes=2, residual=True, extra=0):
    high, low = pool.planes(len(ids), planes, extra)
    of_rows = pool.ints(ids)
    base = pool.normal(len(ids), pool.out) if residual else None
    out = torch.full((len(ids), pool.out), 77.0, device=DEVICE)
    adapt(pool, of_rows, high, low, base, out)
    check(pool, of_rows, high, low, base, out)
    assert pool.error.item() == 0
    return of_rows, high, low, base, out


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 200, 1500])
@pytest.mark.parametrize("adapters,runs", [(1, False), (5, True), (40, False)])
def test_rows_and_adapters(rows, adapters, runs):
    pool = Pool(adapters, 16, 256, 192, seed=rows)
    run(pool, picks(rows, adapters, rows, runs))


@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 56, 64, 72, 96, 104, 128])
def test_ranks(rank, planes):
    pool = Pool(3, rank, 320, 208, seed=rank)
    run(pool, picks(90, 3, rank), planes)


@pytest.mark.parametrize("width,out", [(8, 1), (8, 16), (24, 3), (40, 17), (1000, 63), (1920, 66),
                                       (4096, 130), (11264, 64), (64, 5001), (72, 4096)])
def test_widths(width, out):
    """Widths that end inside a matrix step, columns inside a 16 and inside 16 bytes."""
    pool = Pool(4, 24, width, out, seed=width)
    run(pool, picks(37, 4, out))
    run(pool, [2], planes=1)


def test_ranks_of_their_own():
    """Each adapter's rank, odd ones, all and none of the stored; NaN behind them."""
    ranks = [0, 1, 7, 8, 9, 15, 16, 17, 31, 33, 39, 40]
    pool = Pool(len(ranks), 40, 160, 100, ranks=ranks)
    run(pool, picks(120, len(ranks)) + list(range(len(ranks))))


@pytest.mark.parametrize("scales", [True, False])
@pytest.mark.parametrize("residual", [True, False])
def test_without_scales_or_residual(scales, residual):
    pool = Pool(3, 16, 128, 100, scales=scales)
    of_rows, *_, out = run(pool, picks(50, 3) + [-1], residual=residual)
    if not residual:
        assert (out[of_rows == -1] == 0).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("offset,extra", [(0, 4), (4, 8), (1, 0), (2, 3), (3, 1)])
def test_columns_of_a_wider_projection(offset, extra, in_place):
    """Output rows inside wider ones: what lies beside the columns keeps its bits."""
    pool = Pool(4, 16, 96, 100)
    ids = picks(70, 4) + [-1]
    of_rows = pool.ints(ids)
    high, low = pool.planes(len(ids), 2, extra=8)
    stride = offset + pool.out + extra
    whole = pool.normal(len(ids), stride)
    before = whole.clone()
    part = whole[:, offset:offset + pool.out]
    target = whole.clone() if not in_place else whole
    if not in_place:
        target.fill_(55.0)
    out = target[:, offset:offset + pool.out]
    adapt(pool, of_rows, high, low, part, out)
    check(pool, of_rows, high, low, before[:, offset:], out)
    beside = torch.ones(stride, dtype=torch.bool, device=DEVICE)
    beside[offset:offset + pool.out] = False
    assert torch.equal(target[:, beside], before[:, beside] if in_place else
                       torch.full_like(before[:, beside], 55.0))
    # Rows without an adapter are their residual, bit for bit.
    none = of_rows == -1
    assert torch.equal(out[none], before[none][:, offset:offset + pool.out])


def test_gaps_between_adapters():
    pool = Pool(5, 24, 72, 50, gap=40)
    run(pool, picks(80, 5), extra=16)


def test_offsets_beyond_32_bits():
    """Adapters 2^31 elements apart."""
    pool = Pool(2, 8, 64, 48)
    apart = 1 << 31
    down = torch.empty(apart + 8 * 64, dtype=torch.bfloat16, device=DEVICE)
    up = torch.empty(apart + 48 * 8, dtype=torch.bfloat16, device=DEVICE)
    for a in range(2):
        down[a * apart:][:8 * 64] = pool.down[a].flatten()
        up[a * apart:][:48 * 8] = pool.up[a].flatten()
    ids = [0, 1, 1, -1, 0]
    high, low = pool.planes(5)
    base, out = pool.normal(5, 48), torch.empty(5, 48, device=DEVICE)
    struct = pool.struct
    pool.struct = lambda: struct(down=down.data_ptr(), up=up.data_ptr(), down_stride=apart,
                                 up_stride=apart)
    adapt(pool, pool.ints(ids), high, low, base, out)
    check(pool, pool.ints(ids), high, low, base, out)


def test_infinities_stay_with_their_rows():
    """An infinity in one row's x, a NaN in one adapter: the other rows keep their bits,
    in the same tile too."""
    pool = Pool(3, 16, 128, 64)
    ids = picks(60, 3, seed=5)
    of_rows, high, low, base, out = run(pool, ids)
    high[7, 3] = math.inf
    high[11, 100] = math.nan
    pool.down[2, 1, 5] = math.nan
    spoilt = adapt(pool, of_rows, high, low, base, torch.empty_like(out))
    same = torch.tensor([a != 2 and i not in (7, 11) for i, a in enumerate(ids)], device=DEVICE)
    assert same.any() and torch.equal(out[same], spoilt[same])
    assert spoilt[of_rows == 2].isnan().all()
    if ids[11] >= 0:
        assert spoilt[11].isnan().all()
    if ids[7] in (0, 1):
        assert not torch.isfinite(spoilt[7]).any()


def test_small_ranks_meet_no_infinity():
    """Zeros behind an adapter's rank would make NaN of a row's infinity."""
    pool = Pool(1, 16, 64, 40, ranks=[3], scales=False)
    high, _ = pool.planes(2, 1)
    pool.down[0, :3] = 1.0
    pool.up[0, :, :3] = 1.0
    high[0] = 0.0
    high[0, 0] = math.inf
    out = adapt(pool, pool.ints([0, 0]), high, None, None, torch.empty(2, 40, device=DEVICE))
    assert (out[0] == math.inf).all() and torch.isfinite(out[1]).all()


def test_inner_values_keep_their_bits():
    """Inner values that cancel in the output but for their last bits: 16 bits of them
    would leave nothing."""
    pool = Pool(1, 8, 8, 16, scales=False)
    pool.down.zero_()
    pool.up.zero_()
    pool.down[0, 0, :3] = 1.0   # x0 + x1 + x2
    pool.down[0, 1, 0] = 1.0    # x0
    pool.down[0, 2, 1] = 1.0    # x1
    pool.up[0, :, 0] = 1.0
    pool.up[0, :, 1] = -1.0
    pool.up[0, :, 2] = -1.0
    high = torch.zeros(1, 8, dtype=torch.bfloat16, device=DEVICE)
    high[0, :3] = torch.tensor([1.0, 2.0 ** -10, 2.0 ** -23])
    out = adapt(pool, pool.ints([0]), high, None, None, torch.empty(1, 16, device=DEVICE))
    assert (out == 2.0 ** -23).all()


@pytest.mark.parametrize("bad", [3, 1000, -2, -2 ** 31, 2 ** 31 - 1])
def test_bad_adapters_count_as_none(bad):
    pool = Pool(3, 16, 64, 32)
    ids = [0, bad, 2, 1, bad]
    high, low = pool.planes(5)
    base = pool.normal(5, 32)
    out = adapt(pool, pool.ints(ids), high, low, base, torch.empty(5, 32, device=DEVICE))
    assert pool.error.item() == N.BAD_ADAPTER
    assert torch.equal(out[[1, 4]], base[[1, 4]])
    check(pool, pool.ints(ids), high, low, base, out)


@pytest.mark.parametrize("bad", [-1, 17, 2 ** 31 - 1, -2 ** 31])
def test_bad_ranks_count_as_none(bad):
    pool = Pool(3, 16, 64, 32, ranks=[16, 5, 9])
    pool.ranks[1] = bad
    pool.host_ranks[1] = -1
    high, low = pool.planes(4)
    base = pool.normal(4, 32)
    of_rows = pool.ints([0, 1, 2, 1])
    out = adapt(pool, of_rows, high, low, base, torch.empty(4, 32, device=DEVICE))
    assert pool.error.item() == N.BAD_ADAPTER
    assert torch.equal(out[[1, 3]], base[[1, 3]])
    check(pool, of_rows, high, low, base, out)


@pytest.mark.parametrize("fill", [0, 1, 127, 255])
@pytest.mark.parametrize("rows,adapters,used", [(341, 55, 1), (12, 8192, 3), (40, 300, 2),
                                                (700, 64, 2), (512, 512, 9)])
def test_workspace_without_initial_contents(rows, adapters, used, fill):
    """Fewer tiles than there might be: whatever the workspace held, nothing of it is read."""
    pool = Pool(adapters, 8, 64, 70, seed=rows)
    ids = [i % used for i in range(rows)]
    high, low = pool.planes(rows)
    base, out = pool.normal(rows, 70), torch.empty(rows, 70, device=DEVICE)
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    workspace = torch.full((need,), fill, dtype=torch.uint8, device=DEVICE)
    of_rows = pool.ints(ids)
    adapt(pool, of_rows, high, low, base, out, workspace=workspace)
    check(pool, of_rows, high, low, base, out)


def test_largest_pool():
    """8192 adapters, each on its own row and some on two, beside rows without."""
    pool = Pool(8192, 8, 32, 16)
    ids = list(range(8192)) + list(range(0, 8192, 7)) + [-1] * 100
    random.Random(1).shuffle(ids)
    run(pool, ids, planes=1)


def test_many_rows():
    """More rows than the sort's block has threads, most of one adapter."""
    pool = Pool(3, 8, 40, 20)
    ids = [1] * 40000 + picks(5000, 3) + [2] * 30000 + [-1] * 64
    run(pool, ids, planes=1)


def test_repeated_and_order_of_rows():
    """The same bits again, and for the same rows in another order."""
    pool = Pool(4, 32, 512, 300)
    of_rows, high, low, base, out = run(pool, picks(150, 4))
    again = adapt(pool, of_rows, high, low, base, torch.empty_like(out))
    assert torch.equal(out, again)
    turn = torch.randperm(150, generator=torch.Generator().manual_seed(1)).to(DEVICE)
    turned = adapt(pool, of_rows[turn].contiguous(), high[turn].contiguous(),
                   low[turn].contiguous(), base[turn].contiguous(), torch.empty_like(out))
    assert torch.equal(out[turn], turned)


def test_captured_with_changing_adapters():
    """A graph follows the adapters of the rows; two calls at once have a workspace each."""
    pool = Pool(6, 16, 256, 128)
    high, low = pool.planes(80)
    base, out = pool.normal(80, 128), torch.zeros(80, 128, device=DEVICE)
    of_rows = pool.ints(picks(80, 6))
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), 80)
    workspace = torch.zeros(need, dtype=torch.uint8, device=DEVICE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adapt(pool, of_rows, high, low, base, out, side, workspace)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        adapt(pool, of_rows, high, low, base, out, side, workspace)
    for seed in range(5):
        of_rows.copy_(pool.ints(picks(80, 6, seed=seed, runs=seed % 2 == 0)))
        high.copy_(pool.planes(80)[0])
        graph.replay()
        torch.cuda.synchronize()
        check(pool, of_rows, high, low, base, out)
        eager = adapt(pool, of_rows, high, low, base, torch.empty_like(out))
        assert torch.equal(eager, out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [adapt(pool, of_rows, high, low, base, torch.empty_like(out), s) for s in streams]
    torch.cuda.synchronize()
    assert torch.equal(outs[0], out) and torch.equal(outs[1], out)


def test_beside_the_shared_product():
    """evo_hip_linear and the adapters against one product with the adapter's matrix added."""
    pool = Pool(3, 16, 256, 128)
    of_rows, high, low, *_ = run(pool, picks(20, 3))
    w = pool.normal(128, 256, std=256 ** -0.5).to(torch.bfloat16)
    out = torch.empty(20, 128, device=DEVICE)
    N.call("evo_hip_linear", high.data_ptr(), low.data_ptr(), w.data_ptr(), None, None, 20, 128,
           256, out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    shared = out.clone()
    adapt(pool, of_rows, high, low, out, out)
    expected, far = exact(pool, of_rows, high, low, shared)
    assert ((out.double() - expected).abs() <= far).all()
    x = high.double() + low.double()
    whole = torch.stack([x[i] @ (w.double() + (float(pool.scales[a]) * pool.up[a].double()
                                               @ pool.down[a].double() if a >= 0 else 0)).t()
                         for i, a in enumerate(of_rows.tolist())])
    room = (x.abs() @ w.double().abs().t()) * 2 * 276 * 2.0 ** -23 + far
    assert ((out.double() - whole).abs() <= room).all()
