"""Adapters whose weights are too many for one launch, up to 512 rows (tiles, sorted by every
block), against their definition in 64 bits; and calls at the border between both ways."""
import math
import random

import pytest
import torch

from evo_hip import native as N
from adapter_util import Pool, adapt, check
from paged_util import DEVICE

pytestmark = pytest.mark.gpu
SHAPES = [(16, 8200, 130), (24, 5464, 97), (72, 3648, 260), (128, 2048, 66)]


def picks(rows, adapters, seed=0, runs=False):
    rng = random.Random(seed)
    if not runs:
        return [rng.randint(-1, adapters - 1) for _ in range(rows)]
    ids = []
    while len(ids) < rows:
        ids += [rng.randint(-1, adapters - 1)] * rng.randint(1, max(1, rows // 3))
    return ids[:rows]


def run(pool, ids, planes=2, residual=True):
    high, low = pool.planes(len(ids), planes, 8)
    of_rows = pool.ints(ids)
    base = pool.normal(len(ids), pool.out) if residual else None
    out = torch.full((len(ids), pool.out), 77.0, device=DEVICE)
    adapt(pool, of_rows, high, low, base, out)
    check(pool, of_rows, high, low, base, out)
    assert pool.error.item() == 0
    return of_rows, high, low, base, out


@pytest.mark.parametrize("rank,width,out", SHAPES)
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 32, 33, 64, 65, 200, 512])
@pytest.mark.parametrize("adapters,runs", [(1, False), (5, True), (40, False)])
def test_rows_and_adapters(rank, width, out, rows, adapters, runs):
    pool = Pool(adapters, rank, width, out, seed=rows)
    run(pool, picks(rows, adapters, rows, runs), planes=1 + rows % 2, residual=rows != 32)


@pytest.mark.parametrize("rank,width,out", SHAPES)
@pytest.mark.parametrize("rows", [9, 90])
def test_ranks_of_their_own(rank, width, out, rows):
    """Odd ranks, all and none of the stored; NaN behind them and between the adapters."""
    pool = Pool(6, rank, width, out, ranks=[rank, 0, 1, rank - 3, rank // 2, 7], gap=8)
    run(pool, picks(rows, 6, 1))


@pytest.mark.parametrize("out", [1, 3, 4, 5, 63, 64, 66, 1027])
def test_output_widths(out):
    pool = Pool(3, 16, 8200, out)
    run(pool, picks(5, 3))
    run(pool, picks(300, 3))


@pytest.mark.parametrize("rows", [5, 60, 300])
def test_infinities_stay_with_their_rows(rows):
    pool = Pool(3, 24, 5464, 64)
    ids = picks(rows, 3, seed=5)
    ids[0], ids[1], ids[2], ids[3] = 2, 0, 1, -1
    of_rows, high, low, base, out = run(pool, ids)
    high[1, 3] = math.inf
    high[2, 100] = math.nan
    high[3, 0] = math.inf
    pool.down[2, 1, 5] = math.nan
    spoilt = adapt(pool, of_rows, high, low, base, torch.empty_like(out))
    same = torch.tensor([a != 2 and i not in (1, 2) for i, a in enumerate(ids)], device=DEVICE)
    assert torch.equal(out[same], spoilt[same])
    assert spoilt[of_rows == 2].isnan().all() and spoilt[2].isnan().all()
    assert not torch.isfinite(spoilt[1]).any()


@pytest.mark.parametrize("bad", [3, -2, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [4, 16, 17, 100, 512])
def test_bad_adapters_count_as_none(rows, bad):
    pool = Pool(3, 16, 8200, 32, ranks=[16, 5, 9])
    pool.ranks[1] = 17
    pool.host_ranks[1] = -1
    ids = picks(rows, 3, rows)
    ids[0] = ids[-1] = bad
    high, low = pool.planes(rows)
    base, out = pool.normal(rows, 32), torch.empty(rows, 32, device=DEVICE)
    adapt(pool, pool.ints(ids), high, low, base, out)
    assert pool.error.item() == N.BAD_ADAPTER
    check(pool, pool.ints(ids), high, low, base, out)


@pytest.mark.parametrize("fill", [0, 1, 127, 255])
@pytest.mark.parametrize("rows,adapters,used", [(12, 4096, 3), (40, 300, 2), (341, 55, 1),
                                                (512, 512, 9)])
def test_workspace_without_initial_contents(rows, adapters, used, fill):
    pool = Pool(adapters, 8, 16392, 70, seed=rows)
    ids = [i % used for i in range(rows)]
    high, low = pool.planes(rows, 1)
    base, out = pool.normal(rows, 70), torch.empty(rows, 70, device=DEVICE)
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    workspace = torch.full((need,), fill, dtype=torch.uint8, device=DEVICE)
    of_rows = pool.ints(ids)
    adapt(pool, of_rows, high, low, base, out, workspace=workspace)
    check(pool, of_rows, high, low, base, out)


@pytest.mark.parametrize("rows", [7, 150])
def test_order_in_place_and_captured(rows):
    """The same bits again, in another order of the rows, in place, and from a graph."""
    pool = Pool(4, 72, 3648, 300)
    of_rows, high, low, base, out = run(pool, picks(rows, 4))
    turn = torch.randperm(rows, generator=torch.Generator().manual_seed(1)).to(DEVICE)
    turned = adapt(pool, of_rows[turn].contiguous(), high[turn].contiguous(),
                   low[turn].contiguous(), base[turn].contiguous(), torch.empty_like(out))
    assert torch.equal(out[turn], turned)
    same = base.clone()
    adapt(pool, of_rows, high, low, same, same)
    assert torch.equal(out, same)
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    workspace = torch.zeros(need, dtype=torch.uint8, device=DEVICE)
    side, result = torch.cuda.Stream(), torch.zeros_like(out)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        adapt(pool, of_rows, high, low, base, result, side, workspace)
    for seed in range(4):
        of_rows.copy_(pool.ints(picks(rows, 4, seed)))
        result.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        eager = adapt(pool, of_rows, high, low, base, torch.empty_like(out))
        check(pool, of_rows, high, low, base, result)
        assert torch.equal(eager, result)


@pytest.mark.parametrize("rank,width", [(16, 8192), (16, 8200), (32, 4096), (32, 4104), (8, 8),
                                        (8, 512), (8, 520), (40, 6552), (40, 6560), (64, 4088),
                                        (64, 4096), (48, 1920), (72, 520), (120, 1088), (128, 8),
                                        (128, 2040), (128, 2048)])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_border_of_weights(rank, width, rows):
    """2^17 and 2^18 weights and just more or fewer; slices of the width that end in each
    place."""
    pool = Pool(3, rank, width, 77)
    run(pool, picks(rows, 3, rows))


@pytest.mark.parametrize("rows", [255, 256, 257, 511, 512, 513])
def test_border_of_rows(rows):
    pool = Pool(3, 8, 264, 1100)
    run(pool, picks(rows, 3, rows))


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128])
def test_column_groups(rank):
    """Outputs of one block's columns and more, beside what belongs to others."""
    for rows, out in ((1, 5000), (2, 129), (100, 2100)):
        pool = Pool(2, rank, 136, out)
        ids = picks(rows, 2, rows)
        high, low = pool.planes(rows)
        whole = torch.full((rows, out + 7), 55.0, device=DEVICE)
        part = whole[:, 3:3 + out]
        part.copy_(pool.normal(rows, out))
        base = part.clone()
        adapt(pool, pool.ints(ids), high, low, part, part)
        check(pool, pool.ints(ids), high, low, base, part)
        assert (whole[:, :3] == 55.0).all() and (whole[:, 3 + out:] == 55.0).all()


@pytest.mark.parametrize("rank,width", [(16, 4096), (72, 2056)])
def test_one_launch_keeps_infinities_and_ranks_apart(rank, width):
    """Rows of one launch: an infinity in x, NaN in an adapter, ranks of their own, rows without."""
    pool = Pool(5, rank, width, 70, ranks=[rank, 0, 3, rank - 1, rank // 2 + 1], gap=16)
    ids = [0, 1, 2, 3, 4, -1, 0, 3, 2, -1, 4, 4]
    of_rows, high, low, base, out = run(pool, ids)
    high[0, width - 1] = math.inf
    high[3, 0] = math.nan
    high[5, 7] = math.inf
    high[1, 7] = math.nan
    pool.up[4, 69, 0] = math.inf
    spoilt = adapt(pool, of_rows, high, low, base, torch.empty_like(out))
    same = torch.tensor([i not in (0, 3) and a != 4 for i, a in enumerate(ids)], device=DEVICE)
    assert torch.equal(out[same], spoilt[same])
    assert not torch.isfinite(spoilt[0]).any() and spoilt[3].isnan().all()
    assert torch.equal(out[of_rows == 4][:, :69], spoilt[of_rows == 4][:, :69])
    assert not torch.isfinite(spoilt[of_rows == 4][:, 69]).any()


@pytest.mark.parametrize("fill", [0, 127, 255])
@pytest.mark.parametrize("rows,adapters,used", [(513, 3, 3), (700, 100, 1), (1600, 60, 60),
                                                (4000, 300, 2), (4095, 5, 5), (4096, 2, 2),
                                                (4097, 2, 2), (4096, 2000, 900)])
def test_rows_sorted_by_blocks_or_first(rows, adapters, used, fill):
    """Around the borders between both; words of 64 rows, and tiles that begin inside them."""
    pool = Pool(adapters, 16, 136, 70, seed=rows)
    of_rows = torch.randint(-1, used, (rows,), generator=pool.gen, device=DEVICE).to(torch.int32)
    of_rows[rows // 4: rows // 2] = used - 1
    high, low = pool.planes(rows)
    base, out = pool.normal(rows, 70), torch.empty(rows, 70, device=DEVICE)
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    workspace = torch.full((need,), fill, dtype=torch.uint8, device=DEVICE)
    adapt(pool, of_rows, high, low, base, out, workspace=workspace)
    check(pool, of_rows, high, low, base, out)
    assert pool.error.item() == 0


@pytest.mark.parametrize("fill", [0, 127, 255])
@pytest.mark.parametrize("rows,adapters,used", [(200, 8, 1), (400, 20, 3), (513, 20, 20),
                                                (1600, 20, 1), (2047, 100, 7)])
@pytest.mark.parametrize("rank,width,out", [(16, 8200, 1030), (72, 4104, 516), (128, 4104, 3),
                                            (24, 8200, 129)])
def test_columns_by_the_tiles_found(rows, adapters, used, rank, width, out, fill):
    """Batches that use few adapters of a pool: the second product's chunks get narrower."""
    pool = Pool(adapters, rank, width, out, seed=rows)
    of_rows = torch.randint(-1, used, (rows,), generator=pool.gen, device=DEVICE).to(torch.int32)
    high, low = pool.planes(rows, 1)
    base, result = pool.normal(rows, out), torch.empty(rows, out, device=DEVICE)
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    workspace = torch.full((need,), fill, dtype=torch.uint8, device=DEVICE)
    adapt(pool, of_rows, high, low, base, result, workspace=workspace)
    check(pool, of_rows, high, low, base, result)
    assert pool.error.item() == 0
