"""Adapters and log probabilities at the ends of what they take: offsets beyond 32 bits,
the most rows, rows that all go without, graphs of the larger launches."""
import math
import random

import pytest
import torch

from evo_hip import native as N
from adapter_util import Pool, adapt, check
from paged_util import DEVICE
from test_gpu_logprobs import check as check_logprobs

pytestmark = pytest.mark.gpu


def picks(rows, adapters, seed=0):
    rng = random.Random(seed)
    return [rng.randint(-1, adapters - 1) for _ in range(rows)]


@pytest.mark.parametrize("rows,adapters,stride", [(3, 2, 1 << 31), (100, 1, (1 << 26) + 8),
                                                  (600, 2, (1 << 23) + 8)])
def test_rows_beyond_32_bits(rows, adapters, stride):
    """x and outputs whose last rows lie more than 2^32 elements behind the first, in each
    way of sorting and both of writing."""
    pool = Pool(adapters, 16, 64, 40, seed=rows)
    ids = picks(rows, adapters, rows)
    dense, _ = pool.planes(rows, 1)
    x = torch.empty((rows - 1) * stride + 64, dtype=torch.bfloat16, device=DEVICE)
    high = x.as_strided((rows, 64), (stride, 1))
    high.copy_(dense)
    whole = torch.empty((rows - 1) * stride + 40, device=DEVICE)
    out = whole.as_strided((rows, 40), (stride, 1))
    base = pool.normal(rows, 40)
    out.copy_(base)
    adapt(pool, pool.ints(ids), high, None, out, out)
    check(pool, pool.ints(ids), dense, None, base, out.contiguous())


def test_logits_beyond_32_bits():
    stride = (1 << 31) + 1
    whole = torch.empty(2 * stride + 5000, dtype=torch.bfloat16, device=DEVICE)
    logits = whole.as_strided((3, 5000), (stride, 1))
    gen = torch.Generator(device=DEVICE).manual_seed(1)
    logits.copy_(torch.randn(3, 5000, generator=gen, device=DEVICE) * 2.5)
    tokens = torch.tensor([4999, 0, 2500], dtype=torch.int32, device=DEVICE)
    check_logprobs(logits, tokens, 9)


def test_most_rows_of_adapters():
    """2^20 rows."""
    rows = 1 << 20
    pool = Pool(3, 8, 8, 4)
    of_rows = torch.randint(-1, 3, (rows,), generator=pool.gen, device=DEVICE).to(torch.int32)
    high, low = pool.planes(rows, 2)
    base = pool.normal(rows, 4)
    out = adapt(pool, of_rows, high, low, base, torch.empty_like(base))
    assert pool.error.item() == 0
    x = high.double() + low.double()
    size = high.double().abs() + low.double().abs()
    step = 2.0 ** -23
    for a in range(-1, 3):
        at = of_rows == a
        if a < 0:
            assert torch.equal(out[at], base[at])
            continue
        down, up, scale = pool.down[a].double(), pool.up[a].double(), float(pool.scales[a])
        inner = x[at] @ down.t()
        update = inner @ up.t() * scale
        # Roundings as adapter_util.exact counts them: 16 + 20 terms, 24 in the second product.
        far = ((size[at] @ down.abs().t() * 36 + inner.abs() * 27) @ up.abs().t() * scale
               + (base[at].double() + update).abs() + base[at].double().abs()) * step
        assert ((out[at].double() - base[at].double() - update).abs() <= far).all()


def test_most_rows_of_logits():
    """2^20 rows of one token, of which nothing else can be said."""
    rows = 1 << 20
    logits = torch.randn(rows, 1, device=DEVICE)
    tokens = torch.zeros(rows, dtype=torch.int32, device=DEVICE)
    out = check_logprobs(logits, tokens, 1)
    assert (out["logprob"] == 0).all() and (out["entropy"] == 0).all()


@pytest.mark.parametrize("residual", ["none", "other", "same"])
@pytest.mark.parametrize("rows", [1, 40, 700])
def test_all_rows_without(rows, residual):
    pool = Pool(2, 16, 64, 37)
    high, low = pool.planes(rows)
    base = pool.normal(rows, 37)
    out = base.clone() if residual == "same" else torch.full_like(base, 77.0)
    adapt(pool, pool.ints([-1] * rows), high, low,
          {"none": None, "other": base, "same": out}[residual], out)
    assert torch.equal(out, torch.zeros_like(base) if residual == "none" else base)


@pytest.mark.parametrize("bad", [3, -2, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [16, 17, 512, 513, 9000])
def test_bad_adapters_among_many_rows(rows, bad):
    """A few rows name an adapter that there is not, one an adapter of a bad rank."""
    pool = Pool(3, 16, 64, 32, ranks=[16, 5, 9])
    pool.ranks[1] = 200
    pool.host_ranks[1] = -1
    ids = picks(rows, 3, rows)
    for at in (0, rows // 2, rows - 1):
        ids[at] = bad
    high, low = pool.planes(rows)
    base, out = pool.normal(rows, 32), torch.empty(rows, 32, device=DEVICE)
    adapt(pool, pool.ints(ids), high, low, base, out)
    assert pool.error.item() == N.BAD_ADAPTER
    check(pool, pool.ints(ids), high, low, base, out)


@pytest.mark.parametrize("adapters", [4, 30])
def test_order_of_many_rows(adapters):
    """The same rows in another order, their last tiles filled by others: the same bits."""
    pool = Pool(adapters, 40, 256, 300)
    ids = picks(900, adapters)
    high, low = pool.planes(900)
    base = pool.normal(900, 300)
    out = adapt(pool, pool.ints(ids), high, low, base, torch.empty_like(base))
    check(pool, pool.ints(ids), high, low, base, out)
    for seed in range(3):
        turn = torch.randperm(900, generator=torch.Generator().manual_seed(seed)).to(DEVICE)
        turned = adapt(pool, pool.ints(ids)[turn].contiguous(), high[turn].contiguous(),
                       low[turn].contiguous(), base[turn].contiguous(), torch.empty_like(base))
        assert torch.equal(out[turn], turned)


@pytest.mark.parametrize("rows,rank", [(700, 96), (700, 24), (300, 96), (10, 48)])
def test_captured_launches(rows, rank):
    """Two graphs on one workspace, replayed in turn, of each kind of launch."""
    pool = Pool(5, rank, 128, 96)
    high, low = pool.planes(rows)
    base = pool.normal(rows, 96)
    of_rows = [pool.ints(picks(rows, 5, s)) for s in range(2)]
    outs = [torch.zeros_like(base) for _ in range(2)]
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    workspace = torch.zeros(need, dtype=torch.uint8, device=DEVICE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            adapt(pool, of_rows[i], high, low, base, outs[i], side, workspace)
        graphs.append(graph)
    for seed in range(4):
        for i in range(2):
            of_rows[i].copy_(pool.ints(picks(rows, 5, 10 * seed + i)))
            outs[i].fill_(math.nan)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager = adapt(pool, of_rows[i], high, low, base, torch.empty_like(base))
            check(pool, of_rows[i], high, low, base, outs[i])
            assert torch.equal(eager, outs[i])


@pytest.mark.parametrize("top", [33, 47, 63, 64])
@pytest.mark.parametrize("levels", [0.02, 0.25, 1.0, 40.0])
@pytest.mark.parametrize("vocab", [64, 65, 300, 512, 900, 2000, 4097, 9000, 70001])
def test_long_lists_of_alternatives(vocab, levels, top):
    """About as many alternatives as a wave has lanes, of logits with none, few and many equals
    at the list's end."""
    gen = torch.Generator(device=DEVICE).manual_seed(vocab + top)
    logits = torch.randn(6, vocab, generator=gen, device=DEVICE) * 2.5
    logits = ((logits / levels).round() * levels).to(torch.bfloat16)
    logits[4, vocab // 3:] = -math.inf
    logits[5, 10:] = -math.inf
    tokens = torch.randint(0, vocab, (6,), generator=gen, device=DEVICE).to(torch.int32)
    check_logprobs(logits, tokens, top)


@pytest.mark.parametrize("rows,adapters,used", [(700, 200, 2), (700, 200, 20), (2047, 3, 3),
                                                (2048, 3, 3), (2048, 300, 2), (5000, 40, 40),
                                                (17000, 6, 6)])
@pytest.mark.parametrize("rank,width,out", [(16, 2056, 1030), (72, 1032, 516)])
def test_divisions_of_many_rows(rows, adapters, used, rank, width, out):
    """Full tiles where short ones are expected, and each way to divide widths and columns."""
    pool = Pool(adapters, rank, width, out, seed=rows)
    of_rows = torch.randint(-1, used, (rows,), generator=pool.gen, device=DEVICE).to(torch.int32)
    high, low = pool.planes(rows)
    base = pool.normal(rows, out)
    result = adapt(pool, of_rows, high, low, base, torch.empty_like(base))
    assert pool.error.item() == 0
    check(pool, of_rows, high, low, base, result)
