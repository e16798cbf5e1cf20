"""An infinite weight in an adapter's second matrix, in each way that its product is formed."""
import math

import pytest
import torch

from adapter_util import Pool, adapt, check
from paged_util import DEVICE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank,width,rows", [(16, 4096, 3), (48, 1920, 20), (16, 8200, 3),
                                             (24, 5464, 60), (72, 3648, 300), (128, 2048, 600)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_infinite_weight_stays_in_its_column(rank, width, rows, bad):
    pool = Pool(3, rank, width, 70)
    of_rows = pool.ints([i % 4 - 1 for i in range(rows)])
    high, low = pool.planes(rows)
    base = pool.normal(rows, 70)
    out = adapt(pool, of_rows, high, low, base, torch.empty_like(base))
    check(pool, of_rows, high, low, base, out)
    pool.up[1, 33, 2] = bad
    spoilt = adapt(pool, of_rows, high, low, base, torch.empty_like(base))
    hit = torch.zeros(rows, 70, dtype=torch.bool, device=DEVICE)
    hit[of_rows == 1, 33] = True
    assert hit.any() and not torch.isfinite(spoilt[hit]).any()
    assert torch.equal(out[~hit], spoilt[~hit])
