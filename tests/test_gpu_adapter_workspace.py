"""One workspace of the adapters for calls of fewer rows, and nothing written behind it."""
import pytest
import torch

from evo_hip import native as N
from adapter_util import Pool, check
from paged_util import DEVICE
from test_adapter_workspace_cpu import needed

pytestmark = pytest.mark.gpu


def call(pool, of_rows, high, base, out, workspace, size):
    N.call("evo_hip_adapter_linear", pool.struct(), of_rows.data_ptr(), high.data_ptr(), None,
           high.stride(0), high.shape[0], base.data_ptr(), out.data_ptr(), out.stride(0),
           workspace.data_ptr(), size, torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("adapters,rank,width", [(64, 16, 4096), (20, 64, 2056), (3, 128, 4096)])
def test_serves_fewer_rows(adapters, rank, width):
    pool = Pool(adapters, rank, width, 36)
    most = 4097
    size = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), most)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device=DEVICE)
    high, _ = pool.planes(most, 1)
    base, out = pool.normal(most, 36), torch.empty(most, 36, device=DEVICE)
    of_rows = torch.randint(-1, adapters, (most,), generator=pool.gen,
                            device=DEVICE).to(torch.int32)
    for rows in (4097, 4096, 4095, 2048, 2047, 600, 512, 100, 33, 5, 4, 1):
        call(pool, of_rows[:rows], high[:rows], base[:rows], out[:rows], workspace, size)
        check(pool, of_rows[:rows], high[:rows], None, base[:rows], out[:rows])


@pytest.mark.parametrize("adapters,rank,width", [(64, 16, 4096), (20, 64, 2056), (3, 128, 4096),
                                                 (9, 8, 16392)])
@pytest.mark.parametrize("rows", [1, 4, 5, 60, 512, 513, 1500, 2048, 4096, 4097])
def test_smallest_that_is_taken(adapters, rank, width, rows):
    """What a call uses is enough, a byte less is refused, and what lies behind stays."""
    pool = Pool(adapters, rank, width, 36, seed=rows)
    size = needed()(adapters, rank, width, 36, rows)
    workspace = torch.full((size + 4096,), 99, dtype=torch.uint8, device=DEVICE)
    high, _ = pool.planes(rows, 1)
    base, out = pool.normal(rows, 36), torch.full((rows, 36), 77.0, device=DEVICE)
    of_rows = torch.randint(-1, adapters, (rows,), generator=pool.gen,
                            device=DEVICE).to(torch.int32)
    with pytest.raises(N.OpError, match="workspace"):
        call(pool, of_rows, high, base, out, workspace, size - 1)
    call(pool, of_rows, high, base, out, workspace, size)
    check(pool, of_rows, high, None, base, out)
    assert (workspace[size:] == 99).all()
