"""The workspace of the adapters: one that is large enough for some rows is for fewer too."""
import ctypes
import random

import pytest

from evo_hip import native as N
from test_paged_cpu import TESTLIB

POOLS = [(64, 16, 4096), (256, 64, 11264), (64, 128, 11264), (8, 64, 4096), (1, 8, 8),
         (8192, 8, 64), (8192, 128, 4096), (300, 40, 1920), (2, 24, 1 << 24), (5, 128, 1 << 24)]
# Each side of every border of the rules that divide the work, and sizes between them.
ROWS = sorted({r for at in (0, 4, 16, 32, 64, 256, 512, 513, 640, 1024, 2048, 2049, 4096, 4097,
                            1 << 16, 1 << 20) for r in (at - 1, at, at + 1) if 0 < r <= 1 << 20}
              | {int(1.31 ** i) for i in range(3, 51)})


def query(adapters, rank, width, out, rows):
    struct = N.Adapters(adapters=adapters, rank=rank, in_width=width, out_width=out, down=1 << 20,
                        up=1 << 21)
    return N.call("evo_hip_adapter_linear_workspace_bytes", ctypes.byref(struct), rows)


@pytest.mark.parametrize("adapters,rank,width", POOLS)
def test_grows_with_the_rows(adapters, rank, width):
    sizes = [query(adapters, rank, width, 4096, rows) for rows in ROWS]
    assert all(size > 0 for size in sizes) and sizes == sorted(sizes)


def needed():
    lib = ctypes.CDLL(TESTLIB)
    lib.evo_test_adapter_workspace.argtypes = [ctypes.c_int] * 4 + [ctypes.c_size_t]
    lib.evo_test_adapter_workspace.restype = ctypes.c_size_t
    return lib.evo_test_adapter_workspace


@pytest.mark.parametrize("adapters,rank,width", POOLS)
def test_holds_what_calls_need(adapters, rank, width):
    need = needed()
    for rows in ROWS:
        used = need(adapters, rank, width, 4096, rows)
        assert 0 < used <= query(adapters, rank, width, 4096, rows)


def test_holds_what_calls_of_any_pool_need():
    need, rng = needed(), random.Random(1)
    for _ in range(20000):
        adapters, rank = int(2 ** rng.uniform(0, 13)), 8 * rng.randint(1, 16)
        width = 8 * int(2 ** rng.uniform(0, 21))
        rows = int(2 ** rng.uniform(0, 20))
        assert 0 < need(adapters, rank, width, 64, rows) <= query(adapters, rank, width, 64, rows)
