"""A pool of low-rank adapters on the GPU, the operator's call, and its definition in
64 bits."""
import ctypes
import math

import torch

from evo_hip import native as N
from paged_util import DEVICE


class Pool:
    """ranks: None, or one for each adapter; what lies behind them holds NaN, as do the
    gaps that `gap` leaves behind each adapter's matrices."""

    def __init__(self, adapters, rank, width, out, ranks=None, seed=0, scales=True, gap=0):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)
        self.adapters, self.rank, self.width, self.out = adapters, rank, width, out
        self.down = self.spread(adapters, rank * width, gap, width ** -0.5).unflatten(
            1, (rank, width))
        self.up = self.spread(adapters, out * rank, gap, rank ** -0.5).unflatten(1, (out, rank))
        self.gap = gap
        self.scales = 0.25 + torch.rand(adapters, generator=self.gen, device=DEVICE)
        self.scales = self.scales if scales else None
        self.host_ranks = [rank] * adapters if ranks is None else list(ranks)
        self.ranks = None if ranks is None else self.ints(ranks)
        for a, n in enumerate(self.host_ranks):
            self.down[a, max(0, n):] = math.nan
            self.up[a, :, max(0, n):] = math.nan
        self.error = self.ints([0])

    def spread(self, adapters, size, gap, std):
        whole = torch.full((adapters, size + gap), math.nan, dtype=torch.bfloat16, device=DEVICE)
        whole[:, :size] = self.normal(adapters, size, std=std)
        return whole[:, :size]

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.gen, device=DEVICE) * std

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    def planes(self, rows, planes=2, extra=0):
        """x [rows][width + extra]; behind the width lies NaN."""
        x = self.normal(rows, self.width + extra)
        x[:, self.width:] = math.nan
        high = x.to(torch.bfloat16)
        return high, (x - high.float()).to(torch.bfloat16) if planes == 2 else None

    def struct(self, **change):
        fields = dict(adapters=self.adapters, rank=self.rank, in_width=self.width,
                      out_width=self.out, down=self.down.data_ptr(), up=self.up.data_ptr(),
                      down_stride=self.down.stride(0) if self.gap else 0,
                      up_stride=self.up.stride(0) if self.gap else 0,
                      scales=None if self.scales is None else self.scales.data_ptr(),
                      ranks=None if self.ranks is None else self.ranks.data_ptr(),
                      error=self.error.data_ptr())
        return ctypes.byref(N.Adapters(**{**fields, **change}))


def adapt(pool, of_rows, high, low, residual, out, stream=None, workspace=None, rows=None):
    rows = rows or high.shape[0]
    need = N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), rows)
    if workspace is None:
        workspace = torch.full((need,), 255, dtype=torch.uint8, device=high.device)
    stream = torch.cuda.current_stream(high.device) if stream is None else stream
    N.call("evo_hip_adapter_linear", pool.struct(), of_rows.data_ptr(), high.data_ptr(),
           None if low is None else low.data_ptr(), high.stride(0), rows,
           None if residual is None else residual.data_ptr(), out.data_ptr(), out.stride(0),
           workspace.data_ptr(), workspace.numel(), stream.cuda_stream)
    workspace.record_stream(stream)
    return out


def exact(pool, of_rows, high, low, residual):
    """Outputs in 64 bits, and how far the kernel's may be from each: a sum of n F32 terms
    is off by n 2^-23 of the sum of their sizes at most, whatever its order and whether its
    steps round or truncate (n: the width, twice with two planes, and 20 of waves and parts; the
    rank in three planes); the scale, the residual and the output round once each."""
    step = 2.0 ** -23
    x = high[:, :pool.width].double()
    size = x.abs()
    if low is not None:
        x = x + low[:, :pool.width].double()
        size = size + low[:, :pool.width].double().abs()
    base = torch.zeros(x.shape[0], pool.out, dtype=torch.float64, device=DEVICE) \
        if residual is None else residual[:, :pool.out].double()
    out, far = base.clone(), torch.zeros_like(base)
    ids = of_rows.tolist()
    for a in sorted(set(ids)):
        rank = pool.host_ranks[a] if 0 <= a < pool.adapters else -1
        if not 0 < rank <= pool.rank:
            continue
        rows = torch.tensor([i for i, b in enumerate(ids) if b == a], device=DEVICE)
        down, up = pool.down[a, :rank].double(), pool.up[a, :, :rank].double()
        scale = 1.0 if pool.scales is None else float(pool.scales[a])
        inner = x[rows] @ down.t()
        off = size[rows] @ down.abs().t() * (2 * pool.width + 20) * step + inner.abs() * step
        out[rows] += inner @ up.t() * scale
        far[rows] = (off @ up.abs().t() + inner.abs() @ up.abs().t() * (3 * rank + 2) * step) \
            * abs(scale)
    return out, far + (out.abs() + base.abs()) * step


def check(pool, of_rows, high, low, residual, out):
    expected, far = exact(pool, of_rows, high, low, residual)
    excess = (out[:, :pool.out].double() - expected).abs() - far
    assert torch.isfinite(out[:, :pool.out]).all()
    assert (excess <= 0).all(), f"{excess.max()} beyond the bound"
