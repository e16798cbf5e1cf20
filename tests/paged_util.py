"""A paged cache and a ragged batch on the GPU, and the serving operators in 64
bits, written from their definitions."""
import ctypes
import math
import random

import torch

from evo_hip import native as N

DEVICE = "cuda:0"
KINDS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}


def half_step(kind):
    """Largest relative error of one rounding."""
    return torch.finfo(kind).eps / 2


class Paged:
    """`sequences`: (rows, length) of each, lengths counting the shared positions.
    Slots that belong to no position hold NaN. layout "token": [pages][slot][head][d] with
    keys and values in one buffer; "dense": the default strides."""

    def __init__(self, sequences, heads=4, kv_heads=2, dim=64, page=16, kind="bf16", shared=0,
                 seed=0, layout="dense", trailing=0, spare=2, device=DEVICE):
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        self.kind, self.shared, self.sequences = KINDS[kind], shared, list(sequences)
        self.device = device
        self.gen = torch.Generator(device=device)
        self.gen.manual_seed(seed)
        shared_pages = shared // page
        counts = [max(0, -(-length // page) - shared_pages) for _, length in sequences]
        self.pages = shared_pages + sum(counts) + spare
        order = list(range(self.pages))
        random.Random(seed).shuffle(order)
        self.shared_pages, rest = order[:shared_pages], order[shared_pages:]
        width = shared_pages + max(counts) + 1
        self.rows_of, at = [], 0
        for n in counts:
            # Entries of shared positions are not read: they hold no page.
            row = [-9] * shared_pages + rest[at:at + n]
            self.rows_of.append(row + [-1] * (width - len(row)))
            at += n
        start = [0]
        for n, _ in sequences:
            start.append(start[-1] + n)
        self.tokens = start[-1] + trailing
        self.start = self.ints(start)
        self.lengths = self.ints([length for _, length in sequences])
        self.table = self.ints(self.rows_of)
        self.shared_table = self.ints(self.shared_pages or [0])
        self.error = self.ints([0])
        shape = (self.pages, kv_heads, page, dim)
        if layout == "dense":
            self.keys, self.values = (self.normal(*shape) for _ in range(2))
            self.strides = (0, 0, 0)
        else:
            whole = self.normal(self.pages, page, 2, kv_heads, dim + 8)
            self.keys = whole[:, :, 0, :, :dim].transpose(1, 2)
            self.values = whole[:, :, 1, :, :dim].transpose(1, 2)
            self.strides = (whole.stride(0), whole.stride(3), whole.stride(1))
        for pool in (self.keys, self.values):
            self.spoil(pool)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def normal(self, *shape, std=1.0, kind=None):
        x = torch.randn(*shape, generator=self.gen, device=self.device) * std
        return x.to(kind or self.kind)

    def spoil(self, pool):
        used = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for page in self.shared_pages:
            used[page] = True
        for (_, length), row in zip(self.sequences, self.rows_of):
            for p in range(self.shared, length):
                used[row[p // self.page], p % self.page] = True
        pool.masked_fill_(~used.to(self.device)[:, None, :, None], math.nan)

    def cache(self, **change):
        fields = dict(dtype=CODES[self.kind], key_pages=self.keys.data_ptr(),
                      value_pages=self.values.data_ptr(), pages=self.pages, page_size=self.page,
                      kv_heads=self.kv_heads, head_dim=self.dim, page_stride=self.strides[0],
                      head_stride=self.strides[1], token_stride=self.strides[2])
        return ctypes.byref(N.PagedCache(**{**fields, **change}))

    def batch(self, **change):
        fields = dict(sequences=len(self.sequences), tokens=self.tokens,
                      max_tokens=max(1, max(n for n, _ in self.sequences)),
                      max_length=max(1, self.shared, max(n for _, n in self.sequences)),
                      token_start=self.start.data_ptr(), lengths=self.lengths.data_ptr(),
                      page_table=self.table.data_ptr(), table_stride=self.table.stride(0),
                      shared_length=self.shared,
                      shared_table=self.shared_table.data_ptr() if self.shared else None,
                      error=self.error.data_ptr())
        return ctypes.byref(N.PagedBatch(**{**fields, **change}))

    def page_of(self, sequence, position):
        index = position // self.page
        return (self.shared_pages[index] if position < self.shared
                else self.rows_of[sequence][index])

    def rows(self):
        """(row, sequence, position) of every row of a sequence; padding has a negative one."""
        row = 0
        for s, (n, length) in enumerate(self.sequences):
            for i in range(n):
                yield row, s, length - n + i
                row += 1


def attend(p, query, scale, out=None, stream=None, workspace=None, **change):
    out = torch.full_like(query, 77.0) if out is None else out
    batch = p.batch(**change)
    need = N.call("evo_hip_paged_attention_workspace_bytes", p.cache(), batch, p.heads)
    if workspace is None:
        workspace = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=p.device)
    stream = torch.cuda.current_stream(p.device) if stream is None else stream
    N.call("evo_hip_paged_attention", p.cache(), batch, query.data_ptr(), query.stride(0), p.heads,
           scale, out.data_ptr(), out.stride(0), workspace.data_ptr(), workspace.numel(),
           stream.cuda_stream)
    workspace.record_stream(stream)
    return out


def exact_attention(p, query, scale):
    """Outputs in 64 bits, and how far the kernel's may be from each: both roundings of
    16 bits (weights, whose rounded ones also make the sum: twice their half step of
    sum p |v|; outputs: a half step) and a score's F32 error, (dim + 8) roundings of 2^-24
    of scale * sum |q k| and of the score itself, felt by a weight relatively, twice."""
    heads, kv, dim, group = p.heads, p.kv_heads, p.dim, p.heads // p.kv_heads
    out = torch.zeros(p.tokens, heads, dim, dtype=torch.float64, device=p.device)
    far = torch.zeros_like(out)
    u = half_step(p.kind)
    for s, (n, length) in enumerate(p.sequences):
        first = sum(m for m, _ in p.sequences[:s])
        if n == 0 or length == 0:
            continue
        positions = torch.arange(length)
        pages = torch.tensor([p.page_of(s, q) for q in range(length)], device=p.device)
        slots = (positions % p.page).to(p.device)
        k = p.keys[pages, :, slots].double().repeat_interleave(group, 1)   # [length, heads, dim]
        v = p.values[pages, :, slots].double().repeat_interleave(group, 1)
        q = query[first:first + n].view(n, heads, dim).double()
        score = torch.einsum("nhd,khd->hnk", q, k) * scale
        spread = torch.einsum("nhd,khd->hnk", q.abs(), k.abs()) * scale
        at = torch.arange(length - n, length, device=p.device)
        hidden = positions.to(p.device)[None] > at[:, None]
        score = score.masked_fill(hidden, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_min(-1e300)
        w = (score - top).exp()
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
        loose = ((spread + score.abs()).masked_fill(hidden, 0.0).amax(-1) * (dim + 8) *
                 2.0 ** -24).permute(1, 0)
        out[first:first + n] = torch.einsum("hnk,khd->nhd", w, v)
        size = torch.einsum("hnk,khd->nhd", w, v.abs())
        far[first:first + n] = size * (2 * u * (1 + 4 * u) + 2 * loose[..., None] + 2.0 ** -20)
    smallest = torch.finfo(p.kind).smallest_normal * u * 2
    return out, far * (1 + u) + out.abs() * u + smallest


def check_attention(p, query, scale, out):
    owned = sum(n for n, _ in p.sequences)
    expected, far = exact_attention(p, query, scale)
    got = out.view(p.tokens, p.heads, p.dim).double()
    assert torch.isfinite(got[:owned]).all()
    excess = (got - expected).abs()[:owned] - far[:owned]
    assert excess.max() <= 0, f"{excess.max()} beyond the bound"
    assert (got[owned:] == 77.0).all()  # rows behind the last sequence's


def exact_rotation(x, positions, inv_freq, rotary, interleaved, scale):
    """[rows, heads, dim] rotated in 64 bits, and the bound of a kernel's F32 rotation
    before its rounding: two products and a sum of values whose cosine and sine are off by
    four 2^-24 of one."""
    y, far = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    half = rotary // 2
    for i in range(half):
        low, high = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        angle = (positions.double() / scale * inv_freq[i].double())[:, None]
        a, b = x[..., low].double(), x[..., high].double()
        y[..., low], y[..., high] = (a * angle.cos() - b * angle.sin(),
                                     b * angle.cos() + a * angle.sin())
        far[..., low] = far[..., high] = (a.abs() + b.abs()) * 6 * 2.0 ** -24
    return y, far
