"""Page tables and batch descriptions that hold nonsense, in every form that a launch of the
paged attention takes: 16-row blocks, 128-row blocks, and both."""
import math

import pytest
import torch

from evo_hip import native as N
from paged_util import CODES, DEVICE, Paged, attend, half_step

pytestmark = pytest.mark.gpu
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


def check_without(p, query, scale, out, gone):
    """Rows against the definition in 64 bits over the positions whose (sequence, page index)
    is not in `gone`, within the bounds that paged_util counts; rows that are left none: zero."""
    heads, group, u, row = p.heads, p.heads // p.kv_heads, half_step(p.kind), 0
    got = out.view(p.tokens, heads, p.dim).double()
    for s, (n, length) in enumerate(p.sequences):
        at = [i for i in range(length) if (s, i // p.page) not in gone]
        mine, q = got[row:row + n], query[row:row + n].view(n, heads, p.dim).double()
        first = torch.arange(length - n, length, device=DEVICE)
        row += n
        if n == 0:
            continue
        if not at:
            assert (mine == 0).all()
            continue
        page = torch.tensor([p.page_of(s, i) for i in at], device=DEVICE)
        at = torch.tensor(at, device=DEVICE)
        k, v = (pool[page, :, at % p.page].double().repeat_interleave(group, 1)
                for pool in (p.keys, p.values))
        score = torch.einsum("nhd,khd->hnk", q, k) * scale
        spread = torch.einsum("nhd,khd->hnk", q.abs(), k.abs()) * scale
        hidden = at[None] > first[:, None]
        seen = ~hidden.all(1)
        score = score.masked_fill(hidden, -math.inf)
        w = (score - score.amax(-1, keepdim=True).clamp_min(-1e300)).exp()
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
        loose = ((spread + score.abs()).masked_fill(hidden, 0.0).amax(-1) * (p.dim + 8) *
                 2.0 ** -24).permute(1, 0)[..., None]
        expected, size = (torch.einsum("hnk,khd->nhd", w, x) for x in (v, v.abs()))
        room = size * (2 * u * (1 + 4 * u) + 2 * loose + 2.0 ** -20) * (1 + u) + \
            expected.abs() * u + torch.finfo(p.kind).smallest_normal * u * 2
        assert (mine[~seen] == 0).all()
        assert ((mine - expected).abs() <= room)[seen].all()
    assert (got[row:] == 77.0).all()


# The sequences' rows: 128-row blocks (three layouts of groups), and 16-row blocks.
BATCHES = [([(40, 100), (90, 300), (1, 30)], 2, 1), ([(150, 333), (3, 20)], 1, 1),
           ([(5, 310), (33, 280)], 8, 2), ([(1, 290), (2, 100), (6, 300)], 4, 2)]


@pytest.mark.parametrize("sequences,heads,kv_heads", BATCHES)
@pytest.mark.parametrize("page,kind,dim", [(16, "bf16", 64), (32, "f16", 128), (64, "bf16", 32)])
def test_bad_pages(sequences, heads, kv_heads, page, kind, dim):
    """One bad entry after the other, each of a 64-key tile's groups of 16 among them, then
    whole tiles, the first positions, the last, and all."""
    p = Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=kind, trailing=3)
    query = p.normal(p.tokens, heads * dim)
    longest = max(range(len(sequences)), key=lambda s: sequences[s][1])
    pages = -(-sequences[longest][1] // page)
    whole = [i for i in range(pages) if 64 <= i * page < 128]
    kept = p.table.clone()
    for where, entry in [([i], -1) for i in range(min(pages, 9))] + [
            (whole, -7), ([0, 1], p.pages), ([pages - 1], HIGH), (list(range(pages - 1)), LOW),
            (list(range(0, pages, 2)), p.pages), (list(range(pages)), -1)]:
        p.error.zero_()
        p.table[longest, where] = entry
        out = attend(p, query, dim ** -0.5)
        p.table.copy_(kept)
        assert p.error.item() == N.PAGED_BAD_PAGE
        check_without(p, query, dim ** -0.5, out, {(longest, i) for i in where})


@pytest.mark.parametrize("sequences,heads,kv_heads", [
    ([(1, 300), (1, 420)], 4, 2),                          # 16-row blocks
    ([(40, 300), (90, 500)], 2, 2), ([(20, 333)], 8, 1),   # 128-row blocks
    ([(1, 257 + 3 * i) for i in range(40)], 4, 4)])        # 128-row blocks on the prefix alone
@pytest.mark.parametrize("page,kind,dim", [(16, "bf16", 64), (64, "f16", 128)])
def test_bad_pages_of_the_prefix(sequences, heads, kv_heads, page, kind, dim):
    p = Paged(sequences, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=kind,
              shared=256, trailing=2)
    query = p.normal(p.tokens, heads * dim)
    pages = 256 // page
    kept = p.shared_table.clone()
    for where, entry in [([i], -1) for i in range(pages)] + [
            ([0, pages - 1], p.pages), (list(range(pages // 2)), HIGH), (list(range(pages)), LOW)]:
        p.error.zero_()
        p.shared_table[where] = entry
        out = attend(p, query, dim ** -0.5)
        p.shared_table.copy_(kept)
        assert p.error.item() == N.PAGED_BAD_PAGE
        check_without(p, query, dim ** -0.5, out,
                      {(s, i) for s in range(len(sequences)) for i in where})


@pytest.mark.parametrize("shared", [0, 64])
@pytest.mark.parametrize("counts,heads,kv_heads", [((40, 33, 21), 4, 2), ((70, 150, 1), 1, 1),
                                                   ((1, 100, 20), 8, 2)])
def test_bad_sequences_beside_prompts(shared, counts, heads, kv_heads):
    """Each kind of broken entry in one of three sequences of 128-row blocks: the others keep
    their bits, its own rows and everything else stay as they were, appended keys too."""
    good = [(n, shared + n + extra) for n, extra in zip(counts, (50, 0, 7))]
    broken = [("lengths", 1, -3), ("lengths", 1, 10 ** 6), ("lengths", 1, HIGH), ("start", 3, 999),
              ("start", 3, 2), ("start", 3, LOW), ("start", 0, -1)]
    if shared:
        broken.append(("lengths", 1, shared + counts[1] - 1))
    for name, at, value in broken:
        p = Paged(good, heads=heads, kv_heads=kv_heads, dim=64, shared=shared, trailing=2)
        query = p.normal(p.tokens, heads * 64)
        whole = attend(p, query, 0.125)
        getattr(p, name)[at] = value
        out = attend(p, query, 0.125)
        assert p.error.item() == N.PAGED_BAD_SEQUENCE
        lost = 1 if name == "lengths" else 2 if at == 3 else 0
        first = sum(counts[:lost])
        served = torch.arange(p.tokens) < sum(counts)
        served[first:first + counts[lost]] = False
        assert (out[~served] == 77.0).all()
        assert torch.equal(out[served], whole[served])
        before = p.keys.clone().nan_to_num()
        p.error.zero_()
        projected = p.normal(p.tokens, (heads + 2 * kv_heads) * 64, kind=torch.float32)
        turned = torch.full((p.tokens, heads * 64), 77.0, dtype=p.kind, device=DEVICE)
        N.call("evo_hip_paged_append", p.cache(), p.batch(), CODES[torch.float32],
               projected.data_ptr(), projected.stride(0), heads, 0, None, 0, 0, 1.0,
               turned.data_ptr(), turned.stride(0), torch.cuda.current_stream().cuda_stream)
        assert p.error.item() == N.PAGED_BAD_SEQUENCE
        assert (turned[~served] == 77.0).all()
        assert torch.equal(turned[served], projected[served, :heads * 64].to(p.kind))
        changed = (p.keys.nan_to_num() != before).any(-1).any(1)
        assert changed.sum() == served.sum()
