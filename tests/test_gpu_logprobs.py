"""Log probabilities of given tokens, their rank, the entropy and the first tokens of
a row, against their definitions in 64 bits."""
import math

import pytest
import torch

from evo_hip import native as N
from paged_util import CODES, DEVICE, KINDS

pytestmark = pytest.mark.gpu
NONE = -1  # UINT32_MAX as int32


def logprobs(logits, tokens=None, top=0, wanted=("logprob", "rank", "entropy"), stream=None,
             workspace=None, rows=None, vocab=None):
    rows, vocab = rows or logits.shape[0], vocab or logits.shape[1]
    out = {"logprob": torch.full((rows,), 77.0, device=DEVICE),
           "rank": torch.full((rows,), 77, dtype=torch.int32, device=DEVICE),
           "entropy": torch.full((rows,), 77.0, device=DEVICE),
           "top_tokens": torch.full((rows, top), 77, dtype=torch.int32, device=DEVICE),
           "top_logprobs": torch.full((rows, top), 77.0, device=DEVICE)}
    need = N.call("evo_hip_token_logprobs_workspace_bytes", rows, vocab, top)
    if workspace is None and need:
        workspace = torch.full((need,), 255, dtype=torch.uint8, device=DEVICE)
    stream = torch.cuda.current_stream() if stream is None else stream
    at = {name: out[name].data_ptr() if name in wanted else None
          for name in ("logprob", "rank", "entropy")}
    N.call("evo_hip_token_logprobs", CODES[logits.dtype], logits.data_ptr(), rows, vocab,
           logits.stride(0), None if tokens is None else tokens.data_ptr(), at["logprob"],
           at["rank"], at["entropy"], top, out["top_tokens"].data_ptr() if top else None,
           out["top_logprobs"].data_ptr() if top else None,
           None if workspace is None else workspace.data_ptr(),
           0 if workspace is None else workspace.numel(), stream.cuda_stream)
    if workspace is not None:
        workspace.record_stream(stream)
    return out


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def exact(logits, tokens, top):
    """In 64 bits, for rows that are valid; and `far`, a row's bound of log1p(others) and of
    the entropy: a weight is off by 2^-24 of itself 4 times (exponential, joining) and
    2.5 |d| times (its argument and the difference), a sum of up to 32 + 6 a lane, 512 / 256 + 8
    of segments by one more each: 50; the log by 2, the rest by 4 of its result."""
    x = logits.double()
    first = x.max(1, keepdim=True)
    away = x - first.values
    weight = away.exp().scatter(1, first.indices, 0.0)
    others = weight.sum(1, keepdim=True)
    share = away - others.log1p()
    finite = away.clamp_min(-1e4)
    step = 2.0 ** -24
    loose = (weight * (54 + 2.5 * finite.abs())).sum(1, keepdim=True) * step
    far_log = loose / (1 + others) + 4 * step * others.log1p()
    spread = (weight * finite).sum(1, keepdim=True)
    far_spread = (weight * finite.abs() * (56 + 2.5 * finite.abs())).sum(1, keepdim=True) * step
    entropy = others.log1p() - spread / (1 + others)
    far_entropy = far_log + far_spread / (1 + others) + spread.abs() * loose / (1 + others) ** 2 \
        + 8 * step * entropy
    t = tokens.long()[:, None].clamp(0, x.shape[1] - 1)
    chosen = x.gather(1, t)
    index = torch.arange(x.shape[1], device=x.device)
    rank = ((x > chosen) | ((x == chosen) & (index < t))).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return dict(logprob=share.gather(1, t)[:, 0], rank=rank, entropy=entropy[:, 0],
                top_tokens=order, top_logprobs=share.gather(1, order), far_log=far_log,
                far_entropy=far_entropy[:, 0])


def near(got, expected, far):
    """Infinities in the same places, the rest within `far` and 4 roundings of its size."""
    got = got.double()
    assert torch.equal(got.isinf(), expected.isinf())
    at = ~expected.isinf()
    excess = (got - expected).abs() - far - 4 * 2.0 ** -24 * expected.abs() - 2.0 ** -126
    assert not got[at].isnan().any()
    assert (excess[at] <= 0).all(), f"{excess[at].max()} beyond the bound"


def check(logits, tokens, top, out=None):
    out = logprobs(logits, tokens, top) if out is None else out
    e = exact(logits, tokens, top)
    near(out["logprob"], e["logprob"], e["far_log"][:, 0])
    near(out["entropy"], e["entropy"], e["far_entropy"])
    assert torch.equal(out["rank"].long(), e["rank"])
    if top:
        assert torch.equal(out["top_tokens"].long(), e["top_tokens"])
        near(out["top_logprobs"], e["top_logprobs"], e["far_log"].expand(-1, top))
    return out


def inputs(rows, vocab, kind, seed=0, std=2.5, stride=None, offset=0):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    stride = stride or vocab
    whole = torch.full((offset + rows * stride,), math.nan, dtype=KINDS[kind], device=DEVICE)
    logits = whole[offset:].view(rows, stride)[:, :vocab]
    logits.copy_(torch.randn(rows, vocab, generator=gen, device=DEVICE) * std)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE).to(torch.int32)
    return logits, tokens


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 511, 512, 513, 1024, 1025, 2047, 2048, 2049,
                                   4096, 4099, 30001, 131072, 200003])
def test_vocabularies(vocab, kind):
    rows = 5 if vocab > 10000 else 11
    logits, tokens = inputs(rows, vocab, kind, seed=vocab)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        check(logits, tokens, top)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 512, 2048, 9000])
@pytest.mark.parametrize("extra,offset", [(0, 1), (3, 0), (8, 8), (1, 3)])
def test_strides_and_alignment(kind, vocab, extra, offset):
    """Rows inside a larger tensor; what lies between them holds NaN."""
    logits, tokens = inputs(6, vocab, kind, seed=extra, stride=vocab + extra, offset=offset)
    check(logits, tokens, 7)


@pytest.mark.parametrize("rows,vocab", [(1, 512), (2, 512), (4097, 512), (1, 131072), (700, 3001)])
def test_rows(rows, vocab):
    logits, tokens = inputs(rows, vocab, "f32", seed=rows)
    check(logits, tokens, 4)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [8, 9, 64, 100, 257, 511, 512])
def test_many_rows_of_a_small_vocabulary(vocab, kind):
    """Ragged vocabularies and row counts, rows of equal logits, masked and invalid ones
    among ordinary ones."""
    rows = 1027
    logits, tokens = inputs(rows, vocab, kind, seed=vocab, stride=vocab + 3, offset=1)
    logits[5] = 0.0
    logits[6, ::2] = 1.5
    logits[700:705] = -2.0
    logits[9, 3:] = -math.inf
    logits[11] = torch.arange(vocab, device=DEVICE) / 64
    logits[1026] = logits[1026].round()
    for top in sorted({0, 1, 4, 8}):
        check(logits, tokens, min(top, vocab))
    bad = [2, 3, 64, 801]
    logits[2, 1], logits[3, vocab - 1], logits[64], logits[801, 0] = (math.nan, math.inf,
                                                                      -math.inf, -math.nan)
    tokens[7], tokens[8] = -1, vocab
    out = logprobs(logits, tokens, 8)
    good = torch.ones(rows, dtype=torch.bool, device=DEVICE)
    good[bad] = False
    for name in ("logprob", "entropy", "top_logprobs"):
        assert out[name][bad].isnan().all()
    assert (out["rank"][bad] == NONE).all() and (out["top_tokens"][bad] == NONE).all()
    assert out["logprob"][7:9].isnan().all() and (out["rank"][7:9] == NONE).all()
    good[7:9] = False
    check(logits[good], tokens[good], 8, {name: x[good] for name, x in out.items()})


@pytest.mark.parametrize("vocab", [64, 512, 1500, 2048, 5000, 70000])
def test_ties(vocab):
    """Equal logits come in the order of their index: rows of one value, of two, of few."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(vocab)
    logits = torch.randint(0, 3, (8, vocab), generator=gen, device=DEVICE).float()
    logits[0] = -3.0
    logits[1] = 0.0
    logits[1, ::2] = -0.0          # one value
    logits[2] = 1.0
    logits[2, vocab // 2:] = 2.0
    logits[3] = torch.arange(vocab, device=DEVICE) / 64    # ascending
    logits[4] = -torch.arange(vocab, device=DEVICE) / 64
    logits[5] = torch.arange(vocab, device=DEVICE) // 100  # runs
    tokens = torch.randint(0, vocab, (8,), generator=gen, device=DEVICE).to(torch.int32)
    tokens[0] = vocab - 1
    for top in (1, 2, 33, 64):
        check(logits, tokens, top)
        check(logits.to(torch.bfloat16), tokens, top)


@pytest.mark.parametrize("vocab", [300, 512, 2000, 6000, 40000])
def test_masked_logits(vocab):
    """-infinity: most of a row, all but one, whole segments, the given token."""
    logits, tokens = inputs(6, vocab, "f32", seed=vocab)
    logits[0, 5:] = -math.inf
    logits[1] = -math.inf
    logits[1, vocab - 1] = 3.0
    logits[2, : vocab - 3] = -math.inf
    tokens[3] = 7
    logits[3, 7] = -math.inf
    logits[4, vocab // 3:] = torch.finfo(torch.float32).min  # a mask of the lowest value
    tokens[1] = 0
    out = check(logits, tokens, 12)
    assert out["entropy"][1] == 0 and out["logprob"][1] == -math.inf


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [9, 61, 509, 1021, 2047, 2053, 4100, 30001])
def test_rank_of_masked_tokens(vocab, kind):
    """Among tokens of -infinity the rank counts those in front, at a row's end too."""
    logits, tokens = inputs(12, vocab, kind, seed=vocab)
    for r in range(12):
        logits[r, vocab - 1 - r % 8:] = -math.inf
        logits[r, r % 3] = -math.inf
        tokens[r] = vocab - 1 - r // 4
    check(logits, tokens, 0)


@pytest.mark.parametrize("vocab", [200, 512, 2048, 7000])
def test_rows_without_numbers(vocab):
    """NaN, +infinity, or nothing at all make a row NaN and UINT32_MAX, and no other row."""
    logits, tokens = inputs(12, vocab, "f32", seed=1)
    for r, (at, value) in enumerate([(0, math.nan), (vocab - 1, math.nan), (vocab // 2, math.inf),
                                     (3, math.inf), (7, -math.nan)]):
        logits[2 * r + 1, at] = value
    logits[11] = -math.inf
    tokens[1] = 0      # the given token is the NaN itself
    out = logprobs(logits, tokens, 9)
    for name in ("logprob", "entropy", "top_logprobs"):
        assert out[name][1::2].isnan().all()
    assert (out["rank"][1::2] == NONE).all() and (out["top_tokens"][1::2] == NONE).all()
    even = {name: x[::2] for name, x in out.items()}
    check(logits[::2], tokens[::2], 9, even)
    nan = torch.full_like(logits[:2], math.nan)
    out = logprobs(nan, tokens[:2], 3)
    assert out["logprob"].isnan().all() and (out["top_tokens"] == NONE).all()


@pytest.mark.parametrize("vocab", [512, 5000])
def test_tokens_outside_the_vocabulary(vocab):
    logits, tokens = inputs(4, vocab, "bf16")
    tokens[1], tokens[2] = -1, vocab
    out = logprobs(logits, tokens, 2)
    assert out["logprob"][1:3].isnan().all() and (out["rank"][1:3] == NONE).all()
    tokens[1:3] = 0
    check(logits, tokens, 2, {**out, "logprob": logprobs(logits, tokens)["logprob"],
                              "rank": logprobs(logits, tokens)["rank"]})


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [4.0, 12.0, 24.0, 40.0, 70.0])
def test_sure_rows_keep_their_precision(gap, kind):
    """A token far ahead: ln p is as small as exp(-gap), and relatively as exact as any. The
    logits are multiples of 1/8, so their differences are exact, and the bound holds no
    part that grows with them: 4 roundings of a weight, 46 of the sum, 4 of the log; the
    argument's own part that the exact form leaves out is below one."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(gap))
    logits = (torch.randn(9, 512, generator=gen, device=DEVICE).clamp(-4, 4) * 8).round() / 8
    tokens = torch.randint(0, 512, (9,), generator=gen, device=DEVICE).to(torch.int32)
    logits[torch.arange(9), tokens.long()] = 4.0 + gap
    logits = logits.to(KINDS[kind])
    out = logprobs(logits, tokens, 1)
    e = exact(logits, tokens, 1)
    assert (e["logprob"].abs() < 512 * math.exp(-gap)).all()
    for name in ("logprob", "entropy"):
        far = 56 if name == "logprob" else 64
        assert ((out[name].double() - e[name]).abs() <= far * 2.0 ** -24 * e[name].abs()).all()
    assert (out["rank"] == 0).all() and torch.equal(out["top_tokens"][:, 0], tokens)


def test_large_logits():
    """Values up to F32's ends: differences overflow to no weight."""
    logits, tokens = inputs(4, 3000, "f32", std=1e30)
    logits[1] = 3.4e38
    logits[1, ::3] = -3.4e38
    logits[2, 5] = 3.4e38
    check(logits, tokens, 5)


@pytest.mark.parametrize("vocab", [512, 6000])
def test_outputs_alone(vocab):
    """Each output by itself is what it is with the others."""
    logits, tokens = inputs(5, vocab, "f16")
    whole = logprobs(logits, tokens, 3)
    for name in ("logprob", "rank", "entropy"):
        alone = logprobs(logits, None if name == "entropy" else tokens, 0, wanted=(name,))
        assert torch.equal(alone[name], whole[name])
        for other in ("logprob", "rank", "entropy"):
            assert other == name or (alone[other] == 77).all()
    alone = logprobs(logits, None, 3, wanted=())
    assert torch.equal(alone["top_tokens"], whole["top_tokens"])
    assert torch.equal(alone["top_logprobs"], whole["top_logprobs"])


def test_sampled_greedy_token_has_rank_zero():
    """The sampler's first token is the first alternative."""
    logits, _ = inputs(64, 4000, "bf16", seed=5)
    tokens = torch.empty(64, dtype=torch.int32, device=DEVICE)
    uniform = torch.rand(64, device=DEVICE)
    temperature = torch.zeros(64, device=DEVICE)
    N.call("evo_hip_sample", CODES[logits.dtype], logits.data_ptr(), 64, 4000, 4000,
           temperature.data_ptr(), None, None, None, uniform.data_ptr(), tokens.data_ptr(), None,
           0, torch.cuda.current_stream().cuda_stream)
    out = check(logits, tokens, 1)
    assert (out["rank"] == 0).all() and torch.equal(out["top_tokens"][:, 0], tokens)


@pytest.mark.parametrize("vocab", [512, 9000])
def test_captured_and_on_two_streams(vocab):
    """One graph replayed on changing logits, and two calls at once with a workspace each."""
    logits, tokens = inputs(40, vocab, "f32", seed=2)
    need = max(16, N.call("evo_hip_token_logprobs_workspace_bytes", 40, vocab, 8))
    workspace = torch.zeros(need, dtype=torch.uint8, device=DEVICE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logprobs(logits, tokens, 8, stream=side, workspace=workspace)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = logprobs(logits, tokens, 8, stream=side, workspace=workspace)
    for seed in range(4):
        fresh, other = inputs(40, vocab, "f32", seed=10 + seed)
        logits.copy_(fresh)
        tokens.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        check(logits, tokens, 8, captured)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [logprobs(logits, tokens, 8, stream=s) for s in streams]
    torch.cuda.synchronize()
    for out in outs:
        for name in out:
            assert torch.equal(out[name], captured[name])
