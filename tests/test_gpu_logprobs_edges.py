"""Log probabilities where the search for the first tokens, or the sums, go other ways than
for ordinary rows, against their definitions in 64 bits."""
import pytest
import torch

from paged_util import DEVICE
from test_gpu_logprobs import NONE, check, inputs, logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,top", [(48, 32000, 20), (48, 17449, 10), (16, 100003, 64),
                                            (24, 300001, 3), (24, 300001, 64), (6, 1 << 20, 40)])
@pytest.mark.parametrize("levels", [0.0, 0.5, 100.0])
def test_lists_of_each_round(rows, vocab, top, levels):
    """More segments, groups or logits than are ranked directly, in each round of the search:
    all different, with equal ones, and all equal. Many rows, whose blocks run side by side."""
    gen = torch.Generator(device=DEVICE).manual_seed(vocab + top)
    logits = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2.5
    if levels:
        logits = (logits / levels).round() * levels
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE).to(torch.int32)
    check(logits, tokens, top)


def filled(bits, rows, vocab):
    """F32 logits whose bits are all the same."""
    return torch.full((rows, vocab), bits, dtype=torch.int32, device=DEVICE).view(torch.float32)


def check_invalid(out, rows):
    for name in ("logprob", "entropy", "top_logprobs"):
        assert out[name][rows].isnan().all()
    assert (out["rank"][rows] == NONE).all() and (out["top_tokens"][rows] == NONE).all()


@pytest.mark.parametrize("vocab", [64, 512, 2048, 2049, 5000, 40000])
@pytest.mark.parametrize("top", [1, 9, 64])
def test_rows_of_nan_of_any_bits(vocab, top):
    """Every place of the alternatives is written, whatever the bits of a NaN: all ones are
    the least of all orders."""
    logits, tokens = inputs(8, vocab, "f32", seed=vocab)
    for row, bits in ((1, -1), (3, 0x7fffffff), (4, 0x7f800001), (6, -0x7fffff)):
        logits[row] = filled(bits, 1, vocab)[0]
    logits[5, vocab // 2] = filled(-1, 1, 1)[0, 0]
    bad = [1, 3, 4, 5, 6]
    out = logprobs(logits, tokens, top)
    check_invalid(out, bad)
    good = [0, 2, 7]
    check(logits[good], tokens[good], top, {name: x[good] for name, x in out.items()})


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_one_nan_and_every_token_listed(kind):
    logits, tokens = inputs(3, 64, kind)
    size = torch.int32 if kind == "f32" else torch.int16
    logits.view(size)[1, 17] = -1
    out = logprobs(logits, tokens, 64)
    check_invalid(out, [1])
    check(logits[::2], tokens[::2], 64, {name: x[::2] for name, x in out.items()})


@pytest.mark.parametrize("vocab", [5000, 131072])
@pytest.mark.parametrize("top", [1, 5])
@pytest.mark.parametrize("bits", [-1, 0x7fc00000])
def test_nan_where_maxima_begin(vocab, top, bits):
    """NaN in every logit that the first lane takes: it may stand for a segment's largest."""
    logits, tokens = inputs(4, vocab, "f32", seed=top)
    at = torch.arange(vocab, device=DEVICE) % 256 < 4
    logits[2] = torch.where(at, filled(bits, 1, vocab)[0], logits[2])
    out = logprobs(logits, tokens, top)
    check_invalid(out, [2])
    good = [0, 1, 3]
    check(logits[good], tokens[good], top, {name: x[good] for name, x in out.items()})


@pytest.mark.parametrize("vocab", [300, 512, 2000, 6000, 131072])
@pytest.mark.parametrize("offset", [30.0, -30.0, 200.0, -1000.0, 1000.0, 1e5, -1e6, 3e7])
def test_rows_far_from_zero(vocab, offset):
    """Softmax does not see what is added to all logits: weights are as exact there, within
    the bound of rows about zero."""
    logits, tokens = inputs(6, vocab, "f32", seed=vocab)
    logits += offset
    check(logits, tokens, 4)


@pytest.mark.parametrize("offset", [128.0, -4096.0])
def test_16_bit_rows_far_from_zero(offset):
    logits, tokens = inputs(6, 5000, "f32", std=20.0)
    for kind in (torch.bfloat16, torch.float16):
        check((logits + offset).to(kind), tokens, 4)
