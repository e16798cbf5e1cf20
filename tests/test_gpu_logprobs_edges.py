"""Log probabilities where the search for the first tokens, or the sums, go other ways than
for ordinary rows, against their definitions in 64 bits."""
import pytest
import torch

from paged_util import DEVICE
from test_gpu_logprobs import check

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
