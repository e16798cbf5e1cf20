"""Heads of zeros and of the smallest values beside an eps of any size that is taken."""
import pytest
import torch

from paged_util import Paged
from test_gpu_paged_normed import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("eps", [2.0 ** -149, 1e-42, 1e-39, 2.0 ** -128, 2.0 ** -126, 1e-30, 1.0])
def test_zeros_and_small_heads(eps, inside):
    """Zeros stay zero: 1 / eps may be beyond F32."""
    p = Paged([(6, 9)], dim=64)
    x = p.normal(p.tokens, 8 * 64, kind=torch.float32)
    x[0] = 0.0
    x[2, :128] = 0.0
    x[3, :64] = 0.0
    x[3, 5] = 2.0 ** -149
    x[4, 64:128] *= 2.0 ** -127
    x[5, 4 * 64:5 * 64] = -0.0
    check(p, x, eps=eps, inside=inside, rotary=32)
