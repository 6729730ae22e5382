"""Probabilities far from the largest: what the exponential's argument may be off by."""
import pytest
import torch

from tests import learner_reference as ref
from tests.test_gpu_learner import gen, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('K', [2, 40, 700, 3001])
def test_small_probabilities_to_the_rounding_of_their_exponent(K):
    """Rows of two allowed levels, 0 and -d: the gradient of level 0's log probability at the other one is -p, p = e^-d / (1 + e^-d).
    The exponent's product is rounded once (d u), the exponential is a unit (2 u) off, the sum a rounding (1), its reciprocal a unit
    (2), two products (2): (d + 7) u relative, and what e^-d itself adds to 1 is below u."""
    from sustaingym_amd import learner
    rows = 20000
    # (half of them where the product is little above 64, whose rounding is largest against it)
    d = 44.4 + torch.rand(rows, generator=gen(1), device='cuda') * torch.where(torch.arange(rows, device='cuda') % 2 == 0, 1.0, 42.0)
    z = torch.zeros((rows, K), device='cuda')
    z[:, -1] = -d
    mask = torch.zeros(K, dtype=torch.bool, device='cuda')
    mask[0] = mask[-1] = True
    z.requires_grad_(True)
    s = learner.level_logprobs(z, torch.zeros(rows, dtype=torch.int64, device='cuda'), mask)
    grad = host(torch.autograd.grad(s.logprobs.sum(), z)[0][:, -1]).double()
    dc = host(d).double()
    p = torch.exp(-dc) / (1 + torch.exp(-dc))
    off = (grad + p).abs() / p / ref.U - (dc + 7)
    assert float(off.max()) <= 0, f'{float(off.max()):.2f} u beyond the bound at d = {float(dc[off.argmax()]):.4f}'
