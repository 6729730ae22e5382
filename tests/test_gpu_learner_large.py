"""The learner's row operators with more rows than one line of the grid has workgroups for (2^20): a sample of the rows against
float64, from the first, the last and in between."""
import math

import pytest
import torch

from tests import learner_reference as ref
from tests.test_gpu_learner import gen, host, near

pytestmark = pytest.mark.gpu

LINE = 2 ** 20


def filled(rows, K, dtype, g, make):
    z = torch.empty((rows, K), dtype=dtype, device='cuda')
    for part in z.split(max(1, 2 ** 27 // K)):
        part.copy_(make(part.shape))
    return z


@pytest.mark.parametrize('K,each,dtype,masked', [(5, 256, torch.bfloat16, True), (8, 256, torch.float16, False), (33, 64, torch.float16, False),
                                                 (24, 128, torch.bfloat16, True), (1024, 4, torch.bfloat16, False)])
def test_more_workgroups_than_a_line_of_the_grid(K, each, dtype, masked):
    from sustaingym_amd import learner
    g = gen(K)
    rows = LINE * each + 1                       # one workgroup more, with a single row (up to 9 GB of logits, as much of gradients)
    z = filled(rows, K, dtype, g, lambda s: 2.0 * torch.randn(s, generator=g, device='cuda')).requires_grad_(True)
    mask = filled(rows, K, torch.bool, g, lambda s: torch.rand(s, generator=g, device='cuda') < 0.8) if masked else None
    at = torch.cat([torch.arange(300, device='cuda'), torch.randint(0, rows, (1500,), generator=g, device='cuda'),
                    torch.arange(rows - 300, rows, device='cuda')])
    zc, mc = host(z.detach()[at]), None if mask is None else host(mask[at])
    want, r = ref.choose(zc, None, mc)
    c = learner.choose_levels(z, None, mask)
    assert torch.equal(host(c.levels[at]), want)
    near(c.logprobs[at], *r.of_levels(want), 'chosen log probability')
    del c
    levels = torch.randint(-1, K, (rows,), generator=g, device='cuda')
    lc = host(levels[at])
    s = learner.level_logprobs(z, levels, mask)
    near(s.logprobs[at], *r.of_levels(lc), 'log probability')
    near(s.entropy[at], r.entropy, r.tol_entropy, 'entropy')
    ga, gb = torch.randn(rows, generator=g, device='cuda'), torch.randn(rows, generator=g, device='cuda')
    grad, = torch.autograd.grad((s.logprobs, s.entropy), z, (ga, gb))
    near(grad[at], *r.gradient(lc, host(ga[at]), host(gb[at]), dtype), 'gradient')
    assert not math.isnan(float(grad[-1].float().sum()))
