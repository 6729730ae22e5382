"""Advantages of float64 rewards are float64 arithmetic, rounded once to float32."""
import pytest
import torch

from tests import learner_reference as ref
from tests.test_gpu_learner import gen, host, near

pytestmark = pytest.mark.gpu


def definition(rewards, values, ends, last, gamma, lam):
    """In float64 throughout, the discounts too."""
    r, v, on = rewards.double(), values.double(), (~ends).double()
    run, after, out = torch.zeros_like(last, dtype=torch.float64), last.double(), []
    for t in range(r.shape[0] - 1, -1, -1):
        run = r[t] + gamma * on[t] * after - v[t] + gamma * lam * on[t] * run
        after = v[t]
        out.append(run)
    return torch.stack(out[::-1])


@pytest.mark.parametrize('T,N', [(1, 3), (288, 64), (40, 66000), (2049, 3), (20, 140000), (5, 1), (40000, 1), (700, 2048), (16, 300)])
def test_one_rounding(T, N):
    """Off by half a step of float32 (u relative) and what float64 adds: T terms of 2^-53 of sizes below 1e5, less than 1e-9."""
    from sustaingym_amd import learner
    g = gen(T * 3 + N)
    rewards = torch.randn((T, N), generator=g, device='cuda').double() * 3.7 + 1000.0 / 3.0
    values, last = torch.randn((T, N), generator=g, device='cuda') * 3e3, torch.randn(N, generator=g, device='cuda') * 3e3
    ends = torch.rand((T, N), generator=g, device='cuda') < 0.01
    want = definition(host(rewards), host(values), host(ends), host(last), 0.995, 0.95)
    both = want + host(values).double()
    for laid in (lambda t: t, lambda t: t.t().contiguous().t()):
        got = learner.advantages(laid(rewards), laid(values), laid(ends), last, 0.995, 0.95)
        near(got.advantages, want, ref.U * want.abs() + 1e-9, 'advantages')
        near(got.targets, both, ref.U * both.abs() + 1e-9, 'targets')
