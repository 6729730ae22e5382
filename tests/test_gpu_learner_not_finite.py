"""Gates and gradients that are not finite, in every form of the scan: columns, whole tiles of 64 channels, time as the fast index,
long sequences in parts; a state of 0 does not hide them, a reset does."""
import math

import pytest
import torch

from tests.test_gpu_learner import TYPES, gen, host

pytestmark = pytest.mark.gpu

# (shape, dim, where the gate is not finite)
FORMS = [((1, 3, 5), 0, 0), ((40, 3, 70), 0, 17), ((100, 2, 128), 0, 64), ((5, 30), 1, 9), ((2, 700), 1, 511), ((1, 1, 9000, 8)[1:], 1, 4000),
         ((1, 70001), 1, 40000), ((9, 140000), 0, 3), ((3000, 3, 34), 0, 1500), ((3000, 2, 64), 0, 700)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f64'])
@pytest.mark.parametrize('shape,dim,at', FORMS, ids=['x'.join(map(str, f[0])) for f in FORMS])
def test_a_gate_that_is_not_finite_is_seen_by_a_state_of_0(shape, dim, at, dtype):
    """x is 0 up to the step and 1 behind it: the formula multiplies NaN, or an infinity, by a state of 0."""
    from sustaingym_amd import learner
    kind, T = TYPES[dtype], shape[dim]

    def step(t):
        return (slice(None),) * dim + (t,)
    for bad in (math.nan, math.inf, -math.inf):
        for reverse in (False, True):
            x = torch.zeros(shape, dtype=kind, device='cuda')
            x[step(slice(at + 1, None) if not reverse else slice(0, at))] = 1.0
            gate = torch.ones(shape, dtype=kind, device='cuda')            # (products that become 0 would cut)
            gate[step(at)] = bad
            h, final = (host(t) for t in learner.gated_scan(x, gate, dim=dim, reverse=reverse))
            before, behind = (slice(0, at), slice(at, None)) if not reverse else (slice(at + 1, None), slice(0, at + 1))
            assert not h[step(before)].any() and torch.isnan(h[step(behind)]).all() and torch.isnan(final).all()
            # a reset at that step takes the gate out, one behind it takes the NaN out
            resets = torch.zeros(shape[:2], dtype=torch.bool, device='cuda')
            resets[step(at)] = True
            h, final = (host(t) for t in learner.gated_scan(x, gate, None, resets, dim, reverse))
            assert torch.isfinite(h).all() and torch.isfinite(final).all()
            if 0 < at < T - 1:
                resets[step(at)], resets[step(at + (1 if not reverse else -1))] = False, True
                h, _ = learner.gated_scan(x, gate, None, resets, dim, reverse)
                assert int(torch.isnan(host(h)).sum()) == h.numel() // T


def test_a_constant_that_is_not_finite():
    from sustaingym_amd import learner
    for kind in (torch.float32, torch.float64):
        for bad in (math.nan, math.inf):
            h, final = learner.gated_scan(torch.zeros((20, 3), dtype=kind, device='cuda'), bad)
            assert torch.isnan(host(h)).all() and torch.isnan(host(final)).all()


@pytest.mark.parametrize('shape,dim', [((40, 3, 5), 0), ((3, 40), 1), ((70, 2, 64), 0)])
def test_gradients_behind_a_gate_that_is_not_finite(shape, dim):
    """grad_x of the steps in front of it, and grad_initial, have it as a factor: NaN, also where the gradient behind it is 0."""
    from sustaingym_amd import learner
    g = gen(3)

    def step(t):
        return (slice(None),) * dim + (t,)
    for at in (0, 20):
        x = torch.randn(shape, generator=g, device='cuda').requires_grad_(True)
        gate = torch.rand(shape, generator=g, device='cuda')
        gate[step(at)] = math.nan
        rest = shape[:dim] + shape[dim + 1:]
        init = torch.zeros(rest, device='cuda', requires_grad=True)
        h, _ = learner.gated_scan(x, gate, init, dim=dim)
        gx, gi = torch.autograd.grad(h, (x, init), torch.zeros(shape, device='cuda'))
        gx = host(gx)
        assert torch.isnan(gx[step(slice(0, at))]).all() and not gx[step(slice(at, None))].any() and torch.isnan(host(gi)).all()


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f64'])
@pytest.mark.parametrize('shape,dim,at', [f for f in FORMS if f[0][f[1]] > 1], ids=['x'.join(map(str, f[0])) for f in FORMS if f[0][f[1]] > 1])
def test_the_gate_of_a_reset_has_no_gradient_whatever_comes_in(shape, dim, at, dtype):
    """grad_gate is 0 at a reset, also where the gradient of the step, or the state before it, is NaN or infinite."""
    from sustaingym_amd import learner
    kind = TYPES[dtype]

    def step(t):
        return (slice(None),) * dim + (t,)
    for reverse in (False, True):
        before = at - 1 if not reverse else at + 1
        resets = torch.zeros(shape[:2], dtype=torch.bool, device='cuda')
        resets[step(at)] = True
        x = torch.ones(shape, dtype=kind, device='cuda')
        x[step(before)] = math.nan
        gate = torch.full(shape, 0.5, dtype=kind, device='cuda').requires_grad_(True)
        up = torch.zeros(shape, dtype=kind, device='cuda')
        for bad in (math.nan, math.inf, 0.0):
            up[step(at)] = bad
            gg, = torch.autograd.grad(learner.gated_scan(x, gate, None, resets, dim, reverse)[0], gate, up)
            assert not host(gg)[step(at)].any(), (bad, reverse)
