"""The learner's operators (sustaingym_amd.learner) on the GPU against float64 written out on the CPU
(tests/learner_reference.py says where every bound comes from)."""
import math

import numpy as np
import pytest
import torch

from sustaingym_amd.hostio import to_host
from tests import learner_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16, 'f64': torch.float64}


def host(t):
    """A device tensor as a CPU tensor (16-bit types by way of float32, which holds them)."""
    if t is None:
        return None
    if t.dtype in (torch.bfloat16, torch.float16):
        return torch.from_numpy(to_host(t.detach().float())).to(t.dtype)
    return torch.from_numpy(to_host(t.detach()))


def near(got, want, tol, what):
    got = host(got).double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine]
    lim = tol.expand(want.shape)[fine]
    if off.numel():
        worst = int((off - lim).argmax())
        assert bool((off <= lim).all()), f'{what}: off by {off[worst]:.3g}, bound {lim[worst]:.3g}, value {want[fine][worst]:.6g}'


def gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def make_rows(shape, dtype, seed, mask_kind):
    g = gen(seed)
    z = (3.0 * torch.randn(shape, generator=g, device='cuda')).to(dtype)
    mask = None
    if mask_kind == 'each':
        mask = (torch.rand(shape, generator=g, device='cuda') < 0.7) & (torch.rand((*shape[:-1], 1), generator=g, device='cuda') < 0.8)
    elif mask_kind == 'station':                     # whole rows, one value a row
        mask = torch.rand((*shape[:-1], 1), generator=g, device='cuda') < 0.6
    elif mask_kind == 'level':                       # one row of levels for all
        mask = torch.rand(shape[-1:], generator=g, device='cuda') < 0.6
    return z, mask, g


def full(mask, z):
    return None if mask is None else host(mask.expand(z.shape).contiguous())


SHAPES = [((1, 54), 5), ((7, 52), 2), ((3, 1), 1), ((3, 5), 3), ((65,), 4), ((2, 129), 7), ((5, 13), 8), ((33,), 9), ((11, 3), 16),
          ((9,), 17), ((67,), 31), ((70,), 32), ((19,), 33), ((21,), 63), ((10,), 64), ((10,), 65), ((5,), 127), ((9,), 128), ((6,), 200),
          ((5,), 256), ((4,), 257), ((3,), 511), ((3,), 513), ((5,), 1000), ((3,), 1024), ((3,), 1025), ((2,), 2047), ((3,), 4096),
          ((2,), 8195), ((3,), 20001), ((1,), 65536), ((2,), 131071)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('lead,K', SHAPES, ids=[f'{"x".join(map(str, a))}x{k}' for a, k in SHAPES])
def test_rows_against_float64(lead, K, dtype):
    from sustaingym_amd import learner
    shape = (*lead, K)
    for i, mask_kind in enumerate((None, 'each', 'station', 'level')):
        z, mask, g = make_rows(shape, TYPES[dtype], 17 * K + i, mask_kind)
        zc, mc = host(z), full(mask, z)
        noise = None if i == 2 else -torch.log(-torch.log(torch.rand(shape, generator=g, device='cuda').clamp(1e-7, 1 - 1e-6)))
        got = learner.choose_levels(z, noise, mask)
        want, r = ref.choose(zc, host(noise), mc)
        assert torch.equal(host(got.levels), want), 'levels'
        lp, tol = r.of_levels(want)
        near(got.logprobs, lp, tol, 'chosen log probability')
        near(got.entropy, r.entropy, r.tol_entropy, 'entropy')
        levels = torch.randint(-1, K, lead, generator=g, device='cuda')
        top = min(K, (0, 1, 5, 20)[i])
        z.requires_grad_(True)
        got = learner.level_logprobs(z, levels, mask, top)
        lc = host(levels)
        lp, tol = r.of_levels(lc)
        near(got.logprobs, lp, tol, 'log probability')
        near(got.entropy, r.entropy, r.tol_entropy, 'entropy')
        if top:
            ti, tl, tt = ref.top_levels(r, top)
            assert torch.equal(host(got.top_levels), ti), 'alternatives'
            near(got.top_logprobs, tl, tt, 'alternatives')
        ga, gb = torch.randn(lead, generator=g, device='cuda'), torch.randn(lead, generator=g, device='cuda')
        grad, = torch.autograd.grad((got.logprobs, got.entropy), z, (ga, gb))
        assert grad.dtype == z.dtype
        want, tol = r.gradient(lc, host(ga), host(gb), TYPES[dtype])
        near(grad, want, tol, 'gradient')


def test_what_masked_places_hold_is_never_used():
    from sustaingym_amd import learner
    for K in (5, 33, 300, 5000):
        z, _, g = make_rows((6, 7, K), torch.float32, K, None)
        mask = torch.rand(z.shape, generator=g, device='cuda') < 0.5
        mask[0, 0] = False
        clean = torch.where(mask, z, 0.0)
        levels = mask.int().argmax(-1)
        outs = []
        for fill in (0.0, math.inf, -math.inf, math.nan, torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
            dirty = torch.where(mask, clean, fill).requires_grad_(True)
            s = learner.level_logprobs(dirty, levels, mask, 3)
            grad, = torch.autograd.grad(s.logprobs.sum() + s.entropy.sum(), dirty)
            c = learner.choose_levels(dirty, None, mask)
            outs.append([host(t) for t in (*s, grad, *c)])
        for other in outs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(outs[0], other))
        assert float(outs[0][0][0, 0]) == 0.0 and float(outs[0][1][0, 0]) == 0.0
        assert not outs[0][4][~host(mask)].any(), 'gradient at masked places'
        assert int(outs[0][3][0, 0].max()) == -1 and bool((outs[0][2][0, 0] == -math.inf).all())


@pytest.mark.parametrize('K', [5, 40, 300, 5000])
def test_special_logits(K):
    """Additive masks (-inf and the type's lowest value), rows of one value, NaN and +inf."""
    from sustaingym_amd import learner
    low = torch.finfo(torch.float32).min
    z = torch.zeros((8, K), device='cuda')
    z[0, 1:] = -math.inf                    # one level left
    z[1] = -math.inf                        # none
    z[2] = low                              # all the lowest: uniform
    z[3, 0], z[3, 1:] = 3.0, low
    z[4] = 1e4
    z[5, 1] = math.nan
    z[6, 2] = math.inf
    z[7, 0], z[7, 1:] = 80.0, -80.0
    levels = torch.zeros(8, dtype=torch.int64, device='cuda')
    z.requires_grad_(True)
    s = learner.level_logprobs(z, levels, None, 2)
    grad, = torch.autograd.grad((s.logprobs, s.entropy), z, (torch.ones(8, device='cuda'), torch.ones(8, device='cuda')))
    lp, h, tl, ti, gr = (host(t) for t in (*s, grad))
    r = ref.Rows(host(z)[:5])
    want, tol = r.of_levels(torch.zeros(5, dtype=torch.int64))
    near(s.logprobs[:5], want, tol, 'logprobs')
    near(s.entropy[:5], r.entropy, r.tol_entropy, 'entropy')
    assert torch.isnan(lp[5:7]).all() and torch.isnan(h[5:7]).all() and torch.isnan(gr[5]).all() and torch.isnan(gr[6]).all()
    assert torch.isfinite(gr[:5]).all() and not gr[1].any()
    assert ti[0].tolist() == [0, -1] and ti[1].tolist() == [-1, -1] and ti[2].tolist() == [0, 1] and ti[4].tolist() == [0, 1]
    assert lp[7] == 0.0 and abs(float(h[7])) < 1e-30
    c = learner.choose_levels(z)
    assert bool(((host(c.levels) >= 0) & (host(c.levels) < K)).all())
    # levels that cannot be: beyond the row, and one that the row forbids
    odd = learner.level_logprobs(z.detach()[:2], torch.tensor([1, 0], device='cuda'))
    assert host(odd.logprobs).tolist() == [-math.inf, 0.0]
    odd = learner.level_logprobs(z.detach()[3:5], torch.tensor([K, 2 ** 40], device='cuda'))
    assert torch.isnan(host(odd.logprobs)).all() and torch.isfinite(host(odd.entropy)).all()


@pytest.mark.parametrize('K', [4, 6, 33, 257, 3001])
def test_rows_of_any_stride(K):
    """Slices of a wider head, transposed batches, broadcast masks, misaligned starts."""
    from sustaingym_amd import learner
    g = gen(K)
    wide = torch.randn((10, 6, 2 * K + 3), generator=g, device='cuda')
    bank = torch.randn(60 * K + 1, generator=g, device='cuda')
    stations = torch.rand((6, 1), generator=g, device='cuda') < 0.7
    for dtype in (torch.float32, torch.bfloat16):
        w, b = wide.to(dtype), bank.to(dtype)
        views = [w[..., 1:K + 1], w[..., K:2 * K][::2], w.transpose(0, 1)[..., 3:K + 3], b[1:].view(10, 6, K),
                 b[:6 * K].view(1, 6, K).expand(10, 6, K), w[:, 2:3, :K], torch.randn((10, K, 6), generator=g, device='cuda').to(dtype).transpose(1, 2)]
        for i, v in enumerate(views):
            mask = stations if v.shape[1] == 6 else (torch.rand(v.shape[1:], generator=g, device='cuda') < 0.7 if v.shape[1] != 10 else None)
            noise = torch.randn(v.shape[1:], generator=g, device='cuda')
            want, r = ref.choose(host(v.contiguous()), host(noise.expand(v.shape).contiguous()), full(mask, v))
            c = learner.choose_levels(v, noise, mask)
            assert torch.equal(host(c.levels), want), i
            near(c.logprobs, *r.of_levels(want), i)
            near(c.entropy, r.entropy, r.tol_entropy, i)
            levels = torch.randint(0, K, v.shape[:2][::-1], generator=g, device='cuda').t()
            leaf = v.detach().requires_grad_(True)
            s = learner.level_logprobs(leaf, levels, mask, 2)
            lc = host(levels)
            near(s.logprobs, *r.of_levels(lc), i)
            near(s.entropy, r.entropy, r.tol_entropy, i)
            ti, tl, tt = ref.top_levels(r, 2)
            assert torch.equal(host(s.top_levels), ti), i
            near(s.top_logprobs, tl, tt, i)
            up = torch.randn(v.shape[:2][::-1], generator=g, device='cuda').t()
            grad, = torch.autograd.grad(s.logprobs, leaf, up)
            near(grad, *r.gradient(lc, host(up), torch.zeros(v.shape[:2]), dtype), i)


def test_gradients_of_sums_and_of_one_output():
    """A sum's gradient is one value for all rows; only one of the two outputs may be used; neither copies the other's."""
    from sustaingym_amd import learner
    for K in (5, 700):
        z, mask, g = make_rows((9, 4, K), torch.float32, K, 'each')
        levels = torch.randint(-1, K, (9, 4), generator=g, device='cuda')
        r = ref.Rows(host(z), full(mask, z))
        z.requires_grad_(True)
        for a, b in ((1.0, 0.0), (0.0, 1.0), (2.0, -0.5)):
            s = learner.level_logprobs(z, levels, mask)
            loss = (a * s.logprobs.sum() if a else 0.0) + (b * s.entropy.sum() if b else 0.0)
            # levels that the mask forbids are -inf in the sum; their gradients are the formula's all the same
            grad, = torch.autograd.grad(loss, z)
            want, tol = r.gradient(host(levels), torch.full((9, 4), a), torch.full((9, 4), b), torch.float32)
            near(grad, want, tol, (K, a, b))
    # through a network, with a leaf's own accumulation
    w = torch.randn((8, 15), generator=g, device='cuda', requires_grad=True)
    x = torch.randn((6, 8), generator=g, device='cuda')
    learner.level_logprobs((x @ w).view(6, 3, 5), torch.ones((6, 3), dtype=torch.int64, device='cuda')).logprobs.mean().backward()
    logits = (host(x).double() @ host(w).double()).requires_grad_(True)
    torch.log_softmax(logits.view(6, 3, 5), -1)[..., 1].mean().backward()
    want = host(x).double().t() @ logits.grad
    np.testing.assert_allclose(host(w.grad).numpy(), want.numpy(), rtol=0, atol=1e-5)


@pytest.mark.parametrize('K', [3, 65, 2049])
def test_row_gradient_against_differences(K):
    """Central differences of the definition in float64 along random directions: (f(z + e v) - f(z - e v)) / 2 e is off by
    e^2 / 6 of a third derivative (at most about |v|^3 (1 + log K) <= 1e2 here: 2e-7 at e = 1e-4) and 1e-16 |f| / e = 1e-11."""
    from sustaingym_amd import learner
    z, mask, g = make_rows((4, K), torch.float32, K, 'level' if K > 3 else None)
    zc, mc = host(z).double(), full(mask, z)
    r = ref.Rows(zc, mc)
    levels = r.z.argmax(-1)
    ga, gb = torch.randn(4, generator=g, device='cuda'), torch.randn(4, generator=g, device='cuda')
    z.requires_grad_(True)
    s = learner.level_logprobs(z, levels.cuda(), mask)
    grad = host(torch.autograd.grad((s.logprobs, s.entropy), z, (ga, gb))[0]).double()

    def f(y):
        q = ref.Rows(y, mc)
        return (host(ga).double() * q.of_levels(levels)[0] + host(gb).double() * q.entropy).sum()

    e = 1e-4
    _, tol = r.gradient(levels, host(ga), host(gb), torch.float32)
    for k in range(4):
        v = torch.from_numpy(np.random.default_rng(k).standard_normal(zc.shape)) / math.sqrt(K)
        diff = (f(zc + e * v) - f(zc - e * v)) / (2 * e)
        assert abs(float(diff) - float((grad * v).sum())) <= float((tol * v.abs()).sum()) + 3e-7


SCANS = [((1, 1, 1), 0), ((1, 256, 512), 0), ((2, 3, 5), 0), ((5, 1, 64), 0), ((7, 2, 65), 1), ((288, 4, 3), 0), ((3, 289, 33), 1), ((2, 128, 128), 1),
         ((129, 2, 72), 0), ((1, 1000, 72), 1), ((2, 511, 4), 1), ((17, 200), 0), ((200, 17), 1), ((3, 1025), 1), ((1, 4099), 1), ((4099,), 0),
         ((31,), 0), ((64, 64), 1), ((1, 3000, 8), 1), ((1, 9000, 1), 1), ((4000, 1, 2), 0), ((20, 33, 1), 0), ((40, 70, 1000), 0), ((9, 65540), 0), ((600, 3, 34), 0), ((20, 140000), 0)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16', 'f64'])
@pytest.mark.parametrize('shape,dim', SCANS, ids=[f'{"x".join(map(str, s))}-{d}' for s, d in SCANS])
def test_scan_against_float64(shape, dim, dtype):
    from sustaingym_amd import learner
    kind = TYPES[dtype]
    state = torch.float64 if kind == torch.float64 else torch.float32
    for i, (reverse, with_resets, with_initial) in enumerate(((False, True, True), (True, False, True), (True, True, False))):
        g = gen(100 * len(shape) + i + shape[0])
        x = torch.randn(shape, generator=g, device='cuda').to(kind).requires_grad_(True)
        gate = torch.sigmoid(torch.randn(shape, generator=g, device='cuda') * 2 + 2).to(kind).requires_grad_(True)
        if i == 2:
            gate = (-gate.detach()).requires_grad_(True)
        rest = [n for k, n in enumerate(shape) if k != dim]
        initial = torch.randn(rest, generator=g, device='cuda').to(state).requires_grad_(True) if with_initial else None
        resets = torch.rand(shape[:2], generator=g, device='cuda') < 0.03 if with_resets else None
        gh = torch.randn(shape, generator=g, device='cuda').to(kind)
        gf = torch.randn(rest, generator=g, device='cuda').to(state)
        want = ref.scan(host(x), host(gate), host(initial), host(resets), dim, reverse, host(gh), host(gf))
        h, final = learner.gated_scan(x, gate, initial, resets, dim, reverse)
        assert h.dtype == kind and final.dtype == state and h.is_contiguous()
        near(h, *want['h'], 'h')
        near(final, *want['final'], 'final')
        leaves = [x, gate] + ([initial] if with_initial else [])
        grads = torch.autograd.grad((h, final), leaves, (gh, gf))
        for name, got in zip(('grad_x', 'grad_gate', 'grad_initial'), grads):
            near(got, *want[name], name)
        h2, f2 = learner.gated_scan(x.detach(), gate.detach(), None if initial is None else initial.detach(), resets, dim, reverse)
        assert torch.equal(h, h2) and torch.equal(final, f2)


def test_scan_with_one_discount_is_discounted_returns():
    from sustaingym_amd import learner
    for shape, dim in (((288, 1000), 0), ((1000, 288), 1), ((1, 77), 0), ((5000,), 0)):
        g = gen(3)
        for kind in (torch.float64, torch.float32):
            r = torch.randn(shape, generator=g, device='cuda').to(kind)
            ends = torch.rand(shape, generator=g, device='cuda') < 0.02
            h, final = learner.gated_scan(r, 0.97, resets=ends, dim=dim, reverse=True)
            want = ref.scan(host(r), 0.97, None, host(ends), dim, True)
            near(h, *want['h'], shape)
            near(final, *want['final'], shape)


def test_scan_gradients_when_little_is_asked():
    """Only one output used, a broadcast gate, a constant gate, a sum's (broadcast) gradient."""
    from sustaingym_amd import learner
    g = gen(5)
    for shape, dim in (((40, 6, 70), 0), ((6, 300), 1)):
        x = torch.randn(shape, generator=g, device='cuda').requires_grad_(True)
        rest = [n for k, n in enumerate(shape) if k != dim]
        init = torch.randn(rest, generator=g, device='cuda').requires_grad_(True)
        gshape = (*shape[:2], 1) if len(shape) == 3 else (1, shape[1])
        gate = torch.sigmoid(torch.randn(gshape, generator=g, device='cuda')).requires_grad_(True)
        full_gate = host(gate).expand(shape)
        for use in ('h', 'final'):
            h, final = learner.gated_scan(x, gate, init, dim=dim)
            out = h.sum() if use == 'h' else final.sum()
            gx, gg, gi = torch.autograd.grad(out, (x, gate, init))
            want = ref.scan(host(x), full_gate, host(init), None, dim, False, torch.ones(shape) if use == 'h' else None,
                            torch.ones(rest) if use == 'final' else None)
            near(gx, *want['grad_x'], use)
            near(gi, *want['grad_initial'], use)
            v, tol = want['grad_gate']
            axis = 2 if len(shape) == 3 else 0
            tol = tol + 64 * ref.U * v.abs()          # torch adds at most 70 float32 values up
            near(gg, v.sum(axis, keepdim=True), tol.sum(axis, keepdim=True), use)
        h, _ = learner.gated_scan(x, 0.5, None, dim=dim)
        gx, = torch.autograd.grad(h.sum(), x)
        near(gx, *ref.scan(host(x), 0.5, None, None, dim, False, torch.ones(shape))['grad_x'], 'constant gate')


def test_scan_gradient_against_differences():
    """The scan is linear in x and in the initial state: (f(v + e d) - f(v - e d)) / 2 e is its derivative to rounding; in the gate,
    e^2 / 6 of a third derivative (at most 40^3 times the values' size, ~ 10: 1e-6 at e = 1e-6 ... 1e-5 with float64 noise)."""
    from sustaingym_amd import learner
    g = gen(9)
    x, gate = torch.randn((40, 3, 4), generator=g, device='cuda'), torch.rand((40, 3, 4), generator=g, device='cuda') * 0.9
    init, resets = torch.randn((3, 4), generator=g, device='cuda'), torch.rand((40, 3), generator=g, device='cuda') < 0.05
    gh, gf = torch.randn((40, 3, 4), generator=g, device='cuda').double(), torch.randn((3, 4), generator=g, device='cuda').double()
    leaves = [t.double().requires_grad_(True) for t in (x, gate, init)]
    h, final = learner.gated_scan(*leaves, resets)
    grads = torch.autograd.grad((h, final), leaves, (gh, gf))
    base = [host(t) for t in leaves]

    def f(a, b, c):
        o = ref.scan(a, b, c, host(resets), 0, False)
        return float((o['h'][0] * host(gh)).sum() + (o['final'][0] * host(gf)).sum())

    for k in range(3):
        d = torch.from_numpy(np.random.default_rng(k).standard_normal(tuple(base[k].shape)))
        e = 1e-5
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + e * d, base[k] - e * d
        assert abs((f(*up) - f(*down)) / (2 * e) - float((host(grads[k]) * d).sum())) < 1e-5


def test_scan_resets_let_nothing_through():
    from sustaingym_amd import learner
    for shape, dim in (((50, 4, 3), 0), ((4, 600), 1), ((4, 50, 65), 1)):
        g = gen(11)
        x = torch.randn(shape, generator=g, device='cuda')
        gate = torch.rand(shape, generator=g, device='cuda')
        rest = [n for k, n in enumerate(shape) if k != dim]
        resets = torch.zeros(shape[:2], dtype=torch.bool, device='cuda')
        first, later = (slice(0, 20), slice(20, None)) if dim == 0 else ((slice(None), slice(0, 20)), (slice(None), slice(20, None)))
        resets[20 if dim == 0 else (slice(None), 20)] = True
        clean, _ = learner.gated_scan(x, gate, None, resets, dim)
        x2, gate2 = x.clone(), gate.clone()
        x2[first], gate2[first] = math.nan, math.inf
        gate2[20 if dim == 0 else (slice(None), 20)] = math.nan
        leaves = [t.requires_grad_(True) for t in (x2, gate2)]
        dirty, final = learner.gated_scan(*leaves, torch.full(rest, math.inf, device='cuda'), resets, dim)
        assert torch.equal(clean[later], dirty[later])
        gx, gg = torch.autograd.grad(dirty[later].sum() + final.sum(), leaves)
        assert torch.isfinite(gx[later]).all() and torch.isfinite(gg[later]).all()
        # (in front of the reset the formula itself multiplies a gradient of 0 by infinite gates; with finite ones it is 0)
        gate3 = gate.clone()
        gate3[20 if dim == 0 else (slice(None), 20)] = math.nan
        leaves = [x2.detach().requires_grad_(True), gate3.requires_grad_(True)]
        dirty, final = learner.gated_scan(*leaves, torch.full(rest, math.inf, device='cuda'), resets, dim)
        gx, _ = torch.autograd.grad(dirty[later].sum() + final.sum(), leaves)
        assert torch.equal(clean[later], dirty[later]) and torch.isfinite(gx).all() and not gx[first].any()


def test_scan_in_pieces_and_in_single_steps():
    """The state that one call hands to the next is the whole walk's (bounds as for the whole)."""
    from sustaingym_amd import learner
    g = gen(13)
    x, gate = torch.randn((90, 5, 70), generator=g, device='cuda').bfloat16(), torch.rand((90, 5, 70), generator=g, device='cuda').bfloat16()
    want = ref.scan(host(x), host(gate), None, None, 0, False)
    for cuts in ((0, 33, 33, 34, 90), range(91)):
        cuts, state, parts = list(cuts), None, []
        for a, b in zip(cuts[:-1], cuts[1:]):
            h, state = learner.gated_scan(x[a:b], gate[a:b], state)
            parts.append(h)
        near(torch.cat(parts), *want['h'], 'pieces')
        near(state, *want['final'], 'pieces')
    empty = torch.zeros((0, 5, 70), device='cuda', requires_grad=True)
    init = torch.randn((5, 70), generator=g, device='cuda', requires_grad=True)
    h, final = learner.gated_scan(empty, 0.5, init)
    assert h.shape == (0, 5, 70) and torch.equal(final, init)
    assert torch.equal(torch.autograd.grad(final.sum(), init)[0], torch.ones_like(init))


def test_scan_of_any_stride():
    from sustaingym_amd import learner
    g = gen(15)
    base = torch.randn((6, 40, 2, 34), generator=g, device='cuda')
    gbase = torch.rand((40, 34, 6), generator=g, device='cuda')
    rbase = torch.rand((40, 6), generator=g, device='cuda') < 0.05
    for dtype in (torch.float32, torch.float16):
        x, gate = base.to(dtype)[:, :, 1, 1:33], gbase.to(dtype).permute(2, 0, 1)[..., :32]
        x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
        up = torch.randn((6, 32, 40), generator=g, device='cuda').to(dtype).transpose(1, 2)
        for reverse in (False, True):
            want = ref.scan(host(x), host(gate), None, host(rbase.t()), 1, reverse, host(up))
            h, final = learner.gated_scan(x, gate, None, rbase.t(), 1, reverse)
            near(h, *want['h'], 'h')
            near(final, *want['final'], 'final')
            gx, gg = torch.autograd.grad(h, (x, gate), up)
            near(gx, *want['grad_x'], 'grad_x')
            near(gg, *want['grad_gate'], 'grad_gate')
    one = torch.randn((1,), generator=g, device='cuda').expand(300)
    near(learner.gated_scan(one, 0.5)[0], *ref.scan(host(one.contiguous()), 0.5, None, None, 0, False)['h'], 'expanded')


@pytest.mark.parametrize('T,N', [(1, 1), (288, 1), (5, 64), (100, 1000), (288, 4096), (1, 70000), (2049, 3), (20000, 2), (40, 66000), (20, 65537), (20, 140000)])
def test_advantages_against_float64(T, N):
    from sustaingym_amd import learner
    g = gen(T + N)
    values, last = torch.randn((T, N), generator=g, device='cuda') * 3, torch.randn(N, generator=g, device='cuda')
    ends = torch.rand((T, N), generator=g, device='cuda') < 0.01
    for kind in (torch.float64, torch.float32):
        rewards = torch.randn((T, N), generator=g, device='cuda').to(kind)
        got = learner.advantages(rewards, values, ends, last, 0.995, 0.95)
        want, tol = ref.advantages(host(rewards), host(values), host(ends), host(last), 0.995, 0.95)
        near(got.advantages, want, tol + ref.U * want.abs(), 'advantages')
        near(got.targets, want + host(values).double(), tol + ref.U * (2 * want.abs() + host(values).abs()), 'targets')
        v = learner.advantages(rewards.t().contiguous().t(), values.t().contiguous().t(), ends.t().contiguous().t(), last, 0.995, 0.95)
        near(v.advantages, want, tol + ref.U * want.abs(), 'batch-major storage')
    if N == 1:
        v = learner.advantages(rewards[:, 0], values[:, 0], ends[:, 0], last[0], 0.995, 0.95)
        near(v.advantages, want[:, 0], (tol + ref.U * want.abs())[:, 0], 'one sequence')


def test_advantages_nothing_passes_an_end():
    from sustaingym_amd import learner
    r, v = torch.ones((6, 2), device='cuda'), torch.zeros((6, 2), device='cuda')
    e = torch.zeros((6, 2), dtype=torch.bool, device='cuda')
    e[2] = True
    r[3:], v[3:] = math.nan, math.nan
    a = learner.advantages(r, v, e, torch.full((2,), math.nan, device='cuda'), 1.0, 1.0)
    assert host(a.advantages)[:3, 0].tolist() == [3.0, 2.0, 1.0] and torch.isnan(host(a.targets)[3:]).all()
    z = learner.advantages(r[:0], v[:0], e[:0], torch.zeros(2, device='cuda'))
    assert z.advantages.shape == (0, 2)


def test_empty_batches():
    from sustaingym_amd import learner
    z = torch.zeros((0, 54, 5), device='cuda', requires_grad=True)
    c = learner.choose_levels(z, torch.zeros((0, 54, 5), device='cuda'), torch.ones((0, 54, 5), dtype=torch.bool, device='cuda'))
    assert c.levels.shape == (0, 54)
    s = learner.level_logprobs(z, c.levels, None, 2)
    assert s.top_levels.shape == (0, 54, 2)
    assert torch.autograd.grad(s.logprobs.sum(), z)[0].shape == z.shape
    h, f = learner.gated_scan(torch.zeros((4, 0, 3), device='cuda'), 0.5)
    assert h.shape == (4, 0, 3) and f.shape == (0, 3)


def test_nothing_is_written_beside_the_outputs():
    """Outputs inside larger buffers, through the C-ABI: what lies around them keeps its values."""
    import ctypes as C
    from sustaingym_amd import _lib
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    for rows, K in ((3, 5), (70, 6), (5, 100), (2, 3001), (1, 70001)):
        for code, dtype in ((0, torch.float32), (1, torch.bfloat16)):
            z = torch.randn(rows * K, device='cuda').to(dtype)
            R = _lib.LearnerRows(z.data_ptr(), 1, rows, K, 0, K, None, 0, 0, 0, code)
            lv = torch.full((rows + 8,), -7, dtype=torch.int64, device='cuda')
            lp, en = torch.full((rows + 8,), -7.0, device='cuda'), torch.full((rows + 8,), -7.0, device='cuda')
            stat = torch.full((2 * rows + 8,), -7.0, device='cuda')
            n = lib.lrn_choose_workspace(C.byref(R))
            ws = torch.full((n + 64,), 77, dtype=torch.uint8, device='cuda')
            assert lib.lrn_choose(0, st, C.byref(R), None, 0, 0, lv[4:].data_ptr(), lp[4:].data_ptr(), en[4:].data_ptr(), ws.data_ptr(), n) == 0
            assert bool((ws[n:] == 77).all())
            for t in (lv, lp, en):
                assert bool((t[:4] == -7).all()) and bool((t[rows + 4:] == -7).all())
            top = min(K, 3)
            tl, ti = torch.full((top * rows + 8,), -7.0, device='cuda'), torch.full((top * rows + 8,), -7, dtype=torch.int64, device='cuda')
            n = lib.lrn_score_workspace(C.byref(R), top)
            ws = torch.full((n + 64,), 77, dtype=torch.uint8, device='cuda')
            assert lib.lrn_score(0, st, C.byref(R), lv[4:].data_ptr(), lp[4:].data_ptr(), en[4:].data_ptr(), stat[4:].data_ptr(), top, tl[4:].data_ptr(),
                                 ti[4:].data_ptr(), ws.data_ptr(), n) == 0
            assert bool((ws[n:] == 77).all())
            for t, m in ((lp, 1), (en, 1), (stat, 2), (tl, top), (ti, top)):
                assert bool((t[:4] == -7).all()) and bool((t[m * rows + 4:] == -7).all())
            for lead in (16, 1):                        # an aligned start and one that is not
                grad = torch.full((rows * K + lead + 16,), -7.0, device='cuda').to(dtype)
                assert lib.lrn_score_backward(0, st, C.byref(R), lv[4:].data_ptr(), stat[4:].data_ptr(), en[4:].data_ptr(), lp[4:].data_ptr(), 1, None, 0,
                                              grad[lead:].data_ptr()) == 0
                assert bool((grad[:lead] == -7).all()) and bool((grad[rows * K + lead:] == -7).all())
    for shape in ((3, 5, 7), (300, 1, 66), (1, 9, 130), (5000, 1, 1)):
        T, B, Cn = shape
        x, n = torch.randn(shape, device='cuda'), T * B * Cn
        h, f = torch.full((n + 16,), -7.0, device='cuda'), torch.full((B * Cn + 16,), -7.0, device='cuda')
        seq = _lib.LearnerSeq(T, B, Cn, 0, 0)
        ws = torch.full((lib.lrn_scan_workspace(C.byref(seq)) + 64,), 77, dtype=torch.uint8, device='cuda')

        def view(t, off=0):
            return C.byref(_lib.LearnerView(t.data_ptr() + 4 * off, B * Cn, Cn, 1))
        assert lib.lrn_scan(0, st, C.byref(seq), view(x), view(x), 0.0, None, None, view(h, 8), f[8:].data_ptr(), ws.data_ptr(), ws.numel() - 64) == 0
        for t, m in ((h, n), (f, B * Cn)):
            assert bool((t[:8] == -7).all()) and bool((t[m + 8:] == -7).all())
        assert bool((ws[-64:] == 77).all())


def test_captured_training_step_replays():
    """Forward and backward in one graph; replays with new inputs, eager work and synchronisations between them."""
    from sustaingym_amd import learner
    g = gen(21)
    for K, T in ((5, 40), (3000, 300)):
        z = torch.randn((64, 3, K), generator=g, device='cuda', requires_grad=True)
        mask = torch.rand(z.shape, generator=g, device='cuda') < 0.8
        levels = torch.randint(0, K, (64, 3), generator=g, device='cuda')
        up = torch.randn((64, 3), generator=g, device='cuda')
        x, gate = (torch.rand((2, T, 66), generator=g, device='cuda', requires_grad=True) for _ in range(2))
        long = torch.rand((1, 9000), generator=g, device='cuda', requires_grad=True)
        rewards, values = torch.randn((T, 9), generator=g, device='cuda').double(), torch.randn((T, 9), generator=g, device='cuda')
        ends, last = torch.rand((T, 9), generator=g, device='cuda') < 0.1, torch.randn(9, generator=g, device='cuda')

        def step():
            c = learner.choose_levels(z, None, mask)
            s = learner.level_logprobs(z, levels, mask, 2)
            gz, = torch.autograd.grad((s.logprobs, s.entropy), z, (up, up))
            h, f = learner.gated_scan(x, gate, dim=1)
            gx, gg = torch.autograd.grad((h, f), (x, gate), (h.detach(), f.detach()))
            l, _ = learner.gated_scan(long, 0.9, dim=1, reverse=True)
            gl, = torch.autograd.grad(l, long, l.detach())
            return [*c, *s, gz, h, f, gx, gg, l, gl, *learner.advantages(rewards, values, ends, last)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for k in range(4):
            with torch.no_grad():
                for t in (z, x, gate, long, values):
                    t.copy_(torch.rand(t.shape, generator=g, device='cuda'))
            want = [t.clone() for t in step()]
            if k % 2:
                torch.cuda.synchronize()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_on_another_stream():
    from sustaingym_amd import learner
    g = gen(23)
    side = torch.cuda.Stream()
    z = torch.randn((2000, 54, 5), generator=g, device='cuda', requires_grad=True)
    levels = torch.randint(0, 5, (2000, 54), generator=g, device='cuda')
    x = torch.randn((500, 3000), generator=g, device='cuda', requires_grad=True)

    def work():
        s = learner.level_logprobs(z * 1.5, levels)
        h, _ = learner.gated_scan(x * 2.0, 0.9)
        return (s.logprobs, s.entropy, h, *torch.autograd.grad((s.logprobs.sum() + s.entropy.sum(), h.sum()), (z, x)))

    want = work()
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [work() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_offsets_beyond_32_bits():
    """Rows, sequences and steps that lie more than 2^32 bytes (and elements) apart."""
    from sustaingym_amd import learner
    g = gen(31)
    far = 2 ** 32 + 8
    big = torch.empty(far + 4096 * 8, dtype=torch.float16, device='cuda')          # 8.6 GB, written only where it is read
    for K in (5, 40, 700, 3001):
        rows = big.as_strided((2, K), (far, 1))
        rows.copy_(torch.randn((2, K), generator=g, device='cuda'))
        mask = torch.rand((2, K), generator=g, device='cuda') < 0.9
        levels = mask.int().argmax(-1)
        r = ref.Rows(host(rows.contiguous()), host(mask))
        leaf = rows.detach().requires_grad_(True)
        s = learner.level_logprobs(leaf, levels, mask, 1)
        near(s.logprobs, *r.of_levels(host(levels)), K)
        assert torch.equal(host(s.top_levels), ref.top_levels(r, 1)[0])
        up = torch.ones(2, device='cuda')
        near(torch.autograd.grad(s.logprobs, leaf, up)[0], *r.gradient(host(levels), host(up), torch.zeros(2), torch.float16), K)
        want, _ = ref.choose(host(rows.contiguous()), None, host(mask))
        assert torch.equal(host(learner.choose_levels(rows, None, mask).levels), want)
    for shape, strides, dim in (((2, 30, 70), (far, 70, 1), 1), ((2, 600, 34), (far, 34, 1), 1), ((2, 30, 70), (far, 70, 1), 0), ((2, 3000), (far, 1), 1),
                                ((2, 90), (far, 1), 0), ((3, 20, 8), (far // 2, 8, 1), 1)):
        x = big.as_strided(shape, strides)
        x.copy_(torch.randn(shape, generator=g, device='cuda'))
        gate = torch.rand(shape, generator=g, device='cuda').half()
        up = torch.randn(shape, generator=g, device='cuda').half()
        leaves = x.detach().requires_grad_(True), gate.requires_grad_(True)
        want = ref.scan(host(x.contiguous()), host(gate), None, None, dim, False, host(up))
        h, final = learner.gated_scan(*leaves, dim=dim)
        near(h, *want['h'], (shape, dim))
        near(final, *want['final'], (shape, dim))
        # and as the gradient that comes in
        far_up = big.as_strided(shape, strides)
        kept = x.detach().clone()
        h2, _ = learner.gated_scan(kept.requires_grad_(True), gate, dim=dim)
        far_up.copy_(up)
        gx, gg = torch.autograd.grad(h2, (kept, gate), far_up)
        near(gx, *want['grad_x'], (shape, dim))
        near(gg, *want['grad_gate'], (shape, dim))
    del big


def test_one_dimension_and_no_second_derivative():
    from sustaingym_amd import learner
    z = torch.randn(7, device='cuda', requires_grad=True)
    c = learner.choose_levels(z)
    assert c.levels.shape == () and int(c.levels) == int(z.argmax())
    s = learner.level_logprobs(z, c.levels, top=7)
    assert s.top_levels.shape == (7,) and host(s.top_levels).tolist() == host(z).argsort(descending=True).tolist()
    r = ref.Rows(host(z))
    grad, = torch.autograd.grad(s.logprobs, z, create_graph=True)
    near(grad, *r.gradient(host(c.levels), torch.ones(()), torch.zeros(()), torch.float32), 'one row')
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    x = torch.randn((20, 3), device='cuda', requires_grad=True)
    gx, = torch.autograd.grad(learner.gated_scan(x, 0.5)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_gradients_through_saved_tensor_hooks_and_twice():
    """What backward reads is what was saved (here: moved and brought back), and a kept graph gives the same again."""
    from sustaingym_amd import learner
    g = gen(33)
    for K in (5, 2000):
        z = torch.randn((6, K), generator=g, device='cuda', requires_grad=True)
        levels = torch.randint(0, K, (6,), generator=g, device='cuda')
        x = torch.randn((50, 3), generator=g, device='cuda', requires_grad=True)
        gate = torch.rand((50, 3), generator=g, device='cuda', requires_grad=True)

        def work():
            s = learner.level_logprobs(z * 2.0, levels)
            return s.logprobs.sum() + s.entropy.sum() + learner.gated_scan(x * 1.0, gate * 0.5)[0].sum()
        want = torch.autograd.grad(work(), (z, x, gate))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
            loss = work()
        trash = [torch.full((6, K), 7.0, device='cuda') for _ in range(4)]
        first = torch.autograd.grad(loss, (z, x, gate), retain_graph=True)
        again = torch.autograd.grad(loss, (z, x, gate))
        del trash
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, first, again))


def test_calls_from_two_threads_on_two_streams():
    import threading
    from sustaingym_amd import learner
    g = gen(35)
    z = torch.randn((3, 90000), generator=g, device='cuda')
    x = torch.randn((1, 20000, 6), generator=g, device='cuda')
    levels = torch.randint(0, 90000, (3,), generator=g, device='cuda')
    want = (*learner.level_logprobs(z, levels, None, 5), *learner.gated_scan(x, 0.9, dim=1))
    torch.cuda.synchronize()
    got, wrong = {}, []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[k] = [(*learner.level_logprobs(z, levels, None, 5), *learner.gated_scan(x, 0.9, dim=1)) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            try:
                learner.gated_scan(x, 0.9, dim=2)
            except ValueError:
                wrong.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(wrong) == [0, 1]
    assert all(torch.equal(a, b) for k in got for one in got[k] for a, b in zip(one, want))


@pytest.mark.parametrize('dtype', ['f32', 'f64', 'bf16'])
def test_scan_of_one_long_sequence_in_parts(dtype):
    """70 001 steps of one sequence, written out in Python floats (float64) with the bounds of learner_reference.scan."""
    from sustaingym_amd import learner
    kind, T = TYPES[dtype], 70001
    state = torch.float64 if kind == torch.float64 else torch.float32
    u, half = (2.0 ** -53, 0.0) if kind == torch.float64 else (ref.U, ref.half_step(kind))
    for reverse in (False, True):
        g = gen(41)
        x, gate = (torch.rand((1, T), generator=g, device='cuda').sub(0.3).to(kind).requires_grad_(True) for _ in range(2))
        init = torch.ones(1, dtype=state, device='cuda', requires_grad=True)
        resets = torch.rand((1, T), generator=g, device='cuda') < 1e-3
        up = torch.randn((1, T), generator=g, device='cuda').to(kind)
        h, final = learner.gated_scan(x, gate, init, resets, 1, reverse)
        gx, gg, gi = torch.autograd.grad((h, final), (x, gate, init), (up, torch.ones_like(final)))
        flip = (lambda v: v[::-1]) if reverse else (lambda v: v)
        X, A, R, Up = (flip(host(t)[0].tolist()) for t in (x, gate, resets, up))

        def walk(xs, gates, s):
            out, tol, M, N = [], [], abs(s), 0.0
            for xt, a in zip(xs, gates):
                s = a * s + xt
                N = abs(a) * (N + M)
                M = abs(a) * M + abs(xt)
                out.append(s)
                tol.append(u * (2 * N + 16 * M) + 1e-37)
            return out, tol
        A = [0.0 if r else a for a, r in zip(A, R)]
        H, Ht = walk(X, A, 1.0)
        G, Gt = walk(Up[::-1], [1.0] + A[:0:-1], 1.0)
        G, Gt = G[::-1], Gt[::-1]
        prev, pt = [1.0] + H[:-1], [0.0] + Ht[:-1]
        gate_grad = [0.0 if r else a * b for a, b, r in zip(G, prev, R)]
        gate_tol = [abs(a) * (tb + half * abs(b)) + ta * abs(b) * 2 + 2 * u * abs(a * b) for a, ta, b, tb in zip(G, Gt, prev, pt)]

        def check(got, want, tol, what, rounded=True):
            want, tol = (torch.tensor(flip(v), dtype=torch.float64)[None] for v in (want, tol))
            near(got, want, tol + (half * (want.abs() + tol) if rounded else 0), what)
        check(h, H, Ht, 'h')
        check(gx, G, Gt, 'grad_x')
        check(gg, gate_grad, gate_tol, 'grad_gate')
        assert abs(float(final) - H[-1]) <= Ht[-1]
        assert abs(float(gi) - A[0] * G[0]) <= abs(A[0]) * Gt[0] + 2 * u * abs(A[0] * G[0])


@pytest.mark.parametrize('K', [1, 5, 40, 300, 5000])
def test_noise_never_takes_an_allowed_level_out(K):
    """-log(-log(0)) is -inf: a row's only allowed level, or all of them, may get it.  So may the lowest value as a mask overflow."""
    from sustaingym_amd import learner
    z = torch.zeros((6, K), device='cuda')
    mask = torch.ones((6, K), dtype=torch.bool, device='cuda')
    noise = torch.zeros((6, K), device='cuda')
    last = K - 1
    mask[0, :last] = False
    noise[0] = -math.inf                                             # the only one left
    noise[1] = -math.inf                                             # all: the lowest index
    noise[2], noise[2, last] = -math.inf, -50.0                      # a number is ahead of -inf
    noise[3], noise[3, last] = math.nan, -1e30                       # and of NaN
    z[4], noise[4] = torch.finfo(torch.float32).min, -1e38           # the sum passes float32
    mask[4, :last] = False
    mask[5], noise[5] = False, -math.inf                             # nothing allowed
    c = learner.choose_levels(z, noise, mask)
    assert host(c.levels).tolist() == [last, 0, last, last, last, 0]
    lp = host(c.logprobs)
    assert torch.isfinite(lp).all() and lp[0] == 0.0 and lp[4] == 0.0 and lp[5] == 0.0
    assert float((lp[1:4] + math.log(K)).abs().max()) <= 1e-5        # (17 nats at most: 64 steps of float32)


@pytest.mark.parametrize('K', [5, 40, 3001])
def test_gradient_of_a_level_beyond_the_row(K):
    """NaN where the row allows something, nothing where it does not."""
    from sustaingym_amd import learner
    z = torch.zeros((3, K), device='cuda', requires_grad=True)
    mask = torch.ones((3, K), dtype=torch.bool, device='cuda')
    mask[:, 1] = False
    s = learner.level_logprobs(z, torch.tensor([K, 0, 2 ** 40], device='cuda'), mask)
    gr = host(torch.autograd.grad(s.logprobs, z, torch.ones(3, device='cuda'))[0])
    assert not gr[:, 1].any() and torch.isfinite(gr[1]).all()
    assert torch.isnan(gr[0, [0] + list(range(2, K))]).all() and torch.isnan(gr[2, 0])


@pytest.mark.parametrize('shape,strides,dim', [((20, 3, 5), (3, 1, 2 ** 30), 0), ((600, 2, 60), (2, 1, 2 ** 26), 0), ((3, 40, 70), (64, 1, 2 ** 25 + 6), 1),
                                               ((2, 1200, 5), (2 ** 29, 1, 2 ** 30), 1), ((9, 2, 130), (2, 1, 2 ** 25 - 2), 0)])
def test_channels_far_apart(shape, strides, dim):
    """Channels whose columns of one tile lie more than 2^32 bytes apart, as inputs, incoming gradients and outputs."""
    import ctypes as C
    from sustaingym_amd import _lib, learner
    g = gen(41)
    size = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
    big = torch.empty(size, dtype=torch.float16, device='cuda')                  # up to 9.4 GB, written only where it is read
    x = big.as_strided(shape, strides)
    x.copy_(torch.randn(shape, generator=g, device='cuda'))
    gate = torch.rand(shape, generator=g, device='cuda').half()
    up = torch.randn(shape, generator=g, device='cuda').half()
    resets = torch.rand(shape[:2], generator=g, device='cuda') < 0.1
    want = ref.scan(host(x.contiguous()), host(gate), None, host(resets), dim, False, host(up))
    h, final = learner.gated_scan(x, gate, None, resets, dim)
    near(h, *want['h'], 'h')
    near(final, *want['final'], 'final')
    # an output in that layout
    dense = x.contiguous()
    lib, seq = _lib.load(), learner._sequence(shape, dim, False, torch.float16)
    ws = torch.empty(max(1, lib.lrn_scan_workspace(C.byref(seq))), dtype=torch.uint8, device='cuda')
    state = torch.empty(shape[:dim] + shape[dim + 1:], dtype=torch.float32, device='cuda')
    rc = lib.lrn_scan(x.device.index, learner._stream(x.device), C.byref(seq), C.byref(learner._view(dense, dim)), C.byref(learner._view(gate, dim)), 0.0,
                      C.byref(learner._view(resets, dim)), None, C.byref(learner._view(x, dim)), state.data_ptr(), ws.data_ptr(), ws.numel())
    assert rc == 0
    near(x.contiguous(), *want['h'], 'h in that layout')
    # as the gradient that comes in
    leaves = dense.requires_grad_(True), gate.requires_grad_(True)
    h = learner.gated_scan(*leaves, None, resets, dim)[0]
    x.copy_(up)
    gx, gg = torch.autograd.grad(h, leaves, x)
    near(gx, *want['grad_x'], 'grad_x')
    near(gg, *want['grad_gate'], 'grad_gate')


@pytest.mark.parametrize('far', [1, 2 ** 26])
def test_resets_whose_sequences_lie_far_apart(far):
    """Two columns to a lane and flags that one address cannot reach for both."""
    from sustaingym_amd import learner
    g = gen(43)
    T, N = 1100, 66
    x = torch.randn((T, N), generator=g, device='cuda')
    flags = torch.rand((T, N), generator=g, device='cuda') < 0.05
    if far > 1:
        store = torch.empty(far * (N - 1) + T, dtype=torch.bool, device='cuda')          # 4.4 GB
        resets = store.as_strided((T, N), (1, far))
        resets.copy_(flags)
    else:
        resets = flags
    for reverse in (False, True):
        want = ref.scan(host(x), 0.9, None, host(flags), 0, reverse)
        h, final = learner.gated_scan(x, 0.9, None, resets, 0, reverse)
        near(h, *want['h'], 'h')
        near(final, *want['final'], 'final')


def test_more_sequences_than_a_grid_of_wavefronts():
    from sustaingym_amd import learner
    x = torch.randn((2 ** 25 + 3, 2), generator=gen(44), device='cuda')
    h, final = learner.gated_scan(x, 0.5, dim=1)
    assert torch.equal(h[:, 0], x[:, 0]) and torch.equal(h[:, 1], torch.addcmul(x[:, 1], x[:, 0], torch.full_like(x[:, 0], 0.5)))
    assert torch.equal(final, h[:, 1])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f64'])
@pytest.mark.parametrize('T', [2, 3, 7, 8, 9, 15, 16, 17, 33, 64, 65, 129, 256, 257, 300, 511, 512, 513])
def test_short_sequences_with_time_the_fast_index(T, dtype):
    """Several of them share a wavefront; 67 do not fill the last one."""
    from sustaingym_amd import learner
    kind = TYPES[dtype]
    g = gen(50 + T)
    N = 67
    x = torch.randn((N, T), generator=g, device='cuda').to(kind)
    gate = torch.rand((N, T), generator=g, device='cuda').to(kind)
    resets = torch.rand((N, T), generator=g, device='cuda') < 0.1
    up = torch.randn((N, T), generator=g, device='cuda').to(kind)
    state = torch.float64 if dtype == 'f64' else torch.float32
    initial, g_final = (torch.randn(N, generator=g, device='cuda').to(state) for _ in range(2))
    for reverse in (False, True):
        want = ref.scan(host(x), host(gate), host(initial), host(resets), 1, reverse, host(up), host(g_final))
        leaves = [t.clone().requires_grad_(True) for t in (x, gate, initial)]
        out = learner.gated_scan(*leaves, resets, 1, reverse)
        near(out[0], *want['h'], 'h')
        near(out[1], *want['final'], 'final')
        for name, got in zip(('grad_x', 'grad_gate', 'grad_initial'), torch.autograd.grad(out, leaves, (up, g_final))):
            near(got, *want[name], name)
    if dtype != 'bf16':
        ends, values, last = resets, torch.randn((N, T), generator=g, device='cuda'), torch.randn(N, generator=g, device='cuda')
        a = learner.advantages(x.t(), values.t(), ends.t(), last)
        want, tol = ref.advantages(host(x).t(), host(values).t(), host(ends).t(), host(last), 0.99, 0.95)
        near(a.advantages, want, tol + ref.U * want.abs(), 'advantages')
        assert a.targets.stride() == x.t().stride()


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('shape,dim', [((33, 1, 64), 0), ((64, 3, 128), 0), ((65, 2, 192), 0), ((5, 127, 64), 1), ((2, 130, 320), 1), ((40, 130, 64), 0), ((2, 511, 64), 1),
                                       ((700, 1, 8320), 0)])
def test_channels_by_the_64(shape, dim, dtype):
    """Whole tiles of channels, with and without what each form of the kernel has, also from views that are not aligned."""
    from sustaingym_amd import learner
    kind = TYPES[dtype]
    g = gen(60 + shape[1])
    wide = (*shape[:2], shape[2] + 3)
    x, gate, up = (torch.rand(wide, generator=g, device='cuda').to(kind)[..., k:k + shape[2]] for k in (1, 2, 3))
    resets = torch.rand(shape[:2], generator=g, device='cuda') < 0.05
    rest = shape[:dim] + shape[dim + 1:]
    initial, g_final = (torch.randn(rest, generator=g, device='cuda') for _ in range(2))
    for reverse, a, r, i in ((False, gate, resets, initial), (True, gate, None, None), (False, 0.9, resets, initial), (True, -0.5, None, initial),
                             (True, gate, resets, initial)):
        want = ref.scan(host(x), a if isinstance(a, float) else host(a), host(i), host(r), dim, reverse, host(up), host(g_final))
        leaves = {'grad_x': x, 'grad_gate': a, 'grad_initial': i}
        leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items() if isinstance(v, torch.Tensor)}
        out = learner.gated_scan(leaves['grad_x'], leaves.get('grad_gate', a), leaves.get('grad_initial'), r, dim, reverse)
        near(out[0], *want['h'], 'h')
        near(out[1], *want['final'], 'final')
        for name, got in zip(leaves, torch.autograd.grad(out, list(leaves.values()), (up, g_final), retain_graph=True)):
            near(got, *want[name], name)
        if 'grad_gate' in leaves:                       # the gate as it is, and as a leaf of its own
            only, = torch.autograd.grad(out, [leaves['grad_x']], (up, g_final))
            near(only, *want['grad_x'], 'grad_x again')
    # a gate that needs no gradient: the state in front is not read
    leaf = x.detach().requires_grad_(True)
    want = ref.scan(host(x), host(gate), None, host(resets), dim, False, host(up))
    got, = torch.autograd.grad(learner.gated_scan(leaf, gate, None, resets, dim)[0], leaf, up)
    near(got, *want['grad_x'], 'grad_x alone')
