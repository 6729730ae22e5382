"""The gate's gradient of 16-bit sequences is made of states that are not rounded: held to the bound that float32 sequences have,
and one rounding of the result."""
import pytest
import torch

from tests import learner_reference as ref
from tests.test_gpu_learner import SCANS, TYPES, gen, near

from tests.test_gpu_learner import host

pytestmark = pytest.mark.gpu

FORMS = [f for f in SCANS if f[0] not in ((9, 65540), (20, 140000), (40, 70, 1000))]
FORMS += [((T, 2, C), 0) for T in (7, 8, 9, 16, 23, 33, 65, 130) for C in (5, 64)]                     # columns, whole tiles of channels
FORMS += [((67, T), 1) for T in (1, 2, 7, 8, 9, 15, 16, 17, 64, 513)] + [((3, 4100, 64), 1), ((600, 1, 128), 0), ((1, 33000), 1), ((2, 1100, 33), 1), ((1100, 2, 33), 0),
          ((9, 2500), 0)]


def widened(want, dtype):
    """A bound of float32 arithmetic, and the result's own rounding to ``dtype``."""
    v, tol = want
    return v, tol + ref.half_step(dtype) * (v.abs() + tol) + ref.tiny(dtype)


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('shape,dim', FORMS, ids=[f'{"x".join(map(str, s))}-{d}' for s, d in FORMS])
def test_the_gate_gradient_has_the_states_as_they_are(shape, dim, dtype):
    from sustaingym_amd import learner
    kind = TYPES[dtype]
    rest = shape[:dim] + shape[dim + 1:]
    for i, (reverse, with_resets, with_initial) in enumerate(((False, True, True), (True, False, True), (True, True, False), (False, False, False))):
        g = gen(7 * shape[0] + i)
        x = torch.randn(shape, generator=g, device='cuda').to(kind)
        gate = torch.sigmoid(torch.randn(shape, generator=g, device='cuda') * 2 + 2).to(kind).requires_grad_(True)
        initial = torch.randn(rest, generator=g, device='cuda') if with_initial else None
        resets = torch.rand(shape[:2], generator=g, device='cuda') < 0.03 if with_resets else None
        gh = torch.randn(shape, generator=g, device='cuda').to(kind)
        gf = torch.randn(rest, generator=g, device='cuda')
        want = ref.scan(host(x).float(), host(gate).float(), host(initial), host(resets), dim, reverse, host(gh).float(), host(gf))
        x.requires_grad_(i % 2 == 0)
        out = learner.gated_scan(x, gate, initial, resets, dim, reverse)
        leaves = [gate, x] if i % 2 == 0 else [gate]
        grads = torch.autograd.grad(out, leaves, (gh, gf), retain_graph=True)
        near(grads[0], *widened(want['grad_gate'], kind), 'grad_gate')
        if i % 2 == 0:
            near(grads[1], *widened(want['grad_x'], kind), 'grad_x')
            only, = torch.autograd.grad(out, x, (gh, gf))
            assert torch.equal(only, grads[1])


def test_kept_states_lie_where_they_are_said_to():
    """Through the C-ABI: the state before the step that has (j + 1) 8 - 1 behind it, nothing beside the elements."""
    import ctypes as C
    from sustaingym_amd import _lib, learner
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    g = gen(5)
    for T, N, Cn in ((1, 3, 5), (8, 2, 3), (21, 4, 7), (64, 2, 64), (300, 1, 64), (300, 2, 66), (1100, 1, 66)):
        for reverse in (0, 1):
            x, gate = (torch.rand((T, N, Cn), generator=g, device='cuda').bfloat16() for _ in range(2))
            n = -(-T // _lib.LEARNER_KEEP)
            store = torch.full((n + 2, N, Cn), -7.0, device='cuda')
            h, final = torch.empty_like(x), torch.empty((N, Cn), device='cuda')
            seq = _lib.LearnerSeq(T, N, Cn, reverse, 1)
            ws = torch.empty(max(1, lib.lrn_scan_workspace(C.byref(seq))), dtype=torch.uint8, device='cuda')
            views = [C.byref(learner._view(t, 0)) for t in (x, gate, h, store[1:])]
            assert lib.lrn_scan_keep(0, st, C.byref(seq), views[0], views[1], None, None, views[2], views[3], final.data_ptr(), ws.data_ptr(), ws.numel()) == 0
            want = ref.scan(host(x).float(), host(gate).float(), None, None, 0, bool(reverse))
            order = range(T) if not reverse else range(T - 1, -1, -1)
            order = list(order)
            for j in range(n):
                at = T - (j + 1) * 8                                     # the step in walking order
                if at > 0:
                    v, tol = (w[order[at - 1]] for w in want['h'])
                    near(store[1 + j], v, tol, (T, j))
            assert bool((store[0] == -7).all()) and bool((store[n + 1] == -7).all())


BROADCAST = [((40, 2, 5), 0, (40, 1, 5)), ((70, 2, 64), 0, (70, 1, 64)), ((2, 40, 7), 1, (1, 40, 7)), ((2, 600, 64), 1, (1, 600, 64)), ((2, 300), 1, (300,)),
             ((2, 33000), 1, (1, 33000)), ((2, 1100, 33), 1, (1100, 33)), ((1100, 2, 34), 0, (1100, 1, 34)), ((9, 2, 5), 0, (5,)), ((30, 2, 64), 0, (1, 2, 64)),
             ((30, 2, 3), 0, (30, 2, 1)), ((20, 2), 0, ()), ((20, 2, 130), 0, (1, 1, 1)), ((1, 2, 3), 0, (3,)), ((2, 1, 64), 1, (1, 1, 64))]


@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32', 'f64'])
@pytest.mark.parametrize('shape,dim,gshape', BROADCAST, ids=[f'{"x".join(map(str, s))}-{"x".join(map(str, b))}' for s, _, b in BROADCAST])
def test_the_gradient_of_a_broadcast_gate_is_summed_before_it_is_rounded(shape, dim, gshape, dtype):
    """Two sequences whose terms nearly cancel: rounded to 16 bits first, their sum would be off by more than its own size allows.
    torch adds n float32 values up, at most n u of the sum of their sizes off."""
    from sustaingym_amd import learner
    kind = TYPES[dtype]
    g = gen(sum(shape))
    batch = 1 - dim
    one = list(shape)
    one[batch] = 1
    x, gh = (torch.randn(one, generator=g, device='cuda').to(kind).expand(shape).contiguous() for _ in range(2))
    other = (slice(None),) * batch + (1,)
    x[other] *= 1 + 2.0 ** -6
    gh[other] *= -1
    gate = torch.sigmoid(torch.randn(gshape, generator=g, device='cuda') + 2).to(kind).requires_grad_(True)
    wide = (lambda t: t.double()) if kind == torch.float64 else (lambda t: t.float())
    for reverse in (False, True):
        resets = torch.rand(shape[:2], generator=g, device='cuda') < 0.05 if reverse else None
        want = ref.scan(wide(host(x)), wide(host(gate)).expand(shape), None, host(resets), dim, reverse, wide(host(gh)))
        h, _ = learner.gated_scan(x, gate, None, resets, dim, reverse)
        got, = torch.autograd.grad(h, gate, gh)
        assert got.dtype == kind and got.shape == gshape
        v, tol = want['grad_gate']
        n = v.numel() // max(1, gate.numel())
        u = 2.0 ** -53 if kind == torch.float64 else ref.U
        size = v.abs().sum_to_size(gshape)
        v, tol = v.sum_to_size(gshape), tol.sum_to_size(gshape) + n * u * size
        if kind in (torch.bfloat16, torch.float16):
            v, tol = widened((v, tol), kind)
        near(got, v, tol, 'gate')


def test_kept_states_in_a_captured_step_and_through_hooks():
    """16-bit gates, whole and broadcast, in every layout: replays with new inputs and eager work between them give the eager
    results; what backward reads is what was saved."""
    from sustaingym_amd import learner
    g = gen(21)
    cases = [((2, 40, 66), 1, (2, 40, 66)), ((300, 1, 64), 0, (300, 1, 64)), ((3, 9000), 1, (3, 9000)), ((60, 4, 5), 0, (4, 1)), ((1100, 2, 34), 0, (34,)), ((7, 30), 1, (7, 1))]
    x = [torch.rand(s, generator=g, device='cuda').bfloat16().requires_grad_(True) for s, _, _ in cases]
    gate = [torch.rand(s, generator=g, device='cuda').bfloat16().requires_grad_(True) for _, _, s in cases]

    def step():
        out = []
        for (_, dim, _), a, b in zip(cases, x, gate):
            h, final = learner.gated_scan(a, b, dim=dim)
            # (detached: a capture may not begin while an eager graph of the same leaves lives)
            out += [h.detach(), final.detach(), *torch.autograd.grad((h, final), (a, b), (h.detach(), final.detach()))]
            del h, final
        return out

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().cpu(), lambda t: t.cuda()):
        through = step()
    assert all(torch.equal(a, b) for a, b in zip(through, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(through, step()))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            for t in (*x, *gate):
                t.copy_(torch.rand(t.shape, generator=g, device='cuda'))
        want = [t.clone() for t in step()]
        if k % 2:
            torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
