"""What a learner computes next to the engine, on the device tensors that the vector environments hand out
(include/learner_ops.h; hand-written gfx950 kernels in the same library).

    choose_levels(logits, noise, mask)          -> LevelChoice    the levels that ``step`` takes, from a policy's logits
    level_logprobs(logits, levels, mask, top)   -> LevelScores    log probabilities of levels that were played (differentiable)
    gated_scan(x, gate, initial, resets)        -> (h, final)     h_t = gate_t h_{t-1} + x_t over a trajectory (differentiable)
    advantages(rewards, values, ends, ...)      -> Advantages     generalised advantages and value targets

A *level* is a choice of :class:`DiscreteActionWrapper` (or any other index into a row of logits); a row is one decision, so
a batch of N environments with n stations and K levels is ``logits[N, n, K]``.

Every call runs on the current torch stream of its tensors' device, does not synchronise, and may be captured into a graph.
Tensors of any strides are taken as they are where the last dimension of logits and noise is dense; anything else is copied
first.  Wrong arguments raise ``ValueError`` before anything is launched.  There is no CPU form: CPU tensors are refused.  Gradients are
those of a backward pass, once: second derivatives raise, forward-mode tangents are refused.

To capture a backward pass into a graph, run the forward pass inside the same capture and ask for the gradients there with
``torch.autograd.grad``, for leaves that no eager graph holds at that time (a tensor's ``detach().requires_grad_()`` taken inside
the capture is one): torch orders a leaf's gradient behind the stream that first used the leaf, and a capture cannot wait for a
stream outside it.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SEQ_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}
MAX_TOP = _lib.LEARNER_MAX_TOP
_SHORT_ROW = _lib.LEARNER_SHORT_ROW      # up to here no workspace and no statistics for the backward pass
_KEEP = _lib.LEARNER_KEEP                # of 16-bit sequences every so many steps' state is kept for the backward pass


class LevelChoice(NamedTuple):
    levels: torch.Tensor         # int64 [...]
    logprobs: torch.Tensor       # float32 [...]
    entropy: torch.Tensor        # float32 [...]


class LevelScores(NamedTuple):
    logprobs: torch.Tensor               # float32 [...]
    entropy: torch.Tensor                # float32 [...]
    top_logprobs: torch.Tensor | None    # float32 [..., top]
    top_levels: torch.Tensor | None      # int64 [..., top]


class Advantages(NamedTuple):
    advantages: torch.Tensor     # float32 [T, N]
    targets: torch.Tensor        # float32 [T, N]


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise _lib.EngineLibraryError(f'{what} failed with code {rc}: {_lib.load().lrn_last_error().decode("utf-8", "replace")}')


def _on_device(name: str, t, device=None) -> None:
    if isinstance(t, torch.Tensor) and t.is_cuda and (device is None or t.device == device) and not t.is_neg():
        return
    if not isinstance(t, torch.Tensor):
        raise ValueError(f'{name}: a tensor is needed, not {type(t).__name__}')
    if t.is_neg():
        raise ValueError(f'{name}: its memory holds the negated values (the imaginary part of a conjugate view): resolve_neg() it first')
    if not t.is_cuda:
        raise ValueError(f'{name}: a CUDA tensor is needed (there is no CPU form)')
    raise ValueError(f'{name}: on {t.device}, the first argument is on {device}')


def _no_tangents(**inputs) -> None:
    """A dual tensor does not require a gradient: its tangent would be dropped without a word."""
    for name, t in inputs.items():
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f'{name}: there is no forward-mode derivative')


def _broadcasts(t, shape) -> bool:
    try:
        return torch.broadcast_shapes(t.shape, shape) == shape
    except RuntimeError:
        return False


def _stream(device) -> int:
    """The current stream's handle (``torch.cuda.current_stream(device).cuda_stream`` without the object: 0.1 us instead of 2)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _workspace(nbytes: int, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- rows of logits --------------------------------------------------------------------------------------------------

def _folded(shape, strides):
    """Leading dimensions as (outer, inner) with two strides for each of ``strides``; None if they do not fold that far."""
    dims: list[list] = []
    for i, n in enumerate(shape):
        if n == 1:
            continue
        s = [st[i] for st in strides]
        if dims and all(p == n * q for p, q in zip(dims[-1][1], s)):
            dims[-1] = [dims[-1][0] * n, s]
        else:
            dims.append([n, s])
    if len(dims) > 2:
        return None
    while len(dims) < 2:
        dims.insert(0, [1, [0] * len(strides)])
    return dims[0][0], dims[1][0], list(zip(dims[0][1], dims[1][1]))


class _Rows:
    """logits (and mask, noise) laid out for the C call; keeps the tensors that its pointers belong to alive."""

    __slots__ = ('struct', 'keep', 'noise', 'noise_strides')

    def __init__(self, logits, mask, noise=None):
        shape = logits.shape
        K = shape[-1]
        if logits.is_contiguous() and (mask is None or mask.shape == shape and mask.is_contiguous()) and (
                noise is None or noise.shape == shape and noise.is_contiguous()):
            self.struct = _lib.LearnerRows(logits.data_ptr(), 1, logits.numel() // K, K, 0, K,
                                           None if mask is None else mask.data_ptr(), 0, K, 1, _ROW_TYPES[logits.dtype])
            self.keep = (logits, mask, noise)
            self.noise, self.noise_strides = noise, (0, K)
            return
        mask_level = 1
        if logits.stride(-1) != 1 and K > 1:
            logits = logits.contiguous()
        if mask is not None:
            mask = mask.expand(shape)
            mask_level = mask.stride(-1)
            if mask_level not in (0, 1):
                mask, mask_level = mask.contiguous(), 1
        if noise is not None:
            noise = noise.expand(shape)
            if noise.stride(-1) != 1 and K > 1:
                noise = noise.contiguous()
        folded = _folded(shape[:-1], [t.stride()[:-1] for t in (logits, mask, noise) if t is not None])
        if folded is None:
            logits = logits.contiguous()
            mask = None if mask is None else mask.contiguous()
            noise = None if noise is None else noise.contiguous()
            mask_level = 1
            outer, inner, strides = 1, logits.numel() // K, [(0, K)] * 3
        else:
            outer, inner, strides = folded
            if mask is None:
                strides.insert(1, (0, 0))
            if noise is None:
                strides.append((0, 0))
        self.struct = _lib.LearnerRows(logits.data_ptr(), outer, inner, K, *strides[0], _ptr(mask), *strides[1], mask_level,
                                       _ROW_TYPES[logits.dtype])
        self.keep = (logits, mask, noise)
        self.noise, self.noise_strides = noise, strides[2]


def _check_rows(logits, mask, noise=None):
    _on_device('logits', logits)
    if logits.dtype not in _ROW_TYPES:
        raise ValueError(f'logits: float32, bfloat16 or float16, not {logits.dtype}')
    shape = logits.shape
    if not shape or not 1 <= shape[-1] < 2 ** 30:
        raise ValueError(f'logits: [..., levels], got {tuple(shape)}')
    if mask is None and noise is None:
        return
    for name, t, kind in (('mask', mask, torch.bool), ('noise', noise, torch.float32)):
        if t is None:
            continue
        _on_device(name, t, logits.device)
        if t.dtype != kind:
            raise ValueError(f'{name}: {kind}, not {t.dtype}')
        if t.shape != shape and not _broadcasts(t, shape):
            raise ValueError(f'{name}: {tuple(t.shape)} does not broadcast to the logits\' {tuple(shape)}')


def choose_levels(logits, noise=None, mask=None) -> LevelChoice:
    """One level for every row: the allowed one with the largest ``logits + noise`` (the lowest index among equals).

    logits: ``[..., K]`` float32 / bfloat16 / float16.
    noise: float32, broadcastable to the logits; with Gumbel noise (``-log(-log(u))``) the level is a sample of
        ``softmax(logits)`` over the allowed levels, without noise it is the most probable one.  Noise of -inf or NaN puts a
        level behind all others of its row.
    mask: bool, broadcastable to the logits, True = allowed (``mask[N, n, 1]``: stations without a car).

    Returns int64 levels — what ``EVChargingVectorEnv(discrete_bins=K).step`` takes — with their log probabilities and the
    entropy of every row (of the logits without noise; float32).  A row without an allowed level gives level 0, log
    probability 0 and entropy 0.  No gradient flows: a learner asks :func:`level_logprobs` for the same levels."""
    _check_rows(logits, mask, noise)
    logits = logits.detach()
    lib, device, shape = _lib.load(), logits.device, logits.shape[:-1]
    levels = torch.empty(shape, dtype=torch.int64, device=device)
    logprobs = torch.empty(shape, dtype=torch.float32, device=device)
    entropy = torch.empty(shape, dtype=torch.float32, device=device)
    rows = _Rows(logits, mask, noise)
    ref = C.byref(rows.struct)
    nbytes = 0 if rows.struct.levels <= _SHORT_ROW else lib.lrn_choose_workspace(ref)
    ws = _workspace(nbytes, device)
    _check(lib.lrn_choose(device.index, _stream(device), ref, _ptr(rows.noise), rows.noise_strides[0], rows.noise_strides[1],
                          levels.data_ptr(), logprobs.data_ptr(), entropy.data_ptr(), _ptr(ws), nbytes), 'choose_levels')
    return LevelChoice(levels, logprobs, entropy)


def _score(rows, levels, shape, device, top, want_stat):
    lib = _lib.load()
    ref = C.byref(rows.struct)
    logprobs = torch.empty(shape, dtype=torch.float32, device=device)
    entropy = torch.empty(shape, dtype=torch.float32, device=device)
    stat = torch.empty((*shape, 2), dtype=torch.float32, device=device) if want_stat else None
    tl = torch.empty((*shape, top), dtype=torch.float32, device=device) if top else None
    ti = torch.empty((*shape, top), dtype=torch.int64, device=device) if top else None
    nbytes = 0 if rows.struct.levels <= _SHORT_ROW else lib.lrn_score_workspace(ref, top)
    ws = _workspace(nbytes, device)
    _check(lib.lrn_score(device.index, _stream(device), ref, levels.data_ptr(), logprobs.data_ptr(), entropy.data_ptr(),
                         _ptr(stat), top, _ptr(tl), _ptr(ti), _ptr(ws), nbytes), 'level_logprobs')
    return logprobs, entropy, stat, tl, ti


def _row_gradient(g):
    """A per-row gradient and its element stride: one value for all rows (a sum's gradient) is not spread out."""
    if g is None:
        return None, 0
    if g.is_contiguous():
        return g, 1
    if all(s == 0 or n == 1 for n, s in zip(g.shape, g.stride())):
        return g, 0
    return g.contiguous(), 1


def _no_second(gradient, ctx, *grads):
    """``gradient(ctx, *grads)``; under ``create_graph`` its results say, when differentiated, that they cannot be."""
    return once_differentiable(gradient)(ctx, *grads) if torch.is_grad_enabled() else gradient(ctx, *grads)


class _LevelLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, levels, mask, top):
        rows = _Rows(logits, mask)
        needs = rows.struct.levels > _SHORT_ROW
        logprobs, entropy, stat, tl, ti = _score(rows, levels, logits.shape[:-1], logits.device, top, needs)
        ctx.save_for_backward(logits, levels, mask, stat, entropy if needs else None)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(tl, ti)
        return logprobs, entropy, tl, ti

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy, *_):
        return _no_second(_LevelLogprobs._gradient, ctx, g_logprobs, g_entropy)

    @staticmethod
    def _gradient(ctx, g_logprobs, g_entropy):
        logits, levels, mask, stat, entropy = ctx.saved_tensors
        rows = _Rows(logits, mask)       # (from what was saved: hooks may have moved it meanwhile)
        g_logprobs, s_lp = _row_gradient(g_logprobs)
        g_entropy, s_h = _row_gradient(g_entropy)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _check(_lib.load().lrn_score_backward(logits.device.index, _stream(logits.device), C.byref(rows.struct),
                                              levels.data_ptr(), _ptr(stat), _ptr(entropy), _ptr(g_logprobs), s_lp,
                                              _ptr(g_entropy), s_h, grad.data_ptr()), 'level_logprobs backward')
        return grad, None, None, None


def level_logprobs(logits, levels, mask=None, top: int = 0) -> LevelScores:
    """Log probabilities of given levels under ``softmax(logits)`` over the allowed levels, entropies, and alternatives.

    logits: ``[..., K]`` float32 / bfloat16 / float16; gradients of ``logprobs`` and ``entropy`` flow to them.
    levels: int64 or int32 ``[...]``; a negative level marks a padded row (log probability 0, no gradient through it).  A level
        that the mask forbids has log probability -inf; one ``>= K`` gives NaN (levels are not looked at on the host).
    mask: bool, broadcastable to the logits, True = allowed; what masked places hold is never used.  A row that the mask leaves
        empty has log probability 0, entropy 0 and gradient 0.
    top: 0 .. min(K, 64): the most probable levels of each row in falling order (the lowest index first among equals) with their
        log probabilities, ``[..., top]``; behind the last allowed one -1 and -inf.  No gradient flows through these.

    Log probabilities, entropies and all sums are float32 whatever the logits' type; the gradient has the logits' type."""
    _check_rows(logits, mask)
    if forward_ad._current_level >= 0:
        _no_tangents(logits=logits)
    _on_device('levels', levels, logits.device)
    if levels.shape != logits.shape[:-1]:
        raise ValueError(f'levels: {tuple(levels.shape)}, the logits have rows {tuple(logits.shape[:-1])}')
    if levels.dtype != torch.int64:
        if levels.dtype != torch.int32:
            raise ValueError(f'levels: int64 or int32, not {levels.dtype}')
        levels = levels.to(torch.int64)
    levels = levels.contiguous()
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f'top: 0 .. {min(MAX_TOP, logits.shape[-1])}, got {top}')
    if logits.requires_grad and torch.is_grad_enabled():
        return LevelScores(*_LevelLogprobs.apply(logits, levels, mask, top))
    rows = _Rows(logits.detach(), mask)
    logprobs, entropy, _, tl, ti = _score(rows, levels, logits.shape[:-1], logits.device, top, False)
    return LevelScores(logprobs, entropy, tl, ti)


# ---- recurrences -----------------------------------------------------------------------------------------------------

def _view(t, dim):
    """(time, batch, channel) strides of a tensor whose time dimension is ``dim``."""
    if t is None:
        return None
    st = t.stride()
    if t.dim() == 1:
        return _lib.LearnerView(t.data_ptr(), st[0], 0, 0)
    return _lib.LearnerView(t.data_ptr(), st[dim], st[1 - dim], st[2] if t.dim() > 2 else 0)


def _ref(v):
    return None if v is None else C.byref(v)


def _sequence(shape, dim, reverse, dtype):
    return _lib.LearnerSeq(shape[dim], shape[1 - dim] if len(shape) > 1 else 1, shape[2] if len(shape) > 2 else 1,
                           int(reverse), _SEQ_TYPES[dtype])


def _state_type(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _laid_out(shape, stride, dtype, device):
    """An output in the layout of the input with these strides (a batch-major trajectory stays one); contiguous where that one
    has holes or overlaps."""
    if 0 in shape:
        return torch.empty(shape, dtype=dtype, device=device)
    expect = 1
    for s, n in sorted((s, n) for n, s in zip(shape, stride) if n != 1):
        if s != expect:
            return torch.empty(shape, dtype=dtype, device=device)
        expect *= n
    return torch.empty_strided(shape, stride, dtype=dtype, device=device)


def _spread(gate, shape):
    return gate if gate is None or gate.shape == shape else gate.expand(shape)


def _kept(h, dim):
    """Room for every eighth state of 16-bit ``h``, ``[elements, N, C]``: along time where h is, by columns otherwise."""
    steps, N = h.shape[dim], h.shape[1 - dim] if h.dim() > 1 else 1
    C_, n = h.shape[2] if h.dim() > 2 else 1, -(-steps // _KEEP)
    if C_ == 1 and steps > 1 and h.stride(dim) == 1:
        return torch.empty((N, n, 1), dtype=torch.float32, device=h.device).transpose(0, 1)
    return torch.empty((n, N, C_), dtype=torch.float32, device=h.device)


def _scan(x, gate, gate_const, initial, resets, dim, reverse, keep=False):
    lib, device = _lib.load(), x.device
    h = torch.empty(x.shape, dtype=x.dtype, device=device) if x.is_contiguous() else _laid_out(x.shape, x.stride(), x.dtype, device)
    final = torch.empty(x.shape[:dim] + x.shape[dim + 1:], dtype=_state_type(x.dtype), device=device)
    seq = _sequence(x.shape, dim, reverse, x.dtype)
    ref = C.byref(seq)
    nbytes = lib.lrn_scan_workspace(ref)
    ws = _workspace(nbytes, device)
    stream, views = _stream(device), (_ref(_view(x, dim)), _ref(_view(gate, dim)), _ref(_view(resets, dim)), _ref(_view(h, dim)))
    if keep:
        kept = _kept(h, dim)
        _check(lib.lrn_scan_keep(device.index, stream, ref, views[0], views[1], views[2], _ptr(initial), views[3], _ref(_view(kept, 0)),
                                 final.data_ptr(), _ptr(ws), nbytes), 'gated_scan')
        return h, final, kept
    _check(lib.lrn_scan(device.index, stream, ref, views[0], views[1], gate_const, views[2], _ptr(initial), views[3],
                        final.data_ptr(), _ptr(ws), nbytes), 'gated_scan')
    return h, final


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, resets, gate_const, dim, reverse):
        # The gate's gradient needs the states.  h holds them, but rounded for 16-bit sequences: there every eighth is kept in
        # float32, and the backward pass walks the others again from x.
        keep = ctx.needs_input_grad[1] and x.dtype in (torch.bfloat16, torch.float16)
        h, final, *kept = _scan(x, _spread(gate, x.shape), gate_const, initial, resets, dim, reverse, keep)
        ctx.save_for_backward(gate, resets, initial, (x if keep else h) if ctx.needs_input_grad[1] else None, *kept)
        ctx.args = (gate_const, dim, reverse, x.shape, x.stride(), x.dtype, x.device)
        ctx.set_materialize_grads(False)
        return h, final

    @staticmethod
    def backward(ctx, g_h, g_final):
        return _no_second(_GatedScan._gradient, ctx, g_h, g_final)

    @staticmethod
    def _gradient(ctx, g_h, g_final):
        gate, resets, initial, states, *kept = ctx.saved_tensors
        gate_const, dim, reverse, shape, stride, dtype, device = ctx.args
        want_x, want_gate, want_initial = ctx.needs_input_grad[:3]
        if g_h is None and g_final is None:
            return (None,) * 7
        lib = _lib.load()
        g_final = None if g_final is None else g_final.contiguous()
        if g_h is None:                                              # only the last state was used
            g_h = torch.zeros((), dtype=dtype, device=device).expand(shape)
        gx = _laid_out(shape, stride, dtype, device)
        # (of a broadcast gate: summed before it is rounded)
        spread, kind = gate is not None and gate.shape != shape, dtype
        if spread:
            of, gate, kind = gate.shape, gate.expand(shape), _state_type(dtype)
        gg = _laid_out(shape, stride, kind, device) if want_gate else None
        gi = torch.empty(initial.shape, dtype=initial.dtype, device=device) if want_initial else None
        seq = _sequence(shape, dim, reverse, dtype)
        ref = C.byref(seq)
        nbytes = lib.lrn_scan_workspace(ref)
        ws = _workspace(nbytes, device)
        stream, up, out = _stream(device), (_ref(_view(g_h, dim)), _ptr(g_final), _ref(_view(gx, dim)), _ref(_view(gg, dim))), (_ptr(gi), _ptr(ws), nbytes)
        if kept and want_gate:
            _check(lib.lrn_scan_keep_backward(device.index, stream, ref, _ref(_view(states, dim)), _ref(_view(gate, dim)),
                                              _ref(_view(resets, dim)), _ptr(initial), _ref(_view(kept[0], 0)), *up, _SEQ_TYPES[kind], *out),
                   'gated_scan backward')
        else:
            _check(lib.lrn_scan_backward(device.index, stream, ref, _ref(_view(gate, dim)), gate_const, _ref(_view(resets, dim)),
                                         _ptr(initial), _ref(_view(states, dim)), *up, *out), 'gated_scan backward')
        if spread and want_gate:
            gg = gg.sum_to_size(of).to(dtype)
        return gx if want_x else None, gg, gi, None, None, None, None


def gated_scan(x, gate, initial=None, resets=None, dim: int = 0, reverse: bool = False):
    """``h_t = gate_t * h_{t-1} + x_t`` along ``dim``; returns ``(h, final)``.

    x: ``[T]``, ``[T, N]`` or ``[T, N, C]`` (``dim=0``), ``[N, T]`` or ``[N, T, C]`` (``dim=1``); float32, bfloat16, float16 or
        float64.  T may be 0 (``final`` is the initial state) or 1 (one step of a policy's state).
    gate: a tensor of x's type, broadcastable to x, or a number (discounted returns: ``gated_scan(rewards, gamma,
        resets=ends, reverse=True)``).
    initial: the state before the first step, x's shape without ``dim`` (float32; float64 for float64 x); None = 0.
    resets: bool, x's first two dimensions: the sequence starts anew at this step, ``h_t = x_t`` — nothing from before enters,
        not even a NaN.  Forward, that is the step AFTER an episode's end; with ``reverse`` the step of the end itself.
    reverse: from the last step to the first (``h_t = gate_t * h_{t+1} + x_t``).

    A gate of exactly 0 does what a reset does; a NaN or infinite gate makes the state NaN, also a state of 0.  Steps are joined by
    the products of their gates, which are meant to be at most 1 in size: larger ones are computed as well, but where their product
    over a run of steps leaves float32's range (float64's for float64), so does the state; and behind a product that has become 0, a
    NaN or an infinity of the state may be gone.

    ``h`` has x's type and layout (contiguous where x has holes or is expanded); ``final`` is the last state of the walk in the
    state's own type, what a following call takes as ``initial``.  Differentiable in x, gate and initial; gradients are made of states
    in the state's own type, also where h holds them rounded to 16 bits."""
    _on_device('x', x)
    device, shape = x.device, x.shape
    if x.dtype not in _SEQ_TYPES:
        raise ValueError(f'x: float32, bfloat16, float16 or float64, not {x.dtype}')
    if not 1 <= len(shape) <= 3:
        raise ValueError(f'x: one to three dimensions, got {tuple(shape)}')
    if dim not in (0, 1) or dim >= len(shape):
        raise ValueError(f'dim: 0 or 1 of {tuple(shape)}, got {dim}')
    const = 0.0
    if isinstance(gate, torch.Tensor):
        _on_device('gate', gate, device)
        if gate.dtype != x.dtype:
            raise ValueError(f'gate: {gate.dtype}, x is {x.dtype}')
        if gate.shape != shape:
            if not _broadcasts(gate, shape):
                raise ValueError(f'gate: {tuple(gate.shape)} does not broadcast to x\'s {tuple(shape)}')
    elif isinstance(gate, (int, float)):
        const, gate = float(gate), None
    else:
        raise ValueError(f'gate: a tensor or a number, not {type(gate).__name__}')
    if initial is not None:
        _on_device('initial', initial, device)
        rest = shape[:dim] + shape[dim + 1:]
        if initial.shape != rest:
            raise ValueError(f'initial: {tuple(initial.shape)} instead of {tuple(rest)}')
        if initial.dtype != _state_type(x.dtype):
            raise ValueError(f'initial: {_state_type(x.dtype)}, not {initial.dtype}')
        initial = initial.contiguous()
    if resets is not None:
        _on_device('resets', resets, device)
        if resets.dtype != torch.bool:
            raise ValueError(f'resets: torch.bool, not {resets.dtype}')
        if resets.shape != shape[:2]:
            raise ValueError(f'resets: {tuple(resets.shape)} instead of {tuple(shape[:2])}')
    reverse = bool(reverse)
    if forward_ad._current_level >= 0:
        _no_tangents(x=x, gate=gate, initial=initial)
    if torch.is_grad_enabled() and (x.requires_grad or (gate is not None and gate.requires_grad)
                                    or (initial is not None and initial.requires_grad)):
        return _GatedScan.apply(x, gate, initial, resets, const, dim, reverse)
    return _scan(x.detach(), _spread(gate, shape), const, initial, resets, dim, reverse)


def advantages(rewards, values, ends, last_values, gamma: float = 0.99, lam: float = 0.95) -> Advantages:
    """Generalised advantages ``A_t = d_t + gamma lam (1 - end_t) A_{t+1}``, ``d_t = r_t + gamma (1 - end_t) V_{t+1} - V_t``, and
    the value targets ``A_t + V_t`` of a trajectory.

    rewards: ``[T, N]`` (or ``[T]``) float64, as the engines write them, or float32; values: float32, the same shape;
    ends: bool, the same shape, True where the episode ended with that step; last_values: float32 ``[N]``, the value of the
    state behind the last step.  Float32 results; the arithmetic is float64 where the rewards are.  No gradient flows."""
    _on_device('rewards', rewards)
    device, shape = rewards.device, rewards.shape
    if rewards.dtype not in (torch.float64, torch.float32):
        raise ValueError(f'rewards: float64 or float32, not {rewards.dtype}')
    if not 1 <= len(shape) <= 2:
        raise ValueError(f'rewards: [T, N] or [T], got {tuple(shape)}')
    for name, t, kind, want in (('values', values, torch.float32, shape), ('ends', ends, torch.bool, shape),
                                ('last_values', last_values, torch.float32, shape[1:])):
        _on_device(name, t, device)
        if t.dtype != kind:
            raise ValueError(f'{name}: {kind}, not {t.dtype}')
        if t.shape != want:
            raise ValueError(f'{name}: {tuple(t.shape)} instead of {tuple(want)}')
    lib = _lib.load()
    adv = _laid_out(shape, rewards.stride(), torch.float32, device)
    tgt = _laid_out(shape, rewards.stride(), torch.float32, device)
    seq = _sequence(shape, 0, True, rewards.dtype)
    ref = C.byref(seq)
    nbytes = lib.lrn_advantages_workspace(ref)
    ws = _workspace(nbytes, device)
    last_values = last_values.detach().contiguous()
    _check(lib.lrn_advantages(device.index, _stream(device), ref, _ref(_view(rewards, 0)), _ref(_view(values, 0)), _ref(_view(ends, 0)),
                              last_values.data_ptr(), float(gamma), float(lam), _ref(_view(adv, 0)), _ref(_view(tgt, 0)), _ptr(ws),
                              nbytes),
           'advantages')
    return Advantages(adv, tgt)
