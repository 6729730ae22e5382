"""The learner's operators in float64 on the CPU, written out, with bounds on what float32 arithmetic may add.

u = 2^-24 is half a step of float32.  Bounds count roundings along the longest path of any order of the sums: a kernel that
sums in parts has fewer."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal (float16, float32); bfloat16 results below the smallest normal may become zero."""
    f = torch.finfo(dtype)
    return f.smallest_normal if dtype == torch.bfloat16 else f.smallest_normal * f.eps / 2


class Rows:
    """Everything about rows of logits.  ``chain``: additions that one float32 sum may be strung together from."""

    def __init__(self, logits, mask=None):
        z = logits.double()
        K = z.shape[-1]
        ok = torch.isfinite(z) | torch.isnan(z) | (z > 0)
        if mask is not None:
            ok = ok & mask.expand(z.shape)
        self.ok, self.empty = ok, ~ok.any(-1)
        z = torch.where(ok, z, -math.inf)
        self.z = z
        self.m = torch.where(self.empty, 0.0, z.amax(-1))
        d = z - self.m[..., None]
        e = torch.where(ok, d.exp(), 0.0)
        self.s = torch.where(self.empty, 1.0, e.sum(-1))
        self.logs = self.s.log()
        self.logp = d - self.logs[..., None]
        self.p = e / self.s[..., None]
        dd = torch.where(ok, d, 0.0).abs()
        self.d1, self.d2 = (self.p * dd).sum(-1), (self.p * dd * dd).sum(-1)
        self.entropy = torch.where(self.empty, 0.0, -(self.p * torch.where(ok, self.logp, 0.0)).sum(-1))
        # s: every weight is off by (|d| + 2) u (the product under the exponential, the exponential, a rescaling), the sum by
        # one u for each addition and rescaling; both are relative to s.
        self.chain = K / 64 + 16
        self.rel_s = U * (self.d1 + 4 + self.chain)
        self.tol_logs = self.rel_s + 2 * U * self.logs.abs()
        # t = sum e d: each term |d| (|d| + 4) u, and the additions
        self.tol_entropy = self.tol_logs + U * (self.d2 + (6 + self.chain) * self.d1) + self.d1 * self.rel_s + 2 * U * (self.d1 + self.entropy.abs())

    def tol_logp(self, logp):
        return self.tol_logs[..., None] + U * (2 * torch.where(torch.isfinite(logp), logp, 0.0).abs() + 2 * self.logs.abs()[..., None])

    def of_levels(self, levels):
        """(log probabilities, bound)"""
        K = self.z.shape[-1]
        at = levels.clamp(0, K - 1)[..., None]
        lp = self.logp.gather(-1, at)
        tol = self.tol_logp(lp)[..., 0]
        lp = lp[..., 0]
        lp = torch.where(levels >= K, math.nan, torch.where(self.empty | (levels < 0), 0.0, lp))
        return torch.where(levels >= K, math.nan, lp), tol

    def gradient(self, levels, g_lp, g_h, dtype):
        """(gradient of the logits, bound) in ``dtype``"""
        K = self.z.shape[-1]
        g = torch.where(self.empty | (levels < 0), 0.0, g_lp.double())[..., None]
        gh = g_h.double()[..., None]
        one = torch.nn.functional.one_hot(levels.clamp(0, K - 1), K).double()
        lp = torch.where(self.p > 0, self.logp, 0.0)
        inner = lp + self.entropy[..., None]
        grad = g * torch.where(self.ok, one - self.p, 0.0) - gh * self.p * inner
        # p is off by rel_s and the (|d| + 4) u of its own weight; the products by some u each
        rel_p = self.rel_s[..., None] + U * (lp.abs() + self.logs.abs()[..., None] + 8)
        tol = (self.p * (g.abs() + gh.abs() * (inner.abs() + 1)) * rel_p + gh.abs() * self.p * (self.tol_entropy[..., None] + self.tol_logp(lp))
               + 4 * U * (g.abs() * (one + self.p) + gh.abs() * self.p * inner.abs()))
        return grad, tol + half_step(dtype) * (grad.abs() + tol) + tiny(dtype)


def choose(logits, noise, mask):
    """The level in the arithmetic that is asked for: one float32 addition, compared exactly."""
    z = logits.float()
    r = Rows(logits, mask)
    key = torch.where(r.ok, z if noise is None else z + noise, -math.inf)
    best = key.amax(-1, keepdim=True)
    level = (key == best).int().argmax(-1)
    return torch.where(r.empty, 0, level), r


def top_levels(r, top):
    order = torch.sort(r.z, dim=-1, descending=True, stable=True).indices[..., :top]
    lp = r.logp.gather(-1, order)
    gone = ~r.ok.gather(-1, order)
    return torch.where(gone, -1, order), torch.where(gone, -math.inf, lp), r.tol_logp(lp)


def scan(x, gate, initial, resets, dim, reverse, g_h=None, g_final=None):
    """Time-first walk in float64.  Returns a dict of values and of bounds.  Any association of the products and sums
    rounds a contribution x_s a_{s+1} .. a_t at most 2 (t - s) + 16 times: bound u (2 N_t + 16 M_t) with
    M_t = |a| M + |x| and N_t = |a| (N + M).  Below the smallest normal number a rounding is half the smallest subnormal,
    whatever the value: two for each step, carried on by the gates, D_t = |a| D + 2 tiny."""
    kind = x.dtype
    u = 2.0 ** -53 if kind == torch.float64 else U
    half = 0.0 if kind == torch.float64 else half_step(kind)
    small = tiny(torch.float64 if kind == torch.float64 else torch.float32)

    def first(v):
        return v.movedim(dim, 0) if v.dim() > 1 else v

    X = first(x).double()
    A = torch.full_like(X, float(gate)) if not isinstance(gate, torch.Tensor) else first(gate.expand(x.shape)).double()
    R = torch.zeros(X.shape, dtype=torch.bool)
    if resets is not None:
        R = first(resets)
        R = (R[..., None] if X.dim() == 3 else R).expand(X.shape)
    A = torch.where(R, 0.0, A)
    T = X.shape[0]
    order = list(range(T))[::-1] if reverse else list(range(T))
    s = torch.zeros(X.shape[1:], dtype=torch.float64) if initial is None else initial.double()

    def walk(start, xs, gates, anew):
        h, M, N, D, out, bound = start, start.abs(), torch.zeros_like(start), torch.zeros_like(start), [], []
        for xt, at, new in zip(xs, gates, anew):
            h = torch.where(new, xt, at * h + xt)
            N = torch.where(new, 0.0, at.abs() * (N + M))
            M = torch.where(new, xt.abs(), at.abs() * M + xt.abs())
            D = torch.where(new, 0.0, at.abs() * D) + 2 * small
            out.append(h)
            bound.append(u * (2 * N + 16 * M) + D)
        return out, bound, (h, u * (2 * N + 16 * M) + D)

    hs, hb, (final, fb) = walk(s, [X[t] for t in order], [A[t] for t in order], [R[t] for t in order])

    def laid(vs):
        if not vs:
            return torch.zeros(x.shape, dtype=torch.float64)
        v = torch.stack([vs[order.index(t)] for t in range(T)]) if reverse else torch.stack(vs)
        return v.movedim(0, dim) if v.dim() > 1 else v

    h = laid(hs)
    tol = laid(hb)
    res = {'h': (h, tol + half * (h.abs() + tol) + (0 if kind == torch.float64 else tiny(kind))), 'final': (final, fb)}
    if g_h is None and g_final is None:
        return res
    G0 = torch.zeros_like(s) if g_final is None else g_final.double()
    gh = torch.zeros_like(X) if g_h is None else first(g_h).double()
    back = order[::-1]
    ones = torch.ones_like(s)
    gates = [ones] + [A[t] for t in back[:-1]]
    new = [torch.zeros_like(ones, dtype=torch.bool)] + [R[t] for t in back[:-1]]
    Gs, Gb, (Glast, Glast_tol) = walk(G0, [gh[t] for t in back], gates, new)
    gx = {t: (G, b) for t, G, b in zip(back, Gs, Gb)}
    prev = {t: (s, torch.zeros_like(s)) if i == 0 else (hs[i - 1], hb[i - 1] + half * (hs[i - 1].abs() + hb[i - 1]))
            for i, t in enumerate(order)}
    gg = {t: torch.where(R[t], 0.0, gx[t][0] * prev[t][0]) for t in order}
    ggb = {t: gx[t][0].abs() * prev[t][1] + gx[t][1] * (prev[t][0].abs() + prev[t][1]) + 2 * u * gg[t].abs() for t in order}

    def put(d):
        v = torch.stack([d[t] for t in range(T)]) if T else torch.zeros_like(X)
        return v.movedim(0, dim) if v.dim() > 1 else v

    def rounded(v, tol):
        return v, tol + half * (v.abs() + tol) + (0 if kind == torch.float64 else tiny(kind))

    res['grad_x'] = rounded(put({t: v[0] for t, v in gx.items()}), put({t: v[1] for t, v in gx.items()}))
    res['grad_gate'] = rounded(put(gg), put(ggb))
    if T:
        t0 = order[0]
        gi = torch.where(R[t0], 0.0, A[t0] * Glast)
        res['grad_initial'] = gi, A[t0].abs() * Glast_tol + 2 * u * gi.abs()
    else:
        res['grad_initial'] = G0, torch.zeros_like(G0)
    return res


def advantages(rewards, values, ends, last, gamma, lam):
    r, v, e = rewards.double(), values.double(), ends
    A = torch.zeros(r.shape[1:], dtype=torch.float64)
    M, N = A.clone(), A.clone()
    nxt, adv, tol = last.double(), [], []
    for t in range(r.shape[0] - 1, -1, -1):
        on = torch.where(e[t], 0.0, 1.0)
        d = r[t] + gamma * on * nxt - v[t]
        size = 4 * (r[t].abs() + gamma * on * nxt.abs() + v[t].abs())
        A = d + gamma * lam * on * A
        N = gamma * lam * on * (N + M)
        M = gamma * lam * on * M + size
        adv.append(A)
        tol.append(U * (2 * N + 16 * M))
        nxt = v[t]
    if not adv:
        return torch.zeros(r.shape, dtype=torch.float64), torch.zeros(r.shape, dtype=torch.float64)
    return torch.stack(adv[::-1]), torch.stack(tol[::-1])
