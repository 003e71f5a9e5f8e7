"""The FP8 operators in 64 bits, and bounds on what FP32 arithmetic and the
roundings of the operators' definition may move (shared by the FP8 tests).

e4m3 holds 4 significant bits down to 2^-6 and steps of 2^-9 below, so a value
is off by at most half a step of its binade.  BF16 is off by 2^-8 of the value
at most.  FP32 sums of n terms are off by n 2^-24 times the sum of magnitudes;
a tensor-core sum may cut instead of round (2^-23 per addition).
"""

from __future__ import annotations

import torch

G = 128
TOP = 448.0
TINY = 1e-10
BF = 2.0 ** -8
F32 = 2.0 ** -24


def groups(n: int) -> int:
    return -(-n // G)


def step(v: torch.Tensor) -> torch.Tensor:
    """The distance of neighbouring e4m3 values at |v| (64 bits)."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** -6))[1].double() - 1
    return torch.exp2(e - 3)


def nearest(v: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to even."""
    s = step(v)
    return (torch.round(v / s) * s).clamp(-TOP, TOP)


def tops(y: torch.Tensor) -> torch.Tensor:
    """[.., n] -> the largest magnitude of each group [.., ceil(n / 128)]."""
    return torch.stack([y[..., c:c + G].abs().amax(-1) for c in range(0, y.shape[-1], G)], -1).clamp(min=TINY)


def spread(s: torch.Tensor, n: int, dim: int = -1) -> torch.Tensor:
    """Per-group values repeated over their 128 members along dim, cut to n."""
    return s.repeat_interleave(G, dim).narrow(dim, 0, n)


def rows(y: torch.Tensor):
    """64-bit rows -> (what is rounded: y * 448 / a, its e4m3 value, scales)."""
    a = tops(y)
    v = y * TOP / spread(a, y.shape[-1])
    return v, nearest(v), a / TOP


def blocks(w: torch.Tensor):
    """64-bit [.., N, K] -> (e4m3 values, scales)."""
    n, k = w.shape[-2:]
    a = torch.stack([tops(w[..., r:r + G, :]).amax(-2) for r in range(0, n, G)], -2)
    return nearest(w * TOP / spread(spread(a, k), n, -2)), a / TOP


def widen_rows(q, s):
    return q.double() * spread(s.double(), q.shape[-1])


def widen_blocks(q, s):
    return q.double() * spread(spread(s.double(), q.shape[-1]), q.shape[-2], -2)


def chain(k: int) -> int:
    """Roundings of an FP32 sum over k products: at most 256 of 2^-24 inside a
    group of 128 (a cut counts double), one per group, and eight for the scales
    and the joining of partial sums across lanes."""
    return 256 + groups(k) + 8


def linear(x, xs, w, ws):
    """(exact, bound on |FP32 result - exact|)"""
    xd, wd = widen_rows(x, xs), widen_blocks(w, ws)
    return xd @ wd.T, chain(x.shape[1]) * F32 * (xd.abs() @ wd.abs().T)


def experts(x, xs, gu, gus, dn, dns, idx, weights):
    """(exact, bound): the bound counts the FP32 error of h, the e4m3 value of
    an h that this error may carry over a border (one step), the FP32 sums of
    the down product, each route's row rounded to BF16 and the final rounding."""
    t, k = idx.shape
    e_count, inner, hidden = gu.shape[0], dn.shape[2], x.shape[1]
    xd = widen_rows(x, xs)
    out = torch.zeros(t, hidden, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    for e in range(e_count):
        token, slot = torch.nonzero(idx == e, as_tuple=True)
        if token.numel() == 0:
            continue
        wg, wd = widen_blocks(gu[e], gus[e]), widen_blocks(dn[e], dns[e])
        p, pb = xd[token] @ wg.T, chain(hidden) * F32 * (xd[token].abs() @ wg.abs().T)
        g, u, gb, ub = p[:, :inner], p[:, inner:], pb[:, :inner], pb[:, inner:]
        silu = g * torch.sigmoid(g)
        h = silu * u
        # |silu'| <= 1.1; expf, the division and two products: eight roundings
        hb = 1.1 * gb * (u.abs() + ub) + silu.abs() * ub + 8 * F32 * h.abs()
        v, q, s = rows(h)
        a = s * TOP
        ab = torch.stack([hb[:, c:c + G].amax(-1) for c in range(0, inner, G)], -1) + 4 * F32 * a
        rel = spread(ab / a, inner)
        vb = hb * TOP / spread(a, inner) + v.abs() * rel
        st = step(v)
        near = (v / st - torch.floor(v / st) - 0.5).abs() * st <= 1.01 * vb
        qb = torch.where(near, 1.01 * st + vb, torch.zeros_like(v)) + q.abs() * rel
        act, actb = q * spread(s, inner), qb * spread(s, inner)
        y = act @ wd.T
        yb = actb @ wd.abs().T + chain(inner) * F32 * (act.abs() @ wd.abs().T)
        yb = yb + BF * (y.abs() + yb)
        wt = weights[token, slot].double()[:, None]
        out.index_add_(0, token, y * wt)
        bound.index_add_(0, token, (yb + k * F32 * y.abs()) * wt.abs())
    return out, bound + BF * (out.abs() + bound)
