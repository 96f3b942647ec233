"""CPU oracle of the gated recurrence and of the norm and rotation of queries and keys
-- TEST INFRASTRUCTURE ONLY.

Restates the definitions of ``include/kda_b200.h`` (KdaScanArgs, KdaQkArgs) in
float64 torch, token by token and head by head, each value with a bound on what
fp32 arithmetic may add to it.  Only ``tests/`` may import it.

Bounds of the recurrence.  ``U = 2^-24``.  One token's decay is off by at most ``(4 + 1.5 |g|) U`` of itself (the
exponent ``g log2 e`` by its rounding and its constant's, the power of two by ``4 U``), its product and sum by
``U`` of the magnitudes that go in: ``(5 + 1.5 |g|) U``.  From one run of four tokens to the next a state is multiplied by
the exponential of the run's sum ``G``, off by ``(4 + 1.5 |G|) U`` and by ``3 U |G|`` for the sum, in two roundings: ``(6 + 4.5
|G|) U`` a run.  Joining runs' decays before they meet a state rounds each product: at most ``3 x 27 U`` a run where the
two-part decay has become small (``1 + r >= exp(-4)``), which only a state of 32 runs has, and less than one
``U`` a token before.  So a token adds at most ``(8 + 8 |g|) U`` of the magnitude ``m_t = a_t m_{t-1} + |w_t x_t|``, and the
error obeys ``e_t = a_t e_{t-1} + (8 + 8 |g_t|) U m_t``.  ``1 - a`` is off by ``2.4 U`` of itself nearer than ``|g| = 1/2``, and
beyond by ``(4 + 1.5 |g|) U a / (1 - a) + U <= 8.4 U``; with the product by ``x``, and as a value that is multiplied again,
below ``15 U``.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24


def _gate(g, complement):
    a = torch.exp(g)
    w = -torch.expm1(g) if complement else torch.ones_like(g)
    return a, w


def scan(x, g, s0, complement):
    """One sequence: ``x``, ``g`` [T, D] float64, ``s0`` [D].  ``(h, S)`` and their bounds ``(eh, eS)``,
    with the magnitudes ``m`` [T, D]."""
    a, w = _gate(g, complement)
    h, e, m = s0.clone(), torch.zeros_like(s0), s0.abs()
    hs, es, ms = [], [], []
    for t in range(x.shape[0]):
        v = w[t] * x[t]
        forget = a[t] == 0
        h = torch.where(forget & torch.isfinite(h), v, a[t] * h + v)
        m = a[t] * m + v.abs()
        lg = torch.where(forget, torch.zeros_like(g[t]), g[t].abs())
        e = a[t] * e + (8 + 8 * lg) * U * m + (15 * U * v.abs() if complement else 0)
        hs.append(h)
        es.append(e)
        ms.append(m)
    if not hs:
        z = x.new_zeros(0, x.shape[1])
        return z, h, z, e, z
    return torch.stack(hs), h, torch.stack(es), e, torch.stack(ms)


def scan_grad(x, g, s0, dh, dS, complement):
    """Gradients ``(dx, dg, ds0)`` of one sequence and their bounds."""
    a, w = _gate(g, complement)
    hs, _, es, _, ms = scan(x, g, s0, complement)
    T = x.shape[0]
    u, e, m = dS.clone(), torch.zeros_like(dS), dS.abs()
    out = [torch.empty_like(x) for _ in range(4)]
    dx, dg, ex, eg = out
    for t in range(T - 1, -1, -1):
        prev, pe, pm = (hs[t - 1], es[t - 1], ms[t - 1]) if t else (s0, torch.zeros_like(s0), s0.abs())
        if complement:
            prev, pm = prev - x[t], pm + x[t].abs()
        d = dh[t] + u
        md = dh[t].abs() + m
        ed = e + U * md
        lg = torch.where(torch.isfinite(g[t]), g[t].abs(), torch.zeros_like(g[t]))
        dx[t], ex[t] = w[t] * d, w[t] * ed + (18 if complement else 2) * U * w[t] * md
        dg[t] = a[t] * prev * d
        eg[t] = a[t] * (pm * ed + pe * md) + (10 + 8 * lg) * U * a[t] * pm * md
        u, m = a[t] * d, a[t] * md
        e = a[t] * ed + (8 + 8 * lg) * U * m
    return dx, dg, u, ex, eg, e


def rotation(z, angle, interleaved):
    """Channels of ``z`` [..., D] rotated by ``angle`` [..., R / 2] (float64)."""
    n = angle.shape[-1]
    out = z.clone()
    for i in range(n):
        j, k = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        c, s = torch.cos(angle[..., i]), torch.sin(angle[..., i])
        out[..., j] = z[..., j] * c - z[..., k] * s
        out[..., k] = z[..., k] * c + z[..., j] * s
    return out


def rate(x, norm, eps):
    """``r`` [..., 1] of ``n = x r`` and whether it depends on ``x``."""
    if norm is None:
        return torch.ones_like(x[..., :1]), torch.zeros_like(x[..., :1], dtype=torch.bool)
    sq = (x * x).sum(-1, keepdim=True)
    if norm == "rms":
        return (sq / x.shape[-1] + eps) ** -0.5, torch.ones_like(sq, dtype=torch.bool)
    length = sq.sqrt()
    return 1.0 / torch.clamp(length, min=eps), length > eps


def qk(x, w, norm, eps, angle, interleaved):
    """``y`` of one tensor ``x`` [N, H, D] float64, ``w`` [D], [H, D] or None, ``angle`` [N, 1, R / 2] or None."""
    r, _ = rate(x, norm, eps)
    z = x * r if w is None else x * r * w
    return z if angle is None else rotation(z, angle, interleaved)


def qk_grad(x, w, norm, eps, angle, interleaved, dy):
    """``(dx, dw)``; ``dw`` None without a weight, with its sum of magnitudes behind it."""
    dz = dy if angle is None else rotation(dy, -angle, interleaved)
    r, moves = rate(x, norm, eps)
    n = x * r
    dw = mag = None
    if w is not None:
        along = (0, 1) if w.dim() == 1 else (0,)
        dw, mag = (dz * n).sum(along), (dz.abs() * n.abs()).sum(along)
        dz = dz * w
    dot = (dz * n).sum(-1, keepdim=True) / (x.shape[-1] if norm == "rms" else 1)
    return r * torch.where(moves, dz - n * dot, dz), dw, mag
