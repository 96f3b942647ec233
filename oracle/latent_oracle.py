"""CPU oracle of the 8-bit paged latent cache and its attention -- TEST INFRASTRUCTURE ONLY.

Restates the definitions of ``include/kda_b200.h`` (MlaCacheArgs) token by token
and sequence by sequence in float64 torch; only ``tests/`` may import it.
"""

from __future__ import annotations

import math

import torch

MIN_EXP = -100


def least_exp(amax: float, top: float) -> int:
    """Least whole e with amax <= top * 2^e (amax > 0)."""
    e = math.frexp(amax)[1] - math.frexp(top)[1] - 1
    while amax > math.ldexp(top, e):
        e += 1
    return e


def token_scale(c, k=None) -> float:
    """The power-of-two scale of one token (float64 rows), NaN if not finite."""
    if not bool(torch.isfinite(c).all()) or (k is not None and not bool(torch.isfinite(k).all())):
        return math.nan
    e = MIN_EXP
    a = float(c.abs().max())
    if a > 0:
        e = max(e, least_exp(a, 448.0))
    if k is not None:
        r = float(k.abs().max())
        if r > 0:
            e = max(e, least_exp(r, 32768.0))
    return math.ldexp(1.0, e)


def round_e4m3(x):
    """float64 values with |x| <= 448 on the e4m3 grid, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def slots(table, lens, counts, page):
    """``[(b, position, slot or None)]`` of every new token, in order."""
    out = []
    for b, n in enumerate(counts):
        for i in range(n):
            p = int(lens[b]) - n + i
            out.append((b, p, int(table[b, p // page]) * page + p % page if p >= 0 else None))
    return out


def append(codes, scales, rope, c_kv, k_rope, where):
    """New float64 pools ``[slots, ...]`` with the tokens of ``where`` written."""
    codes, scales = codes.clone(), scales.clone()
    rope = None if rope is None else rope.clone()
    for n, (_, _, slot) in enumerate(where):
        if slot is None:
            continue
        k = None if rope is None else k_rope[n].double()
        s = token_scale(c_kv[n].double(), k)
        scales[slot] = s
        codes[slot] = round_e4m3(c_kv[n].double() / s) if s == s else math.nan
        if rope is not None:
            rope[slot] = (k / s).to(k_rope.dtype).double()
    return codes, scales, rope


def attention(q_lat, q_rope, c, k, counts, lens, scale):
    """float64 ``(out, lse, mag)`` of new tokens ``q_lat`` ``[N, H, KVL]``;
    ``c[b]`` ``[lens[b], KVL]`` and ``k[b]`` the cached values of sequence b.
    ``mag`` is sum softmax |c|, the scale of an error in the weights."""
    outs, lses, mags, first = [], [], [], 0
    N, H, KVL = q_lat.shape
    for b, n in enumerate(counts):
        q = q_lat[first:first + n].double()
        L = max(0, int(lens[b]))
        out = torch.zeros(n, H, KVL, dtype=torch.float64)
        mag = torch.zeros_like(out)
        lse = torch.full((n, H), -math.inf, dtype=torch.float64)
        for i in range(n):
            seen = L - n + i + 1
            if seen <= 0:
                continue
            z = q[i] @ c[b][:seen].double().T
            if k is not None:
                z = z + q_rope[first + i].double() @ k[b][:seen].double().T
            z = z * scale
            lse[i] = torch.logsumexp(z, -1)
            w = torch.exp(z - lse[i][:, None])
            out[i] = w @ c[b][:seen].double()
            mag[i] = w @ c[b][:seen].double().abs()
        outs.append(out)
        lses.append(lse)
        mags.append(mag)
        first += n
    return torch.cat(outs), torch.cat(lses), torch.cat(mags)
