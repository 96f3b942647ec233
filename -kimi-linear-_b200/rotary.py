"""Norm of queries and keys per head and rotation by position, in one pass
(``csrc/kda_qk.cu``).

Every head of a token is normalised (root mean square with an optional weight, as
``HeadwiseRMSNorm``, ``kimi_linear/kda.py:258-279``; or to length one, as ``l2norm``,
``kda.py:313-325``; or not at all), and its first ``R`` channels are rotated by the
token's position: what stands between a layer's projections and its attention or
recurrence (:func:`latent.mla_step` rotates its rope parts with it).

:func:`qk_norm_rope` is differentiable in queries, keys and weights;
:func:`qk_norm_rope_backward` is the gradient that autograd calls.  CUDA tensors only
(no fallback), the current stream, no host synchronisation; positions are only
read on the device, so a captured graph can be replayed with new ones.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DT, _check_tensors, _inner_contig, _launch, _needs_grad, _no_tangents

NORMS = {None: _lib.NORM_NONE, "rms": _lib.NORM_RMS, "l2": _lib.NORM_L2}
MAX_D = 512
_NONE = (0, 0, 0, 0)              # pointer and strides of an operand that is not there


def _bth(t):
    """Pointer and (batch, token, head) strides of a [B, T, H, D] or [N, H, D] tensor."""
    if t is None:
        return _NONE
    return (t.data_ptr(), 0, *t.stride()[:2]) if t.dim() == 3 else (t.data_ptr(), *t.stride()[:3])


def _two(q, k):
    """As the argument block has them: both pointers, then both strides."""
    q, k = _bth(q), _bth(k)
    return (q[0], k[0], *q[1:], *k[1:])


_NONE2 = _two(None, None)


def _check(fn, q, k, wq, wk, norm, eps, positions, inv_freq, others=()):
    _no_tangents(fn, q, k, wq, wk, inv_freq, *(t for _, t in others))
    dev = _check_tensors(fn, [("q", q), ("k", k), ("q_weight", wq), ("k_weight", wk), *others])
    if q is None or q.dim() not in (3, 4):
        raise RuntimeError(f"{fn}: expected q [B, T, H, D] or [N, H, D]")
    D = q.shape[-1]
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != D):
        raise RuntimeError(f"{fn}: q {tuple(q.shape)} and k {tuple(k.shape)} must agree but for the "
                           f"number of heads")
    if k is not None and k.dtype != q.dtype:
        raise TypeError(f"{fn}: q is {q.dtype}, k {k.dtype}")
    if not 1 <= D <= MAX_D:
        raise RuntimeError(f"{fn}: head size {D} not supported (1 to {MAX_D})")
    if norm not in NORMS:
        raise ValueError(f"{fn}: norm must be 'rms', 'l2' or None (got {norm!r})")
    if norm is None and (wq is not None or wk is not None):
        raise RuntimeError(f"{fn}: weights need a norm")
    if norm is not None and not float(eps) >= 1e-12:
        raise ValueError(f"{fn}: eps must be at least 1e-12 (got {eps})")
    if wk is not None and k is None:
        raise RuntimeError(f"{fn}: k_weight without k")
    for name, w, t in (("q_weight", wq, q), ("k_weight", wk, k)):
        if w is not None and tuple(w.shape) not in ((D,), (t.shape[-2], D)):
            raise RuntimeError(f"{fn}: {name} shape {tuple(w.shape)} is neither {(D,)} nor "
                               f"{(t.shape[-2], D)}")
    if wq is not None and wk is not None and (wq.dim() != wk.dim() or wq.dtype != wk.dtype):
        raise RuntimeError(f"{fn}: q_weight and k_weight must have the same type and number of "
                           f"dimensions")
    if inv_freq is not None:
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float32 or \
                inv_freq.dim() != 1 or inv_freq.device != dev or 2 * inv_freq.shape[0] > D:
            raise RuntimeError(f"{fn}: inv_freq must be a float32 tensor of at most {D // 2} values on "
                               f"{dev}")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.device != dev or \
                positions.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{fn}: positions must be an int32 or int64 tensor on {dev}")
        ok = [(q.shape[0],)] if q.dim() == 3 else [(q.shape[0],), tuple(q.shape[:2])]
        if tuple(positions.shape) not in ok:
            raise RuntimeError(f"{fn}: positions shape {tuple(positions.shape)} is none of {ok}")
    return dev


def _args(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved, y=_NONE2, dy=_NONE2, dx=_NONE2, dw=(0, 0)):
    """The argument block, but for the partial sums, and what must stay alive with it."""
    packed = q.dim() == 3
    B, T = (1, q.shape[0]) if packed else q.shape[:2]
    ws = [None if w is None else w.detach().contiguous() for w in (wq, wk)]
    w = ws[0] if ws[0] is not None else ws[1]
    R = 0
    if inv_freq is not None:
        inv_freq = inv_freq.detach().contiguous()
        R = 2 * inv_freq.shape[0]
    pos, wide, step, ps = 0, 0, 1, (0, 0)
    if positions is not None:
        pos, wide, s = positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0, positions.stride()
        if positions.dim() == 2:
            ps, step = s, 0
        elif packed:
            ps, step = (0, s[0]), 0
        else:
            ps = (s[0], 0)
    a = _lib.KdaQkArgs.from_buffer_copy(_lib.KdaQkArgs.PACK.pack(
        _lib.ABI_VERSION, B, T, q.shape[-1], R, q.shape[-2], 0 if k is None else k.shape[-2], _DT[q.dtype],
        _lib.DTYPE_F32 if w is None else _DT[w.dtype], NORMS[norm], 1 if interleaved else 0,
        0 if w is None or w.dim() == 1 else 1, wide, step, float(eps), 0, *_two(q, k),
        *(0 if t is None else t.data_ptr() for t in ws), pos, *ps,
        0 if inv_freq is None else inv_freq.data_ptr(), *y, *dy, *dx, *dw, 0, 0))
    return a, (ws, inv_freq)


def _forward(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved):
    q, k = _inner_contig(q), None if k is None else _inner_contig(k)
    oq, ok = q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
    a, keep = _args(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved, y=_two(oq, ok))
    _launch("qk_norm_rope", _lib.load().kda_qk_fwd, a, q.device)
    return oq, ok


def qk_norm_rope(q, k=None, q_weight=None, k_weight=None, *, norm="rms", eps=1e-6, positions=None,
                 inv_freq=None, interleaved=False):
    """``(q, k)`` normalised per head and rotated, new tensors of the inputs' type.

    ``q`` ``[B, T, H, D]`` and ``k`` ``[B, T, HK, D]`` (or ``[N, H, D]``, ``[N, HK, D]``;
    ``k`` may be None, and so is what comes back for it), any strides, ``D <= 512``.

    * ``norm="rms"``: ``x (mean x^2 + eps)^-1/2``; ``"l2"``: ``x min(1 / |x|, 1 / eps)``; None: ``x``.
      Times ``q_weight`` / ``k_weight`` ``[D]`` or ``[H, D]`` / ``[HK, D]`` where given.
    * ``inv_freq`` fp32 ``[R / 2]`` (None: no rotation): channels ``0 .. R - 1`` are rotated in
      pairs ``(i, i + R / 2)``, or ``(2 i, 2 i + 1)`` with ``interleaved``, by the angle ``p
      inv_freq[i]`` (in 64 bits).
    * ``positions``: ``p`` of every token, int32 or int64 ``[B, T]`` (``[N]``), or for ``[B, T, H, D]``
      the first token's ``[B]``, the others following; None: 0, 1, ... for each sequence.

    Statistics are fp32 and a value is rounded once.  Differentiable in ``q``, ``k`` and the weights."""
    fn = "qk_norm_rope"
    if _needs_grad(inv_freq):
        raise RuntimeError(f"{fn}: inv_freq has no gradient; detach it")
    if _needs_grad(q, k, q_weight, k_weight):
        with torch.no_grad():
            _check(fn, q, k, q_weight, k_weight, norm, eps, positions, inv_freq)
        out = _QkNormRope.apply(q, k, q_weight, k_weight, positions, inv_freq, norm, float(eps),
                                bool(interleaved))
        return out if k is not None else (out, None)
    _check(fn, q, k, q_weight, k_weight, norm, eps, positions, inv_freq)
    return _forward(q, k, q_weight, k_weight, norm, eps, positions, inv_freq, interleaved)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, inv_freq, norm, eps, interleaved):
        ctx.save_for_backward(q, k, wq, wk, positions, inv_freq)
        ctx.plain = (norm, eps, interleaved)
        out = _forward(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved)
        return out if k is not None else out[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        q, k, wq, wk, positions, inv_freq = ctx.saved_tensors
        norm, eps, interleaved = ctx.plain
        need = ctx.needs_input_grad
        grads = _backward(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved, dq, dk, need)
        return (*(gr if need[i] else None for i, gr in enumerate(grads)), None, None, None, None, None)


def _backward(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved, dq, dk, need):
    q, k = _inner_contig(q), None if k is None else _inner_contig(k)
    dq = _inner_contig(dq.to(q.dtype))
    dk = None if k is None else _inner_contig(dk.to(k.dtype))
    oq, ok = q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
    dw = [w.new_empty(w.shape) if w is not None and n else None for w, n in ((wq, need[2]), (wk, need[3]))]
    a, keep = _args(q, k, wq, wk, norm, eps, positions, inv_freq, interleaved, dy=_two(dq, dk), dx=_two(oq, ok),
                    dw=[0 if w is None else w.data_ptr() for w in dw])
    lib = _lib.load()
    if a.dw[0] or a.dw[1]:
        n = int(lib.kda_qk_partial_floats(ctypes.byref(a)))
        partial = q.new_empty((n,), dtype=torch.float32)
        a.partial, a.partial_floats = partial.data_ptr(), n
    _launch("qk_norm_rope_backward", lib.kda_qk_bwd, a, q.device)
    return oq, ok, *dw


def qk_norm_rope_backward(dq, dk, q, k=None, q_weight=None, k_weight=None, *, norm="rms", eps=1e-6,
                          positions=None, inv_freq=None, interleaved=False):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of :func:`qk_norm_rope` of the same
    arguments for output gradients ``dq`` and ``dk`` (None where there is no ``k`` or weight)."""
    fn = "qk_norm_rope_backward"
    _check(fn, q, k, q_weight, k_weight, norm, eps, positions, inv_freq, [("dq", dq), ("dk", dk)])
    for name, d, t in (("dq", dq, q), ("dk", dk, k)):
        if (d is None) != (t is None) or (d is not None and d.shape != t.shape):
            raise RuntimeError(f"{fn}: {name} must have the shape of {name[1:]}")
    return _backward(q, k, q_weight, k_weight, norm, eps, positions, inv_freq, interleaved, dq, dk,
                     (True,) * 4)
