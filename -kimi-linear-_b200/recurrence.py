"""Gated linear recurrence, channel by channel (``csrc/kda_scan.cu``).

Beside the delta-rule recurrence of :mod:`ops` (a K x V state per head), the
elementwise one of gated linear RNN layers, with the same kind of gate::

    h_t = a_t h_{t-1} + w_t x_t,    a_t = exp(g_t),    w_t = 1  or, complement=True,  1 - a_t

``g`` is a log decay (``<= 0``; ``-inf`` forgets everything before the token), fp32 or
in ``x``'s type, as ``kda_prologue`` leaves it for KDA.  States are fp32 throughout.

* :func:`gated_scan`: whole sequences (prompts, training), a batch ``[B, T, D]``
  or sequences packed one behind the other;
* :func:`gated_step`: one token for each row of a serving batch;
* :func:`gated_scan_backward`: the gradient, which autograd calls.

As elsewhere in the package: CUDA tensors only (no fallback), the current
stream of the inputs' device, nothing synchronises or is read on the host, so calls
can be captured in CUDA graphs.  Nothing is kept between calls.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _DT, _check_tensors, _inner_contig, _launch, _needs_grad, _no_tangents

_NONE2, _NONE3 = (0, 0), (0, 0, 0)


def _bt(t, packed):
    """Pointer and (batch, token) strides."""
    if packed:
        return t.data_ptr(), 0, t.stride(0)
    return t.data_ptr(), t.stride(0), t.stride(1)


def _rows(t):
    """Pointer and stride of the rows of a state."""
    return t.data_ptr(), t.stride(0)


def _args(B, T, x, g, complement, xs, gs, state=_NONE2, q_start=0, slots=0, h=_NONE3, S=_NONE2, ckpt=0,
          dh=_NONE3, dS=_NONE2, dx=_NONE3, dg=_NONE3, dstate=_NONE2, num_states=0, scatter=0):
    """The argument block, but for the workspace: pointers with their strides."""
    return _lib.KdaScanArgs.from_buffer_copy(_lib.KdaScanArgs.PACK.pack(
        _lib.ABI_VERSION, B, T, x.shape[-1], _DT[x.dtype], _DT[g.dtype], 1 if complement else 0,
        num_states, scatter, 0, *xs, *gs, *state, q_start, slots, *h, *S, ckpt, *dh, *dS, *dx, *dg, *dstate,
        0, 0))


def _check(fn, x, g, state, rows, others=()):
    """Device of the operands, after checks of types and shapes."""
    _no_tangents(fn, x, g, state, *(t for _, t in others))
    dev = _check_tensors(fn, [("x", x), ("g", g), ("state", state), *others])
    if g is None or x.shape != g.shape:
        raise RuntimeError(f"{fn}: x {tuple(x.shape)} and g "
                           f"{None if g is None else tuple(g.shape)} differ in shape")
    if g.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"{fn}: g must be float32 or {x.dtype} (got {g.dtype})")
    if state is not None and tuple(state.shape) != (rows, x.shape[-1]):
        raise RuntimeError(f"{fn}: state shape {tuple(state.shape)} != {(rows, x.shape[-1])}")
    return dev


def _batch(fn, x, q_start):
    """Number of sequences of ``x``, after checks of what says so."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{fn}: x must be a torch.Tensor")
    if q_start is None:
        if x.dim() != 3:
            raise RuntimeError(f"{fn}: expected x, g [B, T, D] (or [N, D] with q_start); got "
                               f"{tuple(x.shape)}")
        return x.shape[0]
    if x.dim() != 2:
        raise RuntimeError(f"{fn}: expected x, g [N, D] with q_start; got {tuple(x.shape)}")
    if not isinstance(q_start, torch.Tensor) or q_start.dtype != torch.int32 or q_start.dim() != 1 \
            or q_start.device != x.device or q_start.shape[0] < 1 \
            or (q_start.shape[0] > 1 and q_start.stride(0) != 1):
        raise RuntimeError(f"{fn}: q_start must be an int32 tensor [sequences + 1] with a unit stride "
                           f"on {x.device}")
    return q_start.shape[0] - 1


def _read_as_float(state):
    """A floating state of a type that the kernels do not take, in fp32."""
    if isinstance(state, torch.Tensor) and state.is_floating_point() and state.dtype not in _DT:
        return state.float()
    return state


def _workspace(a, q_start):
    """Scratch for a packed batch, set in ``a``; the caller holds it through the call."""
    if q_start is None:
        return None
    need = int(_lib.load().kda_scan_workspace_bytes(ctypes.byref(a)))
    ws = q_start.new_empty(((need + 7) // 8,), dtype=torch.int64)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    return ws


def _forward(x, g, state, q_start, complement, keep):
    """``(h, S, checkpoints)`` for operands that :func:`_check` has passed;
    ``keep``: checkpoints for the backward pass are wanted."""
    packed = q_start is not None
    x, g = _inner_contig(x), _inner_contig(g)
    state = None if state is None else _inner_contig(state.float())
    B, T, D = q_start.shape[0] - 1 if packed else x.shape[0], x.shape[-2], x.shape[-1]
    h = x.new_empty(x.shape)
    S = x.new_empty((B, D), dtype=torch.float32)
    lib = _lib.load()
    a = _args(B, T, x, g, complement, _bt(x, packed), _bt(g, packed), _NONE2 if state is None else _rows(state),
              q_start.data_ptr() if packed else 0, 0, _bt(h, packed), (S.data_ptr(), D))
    ckpt = None
    if keep:
        ckpt = S.new_empty((int(lib.kda_scan_ckpt_floats(ctypes.byref(a))),))
        a.ckpt = ckpt.data_ptr()
    ws = _workspace(a, q_start)  # noqa: F841
    _launch("gated_scan", lib.kda_scan_fwd, a, x.device)
    return h, S, ckpt


def gated_scan(x, g, initial_state=None, q_start=None, *, complement=False):
    """``(h, S)``: every ``h_t``, in ``x``'s type, and every sequence's last one, fp32.

    ``x`` and ``g`` ``[B, T, D]`` with ``initial_state`` ``[B, D]`` (None: zeros), or
    packed: ``x`` and ``g`` ``[N, D]``, ``q_start`` int32 ``[B + 1]`` on the device, ascending:
    sequence ``b`` owns rows ``q_start[b] .. q_start[b + 1] - 1`` and starts from
    ``initial_state[b]``.  Rows before ``q_start[0]`` and from ``q_start[B]`` on belong to
    no sequence and give zeros; a sequence without rows gives its initial state.

    Differentiable in ``x``, ``g`` and ``initial_state``.  ``x`` f32, f16 or bf16,
    ``g`` fp32 or ``x``'s type.  A state of any floating type is read as fp32.  What is not finite
    goes on as the formula has it, but that a decay below 2^-126 counts as zero."""
    fn = "gated_scan"
    B = _batch(fn, x, q_start)
    initial_state = _read_as_float(initial_state)
    if _needs_grad(x, g, initial_state):
        with torch.no_grad():
            _check(fn, x, g, initial_state, B)
        return _GatedScan.apply(x, g, initial_state, q_start, bool(complement))
    _check(fn, x, g, initial_state, B)
    return _forward(x, g, initial_state, q_start, complement, False)[:2]


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, state, q_start, complement):
        h, S, ckpt = _forward(x, g, state, q_start, complement, True)
        ctx.save_for_backward(x, g, state, q_start, ckpt)
        ctx.complement = complement
        ctx.set_materialize_grads(False)
        return h, S

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dS):
        x, g, state, q_start, ckpt = ctx.saved_tensors
        grads = _backward(x, g, state, q_start, ctx.complement, ckpt, dh, dS,
                          ctx.needs_input_grad[:3])
        return (*grads, None, None)


def _backward(x, g, state, q_start, complement, ckpt, dh, dS, need):
    packed = q_start is not None
    x, g = _inner_contig(x), _inner_contig(g)
    state32 = None if state is None else _inner_contig(state.float())
    B, T, D = q_start.shape[0] - 1 if packed else x.shape[0], x.shape[-2], x.shape[-1]
    if dh is not None:
        dh = _inner_contig(dh.to(x.dtype))
    if dS is not None:
        dS = _inner_contig(dS.float())
    dx = x.new_empty(x.shape) if need[0] else None
    dg = g.new_empty(g.shape) if need[1] else None
    dstate = ckpt.new_empty((B, D)) if need[2] and state is not None else None
    three = lambda t: _NONE3 if t is None else _bt(t, packed)  # noqa: E731
    two = lambda t: _NONE2 if t is None else _rows(t)  # noqa: E731
    a = _args(B, T, x, g, complement, _bt(x, packed), _bt(g, packed), two(state32),
              q_start.data_ptr() if packed else 0, ckpt=ckpt.data_ptr(), dh=three(dh), dS=two(dS), dx=three(dx),
              dg=three(dg), dstate=two(dstate))
    ws = _workspace(a, q_start)  # noqa: F841
    _launch("gated_scan_backward", _lib.load().kda_scan_bwd, a, x.device)
    return dx, dg, None if dstate is None else dstate.to(state.dtype)


def gated_scan_backward(x, g, initial_state, dh, dS, q_start=None, *, complement=False):
    """Gradients ``(dx, dg, dinitial_state)`` of :func:`gated_scan` for output
    gradients ``dh`` (of ``h``, or None) and ``dS`` (of ``S``, or None).

    Runs the forward pass again for its checkpoints; autograd keeps those of
    the call that it differentiates."""
    fn = "gated_scan_backward"
    B = _batch(fn, x, q_start)
    given, initial_state = initial_state, _read_as_float(initial_state)
    _check(fn, x, g, initial_state, B, [("dh", dh), ("dS", dS)])
    if dh is not None and dh.shape != x.shape:
        raise RuntimeError(f"{fn}: dh shape {tuple(dh.shape)} != {tuple(x.shape)}")
    if dS is not None and tuple(dS.shape) != (B, x.shape[-1]):
        raise RuntimeError(f"{fn}: dS shape {tuple(dS.shape)} != {(B, x.shape[-1])}")
    ckpt = _forward(x, g, initial_state, q_start, complement, True)[2]
    dx, dg, dstate = _backward(x, g, initial_state, q_start, bool(complement), ckpt, dh, dS, (True, True, True))
    return dx, dg, None if dstate is None else dstate.to(given.dtype)


def gated_step(x, g, state=None, slots=None, *, complement=False, inplace=False):
    """One token: ``(h, S)`` for ``x`` and ``g`` ``[B, D]`` (or ``[B, 1, D]``, then ``h`` is too).

    ``state`` fp32 ``[B, D]`` (None: zeros).  With ``slots`` int32 ``[B]``, row ``b``'s
    state is row ``slots[b]`` of a pool ``state`` ``[num_states, D]``; a negative slot marks an
    idle row, whose ``h`` and ``S`` are zeros.  (A slot past the pool counts as idle and
    sets the device error word: :func:`ops.device_error` returns 8.)  ``S`` ``[B, D]`` is a
    new tensor; ``inplace=True`` writes the new states where the old ones were and
    returns ``state`` itself (idle rows leave it alone; no slot twice in a call).
    Forward only: :func:`gated_scan` with ``T = 1`` is the differentiable form."""
    fn = "gated_step"
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{fn}: x must be a torch.Tensor")
    if x.dim() not in (2, 3) or (x.dim() == 3 and x.shape[1] != 1):
        raise RuntimeError(f"{fn}: expected x, g [B, D] or [B, 1, D]; got {tuple(x.shape)}")
    shape = x.shape
    if not isinstance(g, torch.Tensor) or g.shape != shape:
        raise RuntimeError(f"{fn}: g must be a tensor of x's shape {tuple(shape)}")
    if x.dim() == 3:
        x, g = x[:, 0], g[:, 0]
    B, D = x.shape
    rows = B
    if slots is not None:
        if not isinstance(state, torch.Tensor) or state.dim() != 2:
            raise RuntimeError(f"{fn}: slots need a state [num_states, {D}]")
        if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int32 or \
                tuple(slots.shape) != (B,) or slots.device != x.device or (B > 1 and slots.stride(0) != 1):
            raise RuntimeError(f"{fn}: slots must be an int32 tensor [{B}] with a unit stride on {x.device}")
        rows = state.shape[0]
    dev = _check(fn, x, g, state, rows)
    if state is not None and state.dtype != torch.float32:
        raise TypeError(f"{fn}: state must be float32 (got {state.dtype})")
    if inplace:
        if state is None:
            raise RuntimeError(f"{fn}: inplace needs a state")
        if (D > 1 and state.stride(1) != 1) or (rows > 1 and state.stride(0) < D):
            raise RuntimeError(f"{fn}: inplace needs states with a unit innermost stride that do not "
                               f"overlap")
    elif state is not None:
        state = _inner_contig(state)
    x, g = _inner_contig(x), _inner_contig(g)
    h = x.new_empty(shape)
    S = state if inplace else x.new_empty((B, D), dtype=torch.float32)
    a = _args(B, 1, x, g, complement, (x.data_ptr(), x.stride(0), 0), (g.data_ptr(), g.stride(0), 0),
              _NONE2 if state is None else _rows(state), 0, 0 if slots is None else slots.data_ptr(),
              (h.data_ptr(), D, 0), _rows(S), num_states=0 if slots is None else rows, scatter=1 if inplace else 0)
    _launch(fn, _lib.load().kda_scan_step, a, dev)
    if inplace:
        increment_version(state)     # (autograd notices where it has kept the old states)
    return h, S
