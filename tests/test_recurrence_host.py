"""Gated recurrence and rotation without a GPU: the oracle's gradients against
differences and autograd, no CPU path, and what the C entry points refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import pkg
from oracle import recurrence_oracle as R


@pytest.mark.parametrize("complement", [False, True])
def test_oracle_scan_gradient(complement):
    gen = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    x, g, s0, dh, dS = rnd(11, 3), -rnd(11, 3).abs(), rnd(3), rnd(11, 3), rnd(3)
    f = lambda *a: sum((o * d).sum() for o, d in zip(R.scan(*a, complement)[:2], (dh, dS)))  # noqa: E731
    grads = R.scan_grad(x, g, s0, dh, dS, complement)[:3]
    leaves = [t.clone().requires_grad_() for t in (x, g, s0)]
    for got, want in zip(grads, torch.autograd.grad(f(*leaves), leaves)):
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    dirs = [rnd(*t.shape) for t in (x, g, s0)]
    at = lambda s: f(*(t + s * d for t, d in zip((x, g, s0), dirs)))  # noqa: E731
    slope = (at(1e-5) - at(-1e-5)) / 2e-5
    assert abs(slope - sum((a * d).sum() for a, d in zip(grads, dirs))) < 1e-7


@pytest.mark.parametrize("norm", ["rms", "l2", None])
@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation_gradient(norm, interleaved):
    gen = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    x, w, dy, angle = rnd(4, 2, 10), None if norm is None else rnd(2, 10), rnd(4, 2, 10), rnd(4, 1, 3)
    leaves = [t.clone().requires_grad_() for t in (x, w) if t is not None]
    y = R.qk(leaves[0], leaves[1] if w is not None else None, norm, 1e-6, angle, interleaved)
    want = torch.autograd.grad((y * dy).sum(), leaves)
    got = R.qk_grad(x, w, norm, 1e-6, angle, interleaved, dy)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_no_cpu_path():
    kb = pkg()
    x = torch.zeros(2, 5, 4)
    for call in (lambda: kb.gated_scan(x, x), lambda: kb.gated_scan(x.clone().requires_grad_(), x),
                 lambda: kb.gated_step(x[:, 0], x[:, 0]),
                 lambda: kb.recurrence.gated_scan_backward(x, x, None, x, None),
                 lambda: kb.qk_norm_rope(x[:, :, None]),
                 lambda: kb.qk_norm_rope(x[:, :, None].clone().requires_grad_()),
                 lambda: kb.rotary.qk_norm_rope_backward(x[:, :, None], None, x[:, :, None])):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()
    with pytest.raises(TypeError):
        kb.gated_scan([1.0], x)
    with pytest.raises(RuntimeError):
        kb.gated_scan(x[0], x[0])
    with pytest.raises(RuntimeError):
        kb.gated_scan(x, x, None, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        kb.gated_step(x, x)


FAKE = 1 << 20       # never dereferenced: every call below is refused first


def _scan_args(**kw):
    L = pkg()._lib
    a = L.KdaScanArgs()
    a.abi_version, a.B, a.T, a.D = L.ABI_VERSION, 2, 8, 16
    a.x_dtype, a.g_dtype = L.DTYPE_BF16, L.DTYPE_F32
    for n in ("x", "g", "h", "state_out", "ckpt"):
        setattr(a, n, FAKE)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_scan_entry_points_refuse():
    L = pkg()._lib
    lib = L.load()
    P = ctypes.byref
    for fn in (lib.kda_scan_fwd, lib.kda_scan_bwd, lib.kda_scan_step):
        assert fn(None, None) == L.KDA_ERR_NULL_POINTER
        for kw, want in ((dict(abi_version=1), L.KDA_ERR_SHAPE), (dict(B=-1), L.KDA_ERR_SHAPE),
                         (dict(D=-1), L.KDA_ERR_SHAPE), (dict(T=-1), L.KDA_ERR_SHAPE)):
            assert fn(P(_scan_args(**kw)), None) == want, kw
    for fn in (lib.kda_scan_fwd, lib.kda_scan_bwd):
        for kw, want in ((dict(x_dtype=3), L.KDA_ERR_DTYPE), (dict(g_dtype=L.DTYPE_F16), L.KDA_ERR_DTYPE),
                         (dict(x=None), L.KDA_ERR_NULL_POINTER), (dict(g=None), L.KDA_ERR_NULL_POINTER),
                         (dict(x=FAKE + 1), L.KDA_ERR_ALIGNMENT), (dict(g=FAKE + 2), L.KDA_ERR_ALIGNMENT),
                         (dict(q_start=FAKE + 2), L.KDA_ERR_ALIGNMENT), (dict(B=1 << 25), L.KDA_ERR_SHAPE),
                         (dict(T=(1 << 30) + 1), L.KDA_ERR_SHAPE), (dict(q_start=FAKE), L.KDA_ERR_WORKSPACE)):
            assert fn(P(_scan_args(**kw)), None) == want, kw
        assert fn(P(_scan_args(D=0)), None) == L.KDA_OK
        assert fn(P(_scan_args(B=0)), None) == L.KDA_OK
    assert lib.kda_scan_fwd(P(_scan_args(h=None)), None) == L.KDA_ERR_NULL_POINTER
    assert lib.kda_scan_fwd(P(_scan_args(state_out=None)), None) == L.KDA_ERR_NULL_POINTER
    assert lib.kda_scan_bwd(P(_scan_args(ckpt=None)), None) == L.KDA_ERR_NULL_POINTER
    step = dict(T=1, state_in=FAKE, state_in_stride=16, state_out_stride=16)
    assert lib.kda_scan_step(P(_scan_args()), None) == L.KDA_ERR_SHAPE
    assert lib.kda_scan_step(P(_scan_args(**step, slots=FAKE, num_states=-1)), None) == L.KDA_ERR_SHAPE
    assert lib.kda_scan_step(P(_scan_args(**{**step, "state_in": FAKE + 64}, scatter=1)), None) == L.KDA_ERR_STRIDE
    assert lib.kda_scan_step(P(_scan_args(**{**step, "B": 0})), None) == L.KDA_OK
    assert lib.kda_scan_workspace_bytes(P(_scan_args())) == 0
    assert lib.kda_scan_workspace_bytes(P(_scan_args(T=65, q_start=FAKE))) > 0
    n = lib.kda_scan_ckpt_floats
    assert n(P(_scan_args(T=32))) == 2 * 16 and n(P(_scan_args(T=33))) == 2 * 2 * 16
    assert n(P(_scan_args(T=33, q_start=FAKE))) == 2 * 16 and n(P(_scan_args(T=0))) == 0


def _qk_args(**kw):
    L = pkg()._lib
    a = L.KdaQkArgs()
    a.abi_version, a.B, a.T, a.D, a.R = L.ABI_VERSION, 2, 8, 16, 8
    a.heads[0], a.heads[1] = 4, 2
    a.io_dtype, a.w_dtype, a.norm, a.eps = L.DTYPE_BF16, L.DTYPE_F32, L.NORM_RMS, 1e-6
    a.inv_freq = FAKE
    for n in ("x", "y", "dy", "dx"):
        getattr(a, n)[0] = getattr(a, n)[1] = FAKE
    for n, v in kw.items():
        if n.endswith(("0", "1")) and n != "abi_version":
            getattr(a, n[:-1])[int(n[-1])] = v
        else:
            setattr(a, n, v)
    return a


def test_qk_entry_points_refuse():
    L = pkg()._lib
    lib = L.load()
    P = ctypes.byref
    for fn in (lib.kda_qk_fwd, lib.kda_qk_bwd):
        assert fn(None, None) == L.KDA_ERR_NULL_POINTER
        for kw, want in (
                (dict(abi_version=1), L.KDA_ERR_SHAPE), (dict(D=0), L.KDA_ERR_SHAPE), (dict(D=513), L.KDA_ERR_SHAPE),
                (dict(R=7), L.KDA_ERR_SHAPE), (dict(R=18), L.KDA_ERR_SHAPE), (dict(R=-2), L.KDA_ERR_SHAPE),
                (dict(norm=3), L.KDA_ERR_SHAPE), (dict(eps=0.0), L.KDA_ERR_SHAPE),
                (dict(eps=float("nan")), L.KDA_ERR_SHAPE), (dict(heads0=-1), L.KDA_ERR_SHAPE),
                (dict(B=1 << 16, T=1 << 15), L.KDA_ERR_SHAPE),
                (dict(io_dtype=3), L.KDA_ERR_DTYPE), (dict(w_dtype=-1), L.KDA_ERR_DTYPE),
                (dict(inv_freq=None), L.KDA_ERR_NULL_POINTER), (dict(x0=None), L.KDA_ERR_NULL_POINTER),
                (dict(x1=FAKE + 1), L.KDA_ERR_ALIGNMENT), (dict(w0=FAKE + 2), L.KDA_ERR_ALIGNMENT),
                (dict(positions=FAKE + 4, pos_64=1), L.KDA_ERR_ALIGNMENT)):
            assert fn(P(_qk_args(**kw)), None) == want, kw
        assert fn(P(_qk_args(T=0)), None) == L.KDA_OK
        assert fn(P(_qk_args(heads0=0, heads1=0)), None) == L.KDA_OK
    assert lib.kda_qk_fwd(P(_qk_args(y1=None)), None) == L.KDA_ERR_NULL_POINTER
    assert lib.kda_qk_bwd(P(_qk_args(dy0=None)), None) == L.KDA_ERR_NULL_POINTER
    assert lib.kda_qk_bwd(P(_qk_args(dw0=FAKE)), None) == L.KDA_ERR_NULL_POINTER
    assert lib.kda_qk_bwd(P(_qk_args(dw0=FAKE, w0=FAKE)), None) == L.KDA_ERR_WORKSPACE
    need = lib.kda_qk_partial_floats(P(_qk_args()))
    assert need > 0 and need % 16 == 0
    assert lib.kda_qk_bwd(P(_qk_args(dw0=FAKE, w0=FAKE, partial=FAKE, partial_floats=need - 1)),
                          None) == L.KDA_ERR_WORKSPACE


@pytest.mark.parametrize("rope_dim", [0, 64])
def test_mla_step_with_frequencies_refuses(rope_dim):
    """Frequencies without a rope part, and rope parts on the CPU, before the lengths change."""
    from test_latent_step_host import _step_args

    args = _step_args(DR=rope_dim)
    state = args[6]
    state["inv_freq"] = torch.ones(32)
    if rope_dim:
        state["cache"] = pkg().LatentCache(2, 16, 128, rope_dim, device="cpu")
        args[3], args[5] = torch.zeros(2, 1, 2, rope_dim), torch.zeros(2, 1, rope_dim)
    with pytest.raises(RuntimeError):
        pkg().latent.mla_step(*args, True)
    assert state["lens"].tolist() == [3, 5]


def test_forward_mode_tangents_are_refused():
    """A dual tensor that needs no gradient would come back without its tangent."""
    from torch.autograd import forward_ad

    kb = pkg()
    z = lambda *s: torch.zeros(*s)  # noqa: E731
    calls = [
        (kb.gated_scan, [z(1, 2, 4), z(1, 2, 4), z(1, 4)]),
        (kb.recurrence.gated_scan_backward, [z(1, 2, 4), z(1, 2, 4), z(1, 4), z(1, 2, 4), z(1, 4)]),
        (kb.gated_step, [z(2, 4), z(2, 4), z(2, 4)]),
        (kb.qk_norm_rope, [z(1, 2, 3, 4), z(1, 2, 1, 4), z(4), z(4)]),
        (kb.rotary.qk_norm_rope_backward, [z(1, 2, 3, 4), z(1, 2, 1, 4), z(1, 2, 3, 4), z(1, 2, 1, 4), z(4), z(4)]),
    ]
    for fn, args in calls:
        for i in range(len(args)):
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(lambda t: fn(t, *args[1:])[0], (args[0],), (torch.ones_like(args[0]),))
        # inside a level, tensors without a tangent get as far as without one (no CPU path)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="CUDA"):
            fn(*args)
    with forward_ad.dual_level():
        freq = forward_ad.make_dual(z(2), torch.ones(2))
        with pytest.raises(RuntimeError, match="forward-mode"):
            kb.qk_norm_rope(z(1, 2, 3, 4), inv_freq=freq)


def test_backward_wants_checkpoints_for_rows_without_sequences():
    """Packed rows of no sequence are walked too, from the checkpoints."""
    L = pkg()._lib
    lib = L.load()
    packed = dict(B=0, q_start=FAKE, workspace=FAKE, workspace_bytes=1 << 20, ckpt=None)
    assert lib.kda_scan_bwd(ctypes.byref(_scan_args(**packed)), None) == L.KDA_ERR_NULL_POINTER
    assert lib.kda_scan_bwd(ctypes.byref(_scan_args(**packed, T=0)), None) == L.KDA_OK


@pytest.mark.parametrize("tq,tk", [(torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16),
                                   (torch.float64, torch.float64), (torch.bfloat16, torch.bfloat16)])
def test_mla_step_rotates_in_one_type(tq, tk, monkeypatch):
    """Rope parts of two types, which a step without frequencies takes, reach the rotation in one."""
    from test_latent_step_host import _step_args

    kb, seen = pkg(), []

    def rotation(q, k, **kw):
        seen.append((q.dtype, k.dtype))
        raise InterruptedError

    monkeypatch.setattr(kb.latent, "qk_norm_rope", rotation)
    args = _step_args(DR=64)
    args[6].update(inv_freq=torch.ones(32), cache=kb.LatentCache(2, 16, 128, 64, device="cpu"))
    args[3], args[5] = torch.zeros(2, 1, 2, 64, dtype=tq), torch.zeros(2, 1, 64, dtype=tk)
    with pytest.raises(InterruptedError):
        kb.latent.mla_step(*args, True)
    same = tq == tk and tq != torch.float64
    assert seen == [(tq, tk) if same else (torch.float32,) * 2]
    assert args[6]["lens"].tolist() == [3, 5]
