"""Norm and rotation of queries and keys on the GPU against the 64-bit oracle: values,
gradients, layouts, far positions, extremes, streams, graphs, refusals.

Bars, with U = 2^-24.  A row's r comes from a sum of at most 512 squares added in at most
21 steps a path, halved by the root: 20 U of itself.  A rotation's cosine and sine are off by
4 U + 2^-51 |angle| (a 64-bit angle, reduced; then two units in the last place), its products
and sum by 2 U: at most (8 U + 2^-51 |angle|) of the pair's magnitudes.  A sum of n products
adds (n + 2) U of its magnitudes at most, 30 U where 512 are added by lanes and a tree.  Then half a
step of the result's type."""

from __future__ import annotations

import pytest
import torch

from conftest import pkg
from oracle import recurrence_oracle as R
from test_gpu_recurrence import close

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = R.U


def pairs(m, n, interleaved):
    """Each channel's magnitude plus its partner's ([..., D], R = 2 n channels rotated)."""
    out = m.clone()
    for i in range(n):
        j, k = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        out[..., j] = out[..., k] = m[..., j] + m[..., k]
    return out


def turn_error(pos, freq, D, interleaved):
    """What a rotation may be off by, of the pair's magnitudes ([N, 1, D])."""
    e = torch.zeros(pos.shape[0], 1, D, dtype=torch.float64)
    if freq is not None:
        n = freq.shape[0]
        a = (pos[:, None].double() * freq.double()).abs() * 2.0 ** -51 + 8 * U
        for i in range(n):
            j, k = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
            e[:, 0, j] = e[:, 0, k] = a[:, i]
    return e


def oracle(x, w, norm, eps, pos, freq, interleaved, dy=None):
    """``(y, its bar)`` and with ``dy`` also ``(dx, bar), (dw, bar)``, all [N, H, D] float64."""
    x = x.double()
    w = None if w is None else w.double()
    n = 0 if freq is None else freq.shape[0]
    angle = None if freq is None else (pos[:, None].double() * freq.double())[:, None]
    te = turn_error(pos, freq, x.shape[-1], interleaved)
    r, moves = R.rate(x, norm, eps)
    z = (x * r).abs() * (1 if w is None else w.abs())
    out = [(R.qk(x, w, norm, eps, angle, interleaved), pairs(z, n, interleaved) * (24 * U + te))]
    if dy is None:
        return out
    dy = dy.double()
    dx, dw, mag = R.qk_grad(x, w, norm, eps, angle, interleaved, dy)
    dz = dy if angle is None else R.rotation(dy, -angle, interleaved)
    ez = pairs(dy.abs(), n, interleaved) * te
    ww = 1 if w is None else w.abs()
    v, ev, nn = dz.abs() * ww, ez * ww, (x * r).abs()
    d = x.shape[-1] if norm == "rms" else 1
    md = (v * nn).sum(-1, keepdim=True) / d
    ed = (ev * nn).sum(-1, keepdim=True) / d + 60 * U * md
    ex = r * (ev + 24 * U * v + moves * nn * (ed + 60 * U * md))
    out.append((dx, ex))
    if w is not None:
        along = (0, 1) if w.dim() == 1 else (0,)
        out.append((dw, (ez * nn).sum(along) + (40 + x.shape[0]) * U * mag))
    return out


def make(N, H, HK, D, tx, tw, weight, seed):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    loud = torch.exp(rnd(N, 1, 1))
    q, k = (rnd(N, H, D) * loud).to(tx), (rnd(N, HK, D) * loud).to(tx)
    dq, dk = rnd(N, H, D).to(tx), rnd(N, HK, D).to(tx)
    ws = [None, None]
    if weight:
        ws = [(1 + 0.3 * rnd(*((n, D) if weight == "heads" else (D,)))).to(tw) for n in (H, HK)]
    return q, k, dq, dk, ws


def freqs(R_, base=10000.0):
    return (base ** (-torch.arange(0, R_, 2, dtype=torch.float64) / R_)).float()


CASES = [
    # N, H, HK, D, R, type, weight type, weight, norm, interleaved
    (1, 1, 1, 1, 0, F32, F32, "head_dim", "rms", False),
    (3, 2, 1, 2, 2, F32, F32, "heads", "l2", True),
    (5, 3, 1, 7, 4, BF16, F32, "head_dim", "rms", False),
    (9, 16, 16, 128, 128, F16, F16, "head_dim", "rms", False),
    (9, 16, 4, 128, 64, BF16, BF16, "heads", "rms", True),
    (33, 8, 2, 64, 64, BF16, F32, None, "l2", False),
    (4, 16, 1, 64, 64, BF16, F32, None, None, True),
    (4, 16, 1, 64, 32, F16, F32, None, None, False),
    (130, 5, 5, 96, 48, F32, F32, "head_dim", "rms", False),
    (130, 12, 3, 90, 30, BF16, F32, "heads", "rms", False),
    (17, 3, 3, 192, 64, F16, F32, "heads", "rms", True),
    (11, 4, 2, 256, 256, F32, F32, "head_dim", "l2", False),
    (7, 2, 1, 320, 100, BF16, F32, "head_dim", "rms", False),
    (6, 1, 1, 512, 512, BF16, BF16, "heads", "rms", False),
    (6, 2, 1, 511, 510, F16, F32, "head_dim", "l2", True),
    (700, 20, 4, 80, 20, BF16, F32, "head_dim", "rms", False),
    (300, 33, 1, 128, 0, F16, F16, "head_dim", "rms", False),
    (65, 40, 8, 128, 96, BF16, F32, "heads", "rms", False),
    (2, 2, 2, 72, 16, BF16, F32, "head_dim", "rms", False),
    (21, 6, 2, 40, 40, F32, F32, "heads", "l2", False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_values_and_gradients(cuda_dev, case):
    kb = pkg()
    N, H, HK, D, R_, tx, tw, weight, norm, inter = case
    q, k, dq, dk, ws = make(N, H, HK, D, tx, tw, weight, N + D)
    gen = torch.Generator().manual_seed(2)
    pos = torch.randint(0, 200000, (N,), generator=gen)
    freq = freqs(R_) if R_ else None
    eps = 1e-5
    dev = lambda t: None if t is None else t.to(cuda_dev)  # noqa: E731
    leaves = [dev(t).requires_grad_() for t in (q, k, *ws) if t is not None]
    a = leaves + [None, None] if weight is None else leaves
    oq, ok = kb.qk_norm_rope(*a, norm=norm, eps=eps, positions=dev(pos), inv_freq=dev(freq), interleaved=inter)
    grads = list(torch.autograd.grad([oq, ok], leaves, [dev(dq), dev(dk)]))
    with torch.no_grad():
        again = kb.qk_norm_rope(*a, norm=norm, eps=eps, positions=dev(pos.int()), inv_freq=dev(freq),
                                interleaved=inter)
    assert torch.equal(again[0], oq) and torch.equal(again[1], ok)
    for i, (x, d, w, o, name) in enumerate(((q, dq, ws[0], oq, "q"), (k, dk, ws[1], ok, "k"))):
        want = oracle(x, w, norm, eps, pos, freq, inter, d)
        assert o.dtype == tx
        close(o, *want[0], name)
        close(grads[i], *want[1], "d" + name)
        if w is not None:
            assert grads[2 + i].dtype == tw
            close(grads[2 + i], *want[2], "dw" + name)


def test_positions(cuda_dev):
    """First positions, one a token, none, 32 and 64 bits, negative and far ones."""
    kb = pkg()
    B, T, H, D = 3, 37, 2, 64
    q, k, *_ = make(B * T, H, 1, D, F32, F32, None, 1)
    freq = freqs(D)
    first = torch.tensor([0, -5000, 2 ** 31 - 100])
    each = first[:, None] + torch.arange(T)
    dev = lambda t: t.to(cuda_dev)  # noqa: E731
    q4, k4 = dev(q.view(B, T, H, D)), dev(k.view(B, T, 1, D))
    kw = dict(norm=None, inv_freq=dev(freq))
    outs = [kb.qk_norm_rope(q4, k4, positions=p, **kw)
            for p in (dev(first), dev(first.int()), dev(each), dev(each.int()),
                      dev(each.t().contiguous()).t(), dev(torch.stack([first, first], 1))[:, 0])]
    for o in outs[1:]:
        assert torch.equal(o[0], outs[0][0]) and torch.equal(o[1], outs[0][1])
    pos = each.reshape(-1)
    for x, o in ((q, outs[0][0]), (k, outs[0][1])):
        close(o.reshape(x.shape), *oracle(x, None, None, 1e-6, pos, freq, False)[0], "far")
    none = kb.qk_norm_rope(q4, k4, **kw)
    zero = kb.qk_norm_rope(q4, k4, positions=dev(torch.zeros(B, dtype=torch.int32)), **kw)
    assert torch.equal(none[0], zero[0]) and torch.equal(none[1], zero[1])
    flat = kb.qk_norm_rope(dev(q), dev(k), positions=dev(pos), **kw)
    assert torch.equal(flat[0], outs[0][0].view_as(flat[0]))
    only, nothing = kb.qk_norm_rope(q4, positions=dev(first), **kw)
    assert nothing is None and torch.equal(only, outs[0][0])
    with torch.enable_grad():
        leaf = q4.clone().requires_grad_()
        only, nothing = kb.qk_norm_rope(leaf, positions=dev(first), **kw)
        assert nothing is None
        g, = torch.autograd.grad(only, leaf, torch.ones_like(only))
        g2 = kb.rotary.qk_norm_rope_backward(torch.ones_like(only), None, q4, positions=dev(first), **kw)
        assert torch.equal(g, g2[0]) and g2[1:] == (None, None, None)
    # a rotation keeps a pair's length, whatever the position
    huge = torch.tensor([2 ** 62, -2 ** 62, 2 ** 53 + 1])
    o = kb.qk_norm_rope(q4, k4, positions=dev(huge), **kw)[0].double().cpu().view(-1, H, D)
    a, b = (t.double().view(-1, H, 2, D // 2).norm(dim=2) for t in (o, q.double()))
    assert ((a - b).abs() <= 32 * U * b).all()


def test_strides_and_offsets(cuda_dev):
    """Slices of one projection, odd offsets, transposes, broadcast inputs and gradients."""
    kb = pkg()
    B, T, H, HK, D = 2, 19, 6, 2, 48
    gen = torch.Generator().manual_seed(4)
    first, freq = torch.tensor([7, 100]), freqs(32)
    pos = (first[:, None] + torch.arange(T)).reshape(-1)
    flat = lambda t: t.cpu().reshape(B * T, *t.shape[2:])  # noqa: E731
    for dt in (F32, BF16):
        for pad in (0, 1, 2, 8):
            both = torch.randn(B, T, (H + 2 * HK) * D + pad, generator=gen).to(dt).to(cuda_dev)
            q = both[..., pad:pad + H * D].unflatten(-1, (H, D))
            k = both[..., pad + H * D:pad + (H + HK) * D].unflatten(-1, (HK, D))
            dq, dk = torch.randn_like(q), torch.randn_like(k)
            w = [torch.randn(n, D, generator=gen).to(cuda_dev) for n in (H, HK)]
            kw = dict(inv_freq=freq.to(cuda_dev), positions=first.to(cuda_dev))
            want = [oracle(flat(x), wi.cpu(), "rms", 1e-6, pos, freq, False, flat(d))
                    for x, wi, d in ((q, w[0], dq), (k, w[1], dk))]
            heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
            inner = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731
            for f in (lambda t: t, torch.Tensor.contiguous, heads_first, inner):
                got = (*kb.qk_norm_rope(f(q), f(k), *w, **kw),
                       *kb.rotary.qk_norm_rope_backward(f(dq), f(dk), f(q), f(k), *w, **kw))
                for i in range(2):
                    close(flat(got[i]), *want[i][0], "y")
                    close(flat(got[2 + i]), *want[i][1], "dx")
                    close(got[4 + i], *want[i][2], "dw")
    one = torch.ones((), device=cuda_dev).expand(B, T, H, D)
    x = torch.randn(B, T, 1, D, device=cuda_dev).expand(B, T, H, D)
    a = kb.rotary.qk_norm_rope_backward(one, None, x, **kw)
    b = kb.rotary.qk_norm_rope_backward(one.contiguous(), None, x.contiguous(), **kw)
    assert torch.equal(a[0], b[0])


def test_extremes(cuda_dev):
    """Rows of zeros, rows whose squares over- or underflow, and rows that are not finite."""
    kb = pkg()
    for D in (64, 50):
        x = torch.randn(1, 9, 1, D, generator=torch.Generator().manual_seed(1))
        x[0, 0] = 0.0
        x[0, 1] *= 1e25
        x[0, 2] *= 1e-30
        x[0, 3] *= 3e37
        x[0, 4] *= 1e-7
        x[0, 5, 0, 3] = float("inf")
        x[0, 6, 0, 2] = float("nan")
        dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(2))
        pos = torch.arange(9)
        for norm, eps in (("rms", 1e-6), ("l2", 1e-6), ("rms", 1e-12)):
            y, _ = kb.qk_norm_rope(x.to(cuda_dev), norm=norm, eps=eps)
            dx = kb.rotary.qk_norm_rope_backward(dy.to(cuda_dev), None, x.to(cuda_dev), norm=norm, eps=eps)[0]
            ok = [0, 1, 2, 3, 4, 7, 8]
            want = oracle(x[0, ok], None, norm, eps, pos[ok], None, False, dy[0, ok])
            close(y[0, ok], *want[0], (D, norm))
            close(dx[0, ok], want[1][0], want[1][1] + 1e-44, (D, norm, "dx"))
            assert torch.isnan(y[0, 5, 0, 3]) and torch.isnan(y[0, 6]).all()


def test_gradient_by_differences(cuda_dev):
    kb = pkg()
    N, H, D, R_ = 5, 2, 24, 16
    q, _, dq, _, ws = make(N, H, 1, D, F32, F32, "heads", 3)
    pos, freq = torch.arange(N) * 11, freqs(R_)
    angle = (pos[:, None].double() * freq.double())[:, None]
    gen = torch.Generator().manual_seed(1)
    for norm in ("rms", "l2"):
        d = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (q, ws[0])]
        f = lambda s: (R.qk(q.double() + s * d[0], ws[0].double() + s * d[1], norm, 1e-6, angle, False)  # noqa: E731
                       * dq.double()).sum()
        slope = float((f(1e-6) - f(-1e-6)) / 2e-6)
        g = kb.rotary.qk_norm_rope_backward(
            dq.to(cuda_dev), None, q.to(cuda_dev), None, ws[0].to(cuda_dev), norm=norm,
            positions=pos.to(cuda_dev), inv_freq=freq.to(cuda_dev))
        parts = [g[0].cpu().double() * d[0], g[2].cpu().double() * d[1]]
        assert abs(sum(float(p.sum()) for p in parts) - slope) <= 1e-5 * sum(float(p.abs().sum()) for p in parts)


def test_streams_graphs_and_repeats(cuda_dev):
    kb = pkg()
    q, k, dq, dk, ws = ([u.to(cuda_dev) for u in t] if isinstance(t, list) else t.to(cuda_dev)
                        for t in make(400, 16, 4, 128, BF16, F32, "head_dim", 6))
    freq, pos = freqs(128).to(cuda_dev), torch.arange(400, device=cuda_dev, dtype=torch.int32)
    kw = dict(positions=pos, inv_freq=freq)

    def step():
        a = [t.detach().requires_grad_() for t in (q, k, *ws)]
        o = kb.qk_norm_rope(*a, **kw)
        return [t.detach() for t in o] + list(torch.autograd.grad(o, a, [dq, dk]))

    ref = step()
    for _ in range(2):
        assert all(torch.equal(u, v) for u, v in zip(step(), ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, ref))
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            out = step()
        graphs.append((gr, out))
    for shift in (0, 1000):
        pos.copy_(torch.arange(400, device=cuda_dev) + shift)
        q.copy_(q.flip(0))
        want = step()
        for gr, out in graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, want))


def test_empty(cuda_dev):
    kb = pkg()
    z = lambda *s: torch.zeros(*s, device=cuda_dev)  # noqa: E731
    for shape, n in (((0, 4, 2, 8), 1), ((2, 0, 2, 8), 1), ((3, 4, 0, 8), 1), ((3, 4, 2, 8), 0)):
        q, k = z(*shape), z(*shape[:2], n, 8)
        oq, ok = kb.qk_norm_rope(q, k, z(8), z(8), inv_freq=freqs(8).to(cuda_dev))
        assert oq.shape == q.shape and ok.shape == k.shape
        g = kb.rotary.qk_norm_rope_backward(q, k, q, k, z(8), z(8), inv_freq=freqs(8).to(cuda_dev))
        assert (g[2] == 0).all() and (g[3] == 0).all()
    assert torch.equal(kb.qk_norm_rope(torch.ones(2, 3, 1, 4, device=cuda_dev), norm=None)[0],
                       torch.ones(2, 3, 1, 4, device=cuda_dev))


def test_refusals(cuda_dev):
    kb = pkg()
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device=cuda_dev)  # noqa: E731
    q, k, w = z(2, 3, 4, 8), z(2, 3, 1, 8), z(8)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    for args, kw, exc in [
            ((z(3, 8),), {}, RuntimeError), ((q, z(2, 4, 1, 8)), {}, RuntimeError),
            ((q, z(2, 3, 1, 6)), {}, RuntimeError), ((q, k.half()), {}, TypeError),
            ((q, z(3, 1, 8)), {}, RuntimeError), ((z(2, 3, 4, 513),), {}, RuntimeError),
            ((q, k, w, w), dict(norm="layer"), ValueError), ((q, k, w), dict(norm=None), RuntimeError),
            ((q, k, w), dict(eps=0.0), ValueError), ((q, k, w), dict(eps=float("nan")), ValueError),
            ((q, None, w, w), {}, RuntimeError), ((q, k, z(7)), {}, RuntimeError),
            ((q, k, z(1, 8)), {}, RuntimeError), ((q, k, z(4, 8), w), {}, RuntimeError),
            ((q, k, w, w.half()), {}, RuntimeError), ((q, k, w.cpu()), {}, RuntimeError),
            ((q, k), dict(inv_freq=z(5)), RuntimeError), ((q, k), dict(inv_freq=z(4).double()), RuntimeError),
            ((q, k), dict(inv_freq=z(4).cpu()), RuntimeError), ((q, k), dict(inv_freq=z(2, 2)), RuntimeError),
            ((q, k), dict(inv_freq=z(4), positions=i(3)), RuntimeError),
            ((q, k), dict(inv_freq=z(4), positions=i(3, 2)), RuntimeError),
            ((q, k), dict(inv_freq=z(4), positions=z(2)), RuntimeError),
            ((q, k), dict(inv_freq=z(4), positions=i(2).cpu()), RuntimeError),
            ((q, k), dict(inv_freq=z(4).requires_grad_()), RuntimeError),
            ((q.double(),), {}, TypeError), ((q.cpu(),), {}, RuntimeError)]:
        with pytest.raises(exc):
            kb.qk_norm_rope(*args, **kw)
    with pytest.raises(RuntimeError):
        kb.rotary.qk_norm_rope_backward(q, None, q, k)
    with pytest.raises(RuntimeError):
        kb.rotary.qk_norm_rope_backward(z(2, 3, 4, 6), k, q, k)
