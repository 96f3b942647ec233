"""Gated recurrence on the GPU against the 64-bit oracle: scan, gradient, packed
sequences, single-token step; strides, streams, graphs, special values, refusals.

A value may be off by what fp32 arithmetic adds (the oracle's bounds) and by half a step of
its own type."""

from __future__ import annotations

import pytest
import torch

from conftest import pkg
from oracle import recurrence_oracle as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)]


def close(got, want, bound, what):
    """``got`` within ``bound`` and half a step of its type of the float64 ``want``."""
    dt = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    least = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}[dt]
    bar = bound + (want.abs() + bound) * torch.finfo(dt).eps / 2 + least + 2.0 ** -125
    bad = ~((got - want).abs() <= bar)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], bar[bad][:4])


def gates(shape, gen):
    """Log decays between 1e-4 and 30 a token, some of them zero."""
    g = -torch.exp(torch.empty(shape).uniform_(-9.0, 1.5, generator=gen))
    g[torch.rand(shape, generator=gen) < 0.02] = -30.0
    g[torch.rand(shape, generator=gen) < 0.02] = 0.0
    return g


def inputs(rows, D, tx, tg, seed, seqs, dev):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, D, generator=gen).to(tx)
    g = gates((rows, D), gen).to(tg)
    s0 = torch.randn(seqs, D, generator=gen)
    dh = torch.randn(rows, D, generator=gen).to(tx)
    dS = torch.randn(seqs, D, generator=gen)
    return x, g, s0, dh, dS


def expected(x, g, s0, dh, dS, spans, complement):
    """h, S, dx, dg, ds0 and their bounds, over rows of no sequence zeros."""
    x, g, s0, dh, dS = (t.double() for t in (x, g, s0, dh, dS))
    vals = [torch.zeros_like(x), torch.empty_like(s0), torch.zeros_like(x), torch.zeros_like(x),
            torch.empty_like(s0)]
    errs = [torch.zeros_like(v) for v in vals]
    for b, (lo, hi) in enumerate(spans):
        h, S, eh, eS, _ = R.scan(x[lo:hi], g[lo:hi], s0[b], complement)
        dx, dg, ds, ex, eg, es = R.scan_grad(x[lo:hi], g[lo:hi], s0[b], dh[lo:hi], dS[b], complement)
        vals[0][lo:hi], errs[0][lo:hi] = h, eh
        vals[1][b], errs[1][b] = S, eS
        vals[2][lo:hi], errs[2][lo:hi] = dx, ex
        vals[3][lo:hi], errs[3][lo:hi] = dg, eg
        vals[4][b], errs[4][b] = ds, es
    return vals, errs


NAMES = ("h", "S", "dx", "dg", "ds0")


@pytest.mark.parametrize("tx,tg", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("complement", [False, True], ids=["plain", "complement"])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 7, 3), (1, 63, 64), (3, 64, 60), (2, 65, 130),
                                   (1, 129, 66), (2, 257, 32), (1, 700, 20), (67, 5, 16), (5, 1100, 4)])
def test_batch(cuda_dev, tx, tg, complement, B, T, D):
    kb = pkg()
    x, g, s0, dh, dS = inputs(B * T, D, tx, tg, 11 * T + D, B, cuda_dev)
    want, err = expected(x, g, s0, dh, dS, [(b * T, b * T + T) for b in range(B)], complement)
    leaves = [x.view(B, T, D).to(cuda_dev).requires_grad_(), g.view(B, T, D).to(cuda_dev).requires_grad_(),
              s0.to(cuda_dev).requires_grad_()]
    h, S = kb.gated_scan(*leaves, complement=complement)
    assert h.dtype == tx and S.dtype == F32
    got = [h, S, *torch.autograd.grad([h, S], leaves, [dh.view(B, T, D).to(cuda_dev), dS.to(cuda_dev)])]
    with torch.no_grad():
        plain = kb.gated_scan(*leaves, complement=complement)
    assert torch.equal(plain[0], h) and torch.equal(plain[1], S)
    for n, v, w, e in zip(NAMES, got, want, err):
        close(v.reshape(w.shape), w, e, n)


@pytest.mark.parametrize("tx,tg", [(F32, F32), (F16, F32), (BF16, BF16)], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("B,T,D", [(80, 70, 128), (150, 3, 40), (1, 200, 9536), (76, 1030, 128), (149, 1, 64),
                                   (3, 140, 9480)])
def test_more_blocks_than_the_gpu_takes(cuda_dev, tx, tg, B, T, D):
    """The blocks of many sequences or channels, short and long; as a batch and packed."""
    kb = pkg()
    complement = tx == F16
    x, g, s0, dh, dS = inputs(B * T, D, tx, tg, B + T, B, cuda_dev)
    wide = lambda t: t.view(B, T, D).transpose(0, 1).reshape(T, B * D)  # noqa: E731
    want, err = expected(wide(x), wide(g), s0.view(1, -1), wide(dh), dS.view(1, -1), [(0, T)], complement)
    back = lambda t: t.view(T, B, D).transpose(0, 1)  # noqa: E731
    dev = lambda t: t.to(cuda_dev)  # noqa: E731
    for q in (None, dev(torch.arange(0, B * T + 1, T, dtype=torch.int32))):
        rows = (B, T, D) if q is None else (B * T, D)
        leaves = [dev(x).view(rows).requires_grad_(), dev(g).view(rows).requires_grad_(),
                  dev(s0).requires_grad_()]
        h, S = kb.gated_scan(*leaves, q, complement=complement)
        got = [h, S, *torch.autograd.grad([h, S], leaves, [dev(dh).view(rows), dev(dS)])]
        for i, (n, v) in enumerate(zip(NAMES, got)):
            states = i in (1, 4)
            w, e = (t.view(B, D) if states else back(t) for t in (want[i], err[i]))
            close(v.reshape(w.shape), w, e, n)


STARTS = {
    "one": (50, [0, 50]),
    "ragged": (300, [0, 1, 2, 66, 66, 194, 300]),
    "unowned": (200, [13, 13, 77, 140, 190]),
    "single": (130, list(range(0, 131))),
    "tiles": (256, [0, 64, 128, 128, 192, 256]),
    "inside": (90, [40, 45]),
    "empty": (20, [7, 7, 7]),
    "none": (9, [4]),
    "long": (2600, [0, 1300, 1301, 2590]),
    "no rows": (0, [0, 0, 0]),
}


@pytest.mark.parametrize("tx,tg", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("name", list(STARTS))
@pytest.mark.parametrize("D", [5, 72])
def test_packed(cuda_dev, tx, tg, name, D):
    kb = pkg()
    N, q = STARTS[name]
    complement = D == 72
    x, g, s0, dh, dS = inputs(N, D, tx, tg, len(name) + D, len(q) - 1, cuda_dev)
    want, err = expected(x, g, s0, dh, dS, list(zip(q, q[1:])), complement)
    leaves = [t.to(cuda_dev).requires_grad_() for t in (x, g, s0)]
    q_start = torch.tensor(q, dtype=torch.int32, device=cuda_dev)
    h, S = kb.gated_scan(*leaves, q_start, complement=complement)
    got = [h, S, *torch.autograd.grad([h, S], leaves, [dh.to(cuda_dev), dS.to(cuda_dev)])]
    for n, v, w, e in zip(NAMES, got, want, err):
        close(v, w, e, n)
    mine = torch.zeros(N, dtype=torch.bool)
    for lo, hi in zip(q, q[1:]):
        mine[lo:hi] = True
    for v in (got[0], got[2], got[3]):
        assert (v.cpu()[~mine] == 0).all()


def test_sequences_do_not_leak(cuda_dev):
    """Infinities and NaN stay in their sequence, their channel and behind their token."""
    kb = pkg()
    q = [2, 40, 41, 100, 165, 230]
    x, g, s0, dh, dS = inputs(240, 8, F32, F32, 3, 5, cuda_dev)
    clean = [t.to(cuda_dev) for t in (x, g, s0)]
    q_start = torch.tensor(q, dtype=torch.int32, device=cuda_dev)
    ref = kb.gated_scan(*clean, q_start)
    ref_g = kb.recurrence.gated_scan_backward(*clean, dh.to(cuda_dev), dS.to(cuda_dev), q_start)
    x2, s2, dh2 = x.clone(), s0.clone(), dh.clone()
    x2[0], x2[235] = float("nan"), float("inf")          # rows of no sequence
    x2[60, 3] = float("nan")
    x2[110, 4] = float("inf")
    s2[4, 5] = float("nan")
    dh2[1] = dh2[231] = float("nan")
    bad = [t.to(cuda_dev) for t in (x2, g, s2)]
    got = kb.gated_scan(*bad, q_start)
    keep = torch.ones(240, 8, dtype=torch.bool)
    keep[60:100, 3] = keep[110:165, 4] = keep[165:230, 5] = False
    assert torch.equal(got[0].cpu()[keep], ref[0].cpu()[keep])
    assert torch.isnan(got[0].cpu()[60:100, 3]).all() and torch.isinf(got[0].cpu()[110, 4])
    assert torch.isnan(got[0].cpu()[165:230, 5]).all()
    grads = kb.recurrence.gated_scan_backward(*bad, dh2.to(cuda_dev), dS.to(cuda_dev), q_start)
    assert torch.equal(grads[0], ref_g[0])               # dx does not read x
    ok = keep.clone()
    assert torch.equal(grads[1].cpu()[ok], ref_g[1].cpu()[ok])


def test_special_gates(cuda_dev):
    """-inf forgets, 0 keeps all, and slow decays over thousands of tokens lose nothing."""
    kb = pkg()
    T, D = 6000, 8
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(T, D, generator=gen)
    g = torch.zeros(T, D)
    g[:, 1] = -1e-6
    g[:, 2] = -3.3e-5
    g[:, 3] = -1e-3
    g[:, 4] = -0.2499
    g[:, 5] = -0.2501
    g[:, 6] = -200.0
    g[::97, 7] = float("-inf")
    s0 = torch.randn(1, D, generator=gen)
    dh, dS = torch.randn(T, D, generator=gen), torch.randn(1, D, generator=gen)
    want, err = expected(x, g, s0, dh, dS, [(0, T)], False)
    args = [t.to(cuda_dev) for t in (x[None], g[None], s0)]
    h, S = kb.gated_scan(*args)
    grads = kb.recurrence.gated_scan_backward(*args, dh[None].to(cuda_dev), dS.to(cuda_dev))
    for n, v, w, e in zip(NAMES, [h[0], S, grads[0][0], grads[1][0], grads[2]], want, err):
        close(v, w, e, n)


def test_strides_and_offsets(cuda_dev):
    """Slices of a projection, odd offsets, expanded gradients, transposed batches."""
    kb = pkg()
    B, T, D = 3, 77, 24
    x, g, s0, dh, dS = inputs(B * T, D, BF16, F32, 9, B, cuda_dev)
    x, g, dh = (t.view(B, T, D).to(cuda_dev) for t in (x, g, dh))
    s0, dS = s0.to(cuda_dev), dS.to(cuda_dev)
    ref = kb.gated_scan(x, g, s0)
    ref_g = kb.recurrence.gated_scan_backward(x, g, s0, dh, dS)

    def embed(t, off, extra):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + extra), float("nan"), dtype=t.dtype, device=cuda_dev)
        view = wide[..., off:off + t.shape[-1]]
        view.copy_(t)
        return view

    def check(*a):
        got = kb.gated_scan(*a[:3])
        got_g = kb.recurrence.gated_scan_backward(*a)
        for u, v in zip((*got, *got_g), (*ref, *ref_g)):
            assert torch.equal(u, v)

    for off, extra in ((1, 3), (4, 8), (2, 2), (0, 1)):
        check(embed(x, off, extra), embed(g, off, extra), embed(s0, off, extra), embed(dh, off, extra),
              embed(dS, off, extra))
    tm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    check(tm(x), tm(g), s0, tm(dh), dS)
    inner = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    check(inner(x), inner(g), s0.t().contiguous().t(), inner(dh), dS)
    ones = torch.ones((), device=cuda_dev, dtype=BF16).expand(B, T, D)
    a = kb.recurrence.gated_scan_backward(x, g, s0, ones, None)
    b = kb.recurrence.gated_scan_backward(x, g, s0, ones.contiguous(), torch.zeros_like(dS))
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    c = kb.recurrence.gated_scan_backward(x, g, None, None, dS)
    d = kb.recurrence.gated_scan_backward(x, g, torch.zeros_like(s0), torch.zeros_like(dh), dS)
    assert c[2] is None and all(torch.equal(u, v) for u, v in zip(c[:2], d[:2]))
    # one row for the whole batch
    row = x[:1].expand(B, T, D)
    assert torch.equal(kb.gated_scan(row, g, s0)[0], kb.gated_scan(row.contiguous(), g, s0)[0])


def test_state_types_and_partial_gradients(cuda_dev):
    kb = pkg()
    x, g, s0, dh, dS = inputs(2 * 90, 12, F16, F16, 21, 2, cuda_dev)
    x, g = x.view(2, 90, 12).to(cuda_dev), g.view(2, 90, 12).to(cuda_dev)
    s16 = s0.to(cuda_dev).half()
    assert torch.equal(kb.gated_scan(x, g, s16)[1], kb.gated_scan(x, g, s16.float())[1])
    full = kb.recurrence.gated_scan_backward(x, g, s16, dh.view_as(x).to(cuda_dev), dS.to(cuda_dev))
    assert full[2].dtype == F16
    for i in range(3):
        leaves = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, g, s16))]
        h, S = kb.gated_scan(*leaves)
        got, = torch.autograd.grad([h, S], [leaves[i]], [dh.view_as(x).to(cuda_dev), dS.to(cuda_dev)])
        assert torch.equal(got, full[i])
    # only one of the two outputs used
    leaves = [t.clone().requires_grad_() for t in (x, g)]
    kb.gated_scan(*leaves)[1].backward(dS.to(cuda_dev))
    want = kb.recurrence.gated_scan_backward(x, g, None, None, dS.to(cuda_dev))
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[1].grad, want[1])


def test_gradient_by_differences(cuda_dev):
    """Along random directions, against central differences of the 64-bit forward pass."""
    kb = pkg()
    T, D = 150, 6
    for complement in (False, True):
        x, g, s0, dh, dS = (t.double() for t in inputs(T, D, F32, F32, 31, 1, cuda_dev))
        g = g.clamp(max=-1e-3)
        gen = torch.Generator().manual_seed(1)
        dirs = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (x, g, s0)]

        def loss(step):
            y = [t + step * d for t, d in zip((x, g, s0), dirs)]
            h, S, *_ = R.scan(y[0], y[1], y[2][0], complement)
            return (h * dh).sum() + (S * dS[0]).sum()

        eps = 1e-6
        slope = float((loss(eps) - loss(-eps)) / (2 * eps))
        grads = kb.recurrence.gated_scan_backward(
            x.float()[None].to(cuda_dev), g.float()[None].to(cuda_dev), s0.float().to(cuda_dev),
            dh.float()[None].to(cuda_dev), dS.float().to(cuda_dev), complement=complement)
        parts = [(gr.cpu().double().reshape(d.shape) * d) for gr, d in zip(grads, dirs)]
        got = sum(float(p.sum()) for p in parts)
        # a value's share is off by fp32's 2^-24 some tens of times; the differences by eps^2
        assert abs(got - slope) <= 1e-5 * sum(float(p.abs().sum()) for p in parts)


def test_deterministic_and_other_stream(cuda_dev):
    kb = pkg()
    x, g, s0, dh, dS = (t.to(cuda_dev) for t in inputs(4 * 1000, 96, BF16, F32, 2, 4, cuda_dev))
    x, g, dh = (t.view(4, 1000, 96) for t in (x, g, dh))
    ref = (*kb.gated_scan(x, g, s0), *kb.recurrence.gated_scan_backward(x, g, s0, dh, dS))
    for _ in range(3):
        got = (*kb.gated_scan(x, g, s0), *kb.recurrence.gated_scan_backward(x, g, s0, dh, dS))
        assert all(torch.equal(u, v) for u, v in zip(got, ref))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append((*kb.gated_scan(x, g, s0), *kb.recurrence.gated_scan_backward(x, g, s0, dh, dS)))
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(u, v) for u, v in zip(got, ref))


def test_graphs(cuda_dev):
    """Forward and backward captured, two graphs replayed in turn with new inputs."""
    kb = pkg()
    q = torch.tensor([0, 30, 31, 200], dtype=torch.int32, device=cuda_dev)
    sets = [[t.to(cuda_dev) for t in inputs(210, 40, F32, F32, s, 3, cuda_dev)] for s in (1, 2)]
    static = [t.clone() for t in sets[0]]
    starts = q.clone()

    def step():
        leaves = [t.detach().requires_grad_() for t in static[:3]]
        h, S = kb.gated_scan(*leaves, starts)
        return (h.detach(), S.detach(), *torch.autograd.grad([h, S], leaves, static[3:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            outs.append(step())
        graphs.append(gr)
    q2 = torch.tensor([5, 100, 150, 205], dtype=torch.int32, device=cuda_dev)
    for new_q in (q, q2):
        for data in sets:
            starts.copy_(new_q)
            for s, t in zip(static, data):
                s.copy_(t)
            want = step()
            for gr, out in zip(graphs, outs):
                gr.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(u, v) for u, v in zip(out, want))


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("tx,tg", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("complement", [False, True], ids=["plain", "complement"])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 7), (5, 64), (2, 1030), (130, 12)])
def test_step(cuda_dev, tx, tg, complement, B, D):
    kb = pkg()
    x, g, s0, _, _ = inputs(B, D, tx, tg, B + D, B, cuda_dev)
    h64 = torch.stack([R.scan(x[b:b + 1].double(), g[b:b + 1].double(), s0[b].double(), complement)[1]
                       for b in range(B)])
    err = torch.stack([R.scan(x[b:b + 1].double(), g[b:b + 1].double(), s0[b].double(), complement)[3]
                       for b in range(B)])
    xd, gd, sd = x.to(cuda_dev), g.to(cuda_dev), s0.to(cuda_dev)
    h, S = kb.gated_step(xd, gd, sd, complement=complement)
    assert h.dtype == tx and torch.equal(sd.cpu(), s0)
    close(h, h64, err, "h")
    close(S, h64, err, "S")
    # [B, 1, D], a pool with places in any order, idle rows, in place and not
    gen = torch.Generator().manual_seed(1)
    slots = torch.randperm(B + 3, generator=gen)[:B].int()
    pool = torch.full((B + 3, D), 7.0)
    pool[slots.long()] = s0
    idle = torch.arange(B) % 3 == 2
    slots[idle] = -1 - slots[idle]
    before = pool.to(cuda_dev)
    h2, S2 = kb.gated_step(xd[:, None], gd[:, None], before, slots.to(cuda_dev), complement=complement)
    assert h2.shape == (B, 1, D) and torch.equal(before.cpu(), pool)
    live = ~idle
    assert torch.equal(h2[:, 0].cpu()[live], h.cpu()[live]) and torch.equal(S2.cpu()[live], S.cpu()[live])
    assert (h2[:, 0].cpu()[idle] == 0).all() and (S2.cpu()[idle] == 0).all()
    h3, S3 = kb.gated_step(xd, gd, before, slots.to(cuda_dev), complement=complement, inplace=True)
    assert S3 is before and torch.equal(h3, h2[:, 0])
    want = pool.clone()
    want[slots[live].long()] = S.cpu()[live]
    assert torch.equal(before.cpu(), want)
    h4, S4 = kb.gated_step(xd, gd, complement=complement)
    assert torch.equal(S4, kb.gated_step(xd, gd, torch.zeros_like(sd), complement=complement)[1])


def test_step_strides_and_bad_slots(cuda_dev):
    kb = pkg()
    kb.device_error()
    x, g, s0, _, _ = (t.to(cuda_dev) for t in inputs(6, 20, BF16, BF16, 4, 6, cuda_dev))
    ref = kb.gated_step(x, g, s0)
    wide = torch.zeros(6, 31, device=cuda_dev)
    for off in (0, 1, 4):
        view = wide[:, off:off + 20]
        view.copy_(s0)
        h, S = kb.gated_step(x, g, view)
        assert torch.equal(h, ref[0]) and torch.equal(S, ref[1])
        kb.gated_step(x, g, view, inplace=True)
        assert torch.equal(view, ref[1])
    xt = x.t().contiguous().t()
    assert torch.equal(kb.gated_step(xt, g, s0.t().contiguous().t())[0], ref[0])
    assert torch.equal(kb.gated_step(x[:1].expand(6, 20), g, s0)[1], kb.gated_step(x[:1].repeat(6, 1), g, s0)[1])
    assert kb.device_error() == 0
    slots = torch.tensor([0, 6, 2, 2 ** 31 - 1, 4, 5], dtype=torch.int32, device=cuda_dev)
    h, S = kb.gated_step(x, g, s0, slots)
    live = [0, 2, 4, 5]
    assert torch.equal(h[live], ref[0][live]) and (h[[1, 3]] == 0).all() and (S[[1, 3]] == 0).all()
    assert kb.device_error() == 8 and kb.device_error() == 0
    pool = s0.clone()
    kb.gated_step(x, g, pool, slots, inplace=True)
    assert torch.equal(pool[live], ref[1][live]) and torch.equal(pool[[1, 3]], s0[[1, 3]])
    assert kb.device_error() == 8


def test_steps_continue_a_scan(cuda_dev):
    """A prompt's scan and then single tokens, in a captured step, give the longer scan."""
    kb = pkg()
    B, T, n, D = 3, 70, 9, 48
    x, g, s0, _, _ = inputs(B * (T + n), D, F32, F32, 8, B, cuda_dev)
    want, err = expected(x, g, s0, torch.zeros_like(x), torch.zeros_like(s0),
                         [(b * (T + n), (b + 1) * (T + n)) for b in range(B)], False)
    x, g = (t.view(B, T + n, D).to(cuda_dev) for t in (x, g))
    h, S = kb.gated_scan(x[:, :T], g[:, :T], s0.to(cuda_dev))
    xs, gs, pool = x[:, 0].clone(), g[:, 0].clone(), S.clone()
    kb.gated_step(xs, gs, pool.clone(), inplace=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = kb.gated_step(xs, gs, pool, inplace=True)
    pool.copy_(S)
    hs = [h]
    for t in range(T, T + n):
        xs.copy_(x[:, t])
        gs.copy_(g[:, t])
        graph.replay()
        hs.append(out.clone()[:, None])
    close(torch.cat(hs, 1).reshape(-1, D), want[0], err[0], "h")
    close(pool, want[1], err[1], "S")


def test_empty(cuda_dev):
    kb = pkg()
    z = lambda *s: torch.zeros(*s, device=cuda_dev)  # noqa: E731
    for shape in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        s0 = torch.randn(shape[0], shape[2], device=cuda_dev)
        h, S = kb.gated_scan(z(*shape), z(*shape), s0)
        assert h.shape == shape and torch.equal(S, s0) or shape[1] == 5
        dx, dg, ds = kb.recurrence.gated_scan_backward(z(*shape), z(*shape), s0, z(*shape), s0)
        assert dx.shape == shape and (shape[1] == 5 or torch.equal(ds, s0))
    assert kb.gated_step(z(0, 4), z(0, 4), z(0, 4))[0].shape == (0, 4)
    assert kb.gated_step(z(3, 0), z(3, 0), z(3, 0))[1].shape == (3, 0)


def test_refusals(cuda_dev):
    kb = pkg()
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device=cuda_dev)  # noqa: E731
    x, s = z(2, 5, 4), z(2, 4)
    q = torch.zeros(3, dtype=torch.int32, device=cuda_dev)
    for args, kw, exc in [
            ((x, z(2, 5, 3)), {}, RuntimeError), ((x, x, z(2, 3)), {}, RuntimeError),
            ((x, x, z(3, 4)), {}, RuntimeError), ((z(5, 4), z(5, 4)), {}, RuntimeError),
            ((x, x, s, q), {}, RuntimeError), ((x, z(2, 5, 4, dt=F16)), {}, TypeError),
            ((z(2, 5, 4, dt=F16), z(2, 5, 4, dt=BF16)), {}, TypeError),
            ((z(2, 5, 4, dt=torch.float64), z(2, 5, 4, dt=torch.float64)), {}, TypeError),
            ((z(5, 4), z(5, 4), s, q.long()), {}, RuntimeError), ((z(5, 4), z(5, 4), s, q.cpu()), {}, RuntimeError),
            ((z(5, 4), z(5, 4), s, q[:0]), {}, RuntimeError), ((z(5, 4), z(5, 4), z(3, 4), q), {}, RuntimeError),
            ((x, x.cpu()), {}, RuntimeError), ((x, None), {}, (RuntimeError, AttributeError)),
            ((x.requires_grad_(), z(2, 5, 3)), {}, RuntimeError)]:
        with pytest.raises(exc):
            kb.gated_scan(*args, **kw)
    x = z(2, 4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    for args, kw, exc in [
            ((x, z(2, 3)), {}, RuntimeError), ((x, x, z(3, 4)), {}, RuntimeError),
            ((x, x, z(2, 4, dt=F16)), {}, TypeError), ((x, x, None), dict(inplace=True), RuntimeError),
            ((x, x, None, i32(0, 1)), {}, RuntimeError), ((x, x, z(2, 4), i32(0)), {}, RuntimeError),
            ((x, x, z(2, 4), i32(0, 1).long()), {}, RuntimeError),
            ((x, x, z(1, 4).expand(2, 4)), dict(inplace=True), RuntimeError),
            ((x, x, z(4, 2).t()), dict(inplace=True), RuntimeError),
            ((z(2, 2, 4), z(2, 2, 4), z(2, 4)), {}, RuntimeError),
            ((x.clone().requires_grad_(), x, z(2, 4)), {}, RuntimeError)]:
        with pytest.raises(exc):
            kb.gated_step(*args, **kw)
    with pytest.raises(RuntimeError):
        kb.recurrence.gated_scan_backward(z(2, 5, 4), z(2, 5, 4), None, z(2, 5, 3), None)
    with pytest.raises(RuntimeError):
        kb.recurrence.gated_scan_backward(z(2, 5, 4), z(2, 5, 4), None, None, z(3, 4))
