"""Gated recurrence on the GPU, beyond the ordinary: states and inputs that are not finite."""

from __future__ import annotations

import pytest
import torch

from conftest import pkg
from oracle import recurrence_oracle as R
from test_gpu_recurrence import BF16, F16, F32, NAMES, close, expected

pytestmark = pytest.mark.gpu

INF = float("inf")


def close_or_same(got, want, bound, what):
    """:func:`close` where the 64-bit value is finite, and elsewhere the same infinity or a NaN."""
    finite = torch.isfinite(want)
    g = got.detach().cpu()
    assert torch.isfinite(bound[finite]).all(), what
    close(g[finite], want[finite], bound[finite], what)
    for name, is_it in (("nan", torch.isnan), ("inf", lambda t: t == INF), ("-inf", lambda t: t == -INF)):
        bad = is_it(g.double()) != is_it(want)
        assert not bad.any(), (what, name, int(bad.sum()), bad.nonzero()[:4].tolist())


def sprinkled(rows, D, tx, tg, seqs, seed):
    """Gates down to -3 a token, some of them zero, and infinities in a tenth of the channels of each of
    inputs, states and output gradients."""
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, s0, dh, dS = rnd(rows, D), rnd(seqs, D), rnd(rows, D), rnd(seqs, D)
    g = -torch.exp(torch.empty(rows, D).uniform_(-6.0, 1.1, generator=gen))
    g[:, ::5] = -3.0                                   # (over 128 tokens: a decay of e^-384)
    g[torch.rand(rows, D, generator=gen) < 0.02] = 0.0
    for t in (x, s0, dh, dS):
        some = torch.rand(D, generator=gen) < 0.1
        at = torch.randint(0, t.shape[0], (D,), generator=gen)[some]
        t[at, some] = INF * (1 - 2 * torch.randint(0, 2, (int(some.sum()),), generator=gen)).float()
    # an infinity that a gate of -inf meets
    if rows > 3:
        x[rows // 3, 1], g[rows // 2, 1] = INF, -INF
        dh[rows // 2, 2], g[rows // 3, 2] = INF, -INF
    return x.to(tx), g.to(tg), s0, dh.to(tx), dS


@pytest.mark.parametrize("complement", [False, True], ids=["plain", "complement"])
@pytest.mark.parametrize("tx,tg", [(F32, F32), (F16, F32), (BF16, BF16)], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("B,T,D", [(1, 1, 64), (2, 5, 40), (1, 131, 37), (2, 700, 64), (1, 2300, 128), (100, 300, 64),
                                   (160, 200, 64), (240, 150, 64)])
def test_infinities(cuda_dev, B, T, D, tx, tg, complement):
    """What 64 bits give: infinities stay until they meet their opposite or a decay of zero."""
    kb = pkg()
    data = sprinkled(T, B * D, tx, tg, 1, T + D)       # the batch's channels side by side
    want, err = expected(*data, [(0, T)], complement)
    split = lambda t: t.view(-1, B, D).transpose(0, 1)  # noqa: E731
    dev = lambda t: split(t).contiguous().to(cuda_dev)  # noqa: E731
    x, g, s0, dh, dS = data
    leaves = [dev(x).requires_grad_(), dev(g).requires_grad_(), dev(s0)[:, 0].contiguous().requires_grad_()]
    h, S = kb.gated_scan(*leaves, complement=complement)
    got = [h, S, *torch.autograd.grad([h, S], leaves, [dev(dh), dev(dS)[:, 0]])]
    for i, (n, v, w, e) in enumerate(zip(NAMES, got, want, err)):
        w, e = split(w), split(e)
        close_or_same(v, w[:, 0] if i in (1, 4) else w, e[:, 0] if i in (1, 4) else e, n)


@pytest.mark.parametrize("tx,tg", [(F32, F32), (F16, F32), (BF16, BF16)], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("N,D,q", [(300, 128, [3, 4, 40, 40, 171, 290]), (2600, 64, [0, 1300, 1301, 2590]),
                                   (3000, 40, list(range(0, 3000, 9))), (200, 9536, [0, 77, 200])],
                         ids=["ragged", "long", "short", "wide"])
def test_infinities_packed(cuda_dev, N, D, q, tx, tg):
    kb = pkg()
    data = sprinkled(N, D, tx, tg, len(q) - 1, N)
    want, err = expected(*data, list(zip(q, q[1:])), D == 40)
    x, g, s0, dh, dS = (t.to(cuda_dev) for t in data)
    starts = torch.tensor(q, dtype=torch.int32, device=cuda_dev)
    got = [*kb.gated_scan(x, g, s0, starts, complement=D == 40),
           *kb.recurrence.gated_scan_backward(x, g, s0, dh, dS, starts, complement=D == 40)]
    for n, v, w, e in zip(NAMES, got, want, err):
        close_or_same(v, w, e, n)


@pytest.mark.parametrize("complement", [False, True], ids=["plain", "complement"])
def test_infinities_step(cuda_dev, complement):
    kb = pkg()
    gs = [0.0, -0.01, -0.5, -3.0, -80.0, -INF]
    xs = [0.0, 1.0, INF, -INF, float("nan")]
    ss = [1.0, INF, -INF, float("nan")]
    grid = torch.cartesian_prod(*(torch.tensor(v) for v in (gs, xs, ss)))
    for D in (len(grid), 1):
        g, x, s = (c.view(-1, D) for c in grid.t())
        want = torch.stack([R.scan(x[b:b + 1].double(), g[b:b + 1].double(), s[b].double(), complement)[1]
                            for b in range(x.shape[0])])
        h, S = kb.gated_step(x.contiguous().to(cuda_dev), g.contiguous().to(cuda_dev), s.contiguous().to(cuda_dev),
                             complement=complement)
        for v in (h, S):
            close_or_same(v, want, torch.full_like(want, 32 * R.U), "step")


def test_weight_of_the_complement(cuda_dev):
    """One token from a state of zero, x = 1: the weight 1 - e^g by itself.  Nearer than 1/2 it is a
    product g (1 + g q): U for the product, U for the sum behind it (it is above 0.78, its half step below
    U), 0.2 U for those further in, 0.12 U for what q leaves out: 2.4 U.  Farther out it is 1 - a: a, from
    an exponent off by 1.5 U |g| and an instruction off by 4 U, is off by (4 + 1.5 |g|) U of itself, and
    the difference rounds once.  In the scan and in the step."""
    kb = pkg()
    gen = torch.Generator().manual_seed(3)
    edges = torch.tensor([0.125, 0.25, 0.5, 1.0, 0.03125])
    g = -torch.cat([torch.exp(torch.empty(20000).uniform_(-9.0, 3.0, generator=gen)),
                    torch.empty(20000).uniform_(0.1, 0.6, generator=gen), edges, edges.nextafter(torch.zeros(5)),
                    edges.nextafter(torch.ones(5))])[None]
    want = -torch.expm1(g.double())
    a = torch.exp(g.double())
    bar = torch.where(g > -0.5, 2.4 * want, (4 - 1.5 * g.double()) * a + want) * R.U
    x, gd = torch.ones_like(g, device=cuda_dev), g.to(cuda_dev)
    outs = [*kb.gated_step(x, gd, complement=True), *kb.gated_scan(x[None], gd[None], complement=True)]
    for got in outs:
        err = (got.view_as(g).cpu().double() - want).abs()
        bad = err > bar
        assert not bad.any(), (int(bad.sum()), float((err / want / R.U)[bad].max()), g[bad][:4])


@pytest.mark.parametrize("complement", [False, True], ids=["plain", "complement"])
@pytest.mark.parametrize("packed", [False, True])
def test_steady_gates_at_the_seams(cuda_dev, packed, complement):
    """Gates that stay on either side of where a decay is held in two parts (a run of four tokens: 1/8)
    and where 1 - a is worked out in another way (1/2), over thousands of tokens; and the same by steps."""
    kb = pkg()
    T = 3000
    at = torch.tensor([1 / 32, 1 / 8, 1 / 2, 0.2499, 0.2501, 0.2])
    g = -torch.cat([at, at.nextafter(torch.zeros(6)), at.nextafter(torch.ones(6)), at * (1 - 1e-3), at * (1 + 1e-3)])
    g = torch.cat([g, torch.tensor([-1e-6, -3e-4])])[None].expand(T, -1).contiguous()
    D = g.shape[1]
    gen = torch.Generator().manual_seed(6)
    x, dh = 1 + 0.1 * torch.randn(T, D, generator=gen), torch.randn(T, D, generator=gen)
    q = [0, 1100, 1131, T] if packed else [0, T]
    s0, dS = torch.randn(len(q) - 1, D, generator=gen), torch.randn(len(q) - 1, D, generator=gen)
    want, err = expected(x, g, s0, dh, dS, list(zip(q, q[1:])), complement)
    dev = lambda t: t.to(cuda_dev)  # noqa: E731
    args = [dev(x), dev(g), dev(s0)] if packed else [dev(x)[None], dev(g)[None], dev(s0)]
    starts = dev(torch.tensor(q, dtype=torch.int32)) if packed else None
    got = [*kb.gated_scan(*args, starts, complement=complement),
           *kb.recurrence.gated_scan_backward(*args, dev(dh).view_as(args[0]), dev(dS), starts, complement=complement)]
    for n, v, w, e in zip(NAMES, got, want, err):
        close(v.view_as(w), w, e, n)
    if not packed:
        state = dev(s0).clone()
        for t in range(300):
            h, _ = kb.gated_step(args[0][:, t], args[1][:, t], state, complement=complement, inplace=True)
        close(state, want[0][299:300], err[0][299:300], "steps")


@pytest.mark.parametrize("packed", [False, True])
def test_state_of_64_bits(cuda_dev, packed):
    """Read as fp32, its gradient in its own type."""
    kb = pkg()
    gen = torch.Generator().manual_seed(2)
    x, g = torch.randn(2, 50, 24, generator=gen), -torch.rand(2, 50, 24, generator=gen)
    x, g, s0 = x.to(cuda_dev), g.to(cuda_dev), torch.randn(2, 24, generator=gen, dtype=torch.float64).to(cuda_dev)
    q = torch.tensor([0, 50, 100], dtype=torch.int32, device=cuda_dev) if packed else None
    if packed:
        x, g = x.view(100, 24), g.view(100, 24)
    want = kb.gated_scan(x, g, s0.float(), q)
    assert all(torch.equal(a, b) for a, b in zip(kb.gated_scan(x, g, s0, q), want))
    ones = [torch.ones_like(t) for t in want]
    ref = kb.recurrence.gated_scan_backward(x, g, s0.float(), *ones, q)
    got = kb.recurrence.gated_scan_backward(x, g, s0, *ones, q)
    leaf = s0.clone().requires_grad_()
    auto, = torch.autograd.grad(kb.gated_scan(x, g, leaf, q), leaf, ones)
    assert got[2].dtype == auto.dtype == torch.float64
    assert all(torch.equal(a, b.to(a.dtype)) for a, b in zip((*got, auto), (*ref, ref[2])))
    with pytest.raises(TypeError):
        kb.gated_scan(x, g, s0.long(), q)


def test_step_in_place_is_seen_by_autograd(cuda_dev):
    """A scan's backward pass reads its initial states: written over by a step, it refuses as for any other
    operation in place; a step that writes elsewhere leaves it alone."""
    kb = pkg()
    gen = torch.Generator(device=cuda_dev).manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=cuda_dev)  # noqa: E731
    x, g, pool = rnd(60, 16).requires_grad_(), -rnd(60, 16).abs(), rnd(3, 16)
    q = torch.tensor([0, 20, 20, 60], dtype=torch.int32, device=cuda_dev)
    for inplace in (False, True):
        h, _ = kb.gated_scan(x, g, pool, q)
        with torch.no_grad():
            before = pool._version
            _, S = kb.gated_step(x[:3], g[:3], pool, inplace=inplace)
        assert (pool._version > before) == inplace and (S is pool) == inplace
        if inplace:
            with pytest.raises(RuntimeError, match="inplace"):
                h.sum().backward()
        else:
            h.sum().backward()
    with torch.inference_mode():
        held = rnd(3, 16)
        kb.gated_step(x[:3], g[:3], held, inplace=True)


@pytest.mark.parametrize("tx", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("B,T,D,seqs", [(1, 3000, 128, 0), (2, 700, 64, 0), (100, 700, 64, 0), (160, 300, 64, 0),
                                        (240, 300, 64, 0), (1, 2600, 64, 7), (1, 1000, 37, 0)])
def test_waits_that_give_up(cuda_dev, monkeypatch, B, T, D, seqs, tx):
    """Told not to wait, the kernels give up: the calls return, the error word says so, and the next calls
    give what they gave before."""
    kb = pkg()
    kb.device_error()
    gen = torch.Generator(device=cuda_dev).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=cuda_dev)  # noqa: E731
    rows = (T, D) if seqs else (B, T, D)
    x, g, dh = rnd(rows).to(tx), -rnd(rows).abs(), rnd(rows).to(tx)
    s0, dS = rnd(seqs or B, D), rnd(seqs or B, D)
    q = torch.linspace(0, T, seqs + 1).int().to(cuda_dev) if seqs else None

    def both():
        leaves = [t.clone().requires_grad_() for t in (x, g, s0)]
        h, S = kb.gated_scan(*leaves, q)
        return [h, S, *torch.autograd.grad([h, S], leaves, [dh, dS])]

    want, plain = both(), kb.recurrence._args

    def hasty(*a, **kw):
        out = plain(*a, **kw)
        out.hasty = 1
        return out

    monkeypatch.setattr(kb.recurrence, "_args", hasty)
    for call in (lambda: kb.gated_scan(x, g, s0, q),
                 lambda: kb.recurrence._backward(x, g, s0, q, False, rnd(2 * B * T * D), dh, dS, (True,) * 3)):
        call()
        assert kb.device_error() == 9
    monkeypatch.setattr(kb.recurrence, "_args", plain)
    assert all(torch.equal(a, b) for a, b in zip(both(), want))
    assert kb.device_error() == 0


@pytest.mark.parametrize("tx,tg", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("complement", [False, True], ids=["plain", "complement"])
@pytest.mark.parametrize("B,T,D,packed", [(1, 8 * 128 * 5 + 37, 64, False), (1, 4500, 2048, False), (40, 900, 128, False),
                                          (100, 1021, 64, False), (1, 8 * 128 * 5 + 37, 72, True)])
def test_long_shape_past_its_ring(cuda_dev, B, T, D, packed, complement, tx, tg):
    """Sequences of 16 bits that a block goes through in more turns than it has rows in shared memory for: in
    clusters of eight, four, one; rows by TMA, and 64 channels with a rest of eight.  (Subsets of the channels go
    to the oracle: they do not meet.)"""
    kb = pkg()
    # (a few channels at the edges and in between)
    some = sorted({0, 1, 31, 63, D - 1, D // 2, 64 % D, 65 % D})
    gen = torch.Generator(device=cuda_dev).manual_seed(T + D)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=cuda_dev)  # noqa: E731
    x, dh = rnd(B, T, D).to(tx), rnd(B, T, D).to(tx)
    g = (-torch.exp(torch.empty(B, T, D, device=cuda_dev).uniform_(-9.0, 1.5, generator=gen))).to(tg)
    s0, dS = rnd(B, D), rnd(B, D)
    cuts = [3, 700, 700, 3000, T - 11] if packed else None
    if packed:
        s0, dS = rnd(4, D), rnd(4, D)
    rows = (T, D) if packed else (B, T, D)
    starts = torch.tensor(cuts, dtype=torch.int32, device=cuda_dev) if packed else None
    leaves = [x.view(rows).requires_grad_(), g.view(rows).requires_grad_(), s0.requires_grad_()]
    h, S = kb.gated_scan(*leaves, starts, complement=complement)
    got = [h, S, *torch.autograd.grad([h, S], leaves, [dh.view(rows), dS])]
    for b in ([0] if packed else sorted({0, B // 2, B - 1})):
        pick = lambda t: t.detach().cpu()[..., some]  # noqa: E731
        seq = lambda t: pick(t.view(B, T, D)[b])  # noqa: E731
        st = (lambda t: pick(t)) if packed else (lambda t: pick(t[b:b + 1]))  # noqa: E731
        want, err = expected(seq(x), seq(g), st(s0), seq(dh), st(dS), list(zip(cuts, cuts[1:])) if packed else [(0, T)],
                             complement)
        for i, (n, v, w, e) in enumerate(zip(NAMES, got, want, err)):
            close(st(v) if i in (1, 4) else seq(v), w, e, n)


def test_empty_calls(cuda_dev):
    """Shapes, and states that go through, one by one."""
    kb = pkg()
    for B, T, D in ((0, 5, 4), (2, 0, 4), (2, 5, 0), (0, 0, 4), (2, 0, 0)):
        x, s0 = torch.zeros(B, T, D, device=cuda_dev), torch.randn(B, D, device=cuda_dev)
        h, S = kb.gated_scan(x, x, s0)
        assert h.shape == (B, T, D)
        assert S.shape == (B, D)
        dx, dg, ds = kb.recurrence.gated_scan_backward(x, x, s0, x, s0)
        assert dx.shape == dg.shape == (B, T, D)
        assert ds.shape == (B, D)
        if T == 0:
            assert torch.equal(S, s0)
            assert torch.equal(ds, s0)
        assert all(t.numel() == 0 for t in (h, dx, dg))


def test_refusals_without_a_gradient(cuda_dev):
    """The same refusals on the way that records nothing, and on the one that does."""
    kb = pkg()
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device=cuda_dev)  # noqa: E731
    x, s, q = z(2, 5, 4), z(2, 4), torch.zeros(3, dtype=torch.int32, device=cuda_dev)
    cases = [((x, z(2, 5, 3)), RuntimeError), ((x, x, z(2, 3)), RuntimeError), ((x, x, z(3, 4)), RuntimeError),
             ((z(5, 4), z(5, 4)), RuntimeError), ((x, x, s, q), RuntimeError), ((x, z(2, 5, 4, dt=F16)), TypeError),
             ((z(5, 4), z(5, 4), s, q.long()), RuntimeError), ((z(5, 4), z(5, 4), s, q.cpu()), RuntimeError),
             ((x, x.cpu()), RuntimeError), ((x, x, s.cpu()), RuntimeError)]
    for args, exc in cases:
        assert not any(t.requires_grad for t in args)
        with pytest.raises(exc):
            kb.gated_scan(*args)
        with pytest.raises(exc):
            kb.gated_scan(args[0].clone().requires_grad_(), *args[1:])
