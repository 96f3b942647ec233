"""The gated scan, the norm and rotation of queries and keys, and the operators around them, as
layers use them: sequences with their gradients, the same by single tokens, and MLA steps whose
rope parts are rotated on the way into the cache."""

from __future__ import annotations

import pytest
import torch

from conftest import pkg
from oracle import recurrence_oracle as R
from test_gpu_latent import _module

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rel(a, b):
    b = b.detach()
    return float((a.detach().cpu().double() - b).norm() / b.norm())


def _layer64(x, g, s0, w, gate, beta, angle, H, K):
    """The chain in 64 bits on the CPU, differentiable: h, then KDA of its normalised parts."""
    B, T, D = x.shape
    h, hs = s0, []
    for t in range(T):
        a = torch.exp(g[:, t])
        h = a * h + (1 - a) * x[:, t]
        hs.append(h)
    q, k, v = torch.stack(hs, 1).view(B, T, 3, H, K).unbind(2)
    q = R.qk(q, w, "rms", 1e-6, angle, False)
    k = R.qk(k, None, "l2", 1e-6, angle, False)
    S, out = x.new_zeros(B, H, K, K), []
    for t in range(T):
        S = S * torch.exp(gate[:, t])[..., None]
        u = beta[:, t][..., None] * (v[:, t] - torch.einsum("bhk,bhkv->bhv", k[:, t], S))
        S = S + k[:, t][..., None] * u[..., None, :]
        out.append(torch.einsum("bhkv,bhk->bhv", S, q[:, t]) * K ** -0.5)
    return torch.stack(out, 1), S, h


def test_scan_norm_rotation_and_kda(cuda_dev):
    """Bars: 2e-5 relative for KDA's fp32 values and gradients by themselves; the scan and the
    norm are off by 40 x 2^-24 = 2.4e-6 of their magnitudes at most, which the stages
    between them and the result enlarge less than tenfold (keys of length one, beta below one):
    5e-5 in all."""
    kb = pkg()
    B, T, H, K, bar = 2, 64, 2, 32, 5e-5
    D = 3 * H * K
    gen = torch.Generator().manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, g, s0, w = rnd(B, T, D), -torch.rand(B, T, D, generator=gen), rnd(B, D), 1 + 0.2 * rnd(K)
    gate, beta = -0.1 * torch.rand(B, T, H, K, generator=gen), torch.rand(B, T, H, generator=gen)
    do, first = rnd(B, T, H, K), torch.tensor([0, 1000], dtype=torch.int32)
    freq = (10000.0 ** (-torch.arange(0, K, 2).double() / K)).float()
    pos = first.double()[:, None] + torch.arange(T)
    angle = (pos[..., None] * freq.double())[:, :, None]

    ref = [t.double().requires_grad_() for t in (x, g, s0, w, gate, beta)]
    want, S_want, h_want = _layer64(*ref, angle, H, K)
    want_grads = torch.autograd.grad(want, ref, do.double())

    dev = lambda t: t.to(cuda_dev)  # noqa: E731
    kw = dict(positions=dev(first), inv_freq=dev(freq))
    leaves = [dev(t).requires_grad_() for t in (x, g, s0, w, gate, beta)]
    h, last = kb.gated_scan(leaves[0], leaves[1], leaves[2], complement=True)
    q, k, v = h.view(B, T, 3, H, K).unbind(2)
    q, _ = kb.qk_norm_rope(q, None, leaves[3], **kw)
    k, _ = kb.qk_norm_rope(k, norm="l2", **kw)
    o, S = kb.kda_chunkwise(q, k, v, leaves[4], leaves[5], chunk_size=32)
    grads = torch.autograd.grad(o, leaves, dev(do))
    assert _rel(o, want) < bar and _rel(S, S_want) < bar and _rel(last, h_want) < bar
    for name, a, b in zip(("x", "g", "state", "weight", "gate", "beta"), grads, want_grads):
        assert _rel(a, b) < bar, name

    # the same by single tokens: the scan's states in a pool, both sequences in other rows
    with torch.no_grad():
        pool, slots = torch.full((5, D), float("nan"), device=cuda_dev), dev(torch.tensor([3, 1]).int())
        pool[slots.long()] = leaves[2]
        at, S, outs = dev(first).clone(), None, []
        for t in range(T):
            h1, _ = kb.gated_step(leaves[0][:, t:t + 1], leaves[1][:, t:t + 1], pool, slots, complement=True,
                                  inplace=True)
            q, k, v = h1.view(B, 1, 3, H, K).unbind(2)
            q, _ = kb.qk_norm_rope(q, None, leaves[3], positions=at, inv_freq=kw["inv_freq"])
            k, _ = kb.qk_norm_rope(k, norm="l2", positions=at, inv_freq=kw["inv_freq"])
            o1, S = kb.kda_recurrent(q, k, v, leaves[4][:, t:t + 1], leaves[5][:, t:t + 1], state=S)
            outs.append(o1)
            at += 1
        assert _rel(torch.cat(outs, 1), want) < bar and _rel(S, S_want) < bar
        assert _rel(pool[slots.long()], h_want) < bar
        idle = torch.ones(5, dtype=torch.bool)
        idle[slots.cpu().long()] = False
        assert torch.isnan(pool.cpu()[idle]).all()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_mla_step_rotates(dt, interleaved, cuda_dev):
    """Rope parts given before their rotation: what a caller who rotates them first gets, for a prompt
    and for single tokens in a captured graph, at the positions that the device holds."""
    kb, dev = pkg(), cuda_dev
    B, H, DN, DV, KVL, DR, hidden = 2, 16, 32, 32, 128, 64, 64
    mod = _module(H, DN, DV, KVL, DR, hidden, dev, dt)
    freq = (10000.0 ** (-torch.arange(0, DR, 2).double() / DR)).float().to(dev)
    table = torch.arange(8, dtype=torch.int32, device=dev).view(B, 4)

    def fresh(**kw):
        return {"cache": kb.LatentCache(8, 16, KVL, DR, dtype=dt, device=dev), "block_table": table,
                "lens": torch.tensor([0, 5], dtype=torch.int32, device=dev), **kw}

    def inputs(T, seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=dev).to(dt)  # noqa: E731
        return [torch.zeros(B, T, hidden, device=dev, dtype=dt), r(B, T, H, DN), r(B, T, H, DR),
                r(B, T, KVL), r(B, T, DR)]

    def rotated(args, lens):
        q, k = kb.qk_norm_rope(args[2], args[4][:, :, None], norm=None, positions=lens, inv_freq=freq,
                               interleaved=interleaved)
        return [args[0], args[1], q, args[3], k[:, :, 0]]

    with torch.no_grad():
        got, want = fresh(inv_freq=freq, interleaved=interleaved), fresh()
        # (rows of the pages that no token has reached yet: the other sequence's first five)
        for s in (got, want):
            kb.latent_append(s["cache"], torch.ones(B * 5, KVL, device=dev, dtype=dt), table,
                             torch.full((B,), 5, dtype=torch.int32, device=dev),
                             k_rope=torch.ones(B * 5, DR, device=dev, dtype=dt))
        args = inputs(20, 1)
        a = kb.latent.mla_step(mod, *args, got, False)
        b = kb.latent.mla_step(mod, *rotated(args, want["lens"]), want, False)
        assert torch.equal(a, b) and got["lens"].tolist() == want["lens"].tolist() == [20, 25]
        args = inputs(1, 2)
        warm = dict(got, lens=got["lens"].clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kb.latent.mla_step(mod, *args, warm, False)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kb.latent.mla_step(mod, *args, got, False)
        for step in range(3):
            new = inputs(1, 10 + step)
            for dst, src in zip(args, new):
                dst.copy_(src)
            graph.replay()
            b = kb.latent.mla_step(mod, *rotated(new, want["lens"]), want, False)
            torch.cuda.synchronize()
            assert torch.equal(out, b) and got["lens"].tolist() == want["lens"].tolist()
        del graph
        # a refused rotation leaves the lengths alone
        bad = dict(got, inv_freq=freq.double())
        before = bad["lens"].tolist()
        with pytest.raises(RuntimeError):
            kb.latent.mla_step(mod, *args, bad, False)
        assert bad["lens"].tolist() == before
