"""Norm and rotation on the GPU, beyond the ordinary: MLA steps whose rope parts come in other types, and
calls of thousands of tokens."""

from __future__ import annotations

import pytest
import torch

from conftest import pkg
from test_gpu_latent import _module
from test_gpu_recurrence import close
from test_gpu_rotary import freqs, make, oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("tq,tk", [(F32, BF16), (F16, BF16), (BF16, F32), (torch.float64, F32),
                                   (torch.float64, torch.float64)], ids=lambda t: str(t)[6:])
def test_mla_step_rotates_parts_of_two_types(tq, tk, cuda_dev):
    """As the step without frequencies takes them: rotated in fp32 and then cast to the cache's type."""
    kb, dev, dt = pkg(), cuda_dev, BF16
    B, T, H, DN, DV, KVL, DR, hidden = 2, 3, 16, 32, 32, 128, 64, 64
    mod = _module(H, DN, DV, KVL, DR, hidden, dev, dt)
    freq = (10000.0 ** (-torch.arange(0, DR, 2).double() / DR)).float().to(dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    x, qn, ckv = rnd(B, T, hidden).to(dt), rnd(B, T, H, DN).to(dt), rnd(B, T, KVL).to(dt)
    q, k = rnd(B, T, H, DR).to(tq), rnd(B, T, DR).to(tk)

    def state(**kw):
        return {"cache": kb.LatentCache(4, 16, KVL, DR, dtype=dt, device=dev),
                "block_table": torch.arange(4, dtype=torch.int32, device=dev).view(B, 2),
                "lens": torch.zeros(B, dtype=torch.int32, device=dev), **kw}

    with torch.no_grad():
        got = kb.latent.mla_step(mod, x, qn, q, ckv, k, state(inv_freq=freq), False)
        rq, rk = kb.qk_norm_rope(q.float(), k.float()[:, :, None], norm=None, inv_freq=freq)
        want = kb.latent.mla_step(mod, x, qn, rq, ckv, rk[:, :, 0], state(), False)
    assert torch.equal(got, want)


# Long calls: a block goes through several batches of angles, with a remainder, or through several tokens side
# by side.  (B, T, H, HK, D, R, type, weight, norm, interleaved, gap: values between a batch's sequences, so that
# they do not lie one behind the other)
LONG = [
    # three and more batches of 16 tokens a block
    (1, 23501, 16, 16, 128, 128, F16, "head_dim", "rms", False, 0),
    (2, 12007, 16, 16, 128, 128, BF16, "heads", "rms", True, 64),
    (1, 25013, 12, 4, 128, 64, F32, "heads", "l2", False, 0),
    (3, 10007, 1, 1, 256, 256, BF16, "head_dim", "rms", False, 0),
    # one or two
    (1, 7001, 16, 16, 64, 64, F16, "head_dim", "rms", False, 0),
    (1, 6007, 16, 16, 128, 128, BF16, "heads", "rms", True, 0),
    (1, 5003, 16, 16, 64, 32, F32, "head_dim", "l2", True, 0),
    (1, 4999, 12, 4, 128, 64, F32, "heads", "rms", False, 0),
    (3, 2503, 16, 16, 64, 64, BF16, "heads", "rms", False, 0),
    (3, 2503, 16, 16, 64, 64, BF16, "head_dim", "rms", True, 64),
    (2, 3001, 20, 4, 96, 48, F16, None, "l2", False, 48),
    # tokens side by side
    (1, 149, 1, 1, 64, 64, F16, "head_dim", "rms", False, 0),
    (1, 9001, 1, 1, 64, 32, BF16, "head_dim", "rms", False, 0),
    (1, 20011, 1, 1, 32, 32, F32, "heads", "rms", True, 0),
    (5, 1999, 2, 1, 64, 64, F16, "head_dim", "l2", False, 32),
    (4, 3001, 1, 1, 256, 256, BF16, "head_dim", "rms", False, 0),
    (2, 5001, 3, 1, 40, 0, F32, "heads", "rms", False, 0),
    # rows of a warp each
    (1, 6001, 2, 1, 90, 30, BF16, "heads", "rms", False, 0),
    (2, 2503, 3, 1, 33, 16, F32, "head_dim", "l2", True, 33),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_long_calls(cuda_dev, case):
    """Values and gradients of every row, by the bars of the short ones."""
    kb = pkg()
    B, T, H, HK, D, R_, tx, weight, norm, inter, gap = case
    N = B * T
    q, k, dq, dk, ws = make(N, H, HK, D, tx, F32, weight, N + D)
    gen = torch.Generator().manual_seed(2)
    first = torch.randint(0, 100000, (B,), generator=gen)
    pos = (first[:, None] + torch.arange(T)).reshape(-1)
    freq = freqs(R_) if R_ else None
    dev = lambda t: None if t is None else t.to(cuda_dev)  # noqa: E731

    def batch(t):
        """[B, T, H, D] with `gap` values behind each sequence."""
        n = t[0].numel() * T
        wide = torch.full((B, n + gap), float("nan"), dtype=t.dtype, device=cuda_dev)
        view = wide[:, :n].unflatten(1, (T, *t.shape[1:]))
        view.copy_(t.view(B, T, *t.shape[1:]))
        return view

    leaves = [batch(t).requires_grad_() for t in (q, k)] + [dev(w).requires_grad_() for w in ws if w is not None]
    args = leaves if weight else leaves + [None, None]
    kw = dict(norm=norm, eps=1e-5, positions=dev(first), inv_freq=dev(freq), interleaved=inter)
    oq, ok = kb.qk_norm_rope(*args, **kw)
    grads = torch.autograd.grad([oq, ok], leaves, [batch(dq), batch(dk)])
    for i, (x, d, w, o, name) in enumerate(((q, dq, ws[0], oq, "q"), (k, dk, ws[1], ok, "k"))):
        with torch.device(cuda_dev):                   # (the oracle in 64 bits on the GPU)
            want = [[t.cpu() for t in pair] for pair in oracle(dev(x), dev(w), norm, 1e-5, dev(pos), dev(freq), inter, dev(d))]
        close(o.reshape(x.shape), *want[0], name)
        close(grads[i].reshape(x.shape), *want[1], "d" + name)
        if w is not None:
            close(grads[2 + i], *want[2], "dw" + name)
    # the same rows in another cut: each sequence by itself
    with torch.no_grad():
        for b in range(B):
            one = kb.qk_norm_rope(args[0][b:b + 1], args[1][b:b + 1], *args[2:], **{**kw, "positions": dev(first[b:b + 1])})
            assert torch.equal(one[0][0], oq[b]) and torch.equal(one[1][0], ok[b])
