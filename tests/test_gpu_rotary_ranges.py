"""Norm and rotation on the GPU, beyond the ordinary: MLA steps whose rope parts come in other types."""

from __future__ import annotations

import pytest
import torch

from conftest import pkg
from test_gpu_latent import _module

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
