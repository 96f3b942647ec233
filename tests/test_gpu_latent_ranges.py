"""GPU tests of the latent attention over long ranges: many tiles for one block at
every width, and weights far below the largest.  Bars as in ``test_gpu_latent.py``
where nothing else is said."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import pkg
from oracle import latent_oracle as lo
from test_gpu_latent import BF16, F16, attend, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("KVL,DR,n,page,dt", [
    (128, 0, 1, 128, BF16),
    (128, 0, 1, 256, F16),
    (128, 64, 2, 128, BF16),
    (256, 0, 1, 128, BF16),
    (256, 64, 1, 128, BF16),
    (256, 0, 2, 1024, F16),
    (384, 0, 1, 128, BF16),
    (384, 64, 1, 128, F16),
    (384, 0, 2, 128, BF16),          # three tiles and a third: as many in the making
    (384, 0, 1, 128, F16),
    (256, 64, 2, 128, BF16),
    (256, 64, 2, 128, F16),
])
def test_rings_of_more_than_three_tiles(KVL, DR, n, page, dt, cuda_dev):
    """Narrow latents, whose ring holds more than three tiles: some ten tiles a block, read from
    memory, so that a fifth tile's turn comes while the first may be on its way."""
    lens = [16001 - 7 * i for i in range(12)]
    m = make(lens, [n] * len(lens), KVL=KVL, DR=DR, page=page, dt=dt, seed=KVL + DR + n)
    flush = torch.empty(1 << 27, device=m.dev)
    for _ in range(3):
        flush.fill_(1.0)                          # 512 MB: the cache leaves L2
        out, lse = attend(m)
    check(m, out, lse)


@pytest.mark.parametrize("n", [1, 2])                 # 16 and 32 rows a group
@pytest.mark.parametrize("share", [0.5, 0.9, 0.97])
def test_a_heavy_token_over_a_long_context(share, n, cuda_dev):
    """The first token holds `share` of the weight, 32767 others the rest, each 2^-15 to
    2^-20 of it and nearly the same, and one block has all of them: 148 sequences that
    share one context.  Outside channel 0 the output is the crowd's alone.

    Bar: the output's rounding 2^-11 |out|, and of sum w|c|: 2^-11 for weights rounded to 11
    bits, 2^-12 for sums (1024 additions into an fp32 accumulator, cut at 2^-23: 2^-13) and
    scores of magnitude 20 in fp32 (2^-18).  A weight below the 11 bits' range is off by
    2^-34 of the largest, 2^-19 for all of them together."""
    L, H, KVL = 32768, 16, 128
    m = make([L], [n], H=H, KVL=KVL, page=128, dt=F16, seed=17 + n, q_gain=0.01)
    slot = (m.table[0].long().cpu()[torch.arange(L) // 128] * 128 + torch.arange(L) % 128)
    g = torch.Generator().manual_seed(3)
    c = torch.randn(L, KVL, generator=g) + 0.5
    c[:, 0] = 0.0
    c[0] = 0.0
    c[0, 0] = 24.0
    s = torch.exp2(torch.ceil(torch.log2(c.abs().amax(-1) / 448.0)))
    q8 = (c / s[:, None]).to(torch.float8_e4m3fn)
    m.cache.codes.view(torch.uint8).view(-1, KVL)[slot.to(m.dev)] = q8.view(torch.uint8).to(m.dev)
    m.cache.scales.view(-1)[slot.to(m.dev)] = s.to(m.dev)
    m.c = [q8.double() * s[:, None].double()]
    m.q[..., 0] = math.log(L * share / (1 - share)) / (m.scale * 24.0)
    want, wlse, mag = lo.attention(m.q, None, m.c, None, [n], [L], m.scale)
    B = 148
    out, lse = pkg().latent_attention(
        m.q.to(m.dev).repeat(B, 1, 1), m.cache, m.table.expand(B, -1).contiguous(),
        m.lens.expand(B).contiguous(), m.scale, return_lse=True)
    bar = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mag + 2.0 ** -19 * 24.0 * 2.0 ** -5
    err = (out.double().cpu().view(B, n, H, KVL) - want).abs()
    assert float((err / bar).max()) <= 1.0, float((err / bar).max())
    tol = 2.0 ** -24 * 576 * 20 + 2.0 ** -20 * (1 + wlse.abs())
    assert bool(((lse.double().cpu().view(B, n, H) - wlse).abs() <= tol).all())
    assert pkg().device_error() == 0
