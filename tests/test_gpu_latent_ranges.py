"""GPU tests of the latent attention over long ranges: many tiles for one block at
every width, and weights far below the largest.  Bars as in ``test_gpu_latent.py``
where nothing else is said."""

from __future__ import annotations

import pytest
import torch

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
