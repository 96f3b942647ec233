"""GPU tests of the latent attention over long ranges: many tiles for one block at
every width, and weights far below the largest.  Bars as in ``test_gpu_latent.py``
where nothing else is said."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import pkg
from oracle import latent_oracle as lo
from test_gpu_latent import BF16, F16, _module, attend, check, make

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


def _dirty(dev):
    """What the allocator hands out next reads as NaN."""
    blocks = [torch.full((size,), math.nan, device=dev) for size in [1 << k for k in range(7, 20)] * 3]
    del blocks


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lens,counts", [([700, 90], [1, 1]), ([130, 5, 700], [9, 5, 40])])
def test_rows_of_no_sequence(lens, counts, dt, cuda_dev):
    """Rows before q_start[0] and from q_start[B] on: zeros and -inf from attention, zeros
    from read, skipped by append; the others as without them."""
    kb = pkg()
    m = make(lens, counts, H=5, KVL=128, DR=64, page=64, dt=dt, seed=len(lens))
    N, before, after = sum(counts), 3, 150
    want, wl = attend(m)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(before + N + after, 5, 128, generator=g).to(dt).to(m.dev)
    qr = torch.randn(before + N + after, 5, 64, generator=g).to(dt).to(m.dev)
    q[before:before + N], qr[before:before + N] = m.q.to(m.dev), m.qr.to(m.dev)
    q_start = m.q_start + before
    own = torch.zeros(before + N + after, dtype=torch.bool, device=m.dev)
    own[before:before + N] = True
    for wide in (m.table, torch.cat([m.table] * 20, 1)):        # whole contexts, and split ones
        _dirty(m.dev)
        out, lse = kb.latent_attention(q, m.cache, wide.contiguous(), m.lens, m.scale, q_start=q_start,
                                       q_rope=qr, return_lse=True)
        assert bool((out[~own] == 0).all()) and bool(torch.isneginf(lse[~own]).all())
        assert torch.equal(torch.isneginf(lse[own]), torch.isneginf(wl))
        assert float((out[own].float() - want.float()).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
    c0, _ = kb.latent_read(m.cache, m.table, m.lens, N, q_start=m.q_start)
    _dirty(m.dev)
    c, k = kb.latent_read(m.cache, m.table, m.lens, before + N + after, q_start=q_start)
    assert torch.equal(c[own], c0) and bool((c[~own] == 0).all()) and bool((k[~own] == 0).all())
    codes = m.cache.codes.view(torch.uint8).clone()
    slots = [w[2] for w in lo.slots(m.table.cpu(), lens, counts, 64) if w[2] is not None]
    kb.latent_append(m.cache, q[:, 0].contiguous(), m.table, m.lens, q_start=q_start,
                     k_rope=qr[:, 0].contiguous())
    same = (codes == m.cache.codes.view(torch.uint8)).all(-1).view(-1).cpu()
    same[slots] = True
    assert bool(same.all())
    assert kb.device_error() == 0


def test_no_sequence_at_all(cuda_dev):
    """B = 0 with a q_start of one entry."""
    kb = pkg()
    cache = kb.LatentCache(2, 16, 128, device=cuda_dev)
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    table, lens, q_start = torch.zeros(0, 1, **i32), torch.zeros(0, **i32), torch.zeros(1, **i32)
    x = torch.ones(7, 4, 128, dtype=BF16, device=cuda_dev)
    for t in (table, torch.zeros(0, 4096, **i32)):
        _dirty(cuda_dev)
        out, lse = kb.latent_attention(x, cache, t, lens, 1.0, q_start=q_start, return_lse=True)
        c, _ = kb.latent_read(cache, t, lens, 7, q_start=q_start)
        assert bool((out == 0).all()) and bool(torch.isneginf(lse).all()) and bool((c == 0).all())
    before = cache.codes.view(torch.uint8).clone()
    kb.latent_append(cache, x[:, 0].contiguous(), table, lens, q_start=q_start)
    assert torch.equal(before, cache.codes.view(torch.uint8)) and kb.device_error() == 0


def test_a_padded_batch_in_a_graph(cuda_dev):
    """One captured call of eight rows, replayed with fewer and fewer of them owned."""
    kb = pkg()
    m = make([900, 333], [4, 4], H=16, KVL=128, page=64, seed=5)
    q, q_start = m.q.to(m.dev), m.q_start.clone()
    args = (q, m.cache, m.table, m.lens, m.scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kb.latent_attention(*args, q_start=q_start, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = kb.latent_attention(*args, q_start=q_start, return_lse=True)
    for starts in ([0, 4, 8], [0, 4, 5], [0, 1, 2], [2, 4, 4], [0, 0, 0]):
        q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(math.nan)
        lse.fill_(math.nan)
        graph.replay()
        want, wl = kb.latent_attention(*args, q_start=q_start, return_lse=True)
        own = torch.zeros(8, dtype=torch.bool)
        own[starts[0]:starts[2]] = True
        assert torch.equal(out, want) and torch.equal(lse, wl)
        assert bool((out[~own] == 0).all()) and bool(torch.isneginf(lse[~own]).all())
        assert bool(torch.isfinite(lse[own]).all())
    del graph


@pytest.mark.parametrize("spoil", ["grad", "heads", "table"])
def test_a_refused_layer_step_changes_nothing(spoil, cuda_dev):
    """A step that is refused, before or after its tokens were written, leaves the lengths;
    the next one gives what it would have given without it."""
    kb, dev = pkg(), cuda_dev
    mod = _module(4, 16, 16, 128, 0, 32, dev, BF16)
    cache = kb.LatentCache(4, 16, 128, device=dev)
    state = {"cache": cache, "block_table": torch.arange(4, dtype=torch.int32, device=dev).view(2, 2),
             "lens": torch.zeros(2, dtype=torch.int32, device=dev)}
    g = torch.Generator(device=dev).manual_seed(2)
    x, q, c = (torch.randn(*s, generator=g, device=dev).to(BF16)
               for s in ((2, 3, 32), (2, 3, 4, 16), (2, 3, 128)))
    with torch.no_grad():
        want = kb.latent.mla_step(mod, x, q, None, c, None, dict(state, lens=state["lens"].clone()), False)
    bad = dict(state)
    args = [mod, x, q, None, c, None]
    if spoil == "grad":
        args[4] = c.clone().requires_grad_(True)
    elif spoil == "heads":
        args[2] = torch.cat([q, q], 2)                # found after the tokens are written
    else:
        bad["block_table"] = state["block_table"][:1]
    with pytest.raises(RuntimeError):
        with torch.set_grad_enabled(spoil == "grad"):
            kb.latent.mla_step(*args, bad, True)
    assert state["lens"].tolist() == [0, 0]
    with torch.no_grad():
        out = kb.latent.mla_step(mod, x, q, None, c, None, state, False)
    assert torch.equal(out, want) and state["lens"].tolist() == [3, 3]


@pytest.mark.parametrize("lens", [[40], [4000]])
def test_scores_far_below_zero(lens, cuda_dev):
    """Scores of -1e31 and less: a row has seen something, however low its maximum."""
    m = make(lens, [1], H=3, KVL=128, dt=BF16, seed=23)
    L = lens[0]
    slot = (m.table[0].long().cpu()[torch.arange(L) // 64] * 64 + torch.arange(L) % 64)
    c = torch.zeros(L, 128)
    c[:, 0] = 2.0 ** 41
    c[L // 2, 0] = 2.0 ** 40                          # the least low: all of the weight
    c[:, 1] = torch.arange(L) % 15 * 2.0 ** 38
    s = 2.0 ** 33
    m.cache.codes.view(torch.uint8).view(-1, 128)[slot.to(m.dev)] = \
        (c / s).to(torch.float8_e4m3fn).view(torch.uint8).to(m.dev)
    m.cache.scales.view(-1)[slot.to(m.dev)] = s
    m.c = [c.double()]
    m.q.zero_()
    m.q[..., 0] = -2.0 ** 68
    out, lse = attend(m)
    assert bool((lse < -1e30).all()) and bool(torch.isfinite(lse).all())
    check(m, out, lse)
