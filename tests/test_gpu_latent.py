"""GPU tests of the 8-bit paged latent cache and its attention (``latent.py``)
against the float64 oracle.

Bars, from the formats' roundings (u = 2^-9 for a bf16 output, 2^-11 for fp16):

* append and read are exact: the scale is a power of two, so a code is one
  rounding of an exact quotient, and a value read back is one rounding of an
  exact product;
* attention, per element: |err| <= u |out| (the output's rounding) + eps sum w|c|
  + 2^-16 max|c|, eps = 2^-8 (bf16) / 2^-12 (fp16): the softmax's weights may be
  off by a relative eps each, and tiny ones by a step of 2^-16 of the largest
  one's in all;
* lse: fp32 scores of at most 576 products, so |err| <= 2^-24 * 576 * the largest
  score's sum of magnitudes + 2^-20 (1 + |lse|) for exponentials and sums.
"""

from __future__ import annotations

import math
import types

import pytest
import torch

from conftest import pkg
from oracle import latent_oracle as lo

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(lens, counts, H=16, KVL=512, DR=0, page=64, dt=BF16, seed=0, dev="cuda", q_gain=0.6,
         spare=2):
    """A cache that holds the sequences (written by the oracle's rounding), its
    unwritten slots NaN, and queries for the new tokens."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    need = [-(-max(0, x) // page) for x in lens]
    width = max(1, max(need, default=1))
    P = sum(need) + spare
    perm = torch.randperm(P, generator=g).int()
    table = torch.empty(B, width, dtype=torch.int32)
    for b in range(B):
        own = perm[sum(need[:b]):sum(need[:b]) + need[b]]
        table[b] = torch.cat([own, torch.full((width - need[b],), int(perm[-1]), dtype=torch.int32)])
    codes = torch.full((P * page, KVL), 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.full((P * page,), math.nan)
    rope = torch.full((P * page, DR), math.nan, dtype=dt) if DR else None
    cs, ks = [], []
    gain = torch.exp(0.4 * torch.randn(KVL, generator=g))
    for b in range(B):
        L = max(0, lens[b])
        c = torch.randn(L, KVL, generator=g) * gain
        e = torch.ceil(torch.log2(c.abs().amax(-1) / 448.0)) if L else torch.zeros(0)
        s = torch.exp2(e)
        at = torch.arange(L)
        slot = table[b].long()[at // page] * page + at % page
        q8 = (c / s[:, None]).to(torch.float8_e4m3fn)
        codes.view(torch.uint8)[slot] = q8.view(torch.uint8)
        scales[slot] = s
        cs.append(q8.double() * s[:, None].double())
        if DR:
            r = (torch.randn(L, DR, generator=g) / s[:, None]).to(dt)
            rope[slot] = r
            ks.append(r.double() * s[:, None].double())
    N = sum(counts)
    q = (torch.randn(N, H, KVL, generator=g) * q_gain * (512 / KVL) ** 0.5).to(dt)
    qr = torch.randn(N, H, DR, generator=g).to(dt) if DR else None
    starts = torch.tensor([sum(counts[:b]) for b in range(B + 1)], dtype=torch.int32)
    cache = pkg().LatentCache.from_tensors(
        codes.view(P, page, KVL).to(dev), scales.view(P, page).to(dev),
        None if rope is None else rope.view(P, page, DR).to(dev), dtype=dt)
    return types.SimpleNamespace(
        cache=cache, table=table.to(dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
        q_start=starts.to(dev), q=q, qr=qr, c=cs, k=ks if DR else None, counts=list(counts),
        L=list(lens), dt=dt, scale=(128 + DR) ** -0.5, dev=dev)


def attend(m, q=None, qr=None, q_start=True, scale=None):
    q = m.q.to(m.dev) if q is None else q
    if m.qr is not None and qr is None:
        qr = m.qr.to(m.dev)
    return pkg().latent_attention(q, m.cache, m.table, m.lens, m.scale if scale is None else scale,
                                  q_start=m.q_start if q_start else None, q_rope=qr,
                                  return_lse=True)


def check(m, out, lse, scale=None):
    scale = m.scale if scale is None else scale
    want, wlse, mag = lo.attention(m.q, m.qr, m.c, m.k, m.counts, m.L, scale)
    assert out.dtype == m.dt and tuple(out.shape) == tuple(m.q.shape)
    out, lse = out.double().cpu(), lse.double().cpu()
    u, eps = (2.0 ** -9, 2.0 ** -8) if m.dt is BF16 else (2.0 ** -11, 2.0 ** -12)
    cmax = max([float(c.abs().max()) for c in m.c if c.numel()] + [0.0])
    bar = u * want.abs() + eps * mag + 2.0 ** -16 * cmax + 2.0 ** -24
    # past the type's range the output is an infinity of the same sign
    top = torch.finfo(m.dt).max
    over = torch.isinf(out) & (want.abs() + bar > top) & (out.sign() == want.sign())
    out = torch.where(over, want, out)
    worst = ((out - want).abs() / bar).max().item() if out.numel() else 0.0
    assert worst <= 1.0, f"out: {worst:.3f} of the bar"
    empty = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    assert float(out[empty].abs().sum()) == 0.0
    if (~empty).any():
        qa, ca = m.q.double().abs(), cmax
        mags = abs(scale) * (qa.sum(-1) * ca + (0 if m.qr is None else m.qr.double().abs().sum(-1)
                                                * max(float(k.abs().max()) for k in m.k if k.numel())))
        tol = 2.0 ** -24 * 576 * mags + 2.0 ** -20 * (1 + wlse.abs())
        assert bool(((lse - wlse).abs() <= tol)[~empty].all()), (lse - wlse)[~empty].abs().max()
    assert pkg().device_error() == 0


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [127], [128], [129], [255, 256, 257],
                                  [1000, 1, 63, 640], [0, 5, 0, 300], [0, 0]])
def test_single_token_lengths(lens, dt, cuda_dev):
    m = make(lens, [1] * len(lens), dt=dt, seed=sum(lens))
    check(m, *attend(m, q_start=False))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("KVL,DR", [(128, 0), (256, 64), (384, 0), (384, 64), (512, 0), (512, 64)])
def test_pages_and_widths(page, KVL, DR, cuda_dev):
    m = make([150, 700, 31], [1, 1, 1], KVL=KVL, DR=DR, page=page, dt=F16 if DR else BF16, seed=page)
    check(m, *attend(m))


@pytest.mark.parametrize("H", [1, 3, 8, 16, 17, 32, 40, 64, 128])
@pytest.mark.parametrize("n", [1, 3])
def test_heads(H, n, cuda_dev):
    m = make([333, 64], [n, n], H=H, KVL=256, dt=BF16 if H % 2 else F16, seed=H)
    check(m, *attend(m))


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("DR", [0, 64])
@pytest.mark.parametrize("lens,counts", [
    ([40, 40], [40, 40]),                    # whole prompts: causal from the first position
    ([300], [130]),                          # a chunk on top of a context
    ([129, 5, 260, 0, 64], [4, 5, 1, 0, 33]),  # ragged, a sequence with nothing new
    ([3, 10], [5, 2]),                       # more new tokens than the sequence holds: empty rows
    ([0, 7], [3, 7]),                        # an idle slot's rows are empty
    ([256], [256]),
])
def test_many_tokens_causal(lens, counts, DR, dt, cuda_dev):
    m = make(lens, counts, DR=DR, page=32, dt=dt, seed=len(counts) + DR)
    check(m, *attend(m))


def test_long_context_is_split_and_joined(cuda_dev):
    """Far more tiles than one block takes: the parts join to the same result."""
    for lens, H, dt in (([20001], 16, BF16), ([9000, 1, 4097], 5, F16)):
        m = make(lens, [1] * len(lens), H=H, KVL=128, page=128, dt=dt, seed=H)
        check(m, *attend(m))


def test_many_sequences(cuda_dev):
    lens = [(37 * i) % 211 for i in range(300)]
    m = make(lens, [1] * 300, H=4, KVL=128, page=16, seed=4)
    check(m, *attend(m))


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_scales(scale, cuda_dev):
    """Zero scale: the mean of the latents; a large one: one token takes all."""
    m = make([400], [2], dt=F16, seed=7)
    out, lse = attend(m, scale=scale)
    check(m, out, lse, scale=scale)


def test_growing_scores(cuda_dev):
    """Every later position outweighs all before it: the running maximum moves all the way."""
    m = make([700], [1], dt=F16, KVL=128, seed=8)
    u = m.q[0, 0].double()
    c = m.c[0]
    ramp = torch.linspace(-40, 40, 700, dtype=torch.float64)[:, None] * u / (u @ u) / m.scale
    codes = m.cache.codes.view(-1, 128)
    slot = (m.table[0].long().cpu()[torch.arange(700) // 64] * 64 + torch.arange(700) % 64)
    s = torch.exp2(torch.ceil(torch.log2(ramp.abs().amax(-1).clamp(min=1e-6) / 448)))
    q8 = (ramp / s[:, None]).float().to(torch.float8_e4m3fn)
    codes.view(torch.uint8)[slot.to(m.dev)] = q8.view(torch.uint8).to(m.dev)
    m.cache.scales.view(-1)[slot.to(m.dev)] = s.float().to(m.dev)
    c.copy_(q8.double() * s[:, None])
    check(m, *attend(m))


def test_a_heavy_token_and_a_light_crowd(cuda_dev):
    """One token holds half of the weight, thousands share the rest."""
    m = make([6000], [1], H=2, KVL=128, dt=BF16, seed=9, q_gain=0.02)
    m.q[:, :, 0] = 4.0
    slot = int(m.table[0, 0]) * 64
    c0 = torch.zeros(128)
    c0[0] = 24.0                                     # score 24 * 4 * 128^-0.5 = 8.5 = ln 5000
    m.cache.codes.view(-1, 128)[slot] = (c0 / 0.0625).to(torch.float8_e4m3fn).to(m.dev)
    m.cache.scales.view(-1)[slot] = 0.0625
    m.c[0][0] = c0.double()
    m.c[0][1:, 0] = 0.0
    at = torch.arange(1, 6000)
    rest = m.table[0].long().cpu()[at // 64] * 64 + at % 64
    m.cache.codes.view(torch.uint8).view(-1, 128)[rest.to(m.dev), 0] = 0
    check(m, *attend(m))


def test_tokens_of_very_different_scale(cuda_dev):
    """Scales from 2^-100 (a zero latent) to 2^60 within one sequence."""
    m = make([300], [1], KVL=128, dt=BF16, seed=10)
    at = torch.arange(300)
    slot = (m.table[0].long().cpu()[at // 64] * 64 + at % 64).to(m.dev)
    s = m.cache.scales.view(-1)
    codes = m.cache.codes.view(torch.uint8).view(-1, 128)
    codes[slot[::3]] = 0                             # zero latents,
    s[slot[::3]] = 2.0 ** -100                       # as append would write them
    m.c[0][::3] = 0.0
    s[slot[1::3]] *= 2.0 ** -40
    m.c[0][1::3] *= 2.0 ** -40
    check(m, *attend(m))
    only = make([40], [1], KVL=128, dt=BF16, seed=11)   # nothing but zero latents
    only.cache.codes.view(torch.uint8).zero_()
    only.cache.scales.fill_(2.0 ** -100)
    only.c[0].zero_()
    check(only, *attend(only))
    assert float(attend(only)[0].abs().sum()) == 0.0


def test_masked_places_may_hold_anything(cuda_dev):
    """NaN codes and scales past a sequence's end, and in pages it does not own,
    reach nothing; a NaN token reaches the rows that see it and no others."""
    m = make([100, 190], [3, 2], DR=64, page=64, dt=F16, seed=12)
    out, lse = attend(m)
    check(m, out, lse)                               # make() leaves unwritten slots NaN
    at = 98                                          # seen by the last two of three new tokens
    slot = int(m.table[0, at // 64]) * 64 + at % 64
    m.cache.scales.view(-1)[slot] = math.nan
    out2, lse2 = attend(m)
    assert bool(torch.isnan(out2[1:3]).all()) and bool(torch.isnan(lse2[1:3]).all())
    assert torch.equal(out2[0], out[0]) and torch.equal(out2[3:], out[3:])
    assert torch.equal(lse2[0], lse[0]) and torch.equal(lse2[3:], lse[3:])


def test_non_finite_queries(cuda_dev):
    m = make([70, 70], [1, 1], H=3, KVL=128, dt=BF16, seed=13)
    good, _ = attend(m)
    q = m.q.to(m.dev).clone()
    q[0, 1, 5] = math.inf
    q[1, 2, 0] = math.nan
    out, lse = attend(m, q=q)
    bad = torch.zeros(2, 3, dtype=torch.bool)
    bad[0, 1] = bad[1, 2] = True
    assert bool(torch.isnan(out.cpu()[bad]).all()) and bool(torch.isnan(lse.cpu()[bad]).all())
    assert torch.equal(out.cpu()[~bad], good.cpu()[~bad])


def test_strides_and_alignment(cuda_dev):
    """Head-major queries, rows off the 16-byte grid, pools and tables that are views."""
    m = make([130, 77], [2, 2], H=4, KVL=256, DR=64, dt=F16, seed=14)
    want, wl = attend(m)
    q, qr = m.q.to(m.dev), m.qr.to(m.dev)
    head_major = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(4, 4, 259, dtype=F16, device=m.dev)
    wide[..., 3:] = q
    qr_odd = torch.zeros(4, 4, 65, dtype=F16, device=m.dev)
    qr_odd[..., 1:] = qr
    for a, b in ((head_major, qr), (wide[..., 3:], qr_odd[..., 1:])):
        out, lse = attend(m, q=a, qr=b)
        assert torch.equal(out, want) and torch.equal(lse, wl)
    P, S, KVL = m.cache.codes.shape
    big = torch.full((P, S + 8, KVL + 64), 0x7F, dtype=torch.uint8, device=m.dev)
    big[:, :S, :KVL] = m.cache.codes.view(torch.uint8)
    scales = torch.full((P, S + 3), math.nan, device=m.dev)
    scales[:, :S] = m.cache.scales
    rope = torch.zeros(P, S, 128, dtype=F16, device=m.dev)
    rope[..., :64] = m.cache.rope
    m.cache = pkg().LatentCache.from_tensors(big.view(torch.float8_e4m3fn)[:, :S, :KVL],
                                             scales[:, :S], rope[..., :64])
    table = torch.full((2, 9), -7, dtype=torch.int32, device=m.dev)
    table[:, :m.table.shape[1]] = m.table
    m.table = table[:, :m.table.shape[1]]
    out, lse = attend(m)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    c, k = pkg().latent_read(m.cache, m.table, m.lens, 4, q_start=m.q_start)
    assert torch.equal(c.double().cpu()[:2], m.c[0][128:130].to(F16).double())
    assert torch.equal(k.double().cpu()[2:], m.k[1][75:77].to(F16).double())


def test_offsets_past_32_bits(cuda_dev):
    """Pages in a pool of more than 2^32 bytes of codes (and of rope part)."""
    pages, page, KVL, DR = 8400, 1024, 512, 64
    small = make([900], [1], KVL=KVL, DR=DR, page=page, dt=BF16, seed=15, spare=0)
    dev = small.dev
    codes = torch.empty(pages, page, KVL, dtype=torch.uint8, device=dev)
    scales = torch.full((pages, page), math.nan, device=dev)
    rope = torch.empty(pages, page, 8 * DR, dtype=BF16, device=dev)[..., :DR]
    at = pages - 2
    codes[at] = small.cache.codes.view(torch.uint8)[0]
    scales[at] = small.cache.scales[0]
    rope[at] = small.cache.rope[0]
    want, wl = attend(small)
    small.cache = pkg().LatentCache.from_tensors(codes.view(torch.float8_e4m3fn), scales, rope)
    small.table = torch.tensor([[at]], dtype=torch.int32, device=dev)
    out, lse = attend(small)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    small.lens.fill_(901)
    new = torch.randn(1, KVL, device=dev).to(BF16)
    kn = torch.randn(1, DR, device=dev).to(BF16)
    pkg().latent_append(small.cache, new, small.table, small.lens, k_rope=kn)
    c, k = pkg().latent_read(small.cache, small.table, small.lens, 1)
    assert torch.equal(k, kn) and float((c - new).abs().max()) <= 2.0 ** -4 * float(new.abs().max())
    assert not math.isnan(float(small.cache.scales[at, 900]))


def test_repeated_calls_are_identical_and_streams_are_respected(cuda_dev):
    m = make([5000, 300], [1, 1], seed=16)
    a = attend(m)
    for _ in range(3):
        b = attend(m)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    side = torch.cuda.Stream()
    q = m.q.to(m.dev)
    late = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            torch.empty(1 << 24, device=m.dev).normal_()
        late.copy_(q)                                 # only the side stream knows when
        b = attend(m, q=late)
    side.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_page_outside_the_pool_is_reported(cuda_dev):
    m = make([200, 90], [1, 1], KVL=128, seed=17)
    kb = pkg()
    kb.device_error(clear=True)
    good, _ = attend(m)
    table = m.table.clone()
    table[0, 1] = m.cache.num_pages + 5
    m.table = table
    out, lse = attend(m)
    assert kb.device_error(clear=True) == 6
    assert bool(torch.isnan(out[0]).all()) and torch.equal(out[1], good[1])
    before = m.cache.codes.view(torch.uint8).clone()
    x = torch.ones(2, 128, dtype=BF16, device=m.dev)
    m.lens.copy_(torch.tensor([100, 0]))              # position 99 of sequence 0: the bad page
    kb.latent_append(m.cache, x, m.table, m.lens)
    assert kb.device_error(clear=True) == 6
    assert torch.equal(m.cache.codes.view(torch.uint8), before)
    c, _ = kb.latent_read(m.cache, m.table, m.lens, 2)
    assert float(c.abs().sum()) == 0.0 and kb.device_error(clear=True) == 6
    m.lens.copy_(torch.tensor([200, 64 * m.table.shape[1] + 40]))     # past the table's end
    m.table = table.clone()
    m.table[0] = m.table[1]
    kb.latent_append(m.cache, x, m.table, m.lens)
    assert kb.device_error(clear=True) == 6


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
def pools(cache):
    s = cache.scales.double().cpu().reshape(-1)
    c = cache.codes.double().cpu().reshape(s.numel(), -1)
    r = None if cache.rope is None else cache.rope.double().cpu().reshape(s.numel(), -1)
    return c, s, r


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and \
        torch.equal(torch.nan_to_num(a, nan=0.0), torch.nan_to_num(b, nan=0.0))


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("KVL,DR,page", [(128, 0, 16), (256, 64, 64), (384, 64, 16), (512, 0, 128),
                                         (512, 64, 256)])
@pytest.mark.parametrize("lens,counts", [([1], [1]), ([5, 0, 300, 17], [1, 1, 1, 1]),
                                         ([130, 64, 3], [130, 0, 5]), ([33, 200], [7, 129])])
def test_append_and_read_are_exact(lens, counts, KVL, DR, page, dt, cuda_dev):
    m = make(lens, counts, KVL=KVL, DR=DR, page=page, dt=dt, seed=KVL + DR)
    g = torch.Generator().manual_seed(1)
    N = sum(counts)
    c = torch.randn(N, KVL, generator=g) * torch.exp2(torch.randint(-20, 8, (N, 1), generator=g))
    c[:, ::7] *= 0.01
    if N > 2:
        c[1] = 0.0
        c[2, 1:] = 0.0
    k = (torch.randn(N, DR, generator=g) * 30).to(dt) if DR else None
    c = c.to(dt)
    where = lo.slots(m.table.cpu(), lens, counts, page)
    want = lo.append(*pools(m.cache), c, k, where)
    pkg().latent_append(m.cache, c.cuda(), m.table, m.lens, q_start=m.q_start,
                        k_rope=None if k is None else k.cuda())
    for a, b in zip(pools(m.cache), want):
        assert a is None and b is None or same(a, b)
    got, gk = pkg().latent_read(m.cache, m.table, m.lens, N, q_start=m.q_start)
    rc, rs, rr = want
    for n, (_, _, slot) in enumerate(where):
        ref = torch.zeros(KVL) if slot is None else (rc[slot] * rs[slot]).to(dt)
        assert torch.equal(got[n].double().cpu(), ref.double()), n
        if DR:
            ref = torch.zeros(DR) if slot is None else (rr[slot] * rs[slot]).to(dt)
            assert torch.equal(gk[n].double().cpu(), ref.double()), n
    assert pkg().device_error() == 0


@pytest.mark.parametrize("dt", [BF16, F16])
def test_append_extremes(dt, cuda_dev):
    """The largest and smallest values of the type, exact powers of two and the
    values around 448 2^e, infinities and NaN."""
    KVL = 128
    top = torch.finfo(dt).max
    tiny = torch.finfo(dt).smallest_normal
    firsts = [top, -top, tiny, tiny / 4, 448.0, 450.0, 446.0, 512.0, 1.0, 0.875, 7.0, 1.75, 2.0,
              math.inf, -math.inf, math.nan, 2.0 ** -14]
    c = torch.zeros(len(firsts), KVL, dtype=dt)
    for i, v in enumerate(firsts):
        c[i, 3] = v
        c[i, 4] = v * 0.3 if math.isfinite(v) else 1.0
        c[i, 5] = v * 2.0 ** -9 if math.isfinite(v) else -2.0
    m = make([len(firsts)], [len(firsts)], KVL=KVL, page=16, dt=dt)
    where = lo.slots(m.table.cpu(), m.L, m.counts, 16)
    want = lo.append(*pools(m.cache), c, None, where)
    pkg().latent_append(m.cache, c.cuda(), m.table, m.lens)
    for a, b in zip(pools(m.cache)[:2], want[:2]):
        assert same(a, b)
    got, _ = pkg().latent_read(m.cache, m.table, m.lens, len(firsts))
    for i, v in enumerate(firsts):
        assert bool(torch.isnan(got[i]).all()) == (not math.isfinite(v))


def test_append_strides(cuda_dev):
    """Latents and rope keys as two halves of one projection's rows, and off the grid."""
    m = make([40, 9], [4, 4], DR=64, dt=BF16, seed=3)
    x = torch.randn(8, 512 + 64, device=m.dev).to(BF16)
    pkg().latent_append(m.cache, x[:, :512], m.table, m.lens, k_rope=x[:, 512:])
    want = pools(m.cache)
    m.cache.codes.view(torch.uint8).zero_()
    y = torch.zeros(8, 600, device=m.dev, dtype=BF16)
    y[:, 1:577] = x
    pkg().latent_append(m.cache, y[:, 1:513], m.table, m.lens, k_rope=y[:, 513:577])
    got = pools(m.cache)
    where = [w[2] for w in lo.slots(m.table.cpu(), m.L, m.counts, 64)]
    for a, b in zip(got, want):
        assert torch.equal(a[where], b[where])


def test_empty_calls(cuda_dev):
    kb = pkg()
    cache = kb.LatentCache(2, 16, 128, device=cuda_dev)
    table = torch.zeros(0, 1, dtype=torch.int32, device=cuda_dev)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda_dev)
    x = torch.zeros(0, 128, dtype=BF16, device=cuda_dev)
    kb.latent_append(cache, x, table, lens)
    assert kb.latent_read(cache, table, lens, 0)[0].shape == (0, 128)
    out, lse = kb.latent_attention(x.view(0, 4, 128), cache, table, lens, 1.0, return_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    # a table without pages: every row is empty
    t1, l1 = torch.zeros(3, 0, dtype=torch.int32, device=cuda_dev), lens.new_zeros(3)
    out, lse = kb.latent_attention(torch.ones(3, 2, 128, dtype=BF16, device=cuda_dev), cache, t1, l1,
                                   1.0, return_lse=True)
    assert float(out.abs().sum()) == 0.0 and bool(torch.isneginf(lse).all())


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def _module(H, DN, DV, KVL, DR, hidden, dev, dt):
    torch.manual_seed(0)
    return types.SimpleNamespace(
        num_heads=H, qk_nope_head_dim=DN, qk_rope_head_dim=DR, v_head_dim=DV,
        scale=(DN + DR) ** -0.5,
        kv_b_proj=torch.nn.Linear(KVL, H * (DN + DV), bias=False).to(dev, dt),
        o_proj=torch.nn.Linear(H * DV, hidden, bias=False).to(dev, dt))


def _expanded(m, q, qr, c, k, seen):
    """The layer's attention on expanded keys and values, float64, one sequence."""
    H, DN, DV = m.num_heads, m.qk_nope_head_dim, m.v_head_dim
    kv = (c.double() @ m.kv_b_proj.weight.double().T).view(c.shape[0], H, DN + DV)
    out = []
    for i in range(q.shape[0]):
        s = seen[i]
        z = torch.einsum("hd,lhd->hl", q[i].double(), kv[:s, :, :DN])
        if qr is not None:
            z = z + torch.einsum("hd,ld->hl", qr[i].double(), k[:s].double())
        out.append(torch.einsum("hl,lhd->hd", torch.softmax(z * m.scale, -1), kv[:s, :, DN:]))
    return m.o_proj.weight.double() @ torch.stack(out).reshape(q.shape[0], -1).T


@pytest.mark.parametrize("DR", [0, 64])
@pytest.mark.parametrize("dt,tol", [(F16, 4e-3), (BF16, 2e-2)])
def test_mla_step_prompt_then_tokens(DR, dt, tol, cuda_dev):
    """A prompt in two chunks, then single tokens in a captured graph, against
    the expanded form on the values that the cache holds.  Bar: the folded query,
    the mixed latents, the value product and o_proj's input are each rounded to
    the 16-bit type (2^-9 or 2^-12 rms-like each), the score's error enters
    through the softmax; 4e-3 / 2e-2 is about ten roundings."""
    kb, dev = pkg(), cuda_dev
    B, H, DN, DV, KVL, hidden, page = 2, 16, 128, 128, 512, 256, 64
    mod = _module(H, DN, DV, KVL, DR, hidden, dev, dt)
    cache = kb.LatentCache(20, page, KVL, DR, dtype=dt, device=dev)
    perm = torch.randperm(20, generator=torch.Generator().manual_seed(2)).int()
    state = {"cache": cache, "block_table": perm.view(2, 10).to(dev),
             "lens": torch.zeros(B, dtype=torch.int32, device=dev)}

    def inputs(T, seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=dev).to(dt)  # noqa: E731
        return (torch.zeros(B, T, hidden, device=dev, dtype=dt), r(B, T, H, DN) * 0.5,
                r(B, T, H, DR) if DR else None, r(B, T, KVL), r(B, T, DR) if DR else None)

    def reference(args, total):
        _, q, qr, _, _ = args
        T = q.shape[1]
        c, k = kb.latent_read(cache, state["block_table"], state["lens"], B * total)
        c = c.view(B, total, KVL)
        seen = [total - T + i + 1 for i in range(T)]
        return torch.stack([_expanded(mod, q[b], None if qr is None else qr[b], c[b],
                                      k.view(B, total, DR)[b] if DR else None, seen).T
                            for b in range(B)])

    with torch.no_grad():
        total = 0
        for T in (100, 37):
            args = inputs(T, T)
            out, st = kb.latent.mla_step(mod, *args, state, True)
            total += T
            assert st is state and state["lens"].tolist() == [total] * B
            want = reference(args, total)
            assert float((out.double() - want).norm() / want.norm()) < tol
        args = inputs(1, 5)
        warm = {"cache": cache, "block_table": state["block_table"], "lens": state["lens"].clone()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kb.latent.mla_step(mod, *args, warm, False)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kb.latent.mla_step(mod, *args, state, False)
        for step in range(3):
            for dst, src in zip(args, inputs(1, 50 + step)):
                if dst is not None:
                    dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            total += 1
            assert state["lens"].tolist() == [total] * B
            want = reference(args, total)
            assert float((out.double() - want).norm() / want.norm()) < tol
        del graph


def test_parts_of_a_context_join_by_lse(cuda_dev):
    """Attention over two halves of a context, joined by their lse, is attention over it."""
    m = make([512], [1], KVL=256, dt=F16, page=256, seed=21)
    whole, wl = attend(m)
    kb = pkg()
    parts = []
    for i in range(2):
        lens = torch.full((1,), 256, dtype=torch.int32, device=m.dev)
        parts.append(kb.latent_attention(m.q.to(m.dev), m.cache, m.table[:, i:i + 1].contiguous(),
                                         lens, m.scale, return_lse=True))
    lse = torch.logaddexp(parts[0][1], parts[1][1])
    out = sum(o.float() * torch.exp(x - lse)[..., None] for o, x in parts)
    assert float((lse - wl).abs().max()) < 1e-5
    assert float((out - whole.float()).norm() / whole.float().norm()) < 2.0 ** -10


# ---------------------------------------------------------------------------
# many tiles and many groups for one block
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("H,n,KVL,DR,page,dt", [
    (16, 1, 512, 0, 64, BF16),       # 16 rows a group, the ring's chunks used again and again
    (16, 1, 512, 64, 16, F16),
    (16, 2, 512, 0, 128, BF16),      # 32 rows a group
    (16, 2, 512, 0, 32, F16),        # one buffer of scores
    (8, 4, 512, 64, 128, BF16),
    (16, 2, 512, 64, 256, F16),      # 32 rows would leave too small a ring
    (16, 1, 128, 0, 128, F16),
    (20, 3, 384, 64, 64, BF16),
])
def test_blocks_walk_many_tiles(H, n, KVL, DR, page, dt, cuda_dev):
    """Twelve sequences, the longest of 12000: about ten tiles and several changes of
    sequence for each block."""
    lens = [12000, 4000, 1, 8191, 300, 12000, 0, 6001, 129, 128, 2500, 9000]
    m = make(lens, [n] * len(lens), H=H, KVL=KVL, DR=DR, page=page, dt=dt, seed=KVL + n + DR)
    check(m, *attend(m))


@pytest.mark.parametrize("DR,dt", [(0, F16), (64, BF16)])
def test_blocks_walk_many_groups(DR, dt, cuda_dev):
    """Prompts and chunks of prompts of many row groups, in pairs of unlike length."""
    lens, counts = [700, 1100, 64, 900, 5], [700, 333, 64, 1, 5]
    m = make(lens, counts, H=16, KVL=256, DR=DR, page=64, dt=dt, seed=DR)
    check(m, *attend(m))


def test_maxima_that_move_often(cuda_dev):
    """Loud tokens all along two long sequences: rows outgrow the weights' range at many
    tiles, in both softmax groups."""
    for dt, n in ((BF16, 1), (F16, 1), (F16, 2)):
        m = make([6000, 5000], [n, n], KVL=128, dt=dt, seed=31, q_gain=0.3)
        for b, L in enumerate((6000, 5000)):
            at = torch.arange(L)
            slot = m.table[b].long().cpu()[at // 64] * 64 + at % 64
            grow = torch.exp2(torch.floor(at / 400.0))          # scales double every 400 positions
            m.cache.scales.view(-1)[slot.to(m.dev)] *= grow.float().to(m.dev)
            m.c[b] *= grow.double()[:, None]
        m.q[:, 0] *= 2.0 ** -12                                 # a row that hardly looks
        check(m, *attend(m))
