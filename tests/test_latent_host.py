"""Host-side behaviour of the 8-bit latent cache (no GPU needed): the oracle's
rounding, argument checks of the Python layer and of the C entry points."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from conftest import pkg
from oracle import latent_oracle as lo

BF16 = torch.bfloat16


def test_oracle_rounding_is_e4m3():
    """Every code's value is a fixed point, and midpoints go to the even neighbour."""
    grid = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(lo.round_e4m3(grid), grid) and torch.equal(lo.round_e4m3(-grid), -grid)
    mid = (grid[1:] + grid[:-1]) / 2
    assert torch.equal(lo.round_e4m3(mid), mid.float().to(torch.float8_e4m3fn).double())
    x = torch.linspace(-448, 448, 20011, dtype=torch.float64)
    assert torch.equal(lo.round_e4m3(x), x.float().to(torch.float8_e4m3fn).double())


def test_oracle_scale_is_the_least_power_of_two():
    for a in (1e-3, 1.0, 1.75, 1.7500001, 447.9, 448.0, 448.1, 1e6):
        s = lo.token_scale(torch.tensor([a, 0.0], dtype=torch.float64))
        assert math.log2(s) == int(math.log2(s)) and a <= 448 * s and a > 448 * s / 2
    zero = torch.zeros(4, dtype=torch.float64)
    assert lo.token_scale(zero) == 2.0 ** -100
    assert lo.token_scale(zero, torch.tensor([32769.0], dtype=torch.float64)) == 2.0
    assert math.isnan(lo.token_scale(torch.tensor([math.inf], dtype=torch.float64)))


def cpu_cache(P=2, S=16, KVL=128, DR=0):
    return pkg().LatentCache(P, S, KVL, DR, device="cpu")


def test_cache_layout_and_refusals():
    kb = pkg()
    c = cpu_cache(3, 32, 256, 64)
    assert c.codes.dtype == torch.float8_e4m3fn and tuple(c.codes.shape) == (3, 32, 256)
    assert tuple(c.scales.shape) == (3, 32) and tuple(c.rope.shape) == (3, 32, 64)
    for bad in (dict(kv_lora_rank=64), dict(kv_lora_rank=640), dict(rope_dim=32),
                dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(num_pages=0)):
        a = dict(num_pages=2, page_size=16, kv_lora_rank=128) | bad
        with pytest.raises(RuntimeError, match="not supported"):
            kb.LatentCache(**a, device="cpu")
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        kb.LatentCache(2, 16, 128, dtype=torch.float32, device="cpu")
    with pytest.raises(TypeError, match="dtype is needed"):
        kb.LatentCache.from_tensors(c.codes, c.scales)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        kb.LatentCache.from_tensors(c.codes.float(), c.scales, dtype=BF16)
    with pytest.raises(RuntimeError, match="expected codes"):
        kb.LatentCache.from_tensors(c.codes, c.scales[:2], dtype=BF16)
    with pytest.raises(RuntimeError, match="innermost stride"):
        kb.LatentCache.from_tensors(c.codes, c.scales, c.rope.transpose(1, 2).contiguous()
                                    .transpose(1, 2))


def test_cpu_tensors_raise_no_fallback():
    kb, c = pkg(), cpu_cache()
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 128, dtype=BF16)
    for call in (lambda: kb.latent_append(c, x, table, lens),
                 lambda: kb.latent_read(c, table, lens, 1),
                 lambda: kb.latent_attention(x[:, None], c, table, lens, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


def _args(**kw):
    L = pkg()._lib
    a = L.MlaCacheArgs()
    a.abi_version = L.ABI_VERSION
    a.io_dtype = L.DTYPE_BF16
    a.num_pages, a.page_size, a.KVL, a.DR = 8, 64, 512, 64
    a.B, a.N, a.H, a.max_pages = 2, 4, 16, 4
    a.scale = 0.1
    fake = 1 << 20                       # aligned non-null addresses; validation only
    for f in ("codes", "scales", "rope", "block_table", "lens", "q_start", "c_kv", "k_rope",
              "q_lat", "q_rope", "out", "lse"):
        setattr(a, f, fake)
    i2 = ctypes.c_int64 * 2
    a.codes_stride, a.scales_stride, a.rope_stride = i2(64 * 512, 512), 64, i2(64 * 64, 64)
    a.table_stride, a.c_kv_stride, a.k_rope_stride = 4, 512, 64
    a.q_lat_stride, a.q_rope_stride = i2(16 * 512, 512), i2(16 * 64, 64)
    a.out_stride, a.lse_stride = i2(16 * 512, 512), 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_argument_errors_before_any_launch():
    """Argument errors come back as status codes before anything touches the GPU."""
    L = pkg()._lib
    lib = L.load()
    i2 = ctypes.c_int64 * 2
    for fn in (lib.mla_cache_append, lib.mla_cache_read, lib.mla_cache_attention):
        call = lambda **k: fn(ctypes.byref(_args(**k)), None)  # noqa: E731
        assert fn(None, None) == L.KDA_ERR_NULL_POINTER
        assert call(abi_version=99) == L.KDA_ERR_SHAPE
        assert call(io_dtype=L.DTYPE_F32) == L.KDA_ERR_DTYPE
        for bad in (dict(KVL=64), dict(KVL=640), dict(KVL=200), dict(DR=32), dict(page_size=48),
                    dict(page_size=8), dict(page_size=2048), dict(num_pages=0), dict(B=-1),
                    dict(N=-1), dict(max_pages=-1), dict(num_pages=1 << 26),
                    dict(q_start=None, N=5)):
            assert call(**bad) == L.KDA_ERR_SHAPE, bad
        for bad in (dict(codes=None), dict(scales=None), dict(rope=None), dict(lens=None),
                    dict(block_table=None)):
            assert call(**bad) == L.KDA_ERR_NULL_POINTER, bad
        for bad in (dict(codes=(1 << 20) + 8), dict(codes_stride=i2(64 * 512, 520)),
                    dict(rope=(1 << 20) + 2), dict(rope_stride=i2(64 * 64, 68))):
            assert call(**bad) == L.KDA_ERR_ALIGNMENT, bad
        for bad in (dict(codes_stride=i2(64 * 512, 256)), dict(rope_stride=i2(64 * 64, 32)),
                    dict(codes_stride=i2(-512, 512)), dict(scales_stride=-64),
                    dict(table_stride=-1)):
            assert call(**bad) == L.KDA_ERR_STRIDE, bad
        assert call(B=0, N=0) == L.KDA_OK            # nothing to do, success without a device
    for fn in (lib.mla_cache_append, lib.mla_cache_read):
        assert fn(ctypes.byref(_args(c_kv=None)), None) == L.KDA_ERR_NULL_POINTER
        assert fn(ctypes.byref(_args(k_rope=None)), None) == L.KDA_ERR_NULL_POINTER
        assert fn(ctypes.byref(_args(c_kv=(1 << 20) + 1)), None) == L.KDA_ERR_ALIGNMENT
    att = lambda **k: lib.mla_cache_attention(ctypes.byref(_args(**k)), None)  # noqa: E731
    assert att(q_lat=None) == L.KDA_ERR_NULL_POINTER
    assert att(q_rope=None) == L.KDA_ERR_NULL_POINTER
    assert att(out=None) == L.KDA_ERR_NULL_POINTER
    assert att(H=-1) == L.KDA_ERR_SHAPE and att(H=2000) == L.KDA_ERR_SHAPE
    assert att(out=(1 << 20) + 1) == L.KDA_ERR_ALIGNMENT
    assert att(lse=(1 << 20) + 2) == L.KDA_ERR_ALIGNMENT
    assert att(H=0) == L.KDA_OK


@pytest.mark.gpu
def test_refusals_on_the_gpu(cuda_dev):
    kb, dev = pkg(), cuda_dev
    c = kb.LatentCache(4, 16, 128, 64, device=dev)
    plain = kb.LatentCache(4, 16, 128, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    table, lens = torch.zeros(2, 2, **i32), torch.ones(2, **i32)
    x, r = torch.zeros(2, 128, dtype=BF16, device=dev), torch.zeros(2, 64, dtype=BF16, device=dev)
    q, qr = torch.zeros(2, 3, 128, dtype=BF16, device=dev), torch.zeros(2, 3, 64, dtype=BF16, device=dev)
    with pytest.raises(TypeError, match="cache's type"):
        kb.latent_append(plain, x.half(), table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        kb.latent_append(plain, x.cpu(), table, lens)
    with pytest.raises(RuntimeError, match="c_kv shape"):
        kb.latent_append(plain, x[:, :64], table, lens)
    with pytest.raises(RuntimeError, match="exactly when"):
        kb.latent_append(c, x, table, lens)
    with pytest.raises(RuntimeError, match="exactly when"):
        kb.latent_append(plain, x, table, lens, k_rope=r)
    with pytest.raises(RuntimeError, match="block_table must be"):
        kb.latent_append(plain, x, table.long(), lens)
    with pytest.raises(RuntimeError, match="lens must be"):
        kb.latent_append(plain, x, table, lens.cpu())
    with pytest.raises(RuntimeError, match="one batch"):
        kb.latent_append(plain, x, table[:1], lens)
    with pytest.raises(RuntimeError, match="one batch"):
        kb.latent_append(plain, x, table, lens, q_start=torch.zeros(2, **i32))
    with pytest.raises(RuntimeError, match="do not divide"):
        kb.latent_append(plain, x[:1], table, lens)
    with pytest.raises(RuntimeError, match="negative"):
        kb.latent_read(plain, table, lens, -1)
    with pytest.raises(RuntimeError, match="q_lat shape"):
        kb.latent_attention(x, plain, table, lens, 1.0)
    with pytest.raises(RuntimeError, match="exactly when"):
        kb.latent_attention(q, c, table, lens, 1.0)
    with pytest.raises(RuntimeError, match="q_rope shape"):
        kb.latent_attention(q, c, table, lens, 1.0, q_rope=qr[:, :2])
    with pytest.raises(RuntimeError, match="forward-only"):
        kb.latent_attention(q.clone().requires_grad_(True), plain, table, lens, 1.0)
    odd = torch.zeros(4, 16, 136, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)[..., :128]
    bad = kb.LatentCache.from_tensors(odd, plain.scales, dtype=BF16)
    with pytest.raises(kb.KdaError):
        kb.latent_append(bad, x, table, lens)
