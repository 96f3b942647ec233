"""Paged latent cache in 8 bits and the attention over it (``csrc/mla_cache*.cu``).

For serving the MLA layers: all that such a layer caches per token is its
latent ``c_kv`` (``kv_lora_rank`` channels) and, with a rope part, one rotated
key (``kimi_linear/mla.py:183-288``).  :class:`LatentCache` holds them in pages
of e4m3 codes with one power-of-two scale per token, the rope part in 16 bits:
half the bytes of the 16-bit buffer that :mod:`mla` decodes from, ragged
lengths, and any number of new tokens per sequence and call.

Three operators share the cache.  Each takes ``block_table`` int32
``[B, max_pages]`` (page ``block_table[b, p // page_size]`` holds position
``p`` of sequence ``b``), ``lens`` int32 ``[B]`` (tokens of each sequence, the
new ones included) and ``q_start`` int32 ``[B + 1]`` (sequence ``b`` owns rows
``q_start[b] .. q_start[b + 1] - 1`` of the new tokens; None: ``N / B`` each).
New token ``i`` of the ``n`` of sequence ``b`` sits at position
``lens[b] - n + i``.  Rows before ``q_start[0]`` and from ``q_start[B]`` on (a
batch padded to a fixed ``N``) belong to no sequence: append skips them, read
gives zeros, attention zeros and ``-inf``:

* :func:`latent_append` quantises new tokens into their slots;
* :func:`latent_read` gives tokens back in the 16-bit type;
* :func:`latent_attention` is the absorbed form: scores of ``q_lat`` (and
  ``q_rope``) against the latents up to and with the token's own position,
  softmax, the weighted sum of the latents, and the log-sum-exp.

:func:`mla_step` runs an MLA layer's step on them.  ``block_table``, ``lens``
and ``q_start`` are only read on the device, nothing synchronises and every
kernel runs on the current stream, so a step can be captured in a CUDA graph.
CUDA tensors and 16-bit types only, forward only; anything else raises (no
fallback).  A position past ``max_pages`` or a page outside the pool sets the
device error word (:func:`ops.device_error` returns 6).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DT, _launch
from .rotary import qk_norm_rope

_HALF = (torch.float16, torch.bfloat16)
_I64x2 = ctypes.c_int64 * 2


class LatentCache:
    """The pool: ``codes`` float8_e4m3fn ``[num_pages, page_size, kv_lora_rank]``,
    ``scales`` fp32 ``[num_pages, page_size]`` and ``rope`` ``[num_pages,
    page_size, rope_dim]`` in ``dtype`` (None without a rope part).

    ``page_size``: a power of two from 16 to 1024; ``kv_lora_rank`` 128, 256,
    384 or 512; ``rope_dim`` 0 or 64; ``dtype`` (of the latents, queries and
    outputs) fp16 or bf16.  Slots are written before they are read, so the
    memory starts uninitialised.

    The attributes are read-only (the tensors' values are not): calls pass the
    addresses that the cache was made with.  A pool that moves or grows is
    another cache (:meth:`from_tensors`)."""

    def __init__(self, num_pages, page_size, kv_lora_rank, rope_dim=0, dtype=torch.bfloat16,
                 device="cuda"):
        num_pages, page_size = int(num_pages), int(page_size)
        codes = torch.empty(num_pages, page_size, int(kv_lora_rank), dtype=torch.float8_e4m3fn,
                            device=device)
        scales = torch.empty(num_pages, page_size, dtype=torch.float32, device=device)
        rope = (torch.empty(num_pages, page_size, int(rope_dim), dtype=dtype, device=device)
                if rope_dim else None)
        self._bind(codes, scales, rope, dtype)

    @classmethod
    def from_tensors(cls, codes, scales, rope=None, dtype=None):
        """A cache over tensors that the caller holds (the layout above; rows of
        ``codes`` and ``rope`` start on 16-byte boundaries).  ``dtype`` defaults
        to ``rope.dtype``."""
        if dtype is None:
            if rope is None:
                raise TypeError("LatentCache: dtype is needed without a rope part")
            dtype = rope.dtype
        self = cls.__new__(cls)
        self._bind(codes, scales, rope, dtype)
        return self

    def _bind(self, codes, scales, rope, dtype):
        fn = "LatentCache"
        if dtype not in _HALF:
            raise TypeError(f"{fn}: dtype must be float16 or bfloat16 (got {dtype})")
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32 or \
                (rope is not None and rope.dtype != dtype):
            raise TypeError(f"{fn}: codes must be float8_e4m3fn, scales float32 and rope {dtype}")
        if codes.dim() != 3 or tuple(scales.shape) != tuple(codes.shape[:2]) or \
                (rope is not None and (rope.dim() != 3 or rope.shape[:2] != codes.shape[:2])):
            raise RuntimeError(
                f"{fn}: expected codes [P, S, KVL], scales [P, S], rope [P, S, DR]; got "
                f"{tuple(codes.shape)}, {tuple(scales.shape)}, "
                f"{None if rope is None else tuple(rope.shape)}")
        for name, t in (("codes", codes), ("scales", scales), ("rope", rope)):
            if t is None:
                continue
            if t.device != codes.device:
                raise RuntimeError(f"{fn}: {name} is on {t.device}, expected {codes.device}")
            if t.stride(-1) != 1:
                raise RuntimeError(f"{fn}: {name} needs a unit innermost stride")
        pages, page, kvl = codes.shape
        dr = 0 if rope is None else rope.shape[2]
        if kvl not in (128, 256, 384, 512) or dr not in (0, 64):
            raise RuntimeError(f"{fn}: kv_lora_rank {kvl} / rope_dim {dr} not supported "
                               f"(128, 256, 384 or 512; 0 or 64)")
        if pages < 1 or page < 16 or page > 1024 or page & (page - 1) or pages * page >= 2 ** 31:
            raise RuntimeError(f"{fn}: {pages} pages of {page} tokens not supported (page_size a "
                               f"power of two from 16 to 1024, fewer than 2^31 tokens)")
        a = _lib.MlaCacheArgs()
        a.abi_version = _lib.ABI_VERSION
        a.io_dtype = _DT[dtype]
        a.num_pages, a.page_size, a.KVL, a.DR = pages, page, kvl, dr
        a.codes, a.codes_stride = codes.data_ptr(), _I64x2(*codes.stride()[:2])
        a.scales, a.scales_stride = scales.data_ptr(), scales.stride(0)
        if rope is not None:
            a.rope, a.rope_stride = rope.data_ptr(), _I64x2(*rope.stride()[:2])
        self.__dict__.update(
            codes=codes, scales=scales, rope=rope, dtype=dtype, device=codes.device,
            on_gpu=codes.is_cuda, num_pages=pages, page_size=page, kv_lora_rank=kvl, rope_dim=dr,
            _args=bytes(a))

    def __setattr__(self, name, value):
        raise AttributeError(f"LatentCache.{name} is read-only; make another cache of other "
                             f"tensors with LatentCache.from_tensors")

    def __delattr__(self, name):
        self.__setattr__(name, None)

    def __reduce__(self):        # a copy has the addresses of its own tensors
        return LatentCache.from_tensors, (self.codes, self.scales, self.rope, self.dtype)


def _refuse(fn, cache, name, t):
    """Why operand ``t`` is not a 16-bit tensor of the cache's type on its device."""
    dev, dt = cache.device, cache.dtype
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{fn}: {name} must be a torch.Tensor")
    if dev.type != "cuda" or t.device != dev:
        raise RuntimeError(f"{fn}: {name} is on {t.device}, the cache on {dev}; the B200 kernels "
                           f"need CUDA tensors on one device (there is no CPU path)")
    if t.dtype is not dt:
        raise TypeError(f"{fn}: {name} is {t.dtype}, the cache's type is {dt}")
    raise RuntimeError(f"{fn}: the latent cache is forward-only; call under torch.no_grad() or "
                       f"detach the inputs")


def _operand(fn, cache, name, t):
    if not isinstance(t, torch.Tensor) or t.dtype is not cache.dtype or \
            t.device != cache.device or not t.is_cuda or \
            (t.requires_grad and torch.is_grad_enabled()):
        _refuse(fn, cache, name, t)


def _refuse_index(fn, cache, block_table, lens, q_start):
    if cache.device.type != "cuda":
        raise RuntimeError(f"{fn}: the cache is on {cache.device}; the B200 kernels need CUDA "
                           f"tensors (there is no CPU path)")
    for name, t, dims in (("block_table", block_table, 2), ("lens", lens, 1),
                          ("q_start", q_start, 1)):
        if t is None and name == "q_start":
            continue
        if not _is_index(t, dims, cache.device):
            raise RuntimeError(f"{fn}: {name} must be an int32 tensor of {dims} dimension(s) with "
                               f"a unit innermost stride on {cache.device}")
    raise RuntimeError(
        f"{fn}: block_table {tuple(block_table.shape)}, lens {tuple(lens.shape)} and q_start "
        f"{None if q_start is None else tuple(q_start.shape)} do not describe one batch")


def _is_index(t, dims, dev):
    return isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == dev and \
        t.dim() == dims and (t.stride(-1) == 1 or t.numel() <= 1)


def _args(fn, cache, block_table, lens, q_start, N):
    """The argument block with the pool, the table and the lengths filled in."""
    dev = cache.device
    if not cache.on_gpu or not _is_index(block_table, 2, dev) or not _is_index(lens, 1, dev) or \
            (q_start is not None and not _is_index(q_start, 1, dev)):
        _refuse_index(fn, cache, block_table, lens, q_start)
    B = lens.shape[0]
    rows, width = block_table.shape
    if rows != B or (q_start is not None and q_start.shape[0] != B + 1):
        _refuse_index(fn, cache, block_table, lens, q_start)
    if q_start is None and (N % B if B else N):
        raise RuntimeError(f"{fn}: {N} new tokens do not divide over {B} sequences; pass q_start")
    a = _lib.MlaCacheArgs.from_buffer_copy(cache._args)
    a.B, a.N, a.max_pages = B, N, width
    a.block_table, a.table_stride = block_table.data_ptr(), block_table.stride(0)
    a.lens = lens.data_ptr()
    if q_start is not None:
        a.q_start = q_start.data_ptr()
    return a


def _rows(fn, name, t, N, width):
    if t.dim() != 2 or t.shape[0] != N or t.shape[1] != width:
        raise RuntimeError(f"{fn}: {name} shape {tuple(t.shape)} != {(N, width)}")
    return t if t.stride(1) == 1 else t.contiguous()


def latent_append(cache, c_kv, block_table, lens, q_start=None, k_rope=None):
    """Quantise new tokens into the cache.

    ``c_kv`` ``[N, kv_lora_rank]`` and ``k_rope`` ``[N, rope_dim]`` (rotated) in
    the cache's type.  A token's scale is the least power of two (at least
    2^-100) with ``|c_kv| <= 448 s`` and ``|k_rope| <= 2^15 s``; its codes are
    ``e4m3(c_kv / s)``, rounded to nearest even, its rope part ``k_rope / s``.
    A token with a value that is not finite gets a NaN scale and reads back as
    NaN.  Tokens whose position is negative (``lens[b]`` below the number of new
    tokens) are skipped.  Two tokens of one call must not share a slot."""
    fn = "latent_append"
    _operand(fn, cache, "c_kv", c_kv)
    N = c_kv.shape[0]
    c_kv = _rows(fn, "c_kv", c_kv, N, cache.kv_lora_rank)
    if (k_rope is None) != (cache.rope is None):
        raise RuntimeError(f"{fn}: k_rope must be given exactly when the cache has a rope part")
    a = _args(fn, cache, block_table, lens, q_start, N)
    if N == 0:
        return
    a.c_kv, a.c_kv_stride = c_kv.data_ptr(), c_kv.stride(0)
    if k_rope is not None:
        _operand(fn, cache, "k_rope", k_rope)
        k_rope = _rows(fn, "k_rope", k_rope, N, cache.rope_dim)
        a.k_rope, a.k_rope_stride = k_rope.data_ptr(), k_rope.stride(0)
    _launch(fn, _lib.load().mla_cache_append, a, cache.device)


def latent_read(cache, block_table, lens, num_tokens, q_start=None):
    """``(c_kv [N, kv_lora_rank], k_rope [N, rope_dim] or None)`` of the last
    ``n`` tokens of every sequence, ``N = num_tokens`` in all (``n`` from
    ``q_start``, or ``N / B`` each): what :func:`latent_append` of the same
    arguments wrote, as values (an fp16 latent of 63488 or more may have gone up to
    65536, which reads as infinity).  Zeros for tokens whose position is negative."""
    fn = "latent_read"
    N, dev = int(num_tokens), cache.device
    if N < 0:
        raise RuntimeError(f"{fn}: num_tokens {N} is negative")
    a = _args(fn, cache, block_table, lens, q_start, N)
    c_kv = torch.empty((N, cache.kv_lora_rank), dtype=cache.dtype, device=dev)
    k_rope = None
    a.c_kv, a.c_kv_stride = c_kv.data_ptr(), cache.kv_lora_rank
    if cache.rope is not None:
        k_rope = cache.rope.new_empty((N, cache.rope_dim))
        a.k_rope, a.k_rope_stride = k_rope.data_ptr(), cache.rope_dim
    if N:
        _launch(fn, _lib.load().mla_cache_read, a, dev)
    return c_kv, k_rope


def latent_attention(q_lat, cache, block_table, lens, scale, q_start=None, q_rope=None,
                     return_lse=False):
    """Absorbed-form latent attention of the new tokens over the cache.

    ``q_lat`` ``[N, H, kv_lora_rank]`` (the query folded into the latent space)
    and ``q_rope`` ``[N, H, rope_dim]`` (rotated) in the cache's type.  The
    token at position ``p`` sees positions ``0 .. p`` of its sequence:
    ``softmax(scale * (q_lat . c + q_rope . k_rope))`` over the cached values,
    times ``c``.  Returns ``out`` ``[N, H, kv_lora_rank]`` in the cache's type
    and, with ``return_lse``, ``lse`` fp32 ``[N, H]``, the natural logarithm of
    the sum of the exponentials (attention over other parts of the context joins
    by it).  A row that sees nothing gives zeros and ``-inf``.

    The new tokens' own latents must be in the cache (:func:`latent_append`
    first).  Scores and sums are fp32.  Queries enter the products exactly, but
    for values below 2^-12 of the row's largest, which are off by at most 2^-19
    (bf16) or 2^-23 (fp16) of it.  A softmax weight (times its token's scale) is
    rounded to 11 bits down to 2^-21 (bf16) or 2^-23 (fp16) of the row's largest,
    and is off by at most 2^-32 or 2^-34 of it below that."""
    fn = "latent_attention"
    _operand(fn, cache, "q_lat", q_lat)
    kvl = cache.kv_lora_rank
    if q_lat.dim() != 3 or q_lat.shape[2] != kvl:
        raise RuntimeError(f"{fn}: q_lat shape {tuple(q_lat.shape)} is not [N, H, {kvl}]")
    N, H, _ = q_lat.shape
    if (q_rope is None) != (cache.rope is None):
        raise RuntimeError(f"{fn}: q_rope must be given exactly when the cache has a rope part")
    a = _args(fn, cache, block_table, lens, q_start, N)
    dev = cache.device
    out = q_lat.new_empty((N, H, kvl))
    lse = cache.scales.new_empty((N, H)) if return_lse else None
    if N and H:
        if q_lat.stride(2) != 1:
            q_lat = q_lat.contiguous()
        a.H, a.scale = H, float(scale)
        a.q_lat = q_lat.data_ptr()
        a.q_lat_stride[0], a.q_lat_stride[1] = q_lat.stride(0), q_lat.stride(1)
        if q_rope is not None:
            _operand(fn, cache, "q_rope", q_rope)
            if tuple(q_rope.shape) != (N, H, cache.rope_dim):
                raise RuntimeError(f"{fn}: q_rope shape {tuple(q_rope.shape)} != "
                                   f"{(N, H, cache.rope_dim)}")
            if q_rope.stride(2) != 1:
                q_rope = q_rope.contiguous()
            a.q_rope = q_rope.data_ptr()
            a.q_rope_stride[0], a.q_rope_stride[1] = q_rope.stride(0), q_rope.stride(1)
        a.out = out.data_ptr()
        a.out_stride[0], a.out_stride[1] = H * kvl, kvl
        if lse is not None:
            a.lse, a.lse_stride = lse.data_ptr(), H
        lib = _lib.load()
        need = lib.mla_cache_workspace_bytes(ctypes.byref(a))
        if need:
            ws = lens.new_empty((-(-need // 4),))
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _launch(fn, lib.mla_cache_attention, a, dev)
    return (out, lse) if return_lse else out


def mla_step(module, x, q_nope, q_rope, c_kv, k_rope, state, use_cache):
    """One step of an MLA layer over the 8-bit cache: the arguments and returns
    of ``MLA._decode_step_static`` (``kimi_linear/mla.py:117-181``), for any
    number ``T`` of new tokens per sequence.

    ``q_nope`` ``[B, T, H, DN]``, ``q_rope`` ``[B, T, H, DR]`` and ``k_rope``
    ``[B, T, DR]`` (rotated; None without a rope part), ``c_kv`` ``[B, T, KVL]``.
    ``state``: ``cache`` (a :class:`LatentCache`), ``block_table`` and ``lens``;
    the pages for ``lens + T`` tokens must be in the table.  With ``inv_freq`` fp32
    ``[R / 2]`` in ``state``, ``q_rope`` and ``k_rope`` come before their rotation and are
    rotated by their tokens' positions, ``lens`` and on, read on the device (by
    :func:`rotary.qk_norm_rope`; ``interleaved`` in ``state`` as there; parts of two types
    in fp32).  ``lens`` is advanced
    by ``T`` on the device (a step that raises takes that back), the tokens are
    appended, the queries folded into the latent space by the module's own
    ``kv_b_proj`` weight (cast on every step unless it is in the cache's type),
    attended, and brought out by its value half and ``o_proj``.  The folded queries
    and the mixed latents are in the 16-bit type."""
    B, T = x.shape[:2]
    cache, lens, table = state["cache"], state["lens"], state["block_table"]
    H, DN, DV, KVL = (module.num_heads, module.qk_nope_head_dim, module.v_head_dim,
                      cache.kv_lora_rank)
    if module.qk_rope_head_dim != cache.rope_dim:
        raise RuntimeError(f"mla_step: qk_rope_head_dim {module.qk_rope_head_dim} != the cache's "
                           f"rope_dim {cache.rope_dim}")
    dt = cache.dtype
    w = module.kv_b_proj.weight.detach().to(dt).view(H, DN + DV, KVL)
    inv_freq = state.get("inv_freq")
    if inv_freq is not None:
        if not cache.rope_dim:
            raise RuntimeError("mla_step: inv_freq for a cache without a rope part")
        if q_rope.dtype != k_rope.dtype or q_rope.dtype not in _DT:
            q_rope, k_rope = q_rope.float(), k_rope.float()
        q_rope, k_rope = qk_norm_rope(q_rope.reshape(B, T, H, cache.rope_dim),
                                      k_rope.reshape(B, T, 1, cache.rope_dim), norm=None, positions=lens,
                                      inv_freq=inv_freq, interleaved=state.get("interleaved", False))
    lens.add_(T)
    try:
        if cache.rope_dim:
            k_rope = k_rope.reshape(B * T, cache.rope_dim).to(dt)
            q_rope = q_rope.reshape(B * T, H, cache.rope_dim).to(dt)
        else:
            k_rope = q_rope = None
        latent_append(cache, c_kv.reshape(B * T, KVL).to(dt), table, lens, k_rope=k_rope)
        qn = q_nope.reshape(B * T, H, DN).to(dt)
        q_lat = torch.bmm(qn.transpose(0, 1), w[:, :DN]).transpose(0, 1)           # [N, H, KVL]
        mixed = latent_attention(q_lat, cache, table, lens, module.scale, q_rope=q_rope)
        out = torch.bmm(mixed.transpose(0, 1), w[:, DN:].transpose(1, 2))          # [H, N, DV]
        out = module.o_proj(out.transpose(0, 1).reshape(B, T, H * DV).to(x.dtype))
    except BaseException:
        lens.sub_(T)             # refused: the sequences are as long as they were
        raise
    if use_cache:
        return out, state
    return out
