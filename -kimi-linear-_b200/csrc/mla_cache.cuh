// mla_cache.cuh -- what the latent-cache kernels share: the device-side view
// of MlaCacheArgs, where a new token sits, and the split of values over e4m3.
#pragma once

#include <cuda_fp8.h>

#include "kda_internal.cuh"

namespace kda {
namespace cache {

constexpr int kErrOutside = 6;    // device error word: a position or page outside the pool
constexpr int kErrWait = 7;       // device error word: a bounded wait ran out
constexpr int kMinExp = -100;     // least exponent of a token's scale

// Device-side view of MlaCacheArgs (strides in elements).
struct CacheParams {
  int num_pages, page_size, page_shift, KVL, DR;
  int B, N, H, max_pages;
  float scale;
  uint8_t* codes; int64_t codes_s[2];
  float* scales; int64_t scales_s;
  void* rope; int64_t rope_s[2];
  const int* table; int64_t table_s;
  const int* lens;
  const int* q_start;               // or null: N / B new tokens each
  void* c_kv; int64_t c_s;
  void* k_rope; int64_t k_s;
  const void* q_lat; int64_t ql_s[2];
  const void* q_rope; int64_t qr_s[2];
  void* out; int64_t o_s[2];
  float* lse; int64_t lse_s;
  uint32_t h_mul;                   // 2^32 / H, rounded down (H = 1: 2^32 - 1)
  bool out_vec;                     // out rows start on 4-byte boundaries
  bool vec;                         // c_kv / k_rope (append, read) or q_lat / q_rope (attention)
                                    // rows start on 16-byte boundaries
};

// First new token of sequence b and how many it has.
__device__ __forceinline__ void new_tokens(const CacheParams& p, int b, int& first, int& count) {
  if (p.q_start != nullptr) {
    first = min(max(p.q_start[b], 0), p.N);
    count = max(min(p.q_start[b + 1], p.N) - first, 0);
  } else {
    count = p.N / p.B;
    first = b * count;
  }
}

// Sequence and position of new token n (position < 0: it has none), for all lanes of
// a warp at once; lanes of one half have one n.  (No sequence has it: -1.)  The sequences' starts are counted 32
// at a time: one load's latency, where a search by halves has one for each step.
__device__ __forceinline__ void locate(const CacheParams& p, int n, int& b, int& pos) {
  int first, count;
  if (p.B == 0) {
    b = 0;
    pos = -1;
    return;
  }
  if (p.q_start == nullptr) {
    count = p.N / p.B;
    b = n / count;
    first = b * count;
  } else {
    const int lane = threadIdx.x & 31;
    const int n0 = __shfl_sync(0xffffffffu, n, 0), n1 = __shfl_sync(0xffffffffu, n, 16);
    int c0 = 0, c1 = 0;              // starts 1 .. B - 1 that are <= n
    for (int i = 1; i < p.B; i += 32) {
      const int x = i + lane < p.B ? p.q_start[i + lane] : 0x7fffffff;
      c0 += __popc(__ballot_sync(0xffffffffu, x <= n0));
      c1 += __popc(__ballot_sync(0xffffffffu, x <= n1));
    }
    b = lane < 16 ? c0 : c1;
    new_tokens(p, b, first, count);
  }
  const int i = n - first;
  pos = i >= 0 && i < count ? max(p.lens[b], 0) - count + i : -1;
}

// Page of position pos of sequence b, or -1 where the table or the pool ends.
__device__ __forceinline__ int page_of(const CacheParams& p, int b, int pos) {
  const int i = pos >> p.page_shift;
  if (i >= p.max_pages) return -1;
  const int page = p.table[(int64_t)b * p.table_s + i];
  return page >= 0 && page < p.num_pages ? page : -1;
}

// Exponent of the scale of values with largest magnitudes `amax` (e4m3 part)
// and `rmax` (16-bit rope part), as bit patterns of non-negative floats: the
// least e with amax <= 448 2^e and rmax <= 2^15 2^e, at least kMinExp.  A power
// of two costs e4m3 no relative precision, makes x / s exact, so that codes do
// not depend on how a quotient was rounded, and gives log2 s exactly.
// Not finite (exponent field 255): 128.
__device__ __forceinline__ int scale_exp(uint32_t amax, uint32_t rmax) {
  if (max(amax, rmax) >= 0x7f800000u) return 128;
  const int ea = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u);   // 448 = 1.75 2^8
  const int er = (int)(rmax >> 23) - 127 - 15 + ((rmax & 0x7fffffu) > 0u);
  return max(max(ea, er), kMinExp);
}
// 2^e for -126 <= e <= 127; NaN for e = 128 and e = -128 (scale_exp's mark and its negative)
__device__ __forceinline__ float pow2i(int e) {
  return (e == 128 || e == -128) ? __uint_as_float(0x7fffffffu)
                                 : __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// four floats -> four e4m3 codes (round to nearest even; NaN stays NaN)
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// two e4m3 codes (low 16 bits) -> two floats, exactly
__device__ __forceinline__ float2 from_e4m3x2(uint32_t u) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// eight consecutive 16-bit elements -> fp32; `vec`: the address is 16-byte aligned
template <typename T>
__device__ __forceinline__ void ld8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ld(e + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ld(p + i);
  }
}
template <typename T>
__device__ __forceinline__ void st8(T* p, bool vec, const float (&x)[8]) {
  if (vec) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) st(e + i, x[i]);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) st(p + i, x[i]);
  }
}

size_t attention_workspace_bytes(const CacheParams& p, int io_dtype);
cudaError_t launch_attention(const CacheParams& p, int io_dtype, void* workspace, cudaStream_t s);

}  // namespace cache
}  // namespace kda
