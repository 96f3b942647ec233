// mla_cache.cu -- the 8-bit paged latent cache: tokens quantised as they are
// written, read back in 16 bits, and the C entry points (include/kda_b200.h).
//
// A token is KVL e4m3 codes, DR 16-bit rope channels and one power-of-two
// scale: code = e4m3(c / s), rope = 16-bit(k_rope / s).  Both kernels move each
// byte once and compute next to nothing: memory bounds them at length, the
// launch and one round trip to memory at a few tokens.  Sixteen lanes hold a
// token, eight 16-bit channels (one 16-byte access) a lane and step, so that a
// row of 128 channels is one 256-byte and one 128-byte segment.
//
// Measured (B200, KVL 512, inputs that rotate past L2):
//   append 32768 tokens  10.7 us, 4.7 TB/s of the 6.5 TB/s that a copy reaches; 4 tokens 2.0 us
//   read   18800 tokens  5.5 us, 5.2 TB/s
#include <cstring>

#include "mla_cache.cuh"

namespace kda {
namespace cache {

__device__ int g_cache_device_error = 0;

namespace {

constexpr int kLanes = 16;                 // lanes per token
constexpr int kTokens = 8;                 // tokens per block: small blocks, so that the
                                           // last ones leave no SM idle for long
constexpr int kThreads = kLanes * kTokens;

// eight 16-bit elements as they are; `vec`: the address is 16-byte aligned
template <typename T>
__device__ __forceinline__ uint4 raw8(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// largest magnitude of the halves of `m` and the eight elements, as 16-bit patterns (in
// which infinities and NaN are the largest)
__device__ __forceinline__ uint32_t max8(uint32_t m, const uint4& u) {
  m = __vmaxu2(m, u.x & 0x7fff7fffu);
  m = __vmaxu2(m, u.y & 0x7fff7fffu);
  m = __vmaxu2(m, u.z & 0x7fff7fffu);
  return __vmaxu2(m, u.w & 0x7fff7fffu);
}
template <typename T>
__device__ __forceinline__ uint32_t to_float_bits(uint32_t pattern) {
  const uint16_t h = (uint16_t)pattern;
  return abs_bits(ld(reinterpret_cast<const T*>(&h)));
}

template <typename T, int STEPS>
__global__ void __launch_bounds__(kThreads)
cache_append_kernel(const CacheParams p) {
  const int lane = threadIdx.x % kLanes;
  const int n = blockIdx.x * kTokens + threadIdx.x / kLanes;
  const bool live = n < p.N;
  uint4 x[STEPS], y = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) x[s] = y;
  if (live) {
    const T* c = static_cast<const T*>(p.c_kv) + (int64_t)n * p.c_s + 8 * lane;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) x[s] = raw8(c + 128 * s, p.vec);
    if (p.DR && lane < 8)
      y = raw8(static_cast<const T*>(p.k_rope) + (int64_t)n * p.k_s + 8 * lane, p.vec);
  }
  // where it goes, while its values are on their way
  int b, pos, page = -1;
  locate(p, min(n, p.N - 1), b, pos);
  if (live && pos >= 0) page = page_of(p, b, pos);
  uint32_t amax = 0, rmax = max8(0, y);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) amax = max8(amax, x[s]);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    amax = __vmaxu2(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    rmax = __vmaxu2(rmax, __shfl_xor_sync(0xffffffffu, rmax, o));
  }
  if (!live || pos < 0) return;
  if (page < 0) {
    if (lane == 0) atomicExch(&g_cache_device_error, kErrOutside);
    return;
  }
  const int off = pos & (p.page_size - 1);
  const int e = scale_exp(to_float_bits<T>(max(amax & 0xffffu, amax >> 16)),
                          to_float_bits<T>(max(rmax & 0xffffu, rmax >> 16)));
  const float inv = pow2i(-e);
  uint8_t* q = p.codes + (int64_t)page * p.codes_s[0] + (int64_t)off * p.codes_s[1] + 8 * lane;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const T* v = reinterpret_cast<const T*>(&x[s]);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = ld(v + i) * inv;
    *reinterpret_cast<uint2*>(q + 128 * s) =
        make_uint2(to_e4m3x4(f[0], f[1], f[2], f[3]), to_e4m3x4(f[4], f[5], f[6], f[7]));
  }
  if (p.DR && lane < 8) {
    const T* v = reinterpret_cast<const T*>(&y);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = ld(v + i) * inv;
    st8(static_cast<T*>(p.rope) + (int64_t)page * p.rope_s[0] + (int64_t)off * p.rope_s[1] +
            8 * lane, true, f);
  }
  if (lane == 0) p.scales[(int64_t)page * p.scales_s + off] = pow2i(e);
}

template <typename T, int STEPS>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const CacheParams p) {
  const int lane = threadIdx.x % kLanes;
  const int n = blockIdx.x * kTokens + threadIdx.x / kLanes;
  int b, pos;
  locate(p, min(n, p.N - 1), b, pos);
  if (n >= p.N) return;
  int page = -1;
  if (pos >= 0) {
    page = page_of(p, b, pos);
    if (page < 0 && lane == 0) atomicExch(&g_cache_device_error, kErrOutside);
  }
  T* c = static_cast<T*>(p.c_kv) + (int64_t)n * p.c_s + 8 * lane;
  T* k = static_cast<T*>(p.k_rope) + (int64_t)n * p.k_s + 8 * lane;
  float x[8];
  if (page < 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) st8(c + 128 * s, p.vec, x);
    if (p.DR && lane < 8) st8(k, p.vec, x);
    return;
  }
  const int off = pos & (p.page_size - 1);
  const uint8_t* q = p.codes + (int64_t)page * p.codes_s[0] + (int64_t)off * p.codes_s[1] + 8 * lane;
  uint2 u[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) u[s] = *reinterpret_cast<const uint2*>(q + 128 * s);
  float y[8];
  if (p.DR && lane < 8)
    ld8(static_cast<const T*>(p.rope) + (int64_t)page * p.rope_s[0] + (int64_t)off * p.rope_s[1] +
            8 * lane, true, y);
  const float sc = p.scales[(int64_t)page * p.scales_s + off];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const uint32_t w[4] = {u[s].x, u[s].x >> 16, u[s].y, u[s].y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = from_e4m3x2(w[i]);
      x[2 * i] = f.x * sc;
      x[2 * i + 1] = f.y * sc;
    }
    st8(c + 128 * s, p.vec, x);
  }
  if (p.DR && lane < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= sc;
    st8(k, p.vec, y);
  }
}

template <typename T>
cudaError_t launch_tokens(const CacheParams& p, bool append, cudaStream_t s) {
  const dim3 grid((p.N + kTokens - 1) / kTokens);
  using K = void (*)(CacheParams);
  static const K kernels[2][4] = {
      {cache_read_kernel<T, 1>, cache_read_kernel<T, 2>, cache_read_kernel<T, 3>,
       cache_read_kernel<T, 4>},
      {cache_append_kernel<T, 1>, cache_append_kernel<T, 2>, cache_append_kernel<T, 3>,
       cache_append_kernel<T, 4>}};
  kernels[append ? 1 : 0][p.KVL / 128 - 1]<<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

bool aligned16(const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; }

// The pool, the table and the sizes, whatever the call does with them.
int validate(const MlaCacheArgs* a) {
  if (a == nullptr) return KDA_ERR_NULL_POINTER;
  if (a->abi_version != KDA_B200_ABI_VERSION) return KDA_ERR_SHAPE;
  if (a->io_dtype != KDA_DTYPE_F16 && a->io_dtype != KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
  if (a->KVL < 128 || a->KVL > 512 || a->KVL % 128 != 0) return KDA_ERR_SHAPE;
  if (a->DR != 0 && a->DR != 64) return KDA_ERR_SHAPE;
  if (a->page_size < 16 || a->page_size > 1024 || (a->page_size & (a->page_size - 1)) != 0)
    return KDA_ERR_SHAPE;
  if (a->num_pages < 1 || (int64_t)a->num_pages * a->page_size >= (1ll << 31)) return KDA_ERR_SHAPE;
  if (a->B < 0 || a->N < 0 || a->max_pages < 0 || a->max_pages > (1 << 24)) return KDA_ERR_SHAPE;
  if ((int64_t)a->max_pages * a->page_size > (1ll << 30)) return KDA_ERR_SHAPE;
  if (a->N == 0) return KDA_OK;                            // nothing to do
  if (a->B > 0 && a->q_start == nullptr && a->N % a->B != 0) return KDA_ERR_SHAPE;
  if (!a->codes || !a->scales || (a->DR && !a->rope) ||
      (a->B > 0 && (!a->lens || (a->max_pages > 0 && !a->block_table))))
    return KDA_ERR_NULL_POINTER;
  if (!aligned16(a->codes) || a->codes_stride[0] % 16 || a->codes_stride[1] % 16 ||
      reinterpret_cast<uintptr_t>(a->scales) % 4)
    return KDA_ERR_ALIGNMENT;
  if (a->codes_stride[0] < (a->num_pages > 1) || a->codes_stride[1] < a->KVL || a->scales_stride < 0 ||
      a->table_stride < 0)
    return KDA_ERR_STRIDE;
  if (a->DR) {
    if (!aligned16(a->rope) || a->rope_stride[0] % 8 || a->rope_stride[1] % 8)
      return KDA_ERR_ALIGNMENT;
    if (a->rope_stride[0] < (a->num_pages > 1) || a->rope_stride[1] < a->DR) return KDA_ERR_STRIDE;
  }
  return KDA_OK;
}

CacheParams to_params(const MlaCacheArgs* a) {
  CacheParams p{};
  p.num_pages = a->num_pages; p.page_size = a->page_size;
  while ((1 << p.page_shift) < a->page_size) ++p.page_shift;
  p.KVL = a->KVL; p.DR = a->DR;
  p.B = a->B; p.N = a->N; p.H = a->H; p.max_pages = a->max_pages;
  p.scale = a->scale;
  p.codes = static_cast<uint8_t*>(a->codes);
  std::memcpy(p.codes_s, a->codes_stride, sizeof(p.codes_s));
  p.scales = a->scales; p.scales_s = a->scales_stride;
  p.rope = a->rope; std::memcpy(p.rope_s, a->rope_stride, sizeof(p.rope_s));
  p.table = a->block_table; p.table_s = a->table_stride;
  p.lens = a->lens; p.q_start = a->q_start;
  p.c_kv = a->c_kv; p.c_s = a->c_kv_stride;
  p.k_rope = a->k_rope; p.k_s = a->k_rope_stride;
  p.q_lat = a->q_lat; std::memcpy(p.ql_s, a->q_lat_stride, sizeof(p.ql_s));
  p.q_rope = a->q_rope; std::memcpy(p.qr_s, a->q_rope_stride, sizeof(p.qr_s));
  p.out = a->out; std::memcpy(p.o_s, a->out_stride, sizeof(p.o_s));
  p.lse = a->lse; p.lse_s = a->lse_stride;
  return p;
}

int check_device() {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
    return KDA_ERR_LAUNCH;
  return major == 10 ? KDA_OK : KDA_ERR_ARCH;
}

int run_tokens(const MlaCacheArgs* a, bool append, void* stream) {
  int st = validate(a);
  if (st != KDA_OK) return st;
  if (a->N == 0 || (append && a->B == 0)) return KDA_OK;
  if (!a->c_kv || (a->DR && !a->k_rope)) return KDA_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(a->c_kv) % 2 || reinterpret_cast<uintptr_t>(a->k_rope) % 2)
    return KDA_ERR_ALIGNMENT;
  if ((st = check_device()) != KDA_OK) return st;
  CacheParams p = to_params(a);
  p.vec = aligned16(a->c_kv) && a->c_kv_stride % 8 == 0 &&
          (!a->DR || (aligned16(a->k_rope) && a->k_rope_stride % 8 == 0));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->io_dtype == KDA_DTYPE_F16 ? launch_tokens<__half>(p, append, s)
                                                     : launch_tokens<__nv_bfloat16>(p, append, s);
  return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

int validate_attention(const MlaCacheArgs* a) {
  const int st = validate(a);
  if (st != KDA_OK) return st;
  if (a->H < 0 || a->H > 1024 || (int64_t)a->N * a->H > (1ll << 30)) return KDA_ERR_SHAPE;
  if (a->N == 0 || a->H == 0) return KDA_OK;
  if (!a->q_lat || !a->out || (a->DR && !a->q_rope)) return KDA_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(a->q_lat) % 2 || reinterpret_cast<uintptr_t>(a->q_rope) % 2 ||
      reinterpret_cast<uintptr_t>(a->out) % 2 || reinterpret_cast<uintptr_t>(a->lse) % 4)
    return KDA_ERR_ALIGNMENT;
  return KDA_OK;
}

}  // namespace

int read_device_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_cache_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace cache
}  // namespace kda

extern "C" {

size_t mla_cache_args_size(void) { return sizeof(MlaCacheArgs); }

int mla_cache_append(const MlaCacheArgs* a, void* stream) {
  return kda::cache::run_tokens(a, true, stream);
}

int mla_cache_read(const MlaCacheArgs* a, void* stream) {
  return kda::cache::run_tokens(a, false, stream);
}

size_t mla_cache_workspace_bytes(const MlaCacheArgs* a) {
  using namespace kda::cache;
  if (validate_attention(a) != KDA_OK || a->N == 0 || a->H == 0) return 0;
  return attention_workspace_bytes(to_params(a), a->io_dtype);
}

int mla_cache_attention(const MlaCacheArgs* a, void* stream) {
  using namespace kda::cache;
  int st = validate_attention(a);
  if (st != KDA_OK) return st;
  if (a->N == 0 || a->H == 0) return KDA_OK;
  CacheParams p = to_params(a);
  const size_t need = attention_workspace_bytes(p, a->io_dtype);
  if (need && (a->workspace == nullptr || a->workspace_bytes < need)) return KDA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) % 256) return KDA_ERR_ALIGNMENT;
  if ((st = check_device()) != KDA_OK) return st;
  p.vec = aligned16(a->q_lat) && a->q_lat_stride[0] % 8 == 0 && a->q_lat_stride[1] % 8 == 0 &&
          (!a->DR || (aligned16(a->q_rope) && a->q_rope_stride[0] % 8 == 0 &&
                      a->q_rope_stride[1] % 8 == 0));
  p.h_mul = p.H == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / p.H);
  p.out_vec = reinterpret_cast<uintptr_t>(a->out) % 4 == 0 && a->out_stride[0] % 2 == 0 &&
              a->out_stride[1] % 2 == 0;
  const cudaError_t e =
      launch_attention(p, a->io_dtype, a->workspace, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // extern "C"
