// mla_cache_attn.cu -- absorbed-form latent attention over the 8-bit paged cache.
//
// One block per (new token, head).  Each warp walks every eighth position of
// the sequence with its own running maximum and sum (fp32): the lanes hold the
// query and the accumulator of KVL / 32 channels, a score is one shuffle
// reduction.  The warps join at the end.
#include "mla_cache.cuh"

namespace kda {
namespace cache {

__device__ int g_attn_device_error = 0;

namespace {

constexpr int kWarps = 8;

template <typename T, int STEPS>   // KVL = 128 STEPS
__global__ void __launch_bounds__(kWarps * 32)
cache_attn_kernel(const CacheParams p) {
  constexpr int C = 4 * STEPS;     // channels per lane: 4 lane + 128 s + i
  __shared__ float acc_s[kWarps][128 * STEPS];
  __shared__ float m_s[kWarps], l_s[kWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int n = blockIdx.x, h = blockIdx.y;
  int b, pos;
  locate(p, n, b, pos);
  const int64_t table_end = (int64_t)p.max_pages * p.page_size;
  if (pos >= table_end) {
    if (threadIdx.x == 0) atomicExch(&g_attn_device_error, kErrOutside);
    pos = (int)table_end - 1;
  }
  float q[C], qr[2] = {0.f, 0.f}, acc[C];
  const T* ql = static_cast<const T*>(p.q_lat) + (int64_t)n * p.ql_s[0] + (int64_t)h * p.ql_s[1];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    q[i] = ld(ql + 4 * lane + 128 * (i / 4) + i % 4);
    acc[i] = 0.f;
  }
  if (p.DR) {
    const T* r = static_cast<const T*>(p.q_rope) + (int64_t)n * p.qr_s[0] + (int64_t)h * p.qr_s[1];
    qr[0] = ld(r + 2 * lane);
    qr[1] = ld(r + 2 * lane + 1);
  }
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t <= pos; t += kWarps) {
    const int page = page_of(p, b, t);
    if (page < 0) {
      if (lane == 0) atomicExch(&g_attn_device_error, kErrOutside);
      m = l = __uint_as_float(0x7fffffffu);
      break;
    }
    const int off = t & (p.page_size - 1);
    const uint8_t* c = p.codes + (int64_t)page * p.codes_s[0] + (int64_t)off * p.codes_s[1];
    const float s = p.scales[(int64_t)page * p.scales_s + off];
    float x[C], dot = 0.f;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(c + 128 * k + 4 * lane);
      const float2 lo = from_e4m3x2(u), hi = from_e4m3x2(u >> 16);
      x[4 * k] = lo.x; x[4 * k + 1] = lo.y; x[4 * k + 2] = hi.x; x[4 * k + 3] = hi.y;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      x[i] *= s;
      dot = fmaf(q[i], x[i], dot);
    }
    if (p.DR) {
      const T* r = static_cast<const T*>(p.rope) + (int64_t)page * p.rope_s[0] +
                   (int64_t)off * p.rope_s[1];
      dot = fmaf(qr[0], ld(r + 2 * lane) * s, dot);
      dot = fmaf(qr[1], ld(r + 2 * lane + 1) * s, dot);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float z = dot * p.scale;
    const float mn = fmaxf(m, z);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float a = expf(m - mu), w = expf(z - mu);
    l = l * a + w;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = acc[i] * a + w * x[i];
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < C; ++i) acc_s[warp][4 * lane + 128 * (i / 4) + i % 4] = acc[i];
  if (lane == 0) { m_s[warp] = m; l_s[warp] = l; }
  __syncthreads();
  float mx = -INFINITY, tot = 0.f, wt[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, m_s[w]);
  const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    wt[w] = expf(m_s[w] - mu);
    tot += wt[w] * l_s[w];
  }
  T* o = static_cast<T*>(p.out) + (int64_t)n * p.o_s[0] + (int64_t)h * p.o_s[1];
  for (int c = threadIdx.x; c < p.KVL; c += kWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += wt[w] * acc_s[w][c];
    st(o + c, tot == 0.f ? 0.f : x / tot);
  }
  if (threadIdx.x == 0 && p.lse) p.lse[(int64_t)n * p.lse_s + h] = mu + logf(tot);
}

template <typename T>
cudaError_t launch(const CacheParams& p, cudaStream_t s) {
  using K = void (*)(CacheParams);
  static const K kernels[4] = {cache_attn_kernel<T, 1>, cache_attn_kernel<T, 2>,
                               cache_attn_kernel<T, 3>, cache_attn_kernel<T, 4>};
  kernels[p.KVL / 128 - 1]<<<dim3(p.N, p.H), kWarps * 32, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t attention_workspace_bytes(const CacheParams&) { return 0; }

cudaError_t launch_attention(const CacheParams& p, int io_dtype, void*, cudaStream_t s) {
  return io_dtype == KDA_DTYPE_F16 ? launch<__half>(p, s) : launch<__nv_bfloat16>(p, s);
}

int read_attn_device_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_attn_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace cache
}  // namespace kda
