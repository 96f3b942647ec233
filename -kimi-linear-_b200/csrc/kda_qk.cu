// kda_qk.cu -- queries and keys normalised per head and rotated by position, the
// gradient, and their C entry points (include/kda_b200.h).
//
// Forward, per head of a token: n = x r, z = n w, y = rotation of z by p f_i.
// Gradient: dz = rotation of dy by -p f_i,  dw = sum over tokens (and heads) of dz n,
//   v = dz w,  dx = r (v - n dot),  dot = mean(v n) for the root mean square, sum(v n)
//   for length one, 0 where 1 / eps caps r and without a norm.
// n is computed again from x.  Sums are fp32, dw's last ones fp64, all in a fixed order.
//
// A warp has a row (one head of one token), a lane every 32nd channel.
#include <cstring>

#include "kda_internal.cuh"

namespace kda {
namespace qk {

namespace {

constexpr int kThreads = 128;
constexpr int kMaxD = 512;
constexpr int kItems = kMaxD / 32;

// Device-side view of KdaQkArgs (strides in elements).
struct QkParams {
  int B, T, D, R;
  int64_t tokens;                   // B T
  int heads[2];
  int norm;
  bool interleaved, w_heads, pos_64;
  int w_dtype, pos_step;
  float eps;
  const void* x[2]; int64_t x_s[2][3];
  const void* w[2];
  const void* positions; int64_t pos_s[2];
  const float* inv_freq;
  void* y[2]; int64_t y_s[2][3];
  const void* dy[2]; int64_t dy_s[2][3];
  void* dx[2]; int64_t dx_s[2][3];
  void* dw[2];
  float* partial;                   // [chunks][heads of both][D]
  int chunks, per_chunk;            // tokens of a chunk
};

__device__ __forceinline__ float load_weight(const QkParams& p, int which, int head, int c) {
  if (p.w[which] == nullptr) return 1.f;
  const int64_t i = (p.w_heads ? (int64_t)head * p.D : 0) + c;
  if (p.w_dtype == KDA_DTYPE_F32) return static_cast<const float*>(p.w[which])[i];
  if (p.w_dtype == KDA_DTYPE_F16) return ld(static_cast<const __half*>(p.w[which]) + i);
  return ld(static_cast<const __nv_bfloat16*>(p.w[which]) + i);
}

__device__ __forceinline__ int64_t position(const QkParams& p, int b, int t) {
  const int64_t at = b * p.pos_s[0] + t * p.pos_s[1], step = (int64_t)t * p.pos_step;
  if (p.positions == nullptr) return step;
  return step + (p.pos_64 ? static_cast<const int64_t*>(p.positions)[at]
                          : (int64_t) static_cast<const int32_t*>(p.positions)[at]);
}

// Cosine and sine of pos f.  The angle is reduced in 64 bits, to an eighth of a turn
// either way, so that what is rounded to 32 is below pi / 4 however far the position.
__device__ __forceinline__ float2 angle(int64_t pos, float f) {
  const double quarters = (double)pos * ((double)f * 0.63661977236758134308);   // 2 / pi
  const double whole = rint(quarters);
  float s, c;
  sincospif((float)(quarters - whole) * 0.5f, &s, &c);
  const int q = (int)((long long)whole & 3);
  return q == 0 ? make_float2(c, s) : q == 1 ? make_float2(-s, c)
       : q == 2 ? make_float2(-c, -s) : make_float2(s, -c);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// r of a row with sum of squares ss; where ss has overflowed, `tiny` is the sum of the
// squares of 2^-70 x.  Also whether r depends on x.
struct Rate { float r; bool moves; };
__device__ __forceinline__ Rate rate(const QkParams& p, float ss, float tiny) {
  if (p.norm == KDA_NORM_NONE) return {1.f, false};
  const bool big = !(ss <= 3.4e38f);
  if (p.norm == KDA_NORM_RMS) {
    const float m = big ? tiny / p.D : ss / p.D + p.eps;
    return {__frsqrt_rn(m) * (big ? 0x1p-70f : 1.f), true};
  }
  const float r = __frsqrt_rn(big ? tiny : ss) * (big ? 0x1p-70f : 1.f), cap = 1.f / p.eps;
  return r < cap ? Rate{r, true} : r >= cap ? Rate{cap, false} : Rate{r, true};
}

// A row's sum of squares: x as it is, or where that overflows, of 2^-70 x.
__device__ __forceinline__ Rate rate_of(const QkParams& p, const float (&x)[kItems]) {
  float ss = 0.f;
  if (p.norm == KDA_NORM_NONE) return {1.f, false};
#pragma unroll
  for (int i = 0; i < kItems; ++i) ss = fmaf(x[i], x[i], ss);
  ss = warp_sum(ss);
  float tiny = 0.f;
  if (!(ss <= 3.4e38f)) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) tiny = fmaf(x[i] * 0x1p-70f, x[i] * 0x1p-70f, tiny);
    tiny = warp_sum(tiny);
  }
  return rate(p, ss, tiny);
}

// Channels 0 .. R - 1 rotated by sign p f; `buf`: the warp's own.
__device__ __forceinline__ void rotate(const QkParams& p, float (&z)[kItems], int64_t pos, float sign,
                                       float* buf, int lane) {
  if (p.R == 0) return;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (lane + 32 * i < p.R) buf[lane + 32 * i] = z[i];
  __syncwarp();
  const int half = p.R / 2;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int e = lane + 32 * i;
    if (e >= p.R) continue;
    const bool second = p.interleaved ? e & 1 : e >= half;
    const int pair = p.interleaved ? e >> 1 : second ? e - half : e;
    const int other = p.interleaved ? e ^ 1 : second ? e - half : e + half;
    const float2 cs = angle(pos, p.inv_freq[pair]);
    z[i] = fmaf(second ? sign * cs.y : -sign * cs.y, buf[other], z[i] * cs.x);
  }
}

template <typename T>
__device__ __forceinline__ void load_row(const QkParams& p, const void* base, const int64_t* s, int b, int t,
                                         int head, int lane, float (&v)[kItems]) {
  const T* row = static_cast<const T*>(base) + b * s[0] + t * s[1] + head * s[2];
#pragma unroll
  for (int i = 0; i < kItems; ++i) v[i] = lane + 32 * i < p.D ? ld(row + lane + 32 * i) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_row(const QkParams& p, void* base, const int64_t* s, int b, int t,
                                          int head, int lane, const float (&v)[kItems]) {
  T* row = static_cast<T*>(base) + b * s[0] + t * s[1] + head * s[2];
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (lane + 32 * i < p.D) st(row + lane + 32 * i, v[i]);
}

// Block (chunk, head): the chunk's tokens of one head, a token a warp in turn.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads) qk_kernel(const QkParams p) {
  __shared__ float rows[kThreads / 32][kMaxD];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int which = (int)blockIdx.y >= p.heads[0], head = blockIdx.y - (which ? p.heads[0] : 0);
  float* buf = rows[warp];
  float w[kItems], dw[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    w[i] = lane + 32 * i < p.D ? load_weight(p, which, head, lane + 32 * i) : 0.f;
    dw[i] = 0.f;
  }
  const int64_t first = (int64_t)blockIdx.x * p.per_chunk;
  const int64_t last = min(first + p.per_chunk, p.tokens);
  for (int64_t n = first + warp; n < last; n += kThreads / 32) {
    const int b = (int)(n / p.T), t = (int)(n - (int64_t)b * p.T);
    const int64_t pos = position(p, b, t);
    float x[kItems];
    load_row<T>(p, p.x[which], p.x_s[which], b, t, head, lane, x);
    const Rate rt = rate_of(p, x);
    if constexpr (!GRAD) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) x[i] = x[i] * rt.r * w[i];
      rotate(p, x, pos, 1.f, buf, lane);
      store_row<T>(p, p.y[which], p.y_s[which], b, t, head, lane, x);
    } else {
      float dz[kItems], dot = 0.f;
      load_row<T>(p, p.dy[which], p.dy_s[which], b, t, head, lane, dz);
      rotate(p, dz, pos, -1.f, buf, lane);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        x[i] *= rt.r;
        dw[i] = fmaf(dz[i], x[i], dw[i]);
        dz[i] *= w[i];
        dot = fmaf(dz[i], x[i], dot);
      }
      dot = rt.moves ? warp_sum(dot) / (p.norm == KDA_NORM_RMS ? p.D : 1) : 0.f;
#pragma unroll
      for (int i = 0; i < kItems; ++i) dz[i] = rt.r * (rt.moves ? fmaf(-x[i], dot, dz[i]) : dz[i]);
      store_row<T>(p, p.dx[which], p.dx_s[which], b, t, head, lane, dz);
    }
  }
  if (GRAD && p.dw[which] != nullptr) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kItems; ++i) buf[lane + 32 * i] = dw[i];
    __syncthreads();
    float* out = p.partial + ((int64_t)blockIdx.x * (p.heads[0] + p.heads[1]) + blockIdx.y) * p.D;
    for (int c = threadIdx.x; c < p.D; c += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) s += rows[i][c];
      out[c] = s;
    }
  }
}

// dw = sum of the partials over chunks, and over heads where they share a weight.
// Block: 32 channels of one weight row; thread (r, c) adds every eighth partial.
__global__ void __launch_bounds__(256) qk_weight_kernel(const QkParams p) {
  __shared__ double sums[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, r = threadIdx.x / 32;
  const int q_rows = p.w_heads ? p.heads[0] : 1;
  const int which = (int)blockIdx.y >= q_rows, row = blockIdx.y - (which ? q_rows : 0);
  if (p.dw[which] == nullptr) return;
  const int all = p.heads[0] + p.heads[1];
  const int head0 = (which ? p.heads[0] : 0) + (p.w_heads ? row : 0);
  const int n = p.w_heads ? 1 : p.heads[which];
  double s = 0.;
  if (c < p.D)
    for (int64_t i = r; i < (int64_t)p.chunks * n; i += 8)
      s += p.partial[((i / n) * all + head0 + i % n) * p.D + c];
  sums[r][threadIdx.x % 32] = s;
  __syncthreads();
  if (r > 0 || c >= p.D) return;
  s = 0.;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += sums[i][threadIdx.x % 32];
  const int64_t at = (int64_t)(p.w_heads ? row : 0) * p.D + c;
  if (p.w_dtype == KDA_DTYPE_F32) static_cast<float*>(p.dw[which])[at] = (float)s;
  else if (p.w_dtype == KDA_DTYPE_F16) st(static_cast<__half*>(p.dw[which]) + at, (float)s);
  else st(static_cast<__nv_bfloat16*>(p.dw[which]) + at, (float)s);
}

int size_of(int dt) { return dt == KDA_DTYPE_F32 ? 4 : 2; }
bool misaligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

int validate(const KdaQkArgs* a) {
  if (a == nullptr) return KDA_ERR_NULL_POINTER;
  if (a->abi_version != KDA_B200_ABI_VERSION) return KDA_ERR_SHAPE;
  if (a->B < 0 || a->T < 0 || (int64_t)a->B * a->T > (1ll << 40)) return KDA_ERR_SHAPE;
  if (a->D < 1 || a->D > kMaxD || a->R < 0 || a->R > a->D || a->R % 2) return KDA_ERR_SHAPE;
  if (a->heads[0] < 0 || a->heads[1] < 0 || a->heads[0] > 16384 || a->heads[1] > 16384) return KDA_ERR_SHAPE;
  if (a->io_dtype < KDA_DTYPE_F32 || a->io_dtype > KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
  if (a->w_dtype < KDA_DTYPE_F32 || a->w_dtype > KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
  if (a->norm < KDA_NORM_NONE || a->norm > KDA_NORM_L2) return KDA_ERR_SHAPE;
  if (a->norm != KDA_NORM_NONE && !(a->eps >= 1e-12f)) return KDA_ERR_SHAPE;
  if (a->R > 0 && a->inv_freq == nullptr) return KDA_ERR_NULL_POINTER;
  if (misaligned(a->inv_freq, 4) || misaligned(a->positions, a->pos_64 ? 8 : 4) || misaligned(a->partial, 4))
    return KDA_ERR_ALIGNMENT;
  for (int i = 0; i < 2; ++i) {
    const int e = size_of(a->io_dtype), we = size_of(a->w_dtype);
    if (misaligned(a->x[i], e) || misaligned(a->y[i], e) || misaligned(a->dy[i], e) ||
        misaligned(a->dx[i], e) || misaligned(a->w[i], we) || misaligned(a->dw[i], we))
      return KDA_ERR_ALIGNMENT;
    if (a->dw[i] != nullptr && a->w[i] == nullptr) return KDA_ERR_NULL_POINTER;
  }
  return KDA_OK;
}

// How the tokens are cut: chunks enough for every SM to have several blocks, of at least
// four tokens for each warp.
void cut(QkParams& p) {
  const int heads = p.heads[0] + p.heads[1];
  const int64_t want = max((int64_t)1, (int64_t)(148 * 16) / max(heads, 1));
  int64_t per = (p.tokens + want - 1) / want;
  per = max(per, (int64_t)(kThreads / 32 * 4));
  p.per_chunk = (int)min(per, (int64_t)1 << 30);
  p.chunks = (int)((p.tokens + p.per_chunk - 1) / p.per_chunk);
}

QkParams to_params(const KdaQkArgs* a) {
  QkParams p{};
  p.B = a->B; p.T = a->T; p.D = a->D; p.R = a->R;
  p.tokens = (int64_t)a->B * a->T;
  p.norm = a->norm;
  p.interleaved = a->interleaved != 0; p.w_heads = a->w_heads != 0; p.pos_64 = a->pos_64 != 0;
  p.w_dtype = a->w_dtype; p.pos_step = a->pos_step; p.eps = a->eps;
  p.positions = a->positions; std::memcpy(p.pos_s, a->pos_stride, sizeof(p.pos_s));
  p.inv_freq = a->inv_freq;
  for (int i = 0; i < 2; ++i) {
    p.heads[i] = a->heads[i];
    p.x[i] = a->x[i]; p.w[i] = a->w[i]; p.y[i] = a->y[i];
    p.dy[i] = a->dy[i]; p.dx[i] = a->dx[i]; p.dw[i] = a->dw[i];
  }
  std::memcpy(p.x_s, a->x_stride, sizeof(p.x_s));
  std::memcpy(p.y_s, a->y_stride, sizeof(p.y_s));
  std::memcpy(p.dy_s, a->dy_stride, sizeof(p.dy_s));
  std::memcpy(p.dx_s, a->dx_stride, sizeof(p.dx_s));
  p.partial = a->partial;
  cut(p);
  return p;
}

int check_device() {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
    return KDA_ERR_LAUNCH;
  return major == 10 ? KDA_OK : KDA_ERR_ARCH;
}

template <bool GRAD>
cudaError_t launch(const QkParams& p, int io, cudaStream_t s) {
  const dim3 grid(p.chunks, p.heads[0] + p.heads[1]);
  if (io == KDA_DTYPE_F32) qk_kernel<float, GRAD><<<grid, kThreads, 0, s>>>(p);
  else if (io == KDA_DTYPE_F16) qk_kernel<__half, GRAD><<<grid, kThreads, 0, s>>>(p);
  else qk_kernel<__nv_bfloat16, GRAD><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

size_t partial_floats(const QkParams& p) {
  return (size_t)p.chunks * (p.heads[0] + p.heads[1]) * p.D;
}

int run(const KdaQkArgs* a, bool grad, void* stream) {
  int st = validate(a);
  if (st != KDA_OK) return st;
  const QkParams p = to_params(a);
  const bool weights = grad && (p.dw[0] || p.dw[1]);
  const bool rows = p.tokens > 0 && p.heads[0] + p.heads[1] > 0;
  if (!rows && !weights) return KDA_OK;
  for (int i = 0; i < 2 && p.tokens > 0; ++i) {
    if (p.heads[i] == 0) continue;
    if (!p.x[i] || (grad ? !p.dy[i] || !p.dx[i] : !p.y[i])) return KDA_ERR_NULL_POINTER;
  }
  if (weights && rows && (!p.partial || a->partial_floats < partial_floats(p))) return KDA_ERR_WORKSPACE;
  if ((st = check_device()) != KDA_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (rows) e = grad ? launch<true>(p, a->io_dtype, s) : launch<false>(p, a->io_dtype, s);
  if (e == cudaSuccess && weights) {
    const int n = p.w_heads ? p.heads[0] + p.heads[1] : 2;
    if (n > 0) {
      qk_weight_kernel<<<dim3((p.D + 31) / 32, n), 256, 0, s>>>(p);
      e = cudaGetLastError();
    }
  }
  return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // namespace
}  // namespace qk
}  // namespace kda

extern "C" {

size_t kda_qk_args_size(void) { return sizeof(KdaQkArgs); }

size_t kda_qk_partial_floats(const KdaQkArgs* a) {
  if (kda::qk::validate(a) != KDA_OK) return 0;
  return kda::qk::partial_floats(kda::qk::to_params(a));
}

int kda_qk_fwd(const KdaQkArgs* a, void* stream) { return kda::qk::run(a, false, stream); }
int kda_qk_bwd(const KdaQkArgs* a, void* stream) { return kda::qk::run(a, true, stream); }

}  // extern "C"
