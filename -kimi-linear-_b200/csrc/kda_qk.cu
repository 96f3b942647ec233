// kda_qk.cu -- queries and keys normalised per head and rotated by position, the
// gradient, and their C entry points (include/kda_b200.h).
//
// Forward, per head of a token: n = x r, z = n w, y = rotation of z by p f_i.
// Gradient: dz = rotation of dy by -p f_i,  dw = sum over tokens (and heads) of dz n,
//   v = dz w,  dx = r (v - n dot),  dot = mean(v n) for the root mean square, sum(v n)
//   for length one, 0 where 1 / eps caps r and without a norm.
// n is computed again from x.  Sums are fp32, dw's last ones fp64, all in a fixed order.
//
// Memory bounds both at length.  A lane has two groups of 16 bytes of a row (or 8, where
// the rows are aligned to no more): those that the rotation pairs (i and i + R / 2), or
// neighbours, so that a pair is always in one lane.  (With 8 bytes a group always, instructions,
// 216 for eight channels of 16 bits with their rotation, bound the kernel; now 121.  4 x 8192 tokens of
// 32 heads of 128, f16: 92 us, 89 % of what a copy reaches; gradient 136 us, 90 %.)
// Rows of one token share its angles: a block has the heads of a few tokens side by side and
// puts cosines and sines into shared memory for a batch of tokens.  (head_kernel)  Rows that
// this does not fit (head sizes or strides that are no multiples of the groups) have a warp
// each, a lane every 32nd channel.  (row_kernel)
#include <cstring>
#include <type_traits>

#include "kda_internal.cuh"

namespace kda {
namespace qk {

namespace {

constexpr int kThreads = 128;
constexpr int kMaxD = 512;
constexpr int kItems = kMaxD / 32;
constexpr int kSms = 148;
constexpr int kUnroll = 2;   // rows of a thread on their way in head_kernel

// Device-side view of KdaQkArgs (strides in elements).
struct QkParams {
  int B, T, D, R;
  int tokens;                       // B T
  uint32_t t_mul;                   // 2^32 / T, rounded down (T = 1: 2^32 - 1)
  int heads[2];
  int norm;
  bool interleaved, w_heads, pos_64;
  int w_dtype, pos_step;
  float eps, cap, inv_D;            // cap = 1 / eps
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
  int span, chunks_span;            // (head_kernel) tokens that lie at one step, and their chunks
};

__device__ __forceinline__ float load_weight(const QkParams& p, int which, int head, int c) {
  if (p.w[which] == nullptr) return 1.f;
  const int64_t i = (p.w_heads ? (int64_t)head * p.D : 0) + c;
  if (p.w_dtype == KDA_DTYPE_F32) return static_cast<const float*>(p.w[which])[i];
  if (p.w_dtype == KDA_DTYPE_F16) return ld(static_cast<const __half*>(p.w[which]) + i);
  return ld(static_cast<const __nv_bfloat16*>(p.w[which]) + i);
}

// Token n is token t of sequence b.
struct Token { int b, t; };
__device__ __forceinline__ Token token(const QkParams& p, int n) {
  int b = (int)__umulhi((uint32_t)n, p.t_mul);      // short by one at most
  int t = n - b * p.T;
  if (t >= p.T) {
    ++b;
    t -= p.T;
  }
  return {b, t};
}
__device__ __forceinline__ int64_t offset(const Token& k, const int64_t* s) { return k.b * s[0] + k.t * s[1]; }
__device__ __forceinline__ int64_t position(const QkParams& p, const Token& k) {
  const int64_t at = offset(k, p.pos_s), step = (int64_t)k.t * p.pos_step;
  if (p.positions == nullptr) return step;
  return step + (p.pos_64 ? static_cast<const int64_t*>(p.positions)[at]
                          : (int64_t) static_cast<const int32_t*>(p.positions)[at]);
}

// Cosine and sine of an angle of `quarters` quarter turns.  It is reduced in 64 bits, to an eighth
// of a turn either way, so that what is rounded to 32 is below pi / 4 however far the
// position; there both are their series, up to z^9/9! and z^10/10!, whose first terms left out
// are below 2^-28.
__device__ __forceinline__ double quarter_rate(float f) { return (double)f * 0.63661977236758134308; }   // 2 / pi
__device__ __forceinline__ float2 angle(double quarters) {
  const double whole = rint(quarters);
  const float z = (float)(quarters - whole) * 1.57079632679489662f;
  const float y = z * z;
  float s = fmaf(y, 1.f / 362880.f, -1.f / 5040.f), c = fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
  s = fmaf(s, y, 1.f / 120.f);
  c = fmaf(c, y, -1.f / 720.f);
  s = fmaf(s, y, -1.f / 6.f);
  c = fmaf(c, y, 1.f / 24.f);
  s = fmaf(s * y, z, z);
  c = fmaf(c, y, -0.5f);
  c = fmaf(c, y, 1.f);
  const int q = __double2loint(whole + 6755399441055744.0) & 3;   // 1.5 2^52: whole numbers end in the last bit
  const float a = q & 1 ? s : c, b = q & 1 ? c : s;
  return make_float2(q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// r of a row with sum of squares ss; where ss has overflowed, `tiny` is the sum of the
// squares of 2^-70 x.  Also whether r depends on x.
struct Rate { float r; bool moves; };
__device__ __forceinline__ float rsqrt_fast(float m) {    // off by two units in the last place; infinity for 0
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(m));
  return r;
}
__device__ __forceinline__ Rate rate(const QkParams& p, float ss, float tiny) {
  if (p.norm == KDA_NORM_NONE) return {1.f, false};
  const bool big = !(ss <= 3.4e38f), rms = p.norm == KDA_NORM_RMS;
  // (2^-140 eps is nothing to the mean of squares that overflow)
  float r = rsqrt_fast(rms ? fmaf(big ? tiny : ss, p.inv_D, big ? 0.f : p.eps) : big ? tiny : ss);
  if (big) r *= 0x1p-70f;
  return rms || !(r >= p.cap) ? Rate{r, true} : Rate{p.cap, false};
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
    const float2 cs = angle((double)pos * quarter_rate(p.inv_freq[pair]));
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
__global__ void __launch_bounds__(kThreads) row_kernel(const QkParams p) {
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
  const int first = blockIdx.x * p.per_chunk, last = min(first + p.per_chunk, p.tokens);
  for (int n = first + warp; n < last; n += kThreads / 32) {
    const Token k = token(p, n);
    const int b = k.b, t = k.t;
    const int64_t pos = position(p, k);
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
      dot = rt.moves ? warp_sum(dot) * (p.norm == KDA_NORM_RMS ? p.inv_D : 1.f) : 0.f;
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
    float* out = p.partial + ((int64_t)blockIdx.y * p.chunks + blockIdx.x) * p.D;
    for (int c = threadIdx.x; c < p.D; c += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) s += rows[i][c];
      out[c] = s;
    }
  }
}

// ---------------------------------------------------------------------------
// rows of 2 VEC N channels
// ---------------------------------------------------------------------------
constexpr int kHeadThreads = 256;        // of a block, at most
// Blocks that an SM takes.  4 x 8192 tokens of 32 heads of 128, f16: three blocks 92 us, two
// 111, four (one row of a thread at a time) 100; the gradient with two 136, with three (which
// spill) 178; with one row at a time 158.
template <bool GRAD> constexpr int kHeadBlocks = GRAD ? 2 : 3;

struct HeadShape {
  int vec;                               // channels of a group: 4, or 8 of 16 bits
  int lanes;                             // of a row: 4, 8, 16 or 32
  int heads, groups;                     // heads of a block; blocks that share a token
  int together;                          // tokens side by side in a block
  int threads;
  int batch;                             // tokens whose angles a block has at a time
  size_t smem;
};

// Two groups of VEC channels of a row.
template <int VEC> struct Row {
  float a[VEC], b[VEC];
};
template <int BYTES> struct RawOf;       // VEC values as they come
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };
template <typename T, int VEC> using Raw = typename RawOf<sizeof(T) * VEC>::type;
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Raw<T, VEC>& raw, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += 4) ld4(reinterpret_cast<const T*>(&raw) + i, *reinterpret_cast<float (*)[4]>(v + i));
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> narrow(const float (&v)[VEC]) {
  Raw<T, VEC> raw;
#pragma unroll
  for (int i = 0; i < VEC; i += 4) st4(reinterpret_cast<T*>(&raw) + i, *reinterpret_cast<const float (*)[4]>(v + i));
  return raw;
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int VEC>
__device__ __forceinline__ float dot(const Row<VEC>& x, const Row<VEC>& y) {
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    s = fmaf(x.a[i], y.a[i], s);
    t = fmaf(x.b[i], y.b[i], t);
  }
  return s + t;
}
template <int VEC>
__device__ __forceinline__ void scale(Row<VEC>& x, float r) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    x.a[i] *= r;
    x.b[i] *= r;
  }
}
template <int VEC>
__device__ __forceinline__ void multiply(Row<VEC>& x, const Row<VEC>& y) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    x.a[i] *= y.a[i];
    x.b[i] *= y.b[i];
  }
}
__device__ __forceinline__ void turn_pair(float& u, float& v, float c, float s) {
  const float t = u;
  u = fmaf(-s, v, u * c);
  v = fmaf(s, t, v * c);
}
// The lane's VEC pairs turned by their cosines and sines, pairs 2 i and 2 i + 1 in
// cs[i LANES' turned ones]; SIGN -1: turned back.
template <bool INTERLEAVED, int SIGN, int VEC>
__device__ __forceinline__ void turn(Row<VEC>& z, const float4* cs, int turned) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) {
    const float4 c = cs[i / 2 * turned];
    if constexpr (INTERLEAVED) {
      float* v = 2 * i < VEC ? z.a + 2 * i : z.b + 2 * i - VEC;
      turn_pair(v[0], v[1], c.x, SIGN * c.y);
      turn_pair(v[2], v[3], c.z, SIGN * c.w);
    } else {
      turn_pair(z.a[i], z.b[i], c.x, SIGN * c.y);
      turn_pair(z.a[i + 1], z.b[i + 1], c.z, SIGN * c.w);
    }
  }
}

// A row's r by its lanes: as rate_of().
template <int LANES, int VEC>
__device__ __forceinline__ Rate row_rate(const QkParams& p, const Row<VEC>& x) {
  if (p.norm == KDA_NORM_NONE) return {1.f, false};
  const float ss = row_sum<LANES>(dot(x, x));
  float tiny = 0.f;
  if (__any_sync(0xffffffffu, !(ss <= 3.4e38f))) {
    Row<VEC> y = x;
    scale(y, 0x1p-70f);
    tiny = row_sum<LANES>(dot(y, y));
  }
  return rate(p, ss, tiny);
}

// Threads: rows of LANES lanes; row slot s has head s % heads of the group and every
// `together`-th token from s / heads on.  A block's tokens are of one sequence, or of sequences
// that lie one behind the other (p.span tokens).
template <typename T, int VEC, int LANES, bool GRAD, bool INTERLEAVED>
__global__ void __launch_bounds__(kHeadThreads, kHeadBlocks<GRAD>)
head_kernel(const QkParams p, const HeadShape hs) {
  extern __shared__ __align__(16) unsigned char shared[];
  constexpr int UNROLL = kUnroll;
  using R = Raw<T, VEC>;
  const int pairs = p.R / 2, turned = pairs / VEC;               // of a row: lanes that are turned
  float4* const angles = reinterpret_cast<float4*>(shared);      // [2][batch][VEC / 2][turned]
  double* const rates = reinterpret_cast<double*>(shared + sizeof(float2) * 2 * hs.batch * pairs);   // [pairs]
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const int side = slot / hs.heads, in_group = slot - side * hs.heads;
  const int any = blockIdx.y * hs.heads + in_group;              // head of both tensors
  const bool live = side < hs.together && any < p.heads[0] + p.heads[1];
  const int which = live && any >= p.heads[0], head = live ? any - (which ? p.heads[0] : 0) : 0;
  // the groups of channels: pairs of the rotation, or neighbours
  const bool paired = !INTERLEAVED && lane < turned;
  const int a = (paired ? 1 : 2) * VEC * lane, b = a + (paired ? pairs : VEC);
  const bool on = live && b + VEC <= p.D, turns = on && lane < turned;
  Row<VEC> w = {}, dw = {};
  if (on) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w.a[i] = load_weight(p, which, head, a + i);
      w.b[i] = load_weight(p, which, head, b + i);
    }
  }
  const int seq = blockIdx.x / p.chunks_span, first = (blockIdx.x - seq * p.chunks_span) * p.per_chunk;
  const int last = min(first + p.per_chunk, p.span), before = seq * p.span;
  const int64_t* out_s = GRAD ? p.dx_s[which] : p.y_s[which];
  const int64_t t0 = first + side;
  const T* x = static_cast<const T*>(p.x[which]) + seq * p.x_s[which][0] + t0 * p.x_s[which][1] + head * p.x_s[which][2] + a;
  const T* dy = !GRAD ? nullptr : static_cast<const T*>(p.dy[which]) + seq * p.dy_s[which][0] +
                                      t0 * p.dy_s[which][1] + head * p.dy_s[which][2] + a;
  T* out = static_cast<T*>(GRAD ? p.dx[which] : p.y[which]) + seq * out_s[0] + t0 * out_s[1] + head * out_s[2] + a;
  const int gap = b - a;
  const int64_t x_step = hs.together * p.x_s[which][1], dy_step = hs.together * p.dy_s[which][1],
                out_step = hs.together * out_s[1];
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) rates[i] = quarter_rate(p.inv_freq[i]);
  __syncthreads();
  int buf = 0;
  for (int n0 = first; n0 < last; n0 += hs.batch, buf ^= 1) {
    const int end = min(n0 + hs.batch, last);
    float4* const cs = angles + (size_t)buf * hs.batch * (pairs / 2);
    if (pairs) {
      const int count = (end - n0) * pairs;
      for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const int j = i / pairs, pair = i - j * pairs;           // pair of lane pair / VEC
        const float2 v = angle((double)position(p, token(p, before + n0 + j)) * rates[pair]);
        reinterpret_cast<float2*>(cs + (size_t)j * (pairs / 2) + pair % VEC / 2 * turned + pair / VEC)[pair % 2] = v;
      }
      __syncthreads();
    }
    for (int n1 = n0 + side; n1 - side < end; n1 += UNROLL * hs.together) {
      R xa[UNROLL], xb[UNROLL], da[UNROLL], db[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        xa[u] = xb[u] = da[u] = db[u] = R{};
        if (n1 + u * hs.together < end && on) {
          xa[u] = *reinterpret_cast<const R*>(x);
          xb[u] = *reinterpret_cast<const R*>(x + gap);
          if constexpr (GRAD) {
            da[u] = *reinterpret_cast<const R*>(dy);
            db[u] = *reinterpret_cast<const R*>(dy + gap);
          }
        }
        x += x_step;
        if (GRAD) dy += dy_step;
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int n = n1 + u * hs.together;
        // (rows without a token: angles of another, for nothing)
        const float4* c = cs + (size_t)(n < end ? n - n0 : 0) * (pairs / 2) + lane;
        Row<VEC> v;
        widen<T, VEC>(xa[u], v.a);
        widen<T, VEC>(xb[u], v.b);
        const Rate rt = row_rate<LANES>(p, v);
        if (p.norm != KDA_NORM_NONE) scale(v, rt.r);
        if constexpr (!GRAD) {
          multiply(v, w);
          if (turns) turn<INTERLEAVED, 1>(v, c, turned);
        } else {
          Row<VEC> d;
          widen<T, VEC>(da[u], d.a);
          widen<T, VEC>(db[u], d.b);
          if (turns) turn<INTERLEAVED, -1>(d, c, turned);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            dw.a[i] = fmaf(d.a[i], v.a[i], dw.a[i]);
            dw.b[i] = fmaf(d.b[i], v.b[i], dw.b[i]);
          }
          multiply(d, w);
          if (p.norm != KDA_NORM_NONE) {
            float m = row_sum<LANES>(dot(d, v));
            m = rt.moves ? -(p.norm == KDA_NORM_RMS ? m * p.inv_D : m) : 0.f;
            // (where r does not depend on x, n may be infinite and is not multiplied by the zero)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              v.a[i] = rt.moves ? fmaf(v.a[i], m, d.a[i]) : d.a[i];
              v.b[i] = rt.moves ? fmaf(v.b[i], m, d.b[i]) : d.b[i];
            }
            scale(v, rt.r);
          } else {
            v = d;
          }
        }
        if (n < end && on) {
          *reinterpret_cast<R*>(out) = narrow<T, VEC>(v.a);
          *reinterpret_cast<R*>(out + gap) = narrow<T, VEC>(v.b);
        }
        out += out_step;
      }
    }
  }
  if (GRAD && (p.dw[0] != nullptr || p.dw[1] != nullptr)) {
    // tokens side by side are added in order
    float* sums = reinterpret_cast<float*>(shared);              // [together][heads][D]
    __syncthreads();
    if (on) {
      float* row = sums + ((size_t)side * hs.heads + in_group) * p.D;
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        st4(row + a + i, *reinterpret_cast<const float (*)[4]>(dw.a + i));
        st4(row + b + i, *reinterpret_cast<const float (*)[4]>(dw.b + i));
      }
    }
    __syncthreads();
    const int h0 = blockIdx.y * hs.heads, heads = min(hs.heads, p.heads[0] + p.heads[1] - h0);
    if (p.w_heads) {
      for (int i = threadIdx.x; i < heads * p.D; i += blockDim.x) {
        float s = 0.f;
        for (int j = 0; j < hs.together; ++j) s += sums[(size_t)j * hs.heads * p.D + i];
        p.partial[((int64_t)(h0 + i / p.D) * p.chunks + blockIdx.x) * p.D + i % p.D] = s;
      }
    } else {
      // one weight for the heads of a tensor
      const int edge = max(0, min(heads, p.heads[0] - h0));      // heads of the first tensor
      const int entries = p.chunks * gridDim.y, entry = blockIdx.x * gridDim.y + blockIdx.y;
      for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
        const int second = i >= p.D, c = second ? i - p.D : i;
        float s = 0.f;
        for (int j = 0; j < hs.together; ++j)
          for (int h = second ? edge : 0; h < (second ? heads : edge); ++h)
            s += sums[((size_t)j * hs.heads + h) * p.D + c];
        p.partial[((int64_t)second * entries + entry) * p.D + c] = s;
      }
    }
  }
}

// dw = sum of the partials of a weight row, which lie one behind the other: `each` of the rows' own
// (w_heads) or of the tensor.  Block: 32 channels; thread (r, c) adds every 32nd partial.
__global__ void __launch_bounds__(1024) weight_kernel(const QkParams p, int64_t q_parts, int64_t k_parts) {
  __shared__ double sums[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, r = threadIdx.x / 32;
  const int q_rows = p.w_heads ? p.heads[0] : 1;
  const int which = (int)blockIdx.y >= q_rows, row = blockIdx.y - (which ? q_rows : 0);
  if (p.dw[which] == nullptr) return;
  const int64_t n = which ? k_parts : q_parts, start = (which ? q_rows * q_parts : 0) + row * n;
  double s = 0.;
  if (c < p.D) {
#pragma unroll 8
    for (int64_t i = r; i < n; i += 32) s += p.partial[(start + i) * p.D + c];
  }
  sums[r][threadIdx.x % 32] = s;
  __syncthreads();
  if (r > 0 || c >= p.D) return;
  s = 0.;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += sums[i][threadIdx.x % 32];
  const int64_t at = (int64_t)row * p.D + c;
  if (p.w_dtype == KDA_DTYPE_F32) static_cast<float*>(p.dw[which])[at] = (float)s;
  else if (p.w_dtype == KDA_DTYPE_F16) st(static_cast<__half*>(p.dw[which]) + at, (float)s);
  else st(static_cast<__nv_bfloat16*>(p.dw[which]) + at, (float)s);
}

int validate(const KdaQkArgs* a) {
  if (a == nullptr) return KDA_ERR_NULL_POINTER;
  if (a->abi_version != KDA_B200_ABI_VERSION) return KDA_ERR_SHAPE;
  if (a->B < 0 || a->T < 0 || (int64_t)a->B * a->T > (1 << 30)) return KDA_ERR_SHAPE;
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

// Channels of a group with which head_kernel does it, 0: not at all.  A group is one access.
int group_of(const KdaQkArgs* a, bool grad) {
  const int size = size_of(a->io_dtype);
  for (int vec = 16 / size; vec >= 4; vec /= 2) {
    if (a->D % (2 * vec) || a->D > 64 * vec || a->R % (2 * vec)) continue;
    const auto ok = [&](const void* p, const int64_t* s) {
      return !misaligned(p, vec * size) && s[0] % vec == 0 && s[1] % vec == 0 && s[2] % vec == 0;
    };
    bool all = true;
    for (int i = 0; i < 2; ++i)
      if (a->heads[i] > 0)
        all = all && ok(a->x[i], a->x_stride[i]) &&
              (grad ? ok(a->dy[i], a->dy_stride[i]) && ok(a->dx[i], a->dx_stride[i]) : ok(a->y[i], a->y_stride[i]));
    if (all) return vec;
  }
  return 0;
}

// Sequences that lie one behind the other at the step of their tokens (or have one token
// each) are one of B T tokens.
void join(QkParams& p, bool grad) {
  p.span = p.T;
  bool one = true;
  const auto each = [&](auto f) {
    for (int i = 0; i < 2; ++i) {
      if (p.heads[i] == 0) continue;
      f(p.x_s[i]);
      if (grad) {
        f(p.dy_s[i]);
        f(p.dx_s[i]);
      } else {
        f(p.y_s[i]);
      }
    }
  };
  if (p.T > 1) each([&](int64_t* s) { one = one && s[0] == p.T * s[1]; });
  if (!one && p.B > 1) return;
  if (p.T == 1) each([&](int64_t* s) { s[1] = s[0]; });
  p.span = p.tokens;
}

HeadShape head_shape(const QkParams& p, int vec, bool grad) {
  HeadShape h{};
  h.vec = vec;
  h.lanes = 4;
  while (2 * vec * h.lanes < p.D) h.lanes *= 2;
  const int all = p.heads[0] + p.heads[1], most = kHeadThreads / h.lanes;
  h.groups = (all + most - 1) / most;
  h.heads = (all + h.groups - 1) / h.groups;
  // (small calls get more blocks)
  h.together = max(1, min(most / h.heads, (p.tokens + kSms - 1) / kSms));
  h.threads = (h.heads * h.together * h.lanes + 31) / 32 * 32;
  // angles for several turns, four for every thread or so
  const int turn = h.together * kUnroll;
  h.batch = turn * max(1, min(8, 4 * h.threads / max(1, turn * p.R / 2)));
  h.smem = (size_t)(p.R / 2) * (sizeof(double) + 2 * h.batch * sizeof(float2));
  if (grad) h.smem = max(h.smem, (size_t)h.together * h.heads * p.D * sizeof(float));
  return h;
}

// How the tokens are cut: into chunks of a multiple of `least` tokens, about `blocks` for the GPU.
void cut(QkParams& p, int blocks_per_chunk, int least, int blocks) {
  const int spans = p.span > 0 ? p.tokens / p.span : 1;
  const int64_t want = max(1, blocks / max(blocks_per_chunk, 1) / spans);
  const int64_t per = ((p.span + want - 1) / want + least - 1) / least * least;
  p.per_chunk = (int)max(per, (int64_t)least);
  p.chunks_span = (int)(((int64_t)p.span + p.per_chunk - 1) / p.per_chunk);
  p.chunks = p.chunks_span * spans;
}

QkParams to_params(const KdaQkArgs* a) {
  QkParams p{};
  p.B = a->B; p.T = a->T; p.D = a->D; p.R = a->R;
  p.tokens = a->B * a->T;
  p.t_mul = a->T <= 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / a->T);
  p.norm = a->norm;
  p.interleaved = a->interleaved != 0; p.w_heads = a->w_heads != 0; p.pos_64 = a->pos_64 != 0;
  p.w_dtype = a->w_dtype; p.pos_step = a->pos_step;
  p.eps = a->eps; p.cap = 1.f / a->eps; p.inv_D = 1.f / a->D;
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
  return p;
}

// Cuts the tokens for the kernel that does the call; true: head_kernel, in `h`.
bool plan(const KdaQkArgs* a, QkParams& p, bool grad, HeadShape& h) {
  p.span = p.tokens;
  if (p.tokens == 0 || p.heads[0] + p.heads[1] == 0) {
    cut(p, 1, 1, 1);
    return false;
  }
  const int vec = group_of(a, grad);
  if (vec) {
    join(p, grad);
    h = head_shape(p, vec, grad);
    // as many blocks as the GPU takes at once, so that all end together
    cut(p, h.groups, h.together, kSms * ((grad ? kHeadBlocks<true> : kHeadBlocks<false>) * kHeadThreads / h.threads));
  } else {
    cut(p, p.heads[0] + p.heads[1], kThreads / 32 * 4, kSms * 16);
  }
  return vec != 0;
}

template <bool GRAD>
cudaError_t launch_rows(const QkParams& p, int io, cudaStream_t s) {
  const dim3 grid(p.chunks, p.heads[0] + p.heads[1]);
  if (io == KDA_DTYPE_F32) row_kernel<float, GRAD><<<grid, kThreads, 0, s>>>(p);
  else if (io == KDA_DTYPE_F16) row_kernel<__half, GRAD><<<grid, kThreads, 0, s>>>(p);
  else row_kernel<__nv_bfloat16, GRAD><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int VEC, bool GRAD, bool INTERLEAVED>
cudaError_t launch_heads_of(const QkParams& p, const HeadShape& h, cudaStream_t s) {
  const auto kernel = h.lanes == 4    ? head_kernel<T, VEC, 4, GRAD, INTERLEAVED>
                      : h.lanes == 8  ? head_kernel<T, VEC, 8, GRAD, INTERLEAVED>
                      : h.lanes == 16 ? head_kernel<T, VEC, 16, GRAD, INTERLEAVED>
                                      : head_kernel<T, VEC, 32, GRAD, INTERLEAVED>;
  if (h.smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)h.smem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<dim3(p.chunks, h.groups), h.threads, h.smem, s>>>(p, h);
  return cudaGetLastError();
}
template <bool GRAD>
cudaError_t launch_heads(const QkParams& p, const HeadShape& h, int io, cudaStream_t s) {
  const auto run = [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int VEC = decltype(vec)::value;
    return p.interleaved ? launch_heads_of<T, VEC, GRAD, true>(p, h, s) : launch_heads_of<T, VEC, GRAD, false>(p, h, s);
  };
  using Four = std::integral_constant<int, 4>;
  using Eight = std::integral_constant<int, 8>;
  if (io == KDA_DTYPE_F32) return run(float{}, Four{});
  if (io == KDA_DTYPE_F16) return h.vec == 8 ? run(__half{}, Eight{}) : run(__half{}, Four{});
  return h.vec == 8 ? run(__nv_bfloat16{}, Eight{}) : run(__nv_bfloat16{}, Four{});
}

// Partials of a weight row of tensor i, which lie one behind the other, the queries' rows first.
int64_t parts(const QkParams& p, const HeadShape& h, bool heads, int i) {
  if (p.w_heads) return p.chunks;
  return (int64_t)p.chunks * (heads ? h.groups : p.heads[i]);
}
size_t partial_floats(const QkParams& p, const HeadShape& h, bool heads) {
  const int rows = p.w_heads ? p.heads[0] : 1, k_rows = p.w_heads ? p.heads[1] : 1;
  return (size_t)(rows * parts(p, h, heads, 0) + k_rows * parts(p, h, heads, 1)) * p.D;
}

int run(const KdaQkArgs* a, bool grad, void* stream) {
  int st = validate(a);
  if (st != KDA_OK) return st;
  QkParams p = to_params(a);
  HeadShape h{};
  const bool heads = plan(a, p, grad, h);
  const bool weights = grad && (p.dw[0] || p.dw[1]);
  const bool rows = p.tokens > 0 && p.heads[0] + p.heads[1] > 0;
  if (!rows && !weights) return KDA_OK;
  for (int i = 0; i < 2 && p.tokens > 0; ++i) {
    if (p.heads[i] == 0) continue;
    if (!p.x[i] || (grad ? !p.dy[i] || !p.dx[i] : !p.y[i])) return KDA_ERR_NULL_POINTER;
  }
  if (weights && rows && (!p.partial || a->partial_floats < partial_floats(p, h, heads))) return KDA_ERR_WORKSPACE;
  if ((st = check_device()) != KDA_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (rows && heads)
    e = grad ? launch_heads<true>(p, h, a->io_dtype, s) : launch_heads<false>(p, h, a->io_dtype, s);
  else if (rows)
    e = grad ? launch_rows<true>(p, a->io_dtype, s) : launch_rows<false>(p, a->io_dtype, s);
  if (e == cudaSuccess && weights) {
    const int n = p.w_heads ? p.heads[0] + p.heads[1] : 2;
    if (n > 0) {
      weight_kernel<<<dim3((p.D + 31) / 32, n), 1024, 0, s>>>(p, parts(p, h, heads, 0), parts(p, h, heads, 1));
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
  using namespace kda::qk;
  QkParams p = to_params(a);
  HeadShape h{};
  const bool heads = plan(a, p, true, h);
  return partial_floats(p, h, heads);
}

int kda_qk_fwd(const KdaQkArgs* a, void* stream) { return kda::qk::run(a, false, stream); }
int kda_qk_bwd(const KdaQkArgs* a, void* stream) { return kda::qk::run(a, true, stream); }

}  // extern "C"
