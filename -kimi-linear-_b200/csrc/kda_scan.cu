// kda_scan.cu -- gated linear recurrence h_t = a_t h_{t-1} + w_t x_t: scan, gradient,
// single-token step, and their C entry points (include/kda_b200.h).
//
// Gradient, with u_t what flows into h_t from later tokens (u of the last: dstate_out):
//   d_t = dh_t + u_t,  u_{t-1} = a_t d_t
//   dx_t = w_t d_t,  dg_t = a_t (h_{t-1} - [complement] x_t) d_t,  dstate_in = u_{-1}
// It needs h_{t-1} in 32 bits: h is in x's type, so the states are computed again from
// the checkpoints that the forward pass leaves every kTile tokens.
//
// A thread has a channel and walks its tokens one by one.
#include <cstring>

#include "kda_scan.cuh"

namespace kda {
namespace scan {

__device__ int g_scan_device_error = 0;

namespace {

constexpr int kThreads = 128;

// Where sequence b's rows lie: `row` counts tokens from the tensors' start.
struct Rows {
  int64_t batch;                    // batch index of the tensors (packed: 0)
  int first, last;
  float* ckpt;                      // checkpoint of row 0
};
__device__ __forceinline__ Rows rows_of(const ScanParams& p, int b) {
  Rows r;
  if (p.q_start != nullptr) {
    r.batch = 0;
    owned_rows(p, b, r.first, r.last);
    r.ckpt = p.ckpt;
  } else {
    r.batch = b;
    r.first = 0;
    r.last = p.T;
    r.ckpt = p.ckpt ? p.ckpt + (int64_t)b * p.tiles * p.D : nullptr;
  }
  return r;
}

// Rows of no sequence, shared out over the blocks of the extra sequence B.
template <typename F>
__device__ __forceinline__ void for_unowned(const ScanParams& p, F f) {
  const int lo = min(max(p.q_start[0], 0), p.T), hi = max(lo, min(max(p.q_start[p.B], 0), p.T));
  for (int t = 0; t < lo; ++t) f(t);
  for (int t = hi; t < p.T; ++t) f(t);
}

template <typename TX, typename TG>
__global__ void __launch_bounds__(kThreads) scan_kernel(const ScanParams p) {
  const int c = blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
  if (c >= p.D) return;
  const TX* x = static_cast<const TX*>(p.x) + c;
  const TG* g = static_cast<const TG*>(p.g) + c;
  TX* out = static_cast<TX*>(p.h) + c;
  if (b == p.B) {
    for_unowned(p, [&](int t) { st(out + t * p.h_s[1], 0.f); });
    return;
  }
  const Rows rows = rows_of(p, b);
  x += rows.batch * p.x_s[0];
  g += rows.batch * p.g_s[0];
  out += rows.batch * p.h_s[0];
  float h = p.state_in ? p.state_in[b * p.si_s + c] : 0.f;
  for (int t = rows.first; t < rows.last; ++t) {
    if (rows.ckpt && t % kTile == 0) rows.ckpt[(int64_t)(t / kTile) * p.D + c] = h;
    const float r = decay(ld(g + t * p.g_s[1]));
    float v = ld(x + t * p.x_s[1]);
    if (p.complement) v *= rest(r);
    h = apply(r, h, v);
    st(out + t * p.h_s[1], h);
  }
  p.state_out[b * p.so_s + c] = h;
}

template <typename TX, typename TG>
__global__ void __launch_bounds__(kThreads) scan_grad_kernel(const ScanParams p) {
  const int c = blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
  if (c >= p.D) return;
  const TX* x = static_cast<const TX*>(p.x) + c;
  const TG* g = static_cast<const TG*>(p.g) + c;
  const TX* dh = p.dh ? static_cast<const TX*>(p.dh) + c : nullptr;
  TX* dx = p.dx ? static_cast<TX*>(p.dx) + c : nullptr;
  TG* dg = p.dg ? static_cast<TG*>(p.dg) + c : nullptr;
  if (b == p.B) {
    for_unowned(p, [&](int t) {
      if (dx) st(dx + t * p.dx_s[1], 0.f);
      if (dg) st(dg + t * p.dg_s[1], 0.f);
    });
    return;
  }
  const Rows rows = rows_of(p, b);
  x += rows.batch * p.x_s[0];
  g += rows.batch * p.g_s[0];
  if (dh) dh += rows.batch * p.dh_s[0];
  if (dx) dx += rows.batch * p.dx_s[0];
  if (dg) dg += rows.batch * p.dg_s[0];
  float u = p.dstate_out ? p.dstate_out[b * p.dso_s + c] : 0.f;
  float before[kTile];              // a_t h_{t-1} (complement: a_t (h_{t-1} - x_t))
  for (int end = rows.last; end > rows.first;) {
    const int tile = (end - 1) / kTile, t0 = max(tile * kTile, rows.first);
    float h = t0 == rows.first ? (p.state_in ? p.state_in[b * p.si_s + c] : 0.f)
                               : rows.ckpt[(int64_t)tile * p.D + c];
    for (int t = t0; t < end; ++t) {
      const float r = decay(ld(g + t * p.g_s[1])), v = ld(x + t * p.x_s[1]);
      before[t - t0] = times(r, p.complement ? h - v : h);
      h = apply(r, h, p.complement ? rest(r) * v : v);
    }
    for (int t = end - 1; t >= t0; --t) {
      const float r = decay(ld(g + t * p.g_s[1]));
      const float d = u + (dh ? ld(dh + t * p.dh_s[1]) : 0.f);
      if (dx) st(dx + t * p.dx_s[1], p.complement ? rest(r) * d : d);
      if (dg) st(dg + t * p.dg_s[1], before[t - t0] * d);
      u = times(r, d);
    }
    end = t0;
  }
  if (p.dstate_in) p.dstate_in[b * p.dsi_s + c] = u;
}

// One token: a thread has VEC channels of a row.
template <typename TX, typename TG, int VEC>
__global__ void __launch_bounds__(kThreads) step_kernel(const ScanParams p, int blocks_per_row) {
  const int b = blockIdx.x / blocks_per_row;
  const int c = ((blockIdx.x - b * blocks_per_row) * kThreads + threadIdx.x) * VEC;
  if (c >= p.D) return;
  int64_t row = b;
  bool live = true;
  if (p.slots != nullptr) {
    row = p.slots[b];
    live = row >= 0 && row < p.num_states;
    if (row >= p.num_states) g_scan_device_error = kErrSlot;
  }
  float x[VEC], g[VEC], h[VEC];
  TX* out = static_cast<TX*>(p.h) + b * p.h_s[0] + c;
  if (live) {
    const TX* px = static_cast<const TX*>(p.x) + b * p.x_s[0] + c;
    const TG* pg = static_cast<const TG*>(p.g) + b * p.g_s[0] + c;
    const float* ps = p.state_in + row * p.si_s + c;
    if constexpr (VEC == 4) {
      ld4(px, x);
      ld4(pg, g);
      if (p.state_in) ld4(ps, h);
    } else {
      x[0] = ld(px);
      g[0] = ld(pg);
      if (p.state_in) h[0] = *ps;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if (live) {
      const float r = decay(g[i]);
      h[i] = apply(r, p.state_in ? h[i] : 0.f, p.complement ? rest(r) * x[i] : x[i]);
    } else {
      h[i] = 0.f;
    }
  }
  float* so = p.state_out + (p.scatter ? row : b) * p.so_s + c;
  const bool keep = live || !p.scatter;
  if constexpr (VEC == 4) {
    st4(out, h);
    if (keep) st4(so, h);
  } else {
    st(out, h[0]);
    if (keep) *so = h[0];
  }
}

// Calls f with the types of x and g.
template <typename F>
cudaError_t by_types(int x, int g, F f) {
  if (x == KDA_DTYPE_F32) return f(float{}, float{});
  if (x == KDA_DTYPE_F16)
    return g == KDA_DTYPE_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return g == KDA_DTYPE_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

int size_of(int dt) { return dt == KDA_DTYPE_F32 ? 4 : 2; }
bool misaligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

enum Pass { kForward, kBackward, kStep };

int validate(const KdaScanArgs* a, Pass pass) {
  if (a == nullptr) return KDA_ERR_NULL_POINTER;
  if (a->abi_version != KDA_B200_ABI_VERSION) return KDA_ERR_SHAPE;
  if (a->B < 0 || a->T < 0 || a->D < 0 || a->D > (1 << 24)) return KDA_ERR_SHAPE;
  if ((pass == kStep && a->T != 1) || a->B > (pass == kStep ? 1 << 24 : 65534)) return KDA_ERR_SHAPE;
  if (a->x_dtype < KDA_DTYPE_F32 || a->x_dtype > KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
  if (a->g_dtype != KDA_DTYPE_F32 && a->g_dtype != a->x_dtype) return KDA_ERR_DTYPE;
  if (a->D == 0) return KDA_OK;
  const int xs = size_of(a->x_dtype), gs = size_of(a->g_dtype);
  const bool tokens = a->T > 0 && (a->B > 0 || a->q_start != nullptr);
  if (tokens && (!a->x || !a->g || (pass != kBackward && !a->h))) return KDA_ERR_NULL_POINTER;
  if (a->B > 0 && pass != kBackward && !a->state_out) return KDA_ERR_NULL_POINTER;
  if (tokens && pass == kBackward && a->B > 0 && !a->ckpt) return KDA_ERR_NULL_POINTER;
  if (misaligned(a->x, xs) || misaligned(a->h, xs) || misaligned(a->dh, xs) || misaligned(a->dx, xs) ||
      misaligned(a->g, gs) || misaligned(a->dg, gs) || misaligned(a->state_in, 4) ||
      misaligned(a->state_out, 4) || misaligned(a->dstate_out, 4) || misaligned(a->dstate_in, 4) ||
      misaligned(a->ckpt, 4) || misaligned(a->q_start, 4) || misaligned(a->slots, 4))
    return KDA_ERR_ALIGNMENT;
  if (pass == kStep) {
    if (a->slots && a->num_states < 0) return KDA_ERR_SHAPE;
    if (a->scatter && a->B > 0 && (a->state_in != a->state_out || a->state_in_stride != a->state_out_stride))
      return KDA_ERR_STRIDE;
  }
  return KDA_OK;
}

ScanParams to_params(const KdaScanArgs* a) {
  ScanParams p{};
  p.B = a->B; p.T = a->T; p.D = a->D;
  p.tiles = (a->T + kTile - 1) / kTile;
  p.complement = a->complement != 0;
  p.x = a->x; std::memcpy(p.x_s, a->x_stride, sizeof(p.x_s));
  p.g = a->g; std::memcpy(p.g_s, a->g_stride, sizeof(p.g_s));
  p.state_in = a->state_in; p.si_s = a->state_in_stride;
  p.q_start = a->q_start;
  p.h = a->h; std::memcpy(p.h_s, a->h_stride, sizeof(p.h_s));
  p.state_out = a->state_out; p.so_s = a->state_out_stride;
  p.ckpt = a->ckpt;
  p.dh = a->dh; std::memcpy(p.dh_s, a->dh_stride, sizeof(p.dh_s));
  p.dstate_out = a->dstate_out; p.dso_s = a->dstate_out_stride;
  p.dx = a->dx; std::memcpy(p.dx_s, a->dx_stride, sizeof(p.dx_s));
  p.dg = a->dg; std::memcpy(p.dg_s, a->dg_stride, sizeof(p.dg_s));
  p.dstate_in = a->dstate_in; p.dsi_s = a->dstate_in_stride;
  p.slots = a->slots; p.num_states = a->num_states; p.scatter = a->scatter != 0;
  return p;
}

int check_device() {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
    return KDA_ERR_LAUNCH;
  return major == 10 ? KDA_OK : KDA_ERR_ARCH;
}

int run_scan(const KdaScanArgs* a, Pass pass, void* stream) {
  int st = validate(a, pass);
  if (st != KDA_OK) return st;
  if (a->D == 0 || (a->B == 0 && (a->q_start == nullptr || a->T == 0))) return KDA_OK;
  if ((st = check_device()) != KDA_OK) return st;
  const ScanParams p = to_params(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid((p.D + kThreads - 1) / kThreads, p.B + (p.q_start ? 1 : 0));
  const cudaError_t e = by_types(a->x_dtype, a->g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    if (pass == kForward)
      scan_kernel<TX, TG><<<grid, kThreads, 0, s>>>(p);
    else
      scan_grad_kernel<TX, TG><<<grid, kThreads, 0, s>>>(p);
    return cudaGetLastError();
  });
  return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

int run_step(const KdaScanArgs* a, void* stream) {
  int st = validate(a, kStep);
  if (st != KDA_OK) return st;
  if (a->D == 0 || a->B == 0) return KDA_OK;
  if ((st = check_device()) != KDA_OK) return st;
  const ScanParams p = to_params(a);
  const int xs = size_of(a->x_dtype), gs = size_of(a->g_dtype);
  const bool vec = p.D % 4 == 0 && !misaligned(p.x, 4 * xs) && !misaligned(p.h, 4 * xs) &&
                   !misaligned(p.g, 4 * gs) && !misaligned(p.state_in, 16) &&
                   !misaligned(p.state_out, 16) && p.x_s[0] % 4 == 0 && p.h_s[0] % 4 == 0 &&
                   p.g_s[0] % 4 == 0 && p.si_s % 4 == 0 && p.so_s % 4 == 0;
  const int per_row = (p.D + kThreads * (vec ? 4 : 1) - 1) / (kThreads * (vec ? 4 : 1));
  if ((int64_t)per_row * p.B > 0x7fffffff) return KDA_ERR_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = by_types(a->x_dtype, a->g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    if (vec)
      step_kernel<TX, TG, 4><<<per_row * p.B, kThreads, 0, s>>>(p, per_row);
    else
      step_kernel<TX, TG, 1><<<per_row * p.B, kThreads, 0, s>>>(p, per_row);
    return cudaGetLastError();
  });
  return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // namespace

int read_device_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_scan_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_scan_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace scan
}  // namespace kda

extern "C" {

size_t kda_scan_args_size(void) { return sizeof(KdaScanArgs); }

size_t kda_scan_ckpt_floats(const KdaScanArgs* a) {
  if (kda::scan::validate(a, kda::scan::kForward) != KDA_OK) return 0;
  const size_t tiles = ((size_t)a->T + kda::scan::kTile - 1) / kda::scan::kTile;
  return (a->q_start ? 1 : (size_t)a->B) * tiles * (size_t)a->D;
}

int kda_scan_fwd(const KdaScanArgs* a, void* stream) {
  return kda::scan::run_scan(a, kda::scan::kForward, stream);
}

int kda_scan_bwd(const KdaScanArgs* a, void* stream) {
  return kda::scan::run_scan(a, kda::scan::kBackward, stream);
}

int kda_scan_step(const KdaScanArgs* a, void* stream) { return kda::scan::run_step(a, stream); }

}  // extern "C"
