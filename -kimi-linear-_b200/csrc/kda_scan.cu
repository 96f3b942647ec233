// kda_scan.cu -- gated linear recurrence h_t = a_t h_{t-1} + w_t x_t: scan, single-token
// step, and the C entry points (include/kda_b200.h); its gradient is in kda_scan_grad.cu.
//
// A block walks a sequence's tiles of kTile tokens for kChannels channels: a half warp reads a
// row, a thread has kRun tokens of kVec channels.  Each thread runs over its tokens from a
// state of zero, which gives its piece's decay and its piece's state; the pieces are joined
// (half warps by shuffles, warps through shared memory, and where a sequence has more
// tiles than there are blocks otherwise, the tiles of a cluster's blocks through
// distributed shared memory), and each thread runs over its tokens again from the state that
// enters them.  The gradient does the same in both directions at once.  Rows come by cp.async
// into places that only the thread that asked for them reads, kStages tiles deep, so that
// nothing waits for a load but the tile it is for.
#include <cstring>

#include "kda_scan.cuh"

namespace kda {
namespace scan {

__device__ int g_scan_device_error = 0;

namespace {

// ---------------------------------------------------------------------------
// packed batches: what each row is
// ---------------------------------------------------------------------------
// Blocks 0 .. tiles - 1: a tile each.  The others: a sequence without rows each, whose
// state (gradient) goes through.
__global__ void __launch_bounds__(kTile) mark_kernel(const ScanParams p, Marks* marks, const float* from,
                                                     int64_t from_s, float* to, int64_t to_s) {
  if ((int)blockIdx.x < p.tiles) {
    const int t = blockIdx.x * kTile + threadIdx.x;
    const int b = sequence_at(p.q_start, p.B, t);
    const int end = b >= 0 ? min(p.q_start[b + 1], p.T) : 0;
    const bool owned = end > t;
    const uint32_t first = __ballot_sync(0xffffffffu, owned && p.q_start[max(b, 0)] == t);
    const uint32_t last = __ballot_sync(0xffffffffu, owned && end == t + 1);
    const uint32_t own = __ballot_sync(0xffffffffu, owned);
    if (threadIdx.x % 32 == 0) {
      uint32_t* m = reinterpret_cast<uint32_t*>(marks + blockIdx.x) + threadIdx.x / 32;
      m[0] = first;
      m[2] = last;
      m[4] = own;
    }
    return;
  }
  const int b = blockIdx.x - p.tiles;
  const int lo = min(max(p.q_start[b], 0), p.T), hi = min(p.q_start[b + 1], p.T);
  if (to == nullptr || hi > lo) return;
  for (int c = threadIdx.x; c < p.D; c += kTile) to[b * to_s + c] = from ? from[b * from_s + c] : 0.f;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
constexpr int kStages = 2;

template <typename TX, typename TG, bool WIDE, bool PACKED>
__global__ void __launch_bounds__(kThreads, 3) scan_kernel(const ScanParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint64_t full[2];
  __shared__ __align__(16) float warps[2][kWarps * kPieceFloats];
  using XRing = Ring<TX, WIDE, kStages>;
  using GRing = Ring<TG, WIDE, kStages>;
  const XRing xs(smem);
  const GRing gs(smem + XRing::kBytes);
  const Place w = my_place<WIDE>(p);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % kLanes;
  const bool upper = threadIdx.x % 32 >= kLanes;
  const int turns = (p.tiles + p.cluster - 1) / p.cluster;
  const int t_first = w.rank * kTile + w.run, t_step = p.cluster * kTile;
  const TX* x = static_cast<const TX*>(p.x) + w.b * p.x_s[0] + (int64_t)t_first * p.x_s[1] + w.c;
  const TG* g = static_cast<const TG*>(p.g) + w.b * p.g_s[0] + (int64_t)t_first * p.g_s[1] + w.c;
  TX* out = static_cast<TX*>(p.h) + w.b * p.h_s[0] + (int64_t)t_first * p.h_s[1] + w.c;
  float* ckpt = p.ckpt ? p.ckpt + ((int64_t)w.b * p.tiles + w.rank) * p.D + w.c : nullptr;
  if constexpr (PACKED) ptx::grid_dep_wait();
  float2 carry[kPairs];              // the state that enters the cluster's next tiles
  load_state<WIDE>(PACKED || !p.state_in ? nullptr : p.state_in + w.b * p.si_s + w.c, w.on, carry);
  const auto load = [&](int stage, int tile) {
    const uint32_t there = row_mask<PACKED>(p, w, tile).there;
    xs.load(stage, x, p.x_s[1], there, w.on);
    gs.load(stage, g, p.g_s[1], there, w.on);
    copy_commit();
    x += t_step * p.x_s[1];
    g += t_step * p.g_s[1];
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) load(k, k * p.cluster + w.rank);
  Exchange exchange(full, reinterpret_cast<float*>(smem + XRing::kBytes + GRing::kBytes), p, w.rank,
                    &g_scan_device_error);
  int stage = 0;
  for (int k = 0; k < turns; ++k) {
    const int tile = k * p.cluster + w.rank, t0 = tile * kTile + w.run, buf = k & 1;
    load(stage ? stage - 1 : kStages - 1, tile + (kStages - 1) * p.cluster);
    const RowMask m = row_mask<PACKED>(p, w, tile);
    copy_wait<kStages - 1>();
    // the thread's piece
    Decay a[kRun][kPairs];
    float2 v[kRun][kPairs], sum[kPairs];
    Piece q;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) sum[j] = q.h[j] = both(0.f);
#pragma unroll
    for (int t = 0; t < kRun; ++t) {
      float2 gt[kPairs];
      gs.read(stage, t, gt);
      xs.read(stage, t, v[t]);
      if (PACKED && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, q.h);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        a[t][j] = decay(gt[j]);
        sum[j] = __fadd2_rn(sum[j], gt[j]);
        if (p.complement) v[t][j] = __fmul2_rn(v[t][j], rest(a[t][j]));
        q.h[j] = apply(a[t][j], q.h[j], v[t][j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) q.a[j] = PACKED && m.first ? cut() : decay(sum[j]);
    const Piece low = shuffle(q, lane);            // the lower half warp's
    if (upper) {
      Piece both_halves = low;
      append<PACKED>(both_halves, q);
      put(warps[buf] + warp * kPieceFloats, lane, both_halves);
    }
    __syncthreads();
    // the state that enters the block's tile, and the next turn's
    float2 cur[kPairs], mine[kPairs];
    if (p.cluster > 1) {
      exchange.send<PACKED>(k, warps[buf], false);
      exchange.wait(k);
#pragma unroll 1
      for (int i = 0; i < p.cluster; ++i) {
        if (i == w.rank) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) cur[j] = carry[j];
        }
        pass_on<PACKED>(take(exchange.row(k, i), lane), carry);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) cur[j] = carry[j];
    }
    if (ckpt) {
      if (tile < p.tiles && threadIdx.x < kLanes) store_state<WIDE>(ckpt, w.on, cur);
      ckpt += (int64_t)p.cluster * p.D;
    }
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i == warp) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) mine[j] = cur[j];
      }
      pass_on<PACKED>(take(warps[buf] + i * kPieceFloats, lane), cur);
    }
    if (p.cluster == 1) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) carry[j] = cur[j];
    }
    if (upper) pass_on<PACKED>(low, mine);
    // and the thread's tokens again, from the state that enters them
    TX* row = out;
#pragma unroll
    for (int t = 0; t < kRun; ++t) {
      if (PACKED && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, mine);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) mine[j] = apply(a[t][j], mine[j], v[t][j]);
      if (m.there >> t & 1) {
        write<WIDE>(row, w.on, mine);
      } else if (PACKED && t0 + t < p.T) {
        const float2 zero[kPairs] = {};
        write<WIDE>(row, w.on, zero);
      }
      if (PACKED && (m.last >> t & 1))
        store_state<WIDE>(const_cast<float*>(state_of(p, p.state_out, p.so_s, t0 + t, w.c)), w.on, mine);
      row += p.h_s[1];
    }
    out += t_step * p.h_s[1];
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  if (!PACKED && w.rank == 0 && threadIdx.x < kLanes)
    store_state<WIDE>(p.state_out + w.b * p.so_s + w.c, w.on, carry);
  exchange.leave();
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
  constexpr int N = (VEC + 1) / 2 * 2;   // in pairs
  float x[N] = {}, g[N] = {}, h[N] = {};
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
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const Decay a = decay(make_float2(g[i], g[i + 1]));
      float2 v = make_float2(x[i], x[i + 1]);
      if (p.complement) v = __fmul2_rn(v, rest(a));
      v = apply(a, make_float2(h[i], h[i + 1]), v);
      h[i] = v.x;
      h[i + 1] = v.y;
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

cudaError_t launch_forward(const ScanParams& p, int x_dtype, int g_dtype, bool wide, cudaStream_t s) {
  return by_types(x_dtype, g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    const size_t smem = Ring<TX, true, kStages>::kBytes + Ring<TG, true, kStages>::kBytes + cluster_bytes(p.cluster);
    if (p.q_start)
      return launch_tiles(wide ? scan_kernel<TX, TG, true, true> : scan_kernel<TX, TG, false, true>, p, smem, s);
    return launch_tiles(wide ? scan_kernel<TX, TG, true, false> : scan_kernel<TX, TG, false, false>, p, smem, s);
  });
}

constexpr int kWantBlocks = 512;   // clusters grow until a call has so many blocks

int size_of(int dt) { return dt == KDA_DTYPE_F32 ? 4 : 2; }
bool misaligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

enum Pass { kForward, kBackward, kStep };

int validate_sizes(const KdaScanArgs* a) {
  if (a == nullptr) return KDA_ERR_NULL_POINTER;
  if (a->abi_version != KDA_B200_ABI_VERSION) return KDA_ERR_SHAPE;
  if (a->B < 0 || a->T < 0 || a->D < 0 || a->D > (1 << 24) || a->B > (1 << 24) || a->T > (1 << 30))
    return KDA_ERR_SHAPE;
  return KDA_OK;
}

int validate(const KdaScanArgs* a, Pass pass) {
  const int st = validate_sizes(a);
  if (st != KDA_OK) return st;
  if (pass == kStep && a->T != 1) return KDA_ERR_SHAPE;
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
  p.cluster = 1;
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

size_t workspace_bytes(const KdaScanArgs* a) {
  return a->q_start ? ((size_t)a->T + kTile - 1) / kTile * sizeof(Marks) : 0;
}

// Rows start on kVec values' boundaries.
bool aligned_rows(const void* p, const int64_t* stride, int bytes) {
  return !misaligned(p, 4 * bytes) && stride[0] % 4 == 0 && stride[1] % 4 == 0;
}

int run_scan(const KdaScanArgs* a, Pass pass, void* stream) {
  int st = validate(a, pass);
  if (st != KDA_OK) return st;
  if (a->D == 0 || (a->B == 0 && (a->q_start == nullptr || a->T == 0))) return KDA_OK;
  const size_t need = workspace_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need)) return KDA_ERR_WORKSPACE;
  if (misaligned(a->workspace, 8)) return KDA_ERR_ALIGNMENT;
  if ((st = check_device()) != KDA_OK) return st;
  ScanParams p = to_params(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int xs = size_of(a->x_dtype), gs = size_of(a->g_dtype);
  const bool wide = p.D % kVec == 0 && aligned_rows(p.x, p.x_s, xs) && aligned_rows(p.g, p.g_s, gs) &&
                    (pass == kForward ? aligned_rows(p.h, p.h_s, xs)
                                      : aligned_rows(p.dh, p.dh_s, xs) && aligned_rows(p.dx, p.dx_s, xs) &&
                                            aligned_rows(p.dg, p.dg_s, gs));
  const int64_t blocks = (int64_t)(p.q_start ? 1 : p.B) * ((p.D + kChannels - 1) / kChannels);
  if (blocks * kMaxCluster > 0x7fffffff) return KDA_ERR_SHAPE;
  while (p.cluster < kMaxCluster && p.cluster < p.tiles && blocks * p.cluster < kWantBlocks) p.cluster *= 2;
  cudaError_t e = cudaSuccess;
  if (p.q_start) {
    Marks* marks = static_cast<Marks*>(a->workspace);
    p.marks = marks;
    const bool fwd = pass == kForward;
    mark_kernel<<<p.tiles + p.B, kTile, 0, s>>>(p, marks, fwd ? p.state_in : p.dstate_out,
                                                fwd ? p.si_s : p.dso_s, fwd ? p.state_out : p.dstate_in,
                                                fwd ? p.so_s : p.dsi_s);
    e = cudaGetLastError();
    if (p.tiles == 0) return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
  }
  if (e == cudaSuccess)
    e = pass == kForward ? launch_forward(p, a->x_dtype, a->g_dtype, wide, s)
                         : launch_grad(p, a->x_dtype, a->g_dtype, wide, s);
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
  const int grad = read_grad_device_error(clear);
  if (grad < 0) return grad;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_scan_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_scan_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v ? v : grad;
}

}  // namespace scan
}  // namespace kda

extern "C" {

size_t kda_scan_args_size(void) { return sizeof(KdaScanArgs); }

size_t kda_scan_ckpt_floats(const KdaScanArgs* a) {
  if (kda::scan::validate_sizes(a) != KDA_OK) return 0;
  const size_t tiles = ((size_t)a->T + kda::scan::kTile - 1) / kda::scan::kTile;
  return (a->q_start ? 1 : (size_t)a->B) * tiles * (size_t)a->D;
}

size_t kda_scan_workspace_bytes(const KdaScanArgs* a) {
  if (kda::scan::validate_sizes(a) != KDA_OK) return 0;
  return kda::scan::workspace_bytes(a);
}

int kda_scan_fwd(const KdaScanArgs* a, void* stream) {
  return kda::scan::run_scan(a, kda::scan::kForward, stream);
}

int kda_scan_bwd(const KdaScanArgs* a, void* stream) {
  return kda::scan::run_scan(a, kda::scan::kBackward, stream);
}

int kda_scan_step(const KdaScanArgs* a, void* stream) { return kda::scan::run_step(a, stream); }

}  // extern "C"
