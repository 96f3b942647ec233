// kda_scan_grad.cu -- gradient of the gated linear recurrence.  With u_t what flows into h_t
// from later tokens (u of the last: dstate_out):
//   d_t = dh_t + u_t,  u_{t-1} = a_t d_t
//   dx_t = w_t d_t,  dg_t = a_t (h_{t-1} - [complement] x_t) d_t,  dstate_in = u_{-1}
// It needs h_{t-1} in 32 bits: h is in x's type, so a tile's states are computed again from
// the checkpoint that the forward pass left at its start.  The blocks, threads and pieces are
// those of scan_kernel (kda_scan.cu), the tiles taken from the last to the first.
#include "kda_scan.cuh"

namespace kda {
namespace scan {

__device__ int g_grad_device_error = 0;

namespace {

constexpr int kStages = 2;

template <typename TX, typename TG, bool WIDE, bool PACKED>
__global__ void __launch_bounds__(kThreads, 2) scan_grad_kernel(const ScanParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint64_t full[2];
  __shared__ __align__(16) float warps[2][kWarps * kPieceFloats], back[2][kWarps * kPieceFloats];
  using XRing = Ring<TX, WIDE, kStages>;
  using GRing = Ring<TG, WIDE, kStages>;
  const XRing xs(smem), ds(smem + XRing::kBytes);
  const GRing gs(smem + 2 * XRing::kBytes);
  const Place w = my_place<WIDE>(p);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % kLanes;
  const bool upper = threadIdx.x % 32 >= kLanes;
  const int turns = (p.tiles + p.cluster - 1) / p.cluster;
  const int tile_last = (turns - 1) * p.cluster + w.rank;
  const int64_t t_last = (int64_t)tile_last * kTile + w.run, t_step = (int64_t)p.cluster * kTile;
  const TX* x = static_cast<const TX*>(p.x) + w.b * p.x_s[0] + t_last * p.x_s[1] + w.c;
  const TG* g = static_cast<const TG*>(p.g) + w.b * p.g_s[0] + t_last * p.g_s[1] + w.c;
  const TX* dh = p.dh ? static_cast<const TX*>(p.dh) + w.b * p.dh_s[0] + t_last * p.dh_s[1] + w.c : x;
  TX* dx = p.dx ? static_cast<TX*>(p.dx) + w.b * p.dx_s[0] + t_last * p.dx_s[1] + w.c : nullptr;
  TG* dg = p.dg ? static_cast<TG*>(p.dg) + w.b * p.dg_s[0] + t_last * p.dg_s[1] + w.c : nullptr;
  const float* ckpt = p.ckpt + ((int64_t)w.b * p.tiles + tile_last) * p.D + w.c;
  if constexpr (PACKED) ptx::grid_dep_wait();
  float2 carry[kPairs];              // the gradient that enters the cluster's next tiles
  load_state<WIDE>(PACKED || !p.dstate_out ? nullptr : p.dstate_out + w.b * p.dso_s + w.c, w.on, carry);
  const auto load = [&](int stage, int tile) {
    const uint32_t there = row_mask<PACKED>(p, w, tile).there;
    xs.load(stage, x, p.x_s[1], there, w.on);
    gs.load(stage, g, p.g_s[1], there, w.on);
    ds.load(stage, dh, p.dh_s[1], p.dh ? there : 0, w.on);
    copy_commit();
    x -= t_step * p.x_s[1];
    g -= t_step * p.g_s[1];
    if (p.dh) dh -= t_step * p.dh_s[1];
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) load(k, tile_last - k * p.cluster);
  Exchange exchange(full, reinterpret_cast<float*>(smem + 2 * XRing::kBytes + GRing::kBytes), p, w.rank,
                    &g_grad_device_error);
  int stage = 0;
  for (int turn = 0; turn < turns; ++turn) {
    const int k = turns - 1 - turn;
    const int tile = k * p.cluster + w.rank, t0 = tile * kTile + w.run, buf = k & 1;
    load(stage ? stage - 1 : kStages - 1, tile - (kStages - 1) * p.cluster);
    const RowMask m = row_mask<PACKED>(p, w, tile);
    float2 cur[kPairs];              // the state that enters the tile
    load_state<WIDE>(tile < p.tiles ? ckpt : nullptr, w.on, cur);
    ckpt -= (int64_t)p.cluster * p.D;
    copy_wait<kStages - 1>();
    Decay a[kRun][kPairs];
    float2 v[kRun][kPairs], sum[kPairs];
    Piece q, r;                      // forward; backward
#pragma unroll
    for (int j = 0; j < kPairs; ++j) sum[j] = q.h[j] = r.h[j] = both(0.f);
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
        q.h[j] = apply(a[t][j], q.h[j], p.complement ? __fmul2_rn(rest(a[t][j]), v[t][j]) : v[t][j]);
      }
    }
#pragma unroll
    for (int t = kRun - 1; t >= 0; --t) {
      float2 d[kPairs];
      ds.read(stage, t, d);
      if (PACKED && (m.last >> t & 1))
        load_state<WIDE>(state_of(p, p.dstate_out, p.dso_s, t0 + t, w.c), w.on, r.h);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) r.h[j] = times(a[t][j], __fadd2_rn(d[j], r.h[j]));
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      q.a[j] = r.a[j] = decay(sum[j]);
      if (PACKED && m.first) q.a[j] = cut();
      if (PACKED && m.last) r.a[j] = cut();
    }
    const Piece low = shuffle(q, lane), high = shuffle(r, lane + kLanes);
    if (upper) {
      Piece halves = low;
      append<PACKED>(halves, q);
      put(warps[buf] + warp * kPieceFloats, lane, halves);
    } else {
      Piece halves = high;
      append<PACKED>(halves, r);
      put(back[buf] + warp * kPieceFloats, lane, halves);
    }
    __syncthreads();
    if (p.cluster > 1) exchange.send<PACKED>(turn, back[buf], true);
    // the state that enters the thread's tokens from before
    float2 mine[kPairs], u[kPairs];
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i == warp) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) mine[j] = cur[j];
      }
      if (i + 1 < kWarps) pass_on<PACKED>(take(warps[buf] + i * kPieceFloats, lane), cur);
    }
    if (upper) pass_on<PACKED>(low, mine);
    // and the gradient that enters them from behind
    if (p.cluster > 1) {
      exchange.wait(turn);
#pragma unroll 1
      for (int i = p.cluster - 1; i >= 0; --i) {
        if (i == w.rank) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) cur[j] = carry[j];
        }
        pass_on<PACKED>(take(exchange.row(turn, i), lane), carry);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) cur[j] = carry[j];
    }
#pragma unroll
    for (int i = kWarps - 1; i >= 0; --i) {
      if (i == warp) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) u[j] = cur[j];
      }
      pass_on<PACKED>(take(back[buf] + i * kPieceFloats, lane), cur);
    }
    if (p.cluster == 1) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) carry[j] = cur[j];
    }
    if (!upper) pass_on<PACKED>(high, u);
    // a_t h_{t-1} (complement: a_t (h_{t-1} - x_t)) in the place of x_t
#pragma unroll
    for (int t = 0; t < kRun; ++t) {
      if (PACKED && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, mine);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float2 xt = v[t][j], h = mine[j];
        if (p.complement) {
          v[t][j] = times(a[t][j], __ffma2_rn(xt, both(-1.f), h));
          mine[j] = apply(a[t][j], h, __fmul2_rn(rest(a[t][j]), xt));
        } else {
          v[t][j] = times(a[t][j], h);
          mine[j] = __fadd2_rn(v[t][j], xt);
        }
      }
    }
#pragma unroll
    for (int t = kRun - 1; t >= 0; --t) {
      float2 d[kPairs], ox[kPairs], og[kPairs];
      ds.read(stage, t, d);
      if (PACKED && (m.last >> t & 1))
        load_state<WIDE>(state_of(p, p.dstate_out, p.dso_s, t0 + t, w.c), w.on, u);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        d[j] = __fadd2_rn(d[j], u[j]);
        ox[j] = p.complement ? __fmul2_rn(rest(a[t][j]), d[j]) : d[j];
        og[j] = __fmul2_rn(v[t][j], d[j]);
        u[j] = times(a[t][j], d[j]);
      }
      const bool there = m.there >> t & 1;
      if (PACKED && !there) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) ox[j] = og[j] = both(0.f);
      }
      if (there || (PACKED && t0 + t < p.T)) {
        if (dx) write<WIDE>(dx + t * p.dx_s[1], w.on, ox);
        if (dg) write<WIDE>(dg + t * p.dg_s[1], w.on, og);
      }
      if (PACKED && p.dstate_in && (m.first >> t & 1))
        store_state<WIDE>(const_cast<float*>(state_of(p, p.dstate_in, p.dsi_s, t0 + t, w.c)), w.on, u);
    }
    if (dx) dx -= t_step * p.dx_s[1];
    if (dg) dg -= t_step * p.dg_s[1];
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  if (!PACKED && p.dstate_in && w.rank == 0 && threadIdx.x < kLanes)
    store_state<WIDE>(p.dstate_in + w.b * p.dsi_s + w.c, w.on, carry);
  exchange.leave();
}

}  // namespace

int read_grad_device_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_grad_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_grad_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

cudaError_t launch_grad(const ScanParams& p, int x_dtype, int g_dtype, bool wide, cudaStream_t s) {
  return by_types(x_dtype, g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    const size_t smem =
        2 * Ring<TX, true, kStages>::kBytes + Ring<TG, true, kStages>::kBytes + cluster_bytes(p.cluster);
    if (p.q_start)
      return launch_tiles(wide ? scan_grad_kernel<TX, TG, true, true> : scan_grad_kernel<TX, TG, false, true>, p,
                          smem, s);
    return launch_tiles(wide ? scan_grad_kernel<TX, TG, true, false> : scan_grad_kernel<TX, TG, false, false>, p,
                        smem, s);
  });
}

}  // namespace scan
}  // namespace kda
