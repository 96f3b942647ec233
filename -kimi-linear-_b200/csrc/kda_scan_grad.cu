// kda_scan_grad.cu -- gradient of the gated linear recurrence.  With u_t what flows into h_t
// from later tokens (u of the last: dstate_out):
//   d_t = dh_t + u_t,  u_{t-1} = a_t d_t
//   dx_t = w_t d_t,  dg_t = a_t (h_{t-1} - [complement] x_t) d_t,  dstate_in = u_{-1}
// It needs h_{t-1} in 32 bits: h is in x's type, so a tile's states are computed again from
// the checkpoint that the forward pass left at its start.  The blocks, threads and pieces are
// those of scan_kernel (kda_scan.cu), the tiles taken from the last to the first.
// Memory bounds it: 4 x 8192 x 2048, bf16 with fp32 decays: 157 us, 91 % of what a copy reaches.
#include <type_traits>

#include "kda_scan.cuh"

namespace kda {
namespace scan {

__device__ int g_grad_device_error = 0;

namespace {

// As in the scan; the long shape's tiles are shorter where values have 32 bits, so that they fit.
template <typename TX>
using Long = std::conditional_t<sizeof(TX) == 4, Shape<8, 4, 1>, Shape<12, 4, 1>>;
using Short = Shape<4, 1, 3>;
constexpr int kXSlots = 4, kGSlots = 2;
// A thread's decays of a turn, and 1 - a for the complement.
template <bool COMPLEMENT>
struct Run {
  float2 a[kRun][kPairs], w[COMPLEMENT ? kRun : 1][kPairs];
};
template <typename SHAPE>
struct Shared {
  Parts<SHAPE> parts[2];
  float back[2][SHAPE::kParts][kChannels];   // the parts' gradients from zero, then what enters them
  uint64_t full[kXSlots], exchange[2];
  TileRows<SHAPE> rows;                      // packed
  int lost;                                  // a worker has gone on without its rows
};

template <typename TX, typename TG, typename Bwd, bool WIDE, bool PACKED, bool COMPLEMENT>
__global__ void __launch_bounds__(Bwd::kThreads, Bwd::kBlocks)
scan_grad_kernel(const ScanParams p, const __grid_constant__ CUtensorMap x_map,
                 const __grid_constant__ CUtensorMap g_map, const __grid_constant__ CUtensorMap d_map) {
  extern __shared__ __align__(128) unsigned char smem[];
  using XRing = Ring<TX, Bwd::kTile, kXSlots>;
  using GRing = Ring<TG, Bwd::kTile, kGSlots>;
  const XRing xs{smem}, ds{smem + XRing::kBytes};
  const GRing gs{smem + 2 * XRing::kBytes};
  Shared<Bwd>& sh = *reinterpret_cast<Shared<Bwd>*>(smem + 2 * XRing::kBytes + GRing::kBytes);
  const Place w = my_place<WIDE>(p);
  const Exchange exchange(sh.exchange, reinterpret_cast<float*>(&sh + 1), p, w.rank);
  Patience patience(&g_grad_device_error, &sh.lost, p.hasty);
  const int turns = (p.tiles + p.cluster - 1) / p.cluster;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kXSlots; ++i) ptx::mbar_init(sh.full + i, 1);
    exchange.init();
    sh.lost = 0;
    ptx::fence_mbar_init();
  }
  const auto tile_of = [&](int k) { return (turns - 1 - k) * p.cluster + w.rank; };
  const auto first_row = [&](int k, int part) { return tile_of(k) * Bwd::kTile + part * kRun; };
  if constexpr (PACKED) {
    ptx::grid_dep_wait();
    if (threadIdx.x < 2 * Bwd::kParts) {
      const int k = threadIdx.x / Bwd::kParts, part = threadIdx.x % Bwd::kParts;
      sh.rows.bits[k][part] = packed_rows(p, first_row(k, part));
    }
  }
  __syncthreads();
  exchange.barrier();
  if (threadIdx.x >= Bwd::kWork) {
    // two channels' gradients from turn to turn, their states in a tile, and the copies
    const int at = threadIdx.x % 32, warp = (threadIdx.x - Bwd::kWork) / 32;
    const int ch0 = w.block_c + shared_channel<WIDE>(2 * at), ch1 = w.block_c + shared_channel<WIDE>(2 * at + 1);
    const bool copies = WIDE && warp == 0 && at == 0;
    int asked = 0;                   // turns whose copies have been asked for
    const auto copy = [&](int k) {
      if (k >= turns) return;
      asked = k + 1;
      const int tile = tile_of(k);
      uint64_t* bar = sh.full + k % kXSlots;
      if (tile >= p.tiles) {         // (the first turn's may be missing: its phase passes all the same)
        ptx::mbar_arrive(bar);
        return;
      }
      ptx::mbar_arrive_expect_tx(bar, (p.dh ? 2 : 1) * XRing::kTileBytes + GRing::kTileBytes);
      gs.copy(&g_map, k, w.block_c, tile * Bwd::kTile, w.b, bar);
      xs.copy(&x_map, k, w.block_c, tile * Bwd::kTile, w.b, bar);
      if (p.dh) ds.copy(&d_map, k, w.block_c, tile * Bwd::kTile, w.b, bar);
    };
    if (copies)
      for (int k = 0; k < 2; ++k) copy(k);
    float2 carry = both(0.f);
    if (!PACKED && p.dstate_out) {
      if (ch0 < p.D) carry.x = p.dstate_out[w.b * p.dso_s + ch0];
      if (ch1 < p.D) carry.y = p.dstate_out[w.b * p.dso_s + ch1];
    }
    // the states that enter the parts: a checkpoint's by a warp, the last first, so that the warps that
    // copy and send have the least
    static_assert(Bwd::kTile % kStep == 0 && kStep % kRun == 0, "a tile starts at a checkpoint");
    constexpr int kSteps = Bwd::kTile / kStep, kStepParts = kStep / kRun;
    static_assert(kSteps <= Bwd::kCarryWarps, "a warp for every checkpoint");
    const int step = Bwd::kCarryWarps - 1 - warp;
    // (the first turn's tile may be missing, and the last steps of its last one)
    const auto checkpoint = [&](int k) {
      float2 s = both(0.f);
      const int i = tile_of(k) * kSteps + step;
      if (k >= turns || step >= kSteps || i >= p.steps) return s;
      const float* row = p.ckpt + ((int64_t)w.b * p.steps + i) * p.D;
      if (ch0 < p.D) s.x = row[ch0];
      if (ch1 < p.D) s.y = row[ch1];
      return s;
    };
    float2 next = checkpoint(0);
    for (int k = 0; k < turns; ++k) {
      const int buf = k & 1;
      float2 state = next;
      // (packed: rows of two turns on, asked for while the workers are busy; they are done with turn
      // k - 2, whose place these take, when turn k's pieces are there)
      const bool fetches = PACKED && warp == Bwd::kCarryWarps - 1 && at < Bwd::kParts;
      const uint32_t ahead = fetches ? packed_rows(p, first_row(k + 2, at)) : 0;
      pieces_wait(buf, Bwd::kThreads);
      if (fetches) sh.rows.bits[(k + 2) & 3][at] = ahead;
      // the workers are done with the gates of turn k and with the other rows of turn k - 2
      if (copies && !patience.gone && *const_cast<volatile int*>(&sh.lost) == 0) copy(k + 2);
      next = checkpoint(k + 1);
      uint32_t cuts = 0, starts = 0;
      if constexpr (PACKED) {
        starts = sh.rows.starts(k);
        cuts = sh.rows.ends(k);
      }
      Parts<Bwd>& parts = sh.parts[buf];
      enter_parts<PACKED, true>(exchange, patience, k, parts, sh.back[buf], cuts, carry, warp, at, [&] {
        if (step >= kSteps) return;
#pragma unroll
        for (int j = 0; j < kStepParts; ++j) {
          const int i = step * kStepParts + j;
          const Piece q{pair(parts.c[i], at), PACKED && (starts >> i & 1) ? cut() : pair(parts.r[i], at),
                        pair(parts.h[i], at)};
          pair(parts.h[i], at) = state;
          state = pass_on<PACKED>(q, state);
        }
      });
      states_done(buf, Bwd::kThreads);
    }
    if (!PACKED && p.dstate_in && w.rank == 0 && warp == 0) {
      if (ch0 < p.D) p.dstate_in[w.b * p.dsi_s + ch0] = carry.x;
      if (ch1 < p.D) p.dstate_in[w.b * p.dsi_s + ch1] = carry.y;
    }
    if (copies) {                    // (a worker may have given up)
      for (int k = max(asked - kXSlots, 0); k < asked; ++k) patience.land(sh.full + k % kXSlots, k / kXSlots & 1);
    }
  } else {
    const int part = threadIdx.x / kLanes, row0 = part * kRun;
    const TX* x = static_cast<const TX*>(p.x) + w.b * p.x_s[0] + w.c;
    const TG* g = static_cast<const TG*>(p.g) + w.b * p.g_s[0] + w.c;
    const TX* dh = p.dh ? static_cast<const TX*>(p.dh) + w.b * p.dh_s[0] + w.c : nullptr;
    TX* const dx = p.dx ? static_cast<TX*>(p.dx) + w.b * p.dx_s[0] + w.c : nullptr;
    TG* const dg = p.dg ? static_cast<TG*>(p.dg) + w.b * p.dg_s[0] + w.c : nullptr;
    // d_t = dh_t + u_t in the place of d_{t+1} (for the last token of the run: of u_t)
    const auto add_later = [&](auto each, int k, int t, int t0, const RowMask& m, const Run<COMPLEMENT>& run,
                               float2 (&u)[kPairs]) {
      float2 d[kPairs] = {both(0.f), both(0.f)};
      if (p.dh) ds.read(k, row0 + t, d);
      const bool last = decltype(each)::value && (m.last >> t & 1);
      if (last) load_state<WIDE>(state_of(p, p.dstate_out, p.dso_s, t0 + t, w.c), w.on, u);
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        u[j] = t == kRun - 1 || last ? __fadd2_rn(d[j], u[j]) : __ffma2_rn(run.a[t + 1 < kRun ? t + 1 : t][j], u[j], d[j]);
    };
    const auto pieces = [&](int k, int buf, Run<COMPLEMENT>& run) {
      const int t0 = first_row(k, part);
      Parts<Bwd>& parts = sh.parts[buf];
      if (WIDE) patience.wait(sh.full + k % kXSlots, k / kXSlots & 1);
      if (t0 - row0 >= p.T) {        // no tile: nothing changes
        const float2 one[kPairs] = {both(1.f), both(1.f)}, zero[kPairs] = {};
        put(parts.c[part], one);
        put(parts.r[part], zero);
        put(parts.h[part], zero);
        put(sh.back[buf][part], zero);
        pieces_done(buf, Bwd::kThreads);
        return;
      }
      const RowMask m = PACKED ? sh.rows.of(k, part) : batch_rows(p, t0);
      const bool plain = PACKED && m.plain();
      if constexpr (!WIDE) {
        xs.copy_own(x + (int64_t)t0 * p.x_s[1], p.x_s[1], k, row0, m.there, w.on);
        gs.copy_own(g + (int64_t)t0 * p.g_s[1], p.g_s[1], k, row0, m.there, w.on);
        if (p.dh) ds.copy_own(dh + (int64_t)t0 * p.dh_s[1], p.dh_s[1], k, row0, m.there, w.on);
      }
      // (rows past T are zeros: they change nothing; packed rows of no sequence are not)
      if (PACKED && WIDE && m.there != kAllRows) {
        gs.clear(k, row0, m.there);
        xs.clear(k, row0, m.there);
        ds.clear(k, row0, m.there);
      }
      float2 sum[kPairs], c[kPairs], r[kPairs], h[kPairs], u[kPairs];
      sum[0] = sum[1] = h[0] = h[1] = u[0] = u[1] = both(0.f);
      by_rows<PACKED>(plain, [&](auto each) {
        constexpr bool EACH = decltype(each)::value;
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
          float2 gt[kPairs], v[kPairs];
          gs.read(k, row0 + t, gt);
          xs.read(k, row0 + t, v);
          if (EACH && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, h);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            run.a[t][j] = decay(gt[j]);
            sum[j] = __fadd2_rn(sum[j], gt[j]);
            if (COMPLEMENT) {
              run.w[t][j] = rest(gt[j], run.a[t][j]);
              v[j] = __fmul2_rn(v[j], run.w[t][j]);
            }
            h[j] = __ffma2_rn(run.a[t][j], h[j], v[j]);
          }
        }
#pragma unroll
        for (int t = kRun - 1; t >= 0; --t) add_later(each, k, t, t0, m, run, u);
      });
#pragma unroll
      for (int j = 0; j < kPairs; ++j) u[j] = __fmul2_rn(run.a[0][j], u[j]);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) split_decay(sum[j], c[j], r[j]);
      put(parts.c[part], c);
      put(parts.r[part], r);
      put(parts.h[part], h);
      put(sh.back[buf][part], u);
      pieces_done(buf, Bwd::kThreads);
    };
    const auto grads = [&](int k, int buf, const Run<COMPLEMENT>& run) {
      const int t0 = first_row(k, part);
      states_wait(buf, Bwd::kThreads);
      const RowMask m = PACKED ? sh.rows.of(k, part) : batch_rows(p, t0);
      const bool plain = PACKED && m.plain();      // (before any lane leaves)
      if (t0 >= p.T || (WIDE && !w.on)) return;
      by_rows<PACKED>(plain, [&](auto each) {
        constexpr bool EACH = decltype(each)::value;
        float2 h[kPairs], u[kPairs], v[kRun][kPairs];
        // a_t h_{t-1} (complement: a_t (h_{t-1} - x_t))
        get(sh.parts[buf].h[part], h);
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
          float2 xt[kPairs];
          xs.read(k, row0 + t, xt);
          if (EACH && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, h);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            if (COMPLEMENT) {
              v[t][j] = __fmul2_rn(run.a[t][j], __ffma2_rn(xt[j], both(-1.f), h[j]));
              h[j] = __ffma2_rn(run.a[t][j], h[j], __fmul2_rn(run.w[t][j], xt[j]));
            } else {
              v[t][j] = __fmul2_rn(run.a[t][j], h[j]);
              h[j] = __ffma2_rn(run.a[t][j], h[j], xt[j]);
            }
          }
        }
        get(sh.back[buf][part], u);
        TX* dx_row = dx ? dx + (int64_t)(t0 + kRun - 1) * p.dx_s[1] : nullptr;
        TG* dg_row = dg ? dg + (int64_t)(t0 + kRun - 1) * p.dg_s[1] : nullptr;
#pragma unroll
        for (int t = kRun - 1; t >= 0; --t) {
          float2 ox[kPairs], og[kPairs];
          add_later(each, k, t, t0, m, run, u);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            ox[j] = COMPLEMENT ? __fmul2_rn(run.w[t][j], u[j]) : u[j];
            og[j] = __fmul2_rn(v[t][j], u[j]);
          }
          const bool there = (PACKED && !EACH) || (m.there >> t & 1);
          if (EACH && !there) ox[0] = ox[1] = og[0] = og[1] = both(0.f);
          if (there || (EACH && t0 + t < p.T)) {
            if (dx) write<WIDE>(dx_row, w.on, ox);
            if (dg) write<WIDE>(dg_row, w.on, og);
          }
          if (dx) dx_row -= p.dx_s[1];
          if (dg) dg_row -= p.dg_s[1];
          if (EACH && p.dstate_in && (m.first >> t & 1)) {
            const float2 out[kPairs] = {__fmul2_rn(run.a[t][0], u[0]), __fmul2_rn(run.a[t][1], u[1])};
            store_state<WIDE>(state_of(p, p.dstate_in, p.dsi_s, t0 + t, w.c), w.on, out);
          }
        }
      });
    };
    Run<COMPLEMENT> a, b;
    for (int k = 0; k <= turns; k += 2) {
      if (k < turns) pieces(k, 0, a);
      if (k > 0) grads(k - 1, 1, b);
      if (k + 1 < turns) pieces(k + 1, 1, b);
      if (k < turns) grads(k, 0, a);
    }
  }
  exchange.barrier();                // no block leaves while another may still send to it
  if (exchange.cluster > 1) patience.linger();
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

namespace {
template <typename TX, typename TG, typename Bwd>
cudaError_t launch_shape(ScanParams p, bool wide, cudaStream_t s) {
  choose_cluster<Bwd>(p);
  CUtensorMap mx, mg, md;
  const bool tma = wide && encode<TX>(&mx, p.x, p.x_s, p, Bwd::kTile) && encode<TG>(&mg, p.g, p.g_s, p, Bwd::kTile) &&
                   encode<TX>(&md, p.dh, p.dh_s, p, Bwd::kTile);
  const size_t smem = 2 * Ring<TX, Bwd::kTile, kXSlots>::kBytes + Ring<TG, Bwd::kTile, kGSlots>::kBytes +
                      sizeof(Shared<Bwd>) + cluster_bytes(p.cluster);
  return by_flags(tma, p.q_start != nullptr, p.complement, [&](auto wide_, auto packed, auto complement) {
    return launch_tiles(scan_grad_kernel<TX, TG, Bwd, wide_.value, packed.value, complement.value>, p, Bwd::kThreads,
                        smem, s, mx, mg, md);
  });
}
}  // namespace

cudaError_t launch_grad(const ScanParams& p, int x_dtype, int g_dtype, bool wide, cudaStream_t s) {
  // (us, Long and Short, as the shapes came: 4 x 8192 x 2048 bf16, 128 blocks, 152 and 165; 1 x 4096 x 2048, 32 blocks, 27 and 31;
  // 16 x 2048 x 2048, 512 blocks, 166 and 205; 64 x 512 x 2048, 2048 blocks, 178 and 155)
  const bool is_long =
      (int64_t)(p.q_start ? 1 : p.B) * ((p.D + kChannels - 1) / kChannels) <= kSms || p.T >= 1024;
  return by_types(x_dtype, g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    return is_long ? launch_shape<TX, TG, Long<TX>>(p, wide, s) : launch_shape<TX, TG, Short>(p, wide, s);
  });
}

}  // namespace scan
}  // namespace kda
