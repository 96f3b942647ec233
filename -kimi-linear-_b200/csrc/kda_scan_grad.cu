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

constexpr int kWarps = 4;
constexpr int kXSlots = 4, kGSlots = 2;
using Bwd = Shape<kWarps>;

struct Shared {
  Parts<Bwd::kParts> parts[2];
  float back[2][Bwd::kParts][kChannels];   // the parts' gradients from zero, then what enters them
  uint64_t x_full[kXSlots], d_full[kXSlots], g_full[kGSlots], exchange[2];
  uint8_t ends[2][Bwd::kParts];      // packed: a sequence starts (1), ends (2) in the part
};

template <typename TX, typename TG, bool WIDE, bool PACKED, bool COMPLEMENT>
__global__ void __launch_bounds__(Bwd::kThreads, 3)
scan_grad_kernel(const ScanParams p, const __grid_constant__ CUtensorMap x_map,
                 const __grid_constant__ CUtensorMap g_map, const __grid_constant__ CUtensorMap d_map) {
  extern __shared__ __align__(128) unsigned char smem[];
  using XRing = Ring<TX, Bwd::kTile, kXSlots>;
  using GRing = Ring<TG, Bwd::kTile, kGSlots>;
  const XRing xs{smem}, ds{smem + XRing::kBytes};
  const GRing gs{smem + 2 * XRing::kBytes};
  Shared& sh = *reinterpret_cast<Shared*>(smem + 2 * XRing::kBytes + GRing::kBytes);
  const Place w = my_place<WIDE>(p);
  const Exchange exchange(sh.exchange, reinterpret_cast<float*>(&sh + 1), p, w.rank);
  Patience patience(&g_grad_device_error);
  const int turns = (p.tiles + p.cluster - 1) / p.cluster;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kXSlots; ++i) {
      ptx::mbar_init(sh.x_full + i, 1);
      ptx::mbar_init(sh.d_full + i, 1);
    }
    for (int i = 0; i < kGSlots; ++i) ptx::mbar_init(sh.g_full + i, 1);
    exchange.init();
    ptx::fence_mbar_init();
  }
  __syncthreads();
  exchange.barrier();
  const auto tile_of = [&](int k) { return (turns - 1 - k) * p.cluster + w.rank; };
  if (threadIdx.x >= Bwd::kWork) {
    // a channel's gradient from turn to turn, its states in a tile, and the copies
    const int i_ch = threadIdx.x - Bwd::kWork, ch = w.block_c + shared_channel<WIDE>(i_ch);
    const bool kept = ch < p.D, copies = WIDE && i_ch == 0;
    const auto copy = [&](int k) {
      const int tile = tile_of(k);
      uint64_t *xb = sh.x_full + k % kXSlots, *gb = sh.g_full + k % kGSlots, *db = sh.d_full + k % kXSlots;
      if (k >= turns) return;
      if (tile >= p.tiles) {         // (the first turn's may be missing: its phase passes all the same)
        ptx::mbar_arrive(xb);
        ptx::mbar_arrive(gb);
        if (p.dh) ptx::mbar_arrive(db);
        return;
      }
      xs.copy(&x_map, k, w.block_c, tile * Bwd::kTile, w.b, xb);
      gs.copy(&g_map, k, w.block_c, tile * Bwd::kTile, w.b, gb);
      if (p.dh) ds.copy(&d_map, k, w.block_c, tile * Bwd::kTile, w.b, db);
    };
    if (copies)
      for (int k = 0; k < 2; ++k) copy(k);
    if constexpr (PACKED) ptx::grid_dep_wait();
    float carry = !PACKED && kept && p.dstate_out ? p.dstate_out[w.b * p.dso_s + ch] : 0.f;
    const float* ckpt = p.ckpt + (int64_t)w.b * p.steps * p.D + ch;
    static_assert(Bwd::kTile == kStep, "a tile starts at a checkpoint");
    // (without tokens there is no tile at all; the first turn's may be missing)
    float next = turns > 0 && kept && tile_of(0) < p.tiles ? ckpt[(int64_t)tile_of(0) * p.D] : 0.f;
    for (int k = 0; k < turns; ++k) {
      const int buf = k & 1;
      float state = next;
      pieces_wait(buf, Bwd::kThreads);
      // the workers are done with the gates of turn k and with the other rows of turn k - 2
      if (copies && patience.limit) copy(k + 2);
      if (k + 1 < turns && kept) next = ckpt[(int64_t)tile_of(k + 1) * p.D];
      uint32_t cuts = 0, starts = 0;
      if constexpr (PACKED) {
#pragma unroll
        for (int i = 0; i < Bwd::kParts; ++i) {
          starts |= (uint32_t)(sh.ends[buf][i] & 1) << i;
          cuts |= (uint32_t)(sh.ends[buf][i] >> 1) << i;
        }
      }
#pragma unroll
      for (int i = 0; i < Bwd::kParts; ++i) {
        const Piece q{sh.parts[buf].c[i][i_ch], PACKED && (starts >> i & 1) ? cut() : sh.parts[buf].r[i][i_ch],
                      sh.parts[buf].h[i][i_ch]};
        sh.parts[buf].h[i][i_ch] = state;
        state = pass_on<PACKED>(q, state);
      }
      enter_parts<PACKED, true>(exchange, patience, k, sh.parts[buf], sh.back[buf], cuts, carry, i_ch);
      states_done(buf, Bwd::kThreads);
    }
    if (!PACKED && p.dstate_in && w.rank == 0 && kept) p.dstate_in[w.b * p.dsi_s + ch] = carry;
    if (copies) {                    // (a worker may have given up)
      Patience landed(&g_grad_device_error);
      for (int k = max(turns - 2, 0); k < turns; ++k) {
        landed.wait(sh.x_full + k % kXSlots, k / kXSlots & 1);
        landed.wait(sh.g_full + k % kGSlots, k / kGSlots & 1);
        if (p.dh) landed.wait(sh.d_full + k % kXSlots, k / kXSlots & 1);
      }
    }
  } else {
    if constexpr (PACKED) ptx::grid_dep_wait();
    const int part = threadIdx.x / kLanes, row0 = part * kRun;
    const TX* x = static_cast<const TX*>(p.x) + w.b * p.x_s[0] + w.c;
    const TG* g = static_cast<const TG*>(p.g) + w.b * p.g_s[0] + w.c;
    const TX* dh = p.dh ? static_cast<const TX*>(p.dh) + w.b * p.dh_s[0] + w.c : nullptr;
    TX* const dx = p.dx ? static_cast<TX*>(p.dx) + w.b * p.dx_s[0] + w.c : nullptr;
    TG* const dg = p.dg ? static_cast<TG*>(p.dg) + w.b * p.dg_s[0] + w.c : nullptr;
    // row t of the thread's x or dh of turn k; zeros for a row that is not there
    const auto read = [&](const XRing& ring, int k, int t, uint32_t there, bool tile_there, float2 (&v)[kPairs]) {
      ring.read(k, row0 + t, v);
      if (PACKED ? !(there >> t & 1) : !tile_there) v[0] = v[1] = both(0.f);
    };
    const auto pieces = [&](int k, int buf, Decays<COMPLEMENT>& a) {
      const int t0 = tile_of(k) * Bwd::kTile + row0;
      const RowMask m = row_mask<PACKED>(p, t0);
      const bool tile_there = t0 - row0 < p.T;
      if constexpr (WIDE) {
        patience.wait(sh.g_full + k % kGSlots, k / kGSlots & 1);
        patience.wait(sh.x_full + k % kXSlots, k / kXSlots & 1);
        if (p.dh) patience.wait(sh.d_full + k % kXSlots, k / kXSlots & 1);
      } else {
        xs.copy_own(x + (int64_t)t0 * p.x_s[1], p.x_s[1], k, row0, m.there, w.on);
        gs.copy_own(g + (int64_t)t0 * p.g_s[1], p.g_s[1], k, row0, m.there, w.on);
        if (p.dh) ds.copy_own(dh + (int64_t)t0 * p.dh_s[1], p.dh_s[1], k, row0, m.there, w.on);
      }
      float2 gt[kRun][kPairs], all_c[kPairs], all_r[kPairs], h[kPairs], u[kPairs];
#pragma unroll
      for (int t = 0; t < kRun; ++t) {
        gs.read(k, row0 + t, gt[t]);
        if (PACKED ? !(m.there >> t & 1) : !tile_there) gt[t][0] = gt[t][1] = both(0.f);
      }
      set_decays(a, gt, all_c, all_r);
      h[0] = h[1] = u[0] = u[1] = both(0.f);
#pragma unroll
      for (int t = 0; t < kRun; ++t) {
        float2 v[kPairs];
        read(xs, k, t, m.there, tile_there, v);
        if (PACKED && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, h);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          if (COMPLEMENT) v[j] = __fmul2_rn(v[j], rest(a.c(t, j), a.r[t][j]));
          h[j] = apply(a.c(t, j), a.r[t][j], h[j], v[j]);
        }
      }
#pragma unroll
      for (int t = kRun - 1; t >= 0; --t) {
        float2 d[kPairs] = {both(0.f), both(0.f)};
        if (p.dh) read(ds, k, t, m.there, tile_there, d);
        if (PACKED && (m.last >> t & 1)) load_state<WIDE>(state_of(p, p.dstate_out, p.dso_s, t0 + t, w.c), w.on, u);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) u[j] = times(a.c(t, j), a.r[t][j], __fadd2_rn(d[j], u[j]));
      }
      put(sh.parts[buf].c[part], all_c);
      put(sh.parts[buf].r[part], all_r);
      put(sh.parts[buf].h[part], h);
      put(sh.back[buf][part], u);
      if (PACKED && threadIdx.x % kLanes == 0) sh.ends[buf][part] = (m.first != 0) | (m.last != 0) << 1;
      pieces_done(buf, Bwd::kThreads);
    };
    const auto grads = [&](int k, int buf, const Decays<COMPLEMENT>& a) {
      const int t0 = tile_of(k) * Bwd::kTile + row0;
      const RowMask m = row_mask<PACKED>(p, t0);
      states_wait(buf, Bwd::kThreads);
      if ((WIDE && !w.on) || t0 >= p.T) return;
      float2 h[kPairs], u[kPairs], v[kRun][kPairs];
      // a_t h_{t-1} (complement: a_t (h_{t-1} - x_t))
      get(sh.parts[buf].h[part], h);
#pragma unroll
      for (int t = 0; t < kRun; ++t) {
        float2 xt[kPairs];
        read(xs, k, t, m.there, true, xt);
        if (PACKED && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, h);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const float2 c = a.c(t, j), r = a.r[t][j];
          if (COMPLEMENT) {
            v[t][j] = times(c, r, __ffma2_rn(xt[j], both(-1.f), h[j]));
            h[j] = apply(c, r, h[j], __fmul2_rn(rest(c, r), xt[j]));
          } else {
            v[t][j] = times(c, r, h[j]);
            h[j] = __fadd2_rn(v[t][j], xt[j]);
          }
        }
      }
      get(sh.back[buf][part], u);
#pragma unroll
      for (int t = kRun - 1; t >= 0; --t) {
        float2 d[kPairs] = {both(0.f), both(0.f)}, ox[kPairs], og[kPairs];
        if (p.dh) read(ds, k, t, m.there, true, d);
        if (PACKED && (m.last >> t & 1)) load_state<WIDE>(state_of(p, p.dstate_out, p.dso_s, t0 + t, w.c), w.on, u);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const float2 c = a.c(t, j), r = a.r[t][j];
          d[j] = __fadd2_rn(d[j], u[j]);
          ox[j] = COMPLEMENT ? __fmul2_rn(rest(c, r), d[j]) : d[j];
          og[j] = __fmul2_rn(v[t][j], d[j]);
          u[j] = times(c, r, d[j]);
        }
        const bool there = m.there >> t & 1;
        if (PACKED && !there) ox[0] = ox[1] = og[0] = og[1] = both(0.f);
        if (there || (PACKED && t0 + t < p.T)) {
          if (dx) write<WIDE>(dx + (int64_t)(t0 + t) * p.dx_s[1], w.on, ox);
          if (dg) write<WIDE>(dg + (int64_t)(t0 + t) * p.dg_s[1], w.on, og);
        }
        if (PACKED && p.dstate_in && (m.first >> t & 1))
          store_state<WIDE>(state_of(p, p.dstate_in, p.dsi_s, t0 + t, w.c), w.on, u);
      }
    };
    Decays<COMPLEMENT> a, b;
    for (int k = 0; k <= turns; k += 2) {
      if (k < turns) pieces(k, 0, a);
      if (k > 0) grads(k - 1, 1, b);
      if (k + 1 < turns) pieces(k + 1, 1, b);
      if (k < turns) grads(k, 0, a);
    }
  }
  exchange.barrier();                // no block leaves while another may still send to it
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

cudaError_t launch_grad(ScanParams p, int x_dtype, int g_dtype, bool wide, cudaStream_t s) {
  choose_cluster(p, Bwd::kTile, 3 * 148);
  return by_types(x_dtype, g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    CUtensorMap mx, mg, md;
    const bool tma = wide && encode<TX>(&mx, p.x, p.x_s, p, Bwd::kTile) &&
                     encode<TG>(&mg, p.g, p.g_s, p, Bwd::kTile) && encode<TX>(&md, p.dh, p.dh_s, p, Bwd::kTile);
    const size_t smem = 2 * Ring<TX, Bwd::kTile, kXSlots>::kBytes + Ring<TG, Bwd::kTile, kGSlots>::kBytes +
                        sizeof(Shared) + cluster_bytes(p.cluster);
    return by_flags(tma, p.q_start != nullptr, p.complement, [&](auto wide_, auto packed, auto complement) {
      return launch_tiles(scan_grad_kernel<TX, TG, wide_.value, packed.value, complement.value>, p, Bwd::kThreads,
                          smem, s, mx, mg, md);
    });
  });
}

}  // namespace scan
}  // namespace kda
