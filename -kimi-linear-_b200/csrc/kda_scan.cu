// kda_scan.cu -- gated linear recurrence h_t = a_t h_{t-1} + w_t x_t: scan, single-token
// step, and the C entry points (include/kda_b200.h); its gradient is in kda_scan_grad.cu.
//
// A block walks a sequence's tiles of kTile tokens for kChannels channels.  Its working warps
// read a tile from shared memory, where TMA copies put it two or three turns ahead: a half warp has a
// row, a thread kRun tokens of kVec channels.  Each thread runs over its tokens from a state of
// zero, which gives its piece: a decay and a state.  The carrying warps join the pieces of the
// tile, and of the cluster's blocks that have the sequence's neighbouring tiles (Exchange), and
// give back the state that enters each piece; from it the threads run over their tokens again,
// one turn later, while the carrying warps are busy with the next tile.
//
// Memory bounds it where there are blocks enough: 4 x 8192 x 2048, f16 with fp32 decays, 1 - a:
// 86 us, 96 % of what a copy reaches (without 1 - a 80 us).  A single sequence of 2048 channels has 32 blocks and
// their clusters, 128 SMs, and is bound by the exchange of a turn: 32768 tokens, bf16: 96 us, 64 %.  Packed
// rows cost the marks (4.5 us) and the look at them: 16000 tokens, f16: 74 us, unpacked 50.  Rows that
// TMA cannot address are copied by their threads: 4 x 1000 x 2047: 33 us, 31 %.
#include <cstring>

#include "kda_scan.cuh"

namespace kda {
namespace scan {

__device__ int g_scan_device_error = 0;

namespace {

// ---------------------------------------------------------------------------
// packed batches: what each row is
// ---------------------------------------------------------------------------
// Blocks below `marked`: kMarked rows each.  The others: a sequence without rows each, whose
// state (gradient) goes through.
__global__ void __launch_bounds__(kMarked) mark_kernel(const ScanParams p, int marked, Marks* marks,
                                                       const float* from, int64_t from_s, float* to, int64_t to_s) {
  if ((int)blockIdx.x < marked) {
    const int t = blockIdx.x * kMarked + threadIdx.x;
    const int b = sequence_at(p.q_start, p.B, t);
    const int end = b >= 0 ? min(p.q_start[b + 1], p.T) : 0;
    const bool owned = end > t;
    const uint32_t first = __ballot_sync(0xffffffffu, owned && p.q_start[max(b, 0)] == t);
    const uint32_t last = __ballot_sync(0xffffffffu, owned && end == t + 1);
    const uint32_t own = __ballot_sync(0xffffffffu, owned);
    marks[blockIdx.x].sequence[threadIdx.x] = max(b, 0);
    if (threadIdx.x % 32 == 0) {
      uint32_t* m = reinterpret_cast<uint32_t*>(marks + blockIdx.x) + threadIdx.x / 32;
      m[0] = first;
      m[2] = last;
      m[4] = own;
    }
    return;
  }
  const int b = blockIdx.x - marked;
  const int lo = min(max(p.q_start[b], 0), p.T), hi = min(p.q_start[b + 1], p.T);
  if (to == nullptr || hi > lo) return;
  for (int c = threadIdx.x; c < p.D; c += kMarked) to[b * to_s + c] = from ? from[b * from_s + c] : 0.f;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// Long sequences, one block an SM: fewer and larger exchanges.  Short ones, two blocks: one
// starts or ends while the other works.
using Long = Shape<16, 4, 1>;
using Short = Shape<8, 1, 2>;
// tiles in flight or in use: as many as fit
constexpr int kMaxSlots = 3;
template <typename TX, typename TG, typename SHAPE>
constexpr int kSlotsOf = sizeof(TX) + sizeof(TG) > 6 && SHAPE::kTile == 128 ? 2 : 3;

// A thread's decays and (weighed) inputs of a turn.
struct Run {
  float2 a[kRun][kPairs], v[kRun][kPairs];
};
template <typename SHAPE>
struct Shared {
  Parts<SHAPE> parts[2];             // of two turns
  uint64_t full[kMaxSlots], exchange[2];
  TileRows<SHAPE> rows;              // packed
  int lost;                          // a worker has gone on without its rows
};

template <typename TX, typename TG, typename Fwd, bool WIDE, bool PACKED, bool COMPLEMENT>
__global__ void __launch_bounds__(Fwd::kThreads, Fwd::kBlocks)
scan_kernel(const ScanParams p, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap g_map) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int kSlots = kSlotsOf<TX, TG, Fwd>;
  using XRing = Ring<TX, Fwd::kTile, kSlots>;
  using GRing = Ring<TG, Fwd::kTile, kSlots>;
  const XRing xs{smem};
  const GRing gs{smem + XRing::kBytes};
  Shared<Fwd>& sh = *reinterpret_cast<Shared<Fwd>*>(smem + XRing::kBytes + GRing::kBytes);
  const Place w = my_place<WIDE>(p);
  const Exchange exchange(sh.exchange, reinterpret_cast<float*>(&sh + 1), p, w.rank);
  Patience patience(&g_scan_device_error, &sh.lost, p.hasty);
  const int turns = (p.tiles + p.cluster - 1) / p.cluster;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) ptx::mbar_init(sh.full + i, 1);
    exchange.init();
    sh.lost = 0;
    ptx::fence_mbar_init();
  }
  const auto first_row = [&](int k, int part) { return (k * p.cluster + w.rank) * Fwd::kTile + part * kRun; };
  if constexpr (PACKED) {
    ptx::grid_dep_wait();
    if (threadIdx.x < 2 * Fwd::kParts) {
      const int k = threadIdx.x / Fwd::kParts, part = threadIdx.x % Fwd::kParts;
      sh.rows.bits[k][part] = packed_rows(p, first_row(k, part));
    }
  }
  __syncthreads();
  exchange.barrier();
  if (threadIdx.x >= Fwd::kWork) {
    // two channels' states from turn to turn, and the copies
    const int at = threadIdx.x % 32, warp = (threadIdx.x - Fwd::kWork) / 32;
    const int ch0 = w.block_c + shared_channel<WIDE>(2 * at), ch1 = w.block_c + shared_channel<WIDE>(2 * at + 1);
    const bool copies = WIDE && warp == 0 && at == 0;
    int asked = 0;                   // turns whose copies have been asked for
    const auto copy = [&](int k) {
      const int tile = k * p.cluster + w.rank;
      asked = k + 1;
      if (tile >= p.tiles) return;
      uint64_t* bar = sh.full + k % kSlots;
      ptx::mbar_arrive_expect_tx(bar, XRing::kTileBytes + GRing::kTileBytes);
      gs.copy(&g_map, k, w.block_c, tile * Fwd::kTile, w.b, bar);
      xs.copy(&x_map, k, w.block_c, tile * Fwd::kTile, w.b, bar);
    };
    if (copies)
      for (int k = 0; k < kSlots; ++k) copy(k);
    float2 carry = both(0.f);
    if (!PACKED && p.state_in) {
      if (ch0 < p.D) carry.x = p.state_in[w.b * p.si_s + ch0];
      if (ch1 < p.D) carry.y = p.state_in[w.b * p.si_s + ch1];
    }
    float* const ckpt = p.ckpt ? p.ckpt + (int64_t)w.b * p.steps * p.D : nullptr;
    for (int k = 0; k < turns; ++k) {
      const int buf = k & 1;
      // (packed: rows of two turns on, asked for while the workers are busy; they are done with turn
      // k - 2, whose place these take, when turn k's pieces are there)
      const bool fetches = PACKED && warp == Fwd::kCarryWarps - 1 && at < Fwd::kParts;
      const uint32_t ahead = fetches ? packed_rows(p, first_row(k + 2, at)) : 0;
      pieces_wait(buf, Fwd::kThreads);
      if (fetches) sh.rows.bits[(k + 2) & 3][at] = ahead;
      // the workers have read the rows of turn k
      if (copies && !patience.gone && *const_cast<volatile int*>(&sh.lost) == 0) copy(k + kSlots);
      uint32_t cuts = 0;
      if constexpr (PACKED) {
        cuts = sh.rows.starts(k);
      }
      Parts<Fwd>& parts = sh.parts[buf];
      enter_parts<PACKED, false>(exchange, patience, k, parts, parts.h, cuts, carry, warp, at, [] {});
      if (ckpt) {
        // the checkpoints that are in this warp's share of the parts
        constexpr int N = Fwd::kParts / Fwd::kCarryWarps;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int j = warp * N + i;
          if (j % (kStep / kRun)) continue;
          const int step = (k * p.cluster + w.rank) * (Fwd::kTile / kStep) + j / (kStep / kRun);
          const float2 s = pair(parts.h[j], at);
          if (step < p.steps && ch0 < p.D) ckpt[(int64_t)step * p.D + ch0] = s.x;
          if (step < p.steps && ch1 < p.D) ckpt[(int64_t)step * p.D + ch1] = s.y;
        }
      }
      states_done(buf, Fwd::kThreads);
    }
    if (!PACKED && w.rank == 0 && warp == 0) {
      if (ch0 < p.D) p.state_out[w.b * p.so_s + ch0] = carry.x;
      if (ch1 < p.D) p.state_out[w.b * p.so_s + ch1] = carry.y;
    }
    if (copies) {                    // (a worker may have given up)
      for (int k = max(asked - kSlots, 0); k < asked; ++k)
        if (k * p.cluster + w.rank < p.tiles) patience.land(sh.full + k % kSlots, k / kSlots & 1);
    }
  } else {
    const int part = threadIdx.x / kLanes, row0 = part * kRun;
    const TX* x = static_cast<const TX*>(p.x) + w.b * p.x_s[0] + w.c;
    const TG* g = static_cast<const TG*>(p.g) + w.b * p.g_s[0] + w.c;
    TX* const out = static_cast<TX*>(p.h) + w.b * p.h_s[0] + w.c;
    // turn k's pieces
    const auto pieces = [&](int k, int buf, Run& run) {
      const int t0 = first_row(k, part);
      Parts<Fwd>& parts = sh.parts[buf];
      if (t0 - row0 >= p.T) {        // no tile: nothing changes
        const float2 one[kPairs] = {both(1.f), both(1.f)}, zero[kPairs] = {};
        put(parts.c[part], one);
        put(parts.r[part], zero);
        put(parts.h[part], zero);
        pieces_done(buf, Fwd::kThreads);
        return;
      }
      const RowMask m = PACKED ? sh.rows.of(k, part) : batch_rows(p, t0);
      const bool plain = PACKED && m.plain();
      if constexpr (WIDE) {
        patience.wait(sh.full + k % kSlots, k / kSlots & 1);
      } else {
        xs.copy_own(x + (int64_t)t0 * p.x_s[1], p.x_s[1], k, row0, m.there, w.on);
        gs.copy_own(g + (int64_t)t0 * p.g_s[1], p.g_s[1], k, row0, m.there, w.on);
      }
      // (rows past T are zeros: they change nothing; packed rows of no sequence are not)
      if (PACKED && WIDE && m.there != kAllRows) {
        gs.clear(k, row0, m.there);
        xs.clear(k, row0, m.there);
      }
      float2 sum[kPairs], c[kPairs], r[kPairs], h[kPairs];
      sum[0] = sum[1] = h[0] = h[1] = both(0.f);
      by_rows<PACKED>(plain, [&](auto each) {
        constexpr bool EACH = decltype(each)::value;
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
          float2 gt[kPairs];
          gs.read(k, row0 + t, gt);
          xs.read(k, row0 + t, run.v[t]);
          if (EACH && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, h);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            run.a[t][j] = decay(gt[j]);
            sum[j] = __fadd2_rn(sum[j], gt[j]);
            if (COMPLEMENT) run.v[t][j] = __fmul2_rn(run.v[t][j], rest(gt[j], run.a[t][j]));
            h[j] = __ffma2_rn(run.a[t][j], h[j], run.v[t][j]);
          }
        }
      });
#pragma unroll
      for (int j = 0; j < kPairs; ++j) split_decay(sum[j], c[j], r[j]);
      put(parts.c[part], c);
      put(parts.r[part], r);
      put(parts.h[part], h);
      pieces_done(buf, Fwd::kThreads);
    };
    // turn k's tokens again, from the state that enters them
    const auto states = [&](int k, int buf, const Run& run) {
      const int t0 = first_row(k, part);
      states_wait(buf, Fwd::kThreads);
      const RowMask m = PACKED ? sh.rows.of(k, part) : batch_rows(p, t0);
      const bool plain = PACKED && m.plain();      // (before any lane leaves)
      if (t0 >= p.T || (WIDE && !w.on)) return;
      float2 h[kPairs];
      get(sh.parts[buf].h[part], h);
      TX* row = out + (int64_t)t0 * p.h_s[1];
      by_rows<PACKED>(plain, [&](auto each) {
        constexpr bool EACH = decltype(each)::value;
#pragma unroll
        for (int t = 0; t < kRun; ++t) {
          if (EACH && (m.first >> t & 1)) load_state<WIDE>(state_of(p, p.state_in, p.si_s, t0 + t, w.c), w.on, h);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) h[j] = __ffma2_rn(run.a[t][j], h[j], run.v[t][j]);
          if ((PACKED && !EACH) || (m.there >> t & 1)) {
            write<WIDE>(row, w.on, h);
          } else if (EACH && t0 + t < p.T) {
            const float2 zero[kPairs] = {};
            write<WIDE>(row, w.on, zero);
          }
          if (EACH && (m.last >> t & 1)) store_state<WIDE>(state_of(p, p.state_out, p.so_s, t0 + t, w.c), w.on, h);
          row += p.h_s[1];
        }
      });
    };
    // a turn's pieces before the turn before's states: those come meanwhile
    Run a, b;
    for (int k = 0; k <= turns; k += 2) {
      if (k < turns) pieces(k, 0, a);
      if (k > 0) states(k - 1, 1, b);
      if (k + 1 < turns) pieces(k + 1, 1, b);
      if (k < turns) states(k, 0, a);
    }
  }
  exchange.barrier();                // no block leaves while another may still send to it
  if (exchange.cluster > 1) patience.linger();
}

template <typename Fwd>
cudaError_t launch_shape(const ScanParams& p, int x_dtype, int g_dtype, bool wide, cudaStream_t s) {
  return by_types(x_dtype, g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    constexpr int kSlots = kSlotsOf<TX, TG, Fwd>;
    CUtensorMap mx, mg;
    const bool tma = wide && encode<TX>(&mx, p.x, p.x_s, p, Fwd::kTile) && encode<TG>(&mg, p.g, p.g_s, p, Fwd::kTile);
    const size_t smem = Ring<TX, Fwd::kTile, kSlots>::kBytes + Ring<TG, Fwd::kTile, kSlots>::kBytes +
                        sizeof(Shared<Fwd>) + cluster_bytes(p.cluster);
    return by_flags(tma, p.q_start != nullptr, p.complement, [&](auto wide_, auto packed, auto complement) {
      return launch_tiles(scan_kernel<TX, TG, Fwd, wide_.value, packed.value, complement.value>, p, Fwd::kThreads, smem,
                          s, mx, mg);
    });
  });
}
cudaError_t launch_forward(ScanParams p, int x_dtype, int g_dtype, bool wide, cudaStream_t s) {
  // (blocks: a sequence's channels, before clusters.  us, Long and Short, as the shapes came: 4 x 8192 x 2048
  // f16, 128 blocks, 84 and 127; 1 x 1024 x 2048, 32 blocks, 8.0 and 9.0; 8 x 4096 x 2048 bf16, 256 blocks, 74
  // and 69; 64 x 512 x 2048 f16, 2048 blocks, 100 and 87)
  const bool is_long = (int64_t)(p.q_start ? 1 : p.B) * ((p.D + kChannels - 1) / kChannels) <= kSms;
  if (is_long) {
    choose_cluster<Long>(p);
    return launch_shape<Long>(p, x_dtype, g_dtype, wide, s);
  }
  choose_cluster<Short>(p);
  return launch_shape<Short>(p, x_dtype, g_dtype, wide, s);
}

constexpr int kStepThreads = 128;

// One token: a thread has VEC channels of a row.
template <typename TX, typename TG, int VEC>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const ScanParams p, int blocks_per_row) {
  const int b = blockIdx.x / blocks_per_row;
  const int c = ((blockIdx.x - b * blocks_per_row) * kStepThreads + threadIdx.x) * VEC;
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
      const float2 gi = make_float2(g[i], g[i + 1]);
      float2 v = make_float2(x[i], x[i + 1]), c2, r;
      if (p.complement) v = __fmul2_rn(v, rest(gi, decay(gi)));
      split_decay(gi, c2, r);
      v = pass_on<false>({c2, r, v}, make_float2(h[i], h[i + 1]));
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

enum class Pass { kForward, kBackward, kToken };

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
  if (pass == Pass::kToken && a->T != 1) return KDA_ERR_SHAPE;
  if (a->x_dtype < KDA_DTYPE_F32 || a->x_dtype > KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
  if (a->g_dtype != KDA_DTYPE_F32 && a->g_dtype != a->x_dtype) return KDA_ERR_DTYPE;
  if (a->D == 0) return KDA_OK;
  const int xs = size_of(a->x_dtype), gs = size_of(a->g_dtype);
  const bool tokens = a->T > 0 && (a->B > 0 || a->q_start != nullptr);
  if (tokens && (!a->x || !a->g || (pass != Pass::kBackward && !a->h))) return KDA_ERR_NULL_POINTER;
  if (a->B > 0 && pass != Pass::kBackward && !a->state_out) return KDA_ERR_NULL_POINTER;
  if (tokens && pass == Pass::kBackward && !a->ckpt) return KDA_ERR_NULL_POINTER;
  if (misaligned(a->x, xs) || misaligned(a->h, xs) || misaligned(a->dh, xs) || misaligned(a->dx, xs) ||
      misaligned(a->g, gs) || misaligned(a->dg, gs) || misaligned(a->state_in, 4) ||
      misaligned(a->state_out, 4) || misaligned(a->dstate_out, 4) || misaligned(a->dstate_in, 4) ||
      misaligned(a->ckpt, 4) || misaligned(a->q_start, 4) || misaligned(a->slots, 4))
    return KDA_ERR_ALIGNMENT;
  if (pass == Pass::kToken) {
    if (a->slots && a->num_states < 0) return KDA_ERR_SHAPE;
    if (a->scatter && a->B > 0 && (a->state_in != a->state_out || a->state_in_stride != a->state_out_stride))
      return KDA_ERR_STRIDE;
  }
  return KDA_OK;
}

ScanParams to_params(const KdaScanArgs* a) {
  ScanParams p{};
  p.B = a->B; p.T = a->T; p.D = a->D;
  p.steps = (a->T + kStep - 1) / kStep;
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
  p.hasty = a->hasty != 0;
  p.slots = a->slots; p.num_states = a->num_states; p.scatter = a->scatter != 0;
  return p;
}

size_t workspace_bytes(const KdaScanArgs* a) {
  return a->q_start ? ((size_t)a->T + kMarked - 1) / kMarked * sizeof(Marks) : 0;
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
                    (pass == Pass::kForward ? aligned_rows(p.h, p.h_s, xs)
                                      : aligned_rows(p.dh, p.dh_s, xs) && aligned_rows(p.dx, p.dx_s, xs) &&
                                            aligned_rows(p.dg, p.dg_s, gs));
  if ((int64_t)(p.q_start ? 1 : p.B) * ((p.D + kChannels - 1) / kChannels) * kMaxCluster > 0x7fffffff)
    return KDA_ERR_SHAPE;
  cudaError_t e = cudaSuccess;
  if (p.q_start) {
    Marks* marks = static_cast<Marks*>(a->workspace);
    p.marks = marks;
    const bool fwd = pass == Pass::kForward;
    const int marked = (p.T + kMarked - 1) / kMarked;
    mark_kernel<<<marked + p.B, kMarked, 0, s>>>(p, marked, marks, fwd ? p.state_in : p.dstate_out,
                                                 fwd ? p.si_s : p.dso_s, fwd ? p.state_out : p.dstate_in,
                                                 fwd ? p.so_s : p.dsi_s);
    e = cudaGetLastError();
    if (p.T == 0) return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
  }
  if (e == cudaSuccess)
    e = pass == Pass::kForward ? launch_forward(p, a->x_dtype, a->g_dtype, wide, s)
                         : launch_grad(p, a->x_dtype, a->g_dtype, wide, s);
  return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

int run_step(const KdaScanArgs* a, void* stream) {
  int st = validate(a, Pass::kToken);
  if (st != KDA_OK) return st;
  if (a->D == 0 || a->B == 0) return KDA_OK;
  if ((st = check_device()) != KDA_OK) return st;
  const ScanParams p = to_params(a);
  const int xs = size_of(a->x_dtype), gs = size_of(a->g_dtype);
  const bool vec = p.D % 4 == 0 && !misaligned(p.x, 4 * xs) && !misaligned(p.h, 4 * xs) &&
                   !misaligned(p.g, 4 * gs) && !misaligned(p.state_in, 16) &&
                   !misaligned(p.state_out, 16) && p.x_s[0] % 4 == 0 && p.h_s[0] % 4 == 0 &&
                   p.g_s[0] % 4 == 0 && p.si_s % 4 == 0 && p.so_s % 4 == 0;
  const int per_row = (p.D + kStepThreads * (vec ? 4 : 1) - 1) / (kStepThreads * (vec ? 4 : 1));
  if ((int64_t)per_row * p.B > 0x7fffffff) return KDA_ERR_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = by_types(a->x_dtype, a->g_dtype, [&](auto x, auto g) {
    using TX = decltype(x);
    using TG = decltype(g);
    if (vec)
      step_kernel<TX, TG, 4><<<per_row * p.B, kStepThreads, 0, s>>>(p, per_row);
    else
      step_kernel<TX, TG, 1><<<per_row * p.B, kStepThreads, 0, s>>>(p, per_row);
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
  const size_t steps = ((size_t)a->T + kda::scan::kStep - 1) / kda::scan::kStep;
  return (a->q_start ? 1 : (size_t)a->B) * steps * (size_t)a->D;
}

size_t kda_scan_workspace_bytes(const KdaScanArgs* a) {
  if (kda::scan::validate_sizes(a) != KDA_OK) return 0;
  return kda::scan::workspace_bytes(a);
}

int kda_scan_fwd(const KdaScanArgs* a, void* stream) {
  return kda::scan::run_scan(a, kda::scan::Pass::kForward, stream);
}

int kda_scan_bwd(const KdaScanArgs* a, void* stream) {
  return kda::scan::run_scan(a, kda::scan::Pass::kBackward, stream);
}

int kda_scan_step(const KdaScanArgs* a, void* stream) { return kda::scan::run_step(a, stream); }

}  // extern "C"
