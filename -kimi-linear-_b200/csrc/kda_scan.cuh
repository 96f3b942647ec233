// kda_scan.cuh -- gated linear recurrence: parameters, the arithmetic of its decays, and
// what the scan and its gradient share.
//
// Inside a run of kRun tokens a decay is a = exp(g) in 24 bits.  Over a whole run, where it leads
// from one run to the next, it is held as c + r, c = 1 and r = a - 1 where |sum of g| is small
// and c = 0 (or next to it), r = a elsewhere: a in 24 bits is off by up to 2^-25, always to the same side for a
// steady g, which a state that remembers n runs adds up to n 2^-25.  (Rounding inside a run is not
// carried on.)  c h + r h is one instruction more than a product, and two channels share each
// (fma.f32x2), so a thread works on pairs of channels.
#pragma once

#include <cfloat>
#include <type_traits>

#include "kda_internal.cuh"
#include "tc_ptx.cuh"

namespace kda {
namespace scan {

constexpr int kErrSlot = 8;       // device error word: a step's slot past the pool
constexpr int kErrWait = 9;       // device error word: a wait for a cluster's piece ran out
constexpr int kStep = 32;         // tokens between two checkpoints of the state
constexpr int kMarked = 64;       // rows of a packed batch that one Marks describes

// What kMarked rows of a packed batch are, a bit a row; and each row's sequence.
struct Marks {
  uint64_t first, last, owned;      // of a sequence; by any sequence
  int sequence[kMarked];            // (that of the last row before it where it is not owned, or 0)
};

// Device-side view of KdaScanArgs (strides in elements).
struct ScanParams {
  int B, T, D;
  int tiles;                        // the kernel's tiles of a sequence (packed: of all rows)
  int steps;                        // checkpoints of the same
  bool complement;
  const void* x; int64_t x_s[2];
  const void* g; int64_t g_s[2];
  const float* state_in; int64_t si_s;
  const int* q_start;               // or null: a batch
  void* h; int64_t h_s[2];
  float* state_out; int64_t so_s;
  float* ckpt;                      // [B][steps][D], packed [steps][D]
  const void* dh; int64_t dh_s[2];
  const float* dstate_out; int64_t dso_s;
  void* dx; int64_t dx_s[2];
  void* dg; int64_t dg_s[2];
  float* dstate_in; int64_t dsi_s;
  const Marks* marks;               // packed: of all rows, made by mark_kernel
  int cluster;                      // blocks that share a sequence's tiles
  bool hasty;                       // waits give up at once
  // step
  const int* slots; int num_states; bool scatter;
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp(g) = 2^(g log2 e) by the hardware's instruction: off by 2^-22 of itself, and 2^-24 |g| from
// the rounded exponent.  What is below 2^-126 is zero (which makes an infinite state a NaN).
__device__ __forceinline__ float2 decay(float2 g) {
  const float2 e = __fmul2_rn(g, both(1.4426950408889634f));
  return make_float2(exp2_fast(e.x), exp2_fast(e.y));
}
// exp(g) - 1 by its series up to g^5/5!, of which the first term left out is 2^-24 of the sum at
// |g| = kNear.
constexpr float kNear = 0.125f;
__device__ __forceinline__ float2 decay_less_one(float2 g) {
  float2 p = __ffma2_rn(g, both(1.f / 120.f), both(1.f / 24.f));
  p = __ffma2_rn(p, g, both(1.f / 6.f));
  p = __ffma2_rn(p, g, both(0.5f));
  p = __ffma2_rn(p, g, both(1.f));
  return __fmul2_rn(p, g);
}
// exp(g) as c + r.  c is zero for g = -infinity alone: below kNear it is the smallest number, which
// adds nothing to a finite state and keeps an infinite one (pass_on).
constexpr float kLeast = 0x1p-149f;
__device__ __forceinline__ void split_decay(float2 g, float2& c, float2& r) {
  const float2 p = decay_less_one(g), e = decay(g);
  const bool x = fabsf(g.x) < kNear, y = fabsf(g.y) < kNear;
  c = make_float2(x ? 1.f : g.x < -FLT_MAX ? 0.f : kLeast, y ? 1.f : g.y < -FLT_MAX ? 0.f : kLeast);
  r = make_float2(x ? p.x : e.x, y ? p.y : e.y);
}
// 1 - exp(g), a = exp(g) given.  From |g| = 1/2 on it is 1 - a, off by what a is off times a / (1 - a),
// at most 1.55.  Nearer it is g (1 + g q(g)), q of degree 4 for the least largest error
// relative to 1 - exp(g) over -1/2 .. 1/8 (0.12 of 2^-24, its coefficients in 24 bits): with its roundings
// off by 2.4 x 2^-24.  (1 - a alone would lose three bits at 1/8; of the series in g eight terms would
// be needed.  4 x 8192 x 2048, f16: 86 us, with eight terms 91.)
__device__ __forceinline__ float2 rest(float2 g, float2 a) {
  float2 p = __ffma2_rn(g, both(1.1894653e-3f), both(8.2695400e-3f));
  p = __ffma2_rn(p, g, both(4.1663043e-2f));
  p = __ffma2_rn(p, g, both(0.16666764f));
  p = __ffma2_rn(p, g, both(0.50000006f));
  p = __ffma2_rn(p, g, both(1.f));
  p = __fmul2_rn(p, g);
  const float2 w = __ffma2_rn(a, both(-1.f), both(1.f));
  // -1/2 < g <= -0 by its bits, so that one compare does (g = 0: 1 - a is as right)
  const auto near = [](float v) { return __float_as_int(v) < (int)0xbf000000; };
  return make_float2(near(g.x) ? -p.x : w.x, near(g.y) ? -p.y : w.y);
}

// The last sequence of a packed batch that starts at row t or before it (-1: none).  Of those
// that start at one row only the last can have tokens.
__device__ __forceinline__ int sequence_at(const int* q_start, int B, int t) {
  int lo = 0, hi = B;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (q_start[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

constexpr int kLanes = 16;                    // threads that share a row
constexpr int kVec = 4;                       // channels of a thread
constexpr int kPairs = kVec / 2;
constexpr int kChannels = kLanes * kVec;      // of a block
constexpr int kRun = 4;                       // tokens of a thread in a tile
constexpr int kMaxCluster = 8;
constexpr int kSms = 148;
constexpr uint64_t kWaitNs = 2000000000;      // a wait that takes longer gives up (device error word 9)
constexpr uint64_t kLingerNs = 1000000;

// A block: WORK warps that do the tokens, and CARRY warps that carry states from tile to tile
// (a lane has a pair of channels, a warp its share of the parts).
template <int WORK, int CARRY, int BLOCKS>
struct Shape {
  static constexpr int kWork = WORK * 32, kCarryWarps = CARRY, kCarry = CARRY * 32, kThreads = kWork + kCarry;
  static constexpr int kBlocks = BLOCKS;               // on an SM
  static constexpr int kParts = kWork / kLanes;        // half warps, each with kRun tokens of a tile
  static constexpr int kTile = kParts * kRun;
  static_assert(kParts % CARRY == 0, "shares of the parts");
  static_assert(kParts <= 32, "append() counts on it");
};

// ---------------------------------------------------------------------------
// waits
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool here(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(ptx::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// A thread whose wait runs out goes on, so that the block's other barriers stay matched, and
// waits no more.
struct Patience {
  int* error;
  int* lost;                         // the block's: rows that have not come must not be asked for again
  bool gone;                         // given up
  __device__ Patience(int* error_, int* lost_, bool gone_) : error(error_), lost(lost_), gone(gone_) {}
  __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
    if (here(bar, parity)) return;
    const uint64_t start = ptx::globaltimer_ns();
    while (!gone && !here(bar, parity)) gone = ptx::globaltimer_ns() - start >= kWaitNs;
    if (gone) {
      *error = kErrWait;
      *lost = 1;
    }
  }
  // what is in flight as the block leaves, whoever has given up
  __device__ __forceinline__ void land(uint64_t* bar, uint32_t parity) {
    const uint64_t start = ptx::globaltimer_ns();
    while (!here(bar, parity)) {
      if (ptx::globaltimer_ns() - start < kWaitNs) continue;
      *error = kErrWait;
      return;
    }
  }
  // One that has given up stays, behind the cluster's last barrier, until what the others had sent
  // by then has landed in its block's memory: no barrier of its own counts that any more.
  __device__ __forceinline__ void linger() const {
    if (!gone) return;
    const uint64_t start = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - start < kLingerNs) {}
  }
};
// a barrier of the carrying threads alone
template <int THREADS>
__device__ __forceinline__ void carry_sync() {
  asm volatile("barrier.cta.sync 5, %0;" ::"n"(THREADS) : "memory");
}
// The block's named barriers, two of each kind (buf 0 and 1): the workers' pieces are there (the
// workers go on, the carrying threads wait); the states that enter the parts are there (the
// other way round).
template <int ID>
__device__ __forceinline__ void bar_arrive(int count) {
  asm volatile("barrier.cta.arrive %0, %1;" ::"n"(ID), "r"(count) : "memory");
}
template <int ID>
__device__ __forceinline__ void bar_sync(int count) {
  asm volatile("barrier.cta.sync %0, %1;" ::"n"(ID), "r"(count) : "memory");
}
__device__ __forceinline__ void pieces_done(int buf, int count) { buf ? bar_arrive<2>(count) : bar_arrive<1>(count); }
__device__ __forceinline__ void pieces_wait(int buf, int count) { buf ? bar_sync<2>(count) : bar_sync<1>(count); }
__device__ __forceinline__ void states_done(int buf, int count) { buf ? bar_arrive<4>(count) : bar_arrive<3>(count); }
__device__ __forceinline__ void states_wait(int buf, int count) { buf ? bar_sync<4>(count) : bar_sync<3>(count); }

// ---------------------------------------------------------------------------
// a block's place and its rows in shared memory
// ---------------------------------------------------------------------------
// Shared rows have kChannels values; a thread has kVec next to each other.  WIDE: they are
// channels next to each other too, and a tile comes by one TMA copy.  Else (rows that
// TMA or a thread's stores cannot address) the thread's channels are every kLanes-th, so that
// a half warp reads and writes whole sectors, and it copies them itself.
struct Place {
  int rank;                          // in the cluster: tiles rank, rank + cluster, ...
  int b;                             // sequence (packed: 0)
  int block_c, c;                    // the block's and the thread's first channel
  uint32_t on;                       // which channels exist (WIDE: all or none)
};
template <bool WIDE>
__device__ __forceinline__ int channel(int i) { return WIDE ? i : i * kLanes; }
// where value i of a shared row lies from the block's first channel
template <bool WIDE>
__device__ __forceinline__ int shared_channel(int i) { return WIDE ? i : i / kVec + i % kVec * kLanes; }
template <bool WIDE>
__device__ __forceinline__ Place my_place(const ScanParams& p) {
  Place w;
  const int blocks = (p.D + kChannels - 1) / kChannels;
  const int i = blockIdx.x / p.cluster, lane = threadIdx.x % kLanes;
  w.rank = blockIdx.x - i * p.cluster;
  w.b = i / blocks;
  w.block_c = (i - w.b * blocks) * kChannels;
  w.c = w.block_c + (WIDE ? lane * kVec : lane);
  w.on = 0;
#pragma unroll
  for (int j = 0; j < kVec; ++j)
    if (w.c + channel<WIDE>(j) < p.D) w.on |= 1u << j;
  return w;
}

// Tiles of one tensor in a ring of SLOTS.
template <typename T, int TILE, int SLOTS>
struct Ring {
  static constexpr int kTileBytes = TILE * kChannels * sizeof(T);
  static constexpr int kBytes = SLOTS * kTileBytes;
  unsigned char* base;
  __device__ T* row(int k, int i) const {
    return reinterpret_cast<T*>(base + (k % SLOTS) * kTileBytes) + i * kChannels;
  }
  // one thread: tile k from row t on, its bytes counted on `bar`
  __device__ void copy(const CUtensorMap* map, int k, int c, int t, int b, uint64_t* bar) const {
    ptx::tma_load_3d(base + (k % SLOTS) * kTileBytes, map, c, t, b, bar);
  }
  // a thread: its rows i .. i + kRun - 1 of tile k, those in `mask` (the others: zeros)
  __device__ void copy_own(const T* src, int64_t stride, int k, int i, uint32_t mask, uint32_t on) const {
    T v[kRun][kVec];
#pragma unroll
    for (int t = 0; t < kRun; ++t)
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        v[t][j] = (mask >> t & 1) && (on >> j & 1) ? src[t * stride + channel<false>(j)] : T(0.f);
#pragma unroll
    for (int t = 0; t < kRun; ++t)
#pragma unroll
      for (int j = 0; j < kVec; ++j) row(k, i + t)[threadIdx.x % kLanes * kVec + j] = v[t][j];
  }
  // a thread: zeros for its rows that are not in `mask`
  __device__ void clear(int k, int i, uint32_t mask) const {
#pragma unroll
    for (int t = 0; t < kRun; ++t) {
      const float zero[kVec] = {};
      if (!(mask >> t & 1)) st4(row(k, i + t) + threadIdx.x % kLanes * kVec, zero);
    }
    ptx::fence_proxy_async_smem();   // (TMA writes here again)
  }
  __device__ __forceinline__ void read(int k, int i, float2 (&v)[kPairs]) const {
    float t[kVec];
    ld4(row(k, i) + threadIdx.x % kLanes * kVec, t);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) v[j] = make_float2(t[2 * j], t[2 * j + 1]);
  }
};
template <bool WIDE, typename T>
__device__ __forceinline__ void write(T* p, uint32_t on, const float2 (&v)[kPairs]) {
  float t[kVec];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    t[2 * j] = v[j].x;
    t[2 * j + 1] = v[j].y;
  }
  if constexpr (WIDE) {
    st4(p, t);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (on >> j & 1) st(p + channel<WIDE>(j), t[j]);
  }
}

// A state row of fp32 values, any alignment; zeros without one.
template <bool WIDE>
__device__ __forceinline__ void load_state(const float* row, uint32_t on, float2 (&v)[kPairs]) {
  float t[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) t[j] = row != nullptr && (on >> j & 1) ? row[channel<WIDE>(j)] : 0.f;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) v[j] = make_float2(t[2 * j], t[2 * j + 1]);
}
template <bool WIDE>
__device__ __forceinline__ void store_state(float* row, uint32_t on, const float2 (&v)[kPairs]) {
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    if (on >> (2 * j) & 1) row[channel<WIDE>(2 * j)] = v[j].x;
    if (on >> (2 * j + 1) & 1) row[channel<WIDE>(2 * j + 1)] = v[j].y;
  }
}
// The state of the packed sequence at row t.
__device__ __forceinline__ float* state_of(const ScanParams& p, const float* base, int64_t stride, int t, int c) {
  if (base == nullptr) return nullptr;
  return const_cast<float*>(base) + p.marks[t / kMarked].sequence[t % kMarked] * stride + c;
}

// Which of rows t .. t + kRun - 1 are there (bits), and for packed batches which start and end
// a sequence; held as there | first << kRun | last << 2 kRun.
constexpr uint32_t kAllRows = (1u << kRun) - 1;
struct RowMask {
  uint32_t there, first, last;
  __device__ RowMask() : there(0), first(0), last(0) {}
  __device__ explicit RowMask(uint32_t bits)
      : there(bits & kAllRows), first(bits >> kRun & kAllRows), last(bits >> 2 * kRun & kAllRows) {}
  // (warp-wide: all lanes of the warp have to ask) all rows are there, and no sequence starts or ends
  __device__ __forceinline__ bool plain() const {
    return __all_sync(0xffffffffu, there == kAllRows && (first | last) == 0);
  }
};
// Calls f with whether the rows have to be looked at one by one: branches between the rows of a
// run keep the next rows' reads behind them.  (Packed 16000 tokens of 2048 channels, f16: 23
// sequences, gradient 132 us to 120; of one 130 to 113; of 128, where most tiles have a boundary,
// 152 to 176: documents of 100 tokens pay for those of 700 and more.)
template <bool PACKED, typename F>
__device__ __forceinline__ void by_rows(bool plain, F f) {
  if constexpr (PACKED) {
    if (plain) f(std::false_type{});
    else f(std::true_type{});
  } else {
    f(std::false_type{});
  }
}
__device__ __forceinline__ uint32_t packed_rows(const ScanParams& p, int t) {
  if (t < 0 || t >= p.T) return 0;
  static_assert(kMarked % kRun == 0, "a run is inside one Marks");
  const Marks& k = p.marks[t / kMarked];
  const int at = t % kMarked;
  return (uint32_t)(k.owned >> at) & kAllRows | ((uint32_t)(k.first >> at) & kAllRows) << kRun |
         ((uint32_t)(k.last >> at) & kAllRows) << 2 * kRun;
}
__device__ __forceinline__ RowMask batch_rows(const ScanParams& p, int t) {
  RowMask m;
  const int left = t < 0 ? 0 : p.T - t;
  m.there = left >= kRun ? kAllRows : left > 0 ? (1u << left) - 1 : 0;
  return m;
}
// A packed tile's rows, by part, fetched two turns ahead by the carrying threads: a worker that
// fetched its own would wait for memory in every turn.
template <typename SHAPE>
struct TileRows {
  uint16_t bits[4][SHAPE::kParts];   // of turn k at k & 3
  __device__ RowMask of(int k, int part) const { return RowMask(bits[k & 3][part]); }
  // (warp-wide) which parts have a row in which a sequence starts (ends)
  __device__ uint32_t starts(int k) const { return parts_with(k, kRun); }
  __device__ uint32_t ends(int k) const { return parts_with(k, 2 * kRun); }
  __device__ uint32_t parts_with(int k, int shift) const {
    const int lane = threadIdx.x % 32;
    const uint32_t b = lane < SHAPE::kParts ? bits[k & 3][lane] : 0;
    return __ballot_sync(0xffffffffu, (b >> shift & kAllRows) != 0);
  }
};

// ---------------------------------------------------------------------------
// pieces: the decay over some tokens, and the state they give from a state of zero
// ---------------------------------------------------------------------------
struct Piece {                       // of a pair of channels
  float2 c, r, h;
};
// A piece inside which a packed sequence starts passes nothing on of what came before it,
// not even a NaN: r = -infinity (in both channels).
__device__ __forceinline__ float2 cut() { return both(__int_as_float((int)0xff800000)); }
__device__ __forceinline__ bool is_cut(float2 r) { return __float_as_int(r.x) == (int)0xff800000; }
// What a state h in front of a piece is behind it.  An infinite h stays infinite under any decay but
// zero: c h says so, and r h, which may be infinite the other way or no number, is left out.  (The
// choice is four cycles in a chain of some twenty a turn: 4 x 8192 x 2048 f16 85 us, without 82.)
template <bool PACKED>
__device__ __forceinline__ float2 pass_on(const Piece& q, float2 h) {
  const float2 t = __ffma2_rn(q.c, h, q.h), n = __ffma2_rn(q.r, h, t);
  const float2 v = make_float2(isinf(h.x) ? t.x : n.x, isinf(h.y) ? t.y : n.y);
  return PACKED && is_cut(q.r) ? q.h : v;
}
// `q`, and `next` behind it in the direction of the walk: (c1 + r1) (c2 + r2).  (Where c stays 1 through a tile its
// 32 parts or less have decays of exp(-1/8) at least: of 1 + r >= exp(-4) a rounding of r costs six
// bits at most, 27 x 2^-24 of what a state of 128 tokens keeps; those tokens' own roundings come to more.)
template <bool PACKED>
__device__ __forceinline__ void append(Piece& q, const Piece& next) {
  q.h = pass_on<PACKED>(next, q.h);
  const bool none = PACKED && (is_cut(q.r) || is_cut(next.r));
  const float2 r = __ffma2_rn(q.c, next.r, __ffma2_rn(next.c, q.r, __fmul2_rn(q.r, next.r)));
  q.c = make_float2(fminf(q.c.x, next.c.x), fminf(q.c.y, next.c.y));   // (of 1, kLeast and 0: the product)
  q.r = none ? cut() : r;
}

// The parts' pieces of a tile, and those of the carrying warps' shares of them.
template <typename SHAPE>
struct Parts {
  float c[SHAPE::kParts][kChannels], r[SHAPE::kParts][kChannels], h[SHAPE::kParts][kChannels];
  float share[SHAPE::kCarryWarps][3][kChannels];
};
__device__ __forceinline__ void put(float* row, const float2 (&v)[kPairs]) {
  static_assert(kVec == 4, "a thread's channels are one float4");
  reinterpret_cast<float4*>(row)[threadIdx.x % kLanes] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
}
__device__ __forceinline__ void get(const float* row, float2 (&v)[kPairs]) {
  const float4 t = reinterpret_cast<const float4*>(row)[threadIdx.x % kLanes];
  v[0] = make_float2(t.x, t.y);
  v[1] = make_float2(t.z, t.w);
}
__device__ __forceinline__ float2& pair(float* row, int i) { return reinterpret_cast<float2*>(row)[i]; }

// ---------------------------------------------------------------------------
// pieces between the blocks of a cluster
// ---------------------------------------------------------------------------
// Every block sends its tile's piece to all of them (itself too) by st.async, which counts its
// bytes on the receiver's barrier: nothing is fenced, so no block waits for its own stores
// to memory as a cluster's barrier would (in the first tiled kernel, 4 x 8192 x 2048: 189 us with a
// barrier, 145 with this).
// Two turns of pieces, a barrier each: a block sends turn k + 2 when it has all of turn k + 1,
// which every block sends when it is done with turn k.
constexpr int kRowFloats = 3 * kChannels;
__host__ __device__ constexpr size_t cluster_bytes(int cluster) {
  return cluster > 1 ? (size_t)2 * cluster * kRowFloats * sizeof(float) : 0;
}

struct Exchange {
  uint64_t* full;                    // [2] in shared memory
  float* pieces;                     // [2][cluster][c, r, h][kChannels]
  int cluster, rank;
  __device__ Exchange(uint64_t* full_, float* pieces_, const ScanParams& p, int rank_)
      : full(full_), pieces(pieces_), cluster(p.cluster), rank(rank_) {}
  __device__ void init() const {     // one thread, before a barrier of the block and one of the cluster
    ptx::mbar_init(full, 1);
    ptx::mbar_init(full + 1, 1);
  }
  __device__ void barrier() const {  // all threads
    if (cluster > 1) asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
  }
  __device__ float* row(int turn, int i) const { return pieces + ((turn & 1) * cluster + i) * kRowFloats; }
  __device__ Piece get(int turn, int i, int at) const {
    float* s = row(turn, i);
    return {pair(s, at), pair(s + kChannels, at), pair(s + 2 * kChannels, at)};
  }
  // carrying warp `warp` of `warps` sends to blocks warp, warp + warps, ...  (A thread that has given up
  // must not: the turn's barriers might still be in use by the turn before the last.)
  __device__ void send(int turn, int warp, int warps, int at, const Piece& q) const {
    uint64_t* bar = full + (turn & 1);
    if (warp == 0 && at == 0) ptx::mbar_arrive_expect_tx(bar, cluster * kRowFloats * sizeof(float));
    const uint32_t dst = ptx::smem_u32(&pair(row(turn, rank), at)), mine = ptx::smem_u32(bar);
    for (int i = warp; i < cluster; i += warps) {
      uint32_t d, m;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(dst), "r"(i));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(mine), "r"(i));
      post(d, m, q.c);
      post(d + 4 * kChannels, m, q.r);
      post(d + 8 * kChannels, m, q.h);
    }
  }
  static __device__ __forceinline__ void post(uint32_t dst, uint32_t bar, float2 v) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(dst),
                 "f"(v.x), "f"(v.y), "r"(bar) : "memory");
  }
};

// Puts what enters part i of a tile in the place of h[i]: lane `at` of carrying warp `warp` has a pair
// of channels in its share of the parts; BACK: from the last part to the first.  `carry` (the
// same in all warps) enters the cluster's first tile of the turn and becomes what leaves its
// last one.  `meanwhile` is done while the other blocks' pieces are on their way.
template <bool PACKED, bool BACK, typename SHAPE, typename F>
__device__ __forceinline__ void enter_parts(const Exchange& exchange, Patience& patience, int turn,
                                            Parts<SHAPE>& parts, float (*h)[kChannels], uint32_t cuts, float2& carry,
                                            int warp, int at, F meanwhile) {
  constexpr int W = SHAPE::kCarryWarps, N = SHAPE::kParts / W;
  const int share = BACK ? W - 1 - warp : warp;        // the warp-th in the direction of the walk
  const auto place = [&](int i) { return share * N + (BACK ? N - 1 - i : i); };
  const auto part = [&](int j) {
    return Piece{pair(parts.c[j], at), PACKED && (cuts >> j & 1) ? cut() : pair(parts.r[j], at), pair(h[j], at)};
  };
  float2 s = carry;
  const bool alone = exchange.cluster == 1;
  if (W > 1 || !alone) {
    Piece all, before{both(1.f), both(0.f), both(0.f)};   // of the tile; of the shares before this warp's (none)
    all = part(place(0));
    if (PACKED && cuts != 0) {
#pragma unroll
      for (int i = 1; i < N; ++i) append<PACKED>(all, part(place(i)));
    } else {
#pragma unroll
      for (int i = 1; i < N; ++i) append<false>(all, part(place(i)));
    }
    if constexpr (W > 1) {
      pair(parts.share[warp][0], at) = all.c;
      pair(parts.share[warp][1], at) = all.r;
      pair(parts.share[warp][2], at) = all.h;
      carry_sync<SHAPE::kCarry>();
      const auto share_of = [&](int i) {
        return Piece{pair(parts.share[i][0], at), pair(parts.share[i][1], at), pair(parts.share[i][2], at)};
      };
      all = share_of(0);
#pragma unroll
      for (int i = 1; i < W; ++i) {
        if (i == warp) before = all;
        append<PACKED>(all, share_of(i));
      }
    }
    if (alone) {
      carry = pass_on<PACKED>(all, carry);
      meanwhile();
    } else {
      if (!patience.gone) exchange.send(turn, warp, W, at, all);
      meanwhile();
      patience.wait(exchange.full + (turn & 1), (turn >> 1) & 1);
      Piece others[kMaxCluster];
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i)
        if (i < exchange.cluster) others[i] = exchange.get(turn, BACK ? exchange.cluster - 1 - i : i, at);
      const int me = BACK ? exchange.cluster - 1 - exchange.rank : exchange.rank;
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i) {
        if (i == me) s = carry;
        if (i < exchange.cluster) carry = pass_on<PACKED>(others[i], carry);
      }
    }
    s = pass_on<PACKED>(before, s);
  } else {
    meanwhile();
  }
  const auto enter = [&](auto cut_) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = place(i);
      const Piece q = part(j);
      pair(h[j], at) = s;
      s = pass_on<decltype(cut_)::value>(q, s);
    }
  };
  if (PACKED && cuts != 0) enter(std::true_type{});
  else enter(std::false_type{});
  if (W == 1 && alone) carry = s;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Calls f with the types of x and g.
template <typename F>
cudaError_t by_types(int x, int g, F f) {
  if (x == KDA_DTYPE_F32) return f(float{}, float{});
  if (x == KDA_DTYPE_F16)
    return g == KDA_DTYPE_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return g == KDA_DTYPE_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

// Calls f with the three flags as types.
template <typename F>
cudaError_t by_flags(bool a, bool b, bool c, F f) {
  using Yes = std::true_type;
  using No = std::false_type;
  if (a) return b ? (c ? f(Yes{}, Yes{}, Yes{}) : f(Yes{}, Yes{}, No{})) : (c ? f(Yes{}, No{}, Yes{}) : f(Yes{}, No{}, No{}));
  return b ? (c ? f(No{}, Yes{}, Yes{}) : f(No{}, Yes{}, No{})) : (c ? f(No{}, No{}, Yes{}) : f(No{}, No{}, No{}));
}

// Sets tiles and cluster: as many blocks to a sequence as there are SMs for, and tiles.  (The SMs of a cluster lie
// together, so that not every count of clusters that 148 SMs have room for is there at once: 32768 tokens,
// bf16, take 96 us with 32 x 4 blocks of 2048 channels, but 157 with 29 x 5 of 1856.)
template <typename SHAPE>
void choose_cluster(ScanParams& p) {
  p.tiles = (p.T + SHAPE::kTile - 1) / SHAPE::kTile;
  const int64_t blocks = (int64_t)(p.q_start ? 1 : p.B) * ((p.D + kChannels - 1) / kChannels);
  p.cluster = (int)max((int64_t)1, min((int64_t)min(kMaxCluster, p.tiles), kSms * SHAPE::kBlocks / blocks));
}

// The map of x, g or dh for tiles of `tile` rows; false where TMA cannot address its rows.
template <typename T>
bool encode(CUtensorMap* m, const void* base, const int64_t* stride, const ScanParams& p, int tile) {
  if (base == nullptr) return true;
  const EncodeTiled enc = encode_tiled();
  const int64_t token = stride[1] * (int64_t)sizeof(T), batch = p.q_start ? 0 : stride[0] * (int64_t)sizeof(T);
  if (!enc || reinterpret_cast<uintptr_t>(base) % 16 || token % 16 || batch % 16 || token < 0 || batch < 0)
    return false;
  const bool one = p.q_start != nullptr || p.B == 1;
  if ((p.T > 1 && token == 0) || (!one && batch == 0)) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)p.D, (cuuint64_t)p.T, (cuuint64_t)(one ? 1 : p.B)};
  const cuuint64_t strides[2] = {(cuuint64_t)(p.T > 1 ? token : 16), (cuuint64_t)(one ? 16 : batch)};
  const cuuint32_t box[3] = {(cuuint32_t)kChannels, (cuuint32_t)tile, 1}, ones[3] = {1, 1, 1};
  const CUtensorMapDataType dt = std::is_same<T, float>::value    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(m, dt, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A kernel over all channels and sequences, in clusters of p.cluster blocks, behind
// mark_kernel where the batch is packed.
template <typename... Maps>
cudaError_t launch_tiles(void (*kernel)(ScanParams, Maps...), const ScanParams& p, int threads, size_t smem,
                         cudaStream_t s, const Maps&... maps) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.D + kChannels - 1) / kChannels * (p.q_start ? 1 : p.B) * p.cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (p.cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = p.cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (p.q_start) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, p, maps...);
}

int read_grad_device_error(bool clear);   // kda_scan_grad.cu's error word
cudaError_t launch_grad(const ScanParams& p, int x_dtype, int g_dtype, bool wide, cudaStream_t s);

}  // namespace scan
}  // namespace kda
