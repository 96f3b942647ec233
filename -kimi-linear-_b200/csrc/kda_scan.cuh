// kda_scan.cuh -- gated linear recurrence: parameters, the arithmetic of its decays, and
// what the scan and its gradient share.
//
// A decay a = exp(g) is held as c + r with c = 1, r = a - 1 where |g| < 1/4 and c = 0, r = a
// elsewhere: rounding a itself to 24 bits is off by up to 2^-25 per token, always to the
// same side for a steady g, which a state that remembers n tokens adds up to n 2^-25.
// c h + r h is one instruction more than a product, and two channels share each
// (fma.f32x2), so a thread works on pairs of channels.
#pragma once

#include "kda_internal.cuh"
#include "tc_ptx.cuh"

namespace kda {
namespace scan {

constexpr int kErrSlot = 8;       // device error word: a step's slot past the pool
constexpr int kErrWait = 9;       // device error word: a wait for a cluster's piece ran out
constexpr int kTile = 64;         // tokens between two checkpoints of the state

// What the rows of a tile of a packed batch are, a bit a row.
struct Marks {
  uint64_t first, last, owned;      // of a sequence; by any sequence
};

// Device-side view of KdaScanArgs (strides in elements).
struct ScanParams {
  int B, T, D;
  int tiles;                        // checkpoints of a sequence (packed: of all rows)
  bool complement;
  const void* x; int64_t x_s[2];
  const void* g; int64_t g_s[2];
  const float* state_in; int64_t si_s;
  const int* q_start;               // or null: a batch
  void* h; int64_t h_s[2];
  float* state_out; int64_t so_s;
  float* ckpt;                      // [B][tiles][D], packed [tiles][D]
  const void* dh; int64_t dh_s[2];
  const float* dstate_out; int64_t dso_s;
  void* dx; int64_t dx_s[2];
  void* dg; int64_t dg_s[2];
  float* dstate_in; int64_t dsi_s;
  const Marks* marks;               // packed: [tiles], made by mark_kernel
  int cluster;                      // blocks that share a sequence's tiles
  // step
  const int* slots; int num_states; bool scatter;
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

struct Decay {                      // of a pair of channels
  float2 c, r;
};

// exp(g).  Near zero the series of exp(g) - 1 up to g^6/6!, of which the first term left out
// is 2^-24 of the sum at |g| = 1/4; elsewhere 2^(g log2 e) by the hardware's instruction
// (2^-22 of itself, and 2^-24 |g| from the rounded exponent).  What is below 2^-126 is zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ Decay decay(float2 g) {
  float2 p = __ffma2_rn(g, both(1.f / 720.f), both(1.f / 120.f));
  p = __ffma2_rn(p, g, both(1.f / 24.f));
  p = __ffma2_rn(p, g, both(1.f / 6.f));
  p = __ffma2_rn(p, g, both(0.5f));
  p = __ffma2_rn(p, g, both(1.f));
  p = __fmul2_rn(p, g);
  const float2 e = __fmul2_rn(g, both(1.4426950408889634f));
  const bool x = fabsf(g.x) < 0.25f, y = fabsf(g.y) < 0.25f;
  return {make_float2(x ? 1.f : 0.f, y ? 1.f : 0.f),
          make_float2(x ? p.x : exp2_fast(e.x), y ? p.y : exp2_fast(e.y))};
}
// a h + b
__device__ __forceinline__ float2 apply(const Decay& a, float2 h, float2 b) {
  return __ffma2_rn(a.r, h, __ffma2_rn(a.c, h, b));
}
// a v
__device__ __forceinline__ float2 times(const Decay& a, float2 v) {
  return __ffma2_rn(a.r, v, __fmul2_rn(a.c, v));
}
// 1 - a
__device__ __forceinline__ float2 rest(const Decay& a) {
  return __ffma2_rn(a.r, both(-1.f), __ffma2_rn(a.c, both(-1.f), both(1.f)));
}
// Decay over two pieces: (c1 + r1) (c2 + r2).
__device__ __forceinline__ void renew(float& c, float& r) {
  if (c == 1.f && r < -0.5f) {
    c = 0.f;
    r += 1.f;
  }
}
__device__ __forceinline__ Decay join(const Decay& a, const Decay& b) {
  Decay d{__fmul2_rn(a.c, b.c),
          __ffma2_rn(a.c, b.r, __ffma2_rn(b.c, a.r, __fmul2_rn(a.r, b.r)))};
  renew(d.c.x, d.r.x);
  renew(d.c.y, d.r.y);
  return d;
}

// A piece inside which a packed sequence starts passes nothing on of what came before it,
// not even a NaN: c = 0, r = -infinity in both channels.
__device__ __forceinline__ Decay cut() { return {both(0.f), both(__int_as_float((int)0xff800000))}; }
__device__ __forceinline__ bool is_cut(const Decay& a) { return __float_as_int(a.r.x) == (int)0xff800000; }
template <bool PACKED>
__device__ __forceinline__ float2 pass_on(const Decay& a, float2 h, float2 b) {
  const float2 n = apply(a, h, b);
  return PACKED && is_cut(a) ? b : n;
}
template <bool PACKED>
__device__ __forceinline__ Decay join_pieces(const Decay& a, const Decay& b) {
  return PACKED && (is_cut(a) || is_cut(b)) ? cut() : join(a, b);
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

constexpr int kThreads = 128;                 // of every kernel here
constexpr int kWarps = kThreads / 32;
constexpr int kLanes = 16;                    // threads that share a row
constexpr int kVec = 4;                       // channels of a thread
constexpr int kPairs = kVec / 2;
constexpr int kChannels = kLanes * kVec;      // of a block
constexpr int kRun = kTile / (kWarps * 2);    // tokens of a thread
constexpr int kMaxCluster = 8;

// ---------------------------------------------------------------------------
// rows into a thread's own places in shared memory
// ---------------------------------------------------------------------------
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool ok) {
  const int n = ok ? BYTES : 0;               // 0: the place is filled with zeros
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src),
                 "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src),
                 "r"(n), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's channels.  WIDE: kVec next to each other, in one access; else (rows that
// do not start on such a boundary) every kLanes-th, one by one, so that a half warp
// still reads whole sectors.
struct Place {
  int rank;                          // in the cluster: tiles rank, rank + cluster, ...
  int b;                             // sequence (packed: 0)
  int c;                             // first channel
  int run;                           // first token in a tile
  uint32_t on;                       // which channels exist (WIDE: all or none)
};
template <bool WIDE>
__device__ __forceinline__ int channel(int i) { return WIDE ? i : i * kLanes; }
template <bool WIDE>
__device__ __forceinline__ Place my_place(const ScanParams& p) {
  Place w;
  const int blocks = (p.D + kChannels - 1) / kChannels;
  const int i = blockIdx.x / p.cluster, lane = threadIdx.x % kLanes;
  w.rank = blockIdx.x - i * p.cluster;
  w.b = i / blocks;
  w.c = (i - w.b * blocks) * kChannels + (WIDE ? lane * kVec : lane);
  w.run = threadIdx.x / kLanes * kRun;
  w.on = 0;
#pragma unroll
  for (int j = 0; j < kVec; ++j)
    if (w.c + channel<WIDE>(j) < p.D) w.on |= 1u << j;
  return w;
}

// A thread's kRun rows of one tensor, in a ring of STAGES tiles.
template <typename T, bool WIDE, int STAGES>
struct Ring {
  static constexpr int kBytes = STAGES * kRun * kThreads * kVec * sizeof(T);
  T* at;
  __device__ Ring(void* base) : at(static_cast<T*>(base) + threadIdx.x * kVec) {}
  __device__ T* place(int stage, int i) const { return at + (stage * kRun + i) * kThreads * kVec; }
  // rows row, row + stride, ..., of which those in `mask` are wanted (the others: zeros)
  __device__ void load(int stage, const T* row, int64_t stride, uint32_t mask, uint32_t on) const {
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      T* dst = place(stage, i);
      const bool ok = mask >> i & 1;
      if constexpr (WIDE) {
        copy_async<kVec * sizeof(T)>(dst, row, ok);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const bool has = ok && (on >> j & 1);
          if constexpr (sizeof(T) == 4) copy_async<4>(dst + j, row + channel<WIDE>(j), has);
          else dst[j] = has ? row[channel<WIDE>(j)] : T(0.f);
        }
      }
      row += stride;
    }
  }
  __device__ __forceinline__ void read(int stage, int i, float2 (&v)[kPairs]) const {
    float t[kVec];
    ld4(place(stage, i), t);
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
    if (on) st4(p, t);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (on >> j & 1) st(p + channel<WIDE>(j), t[j]);
  }
}

// A state (or checkpoint) row of fp32 values, any alignment; zeros without one.
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
__device__ __forceinline__ const float* state_of(const ScanParams& p, const float* base, int64_t stride, int t,
                                                 int c) {
  return base == nullptr ? nullptr : base + (int64_t)max(sequence_at(p.q_start, p.B, t), 0) * stride + c;
}

// Which of a thread's rows are there (bits), and for packed batches which start and end a sequence.
struct RowMask { uint32_t there, first, last; };
template <bool PACKED>
__device__ __forceinline__ RowMask row_mask(const ScanParams& p, const Place& w, int tile) {
  constexpr uint32_t all = (1u << kRun) - 1;
  RowMask m{0, 0, 0};
  if (tile >= p.tiles || tile < 0 || !w.on) return m;
  if constexpr (PACKED) {
    const Marks k = p.marks[tile];
    m.there = (uint32_t)(k.owned >> w.run) & all;
    m.first = (uint32_t)(k.first >> w.run) & all;
    m.last = (uint32_t)(k.last >> w.run) & all;
  } else {
    const int left = p.T - (tile * kTile + w.run);
    m.there = left >= kRun ? all : left > 0 ? (1u << left) - 1 : 0;
  }
  return m;
}

// ---------------------------------------------------------------------------
// pieces: the decay over some tokens, and the state they give from a state of zero
// ---------------------------------------------------------------------------
struct Piece {
  Decay a[kPairs];
  float2 h[kPairs];
};
template <bool PACKED>
__device__ __forceinline__ void pass_on(const Piece& q, float2 (&h)[kPairs]) {
#pragma unroll
  for (int j = 0; j < kPairs; ++j) h[j] = pass_on<PACKED>(q.a[j], h[j], q.h[j]);
}
// `q`, and `next` behind it in the direction of the walk
template <bool PACKED>
__device__ __forceinline__ void append(Piece& q, const Piece& next) {
  pass_on<PACKED>(next, q.h);
#pragma unroll
  for (int j = 0; j < kPairs; ++j) q.a[j] = join_pieces<PACKED>(q.a[j], next.a[j]);
}
// Pieces in shared memory: a row of kLanes threads' c, then r, then h.
constexpr int kPieceFloats = 3 * kChannels;
__device__ __forceinline__ void put(float* row, int lane, const Piece& q) {
  static_assert(kVec == 4, "a thread's channels are one float4");
  float4* d = reinterpret_cast<float4*>(row) + lane;
  d[0] = make_float4(q.a[0].c.x, q.a[0].c.y, q.a[1].c.x, q.a[1].c.y);
  d[kLanes] = make_float4(q.a[0].r.x, q.a[0].r.y, q.a[1].r.x, q.a[1].r.y);
  d[2 * kLanes] = make_float4(q.h[0].x, q.h[0].y, q.h[1].x, q.h[1].y);
}
__device__ __forceinline__ Piece take(const float* row, int lane) {
  const float4* s = reinterpret_cast<const float4*>(row) + lane;
  const float4 c = s[0], r = s[kLanes], h = s[2 * kLanes];
  Piece q;
  q.a[0] = {make_float2(c.x, c.y), make_float2(r.x, r.y)};
  q.a[1] = {make_float2(c.z, c.w), make_float2(r.z, r.w)};
  q.h[0] = make_float2(h.x, h.y);
  q.h[1] = make_float2(h.z, h.w);
  return q;
}
// The piece of lane `from` (decays of a cut piece included).
__device__ __forceinline__ float2 shuffle(float2 v, int from) {
  return make_float2(__shfl_sync(0xffffffffu, v.x, from), __shfl_sync(0xffffffffu, v.y, from));
}
__device__ __forceinline__ Piece shuffle(const Piece& q, int from) {
  Piece o;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    o.a[j].c = shuffle(q.a[j].c, from);
    o.a[j].r = shuffle(q.a[j].r, from);
    o.h[j] = shuffle(q.h[j], from);
  }
  return o;
}
// ---------------------------------------------------------------------------
// pieces between the blocks of a cluster
// ---------------------------------------------------------------------------
// Every block sends its tile's piece to all of them (itself too) by st.async, which counts its
// bytes on the receiver's barrier: nothing is fenced, so no block waits for its own stores
// to memory as a cluster's barrier would (B = 4, T = 8192, D = 2048: 189 us with one).
// Two turns of pieces, a barrier each: a block sends turn k + 2 when it has all of turn k + 1,
// which every block sends when all its threads are done with turn k.
__host__ __device__ constexpr size_t cluster_bytes(int cluster) {
  return cluster > 1 ? (size_t)2 * cluster * kPieceFloats * sizeof(float) : 0;
}
constexpr uint64_t kWaitNs = 2000000000;    // a wait that takes longer gives up (device error word 9)

struct Exchange {
  uint64_t* full;                    // [2] in shared memory
  float* pieces;                     // [2][cluster][kPieceFloats]
  int cluster, rank;
  int* error;
  uint64_t limit;
  __device__ Exchange(uint64_t* full_, float* pieces_, const ScanParams& p, int rank_, int* error_)
      : full(full_), pieces(pieces_), cluster(p.cluster), rank(rank_), error(error_), limit(kWaitNs) {
    if (cluster == 1) return;
    if (threadIdx.x == 0) {
      ptx::mbar_init(full, 1);
      ptx::mbar_init(full + 1, 1);
      ptx::fence_mbar_init();
    }
    barrier();
  }
  static __device__ void barrier() {
    asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
  }
  __device__ float* row(int turn, int i) const { return pieces + ((turn & 1) * cluster + i) * kPieceFloats; }
  // The warps' pieces joined in the direction of the walk (`back`: the last warp first), to
  // every block: sixteen threads to a block.
  template <bool PACKED>
  __device__ void send(int turn, const float* warps, bool back) const {
    uint64_t* bar = full + (turn & 1);
    if (threadIdx.x == 0 && limit) ptx::mbar_arrive_expect_tx(bar, cluster * kPieceFloats * sizeof(float));
    const int lane = threadIdx.x % kLanes;
    Piece q = take(warps + (back ? kWarps - 1 : 0) * kPieceFloats, lane);
#pragma unroll
    for (int i = 1; i < kWarps; ++i)
      append<PACKED>(q, take(warps + (back ? kWarps - 1 - i : i) * kPieceFloats, lane));
    const uint32_t dst = ptx::smem_u32(row(turn, rank)) + 16 * lane, at = ptx::smem_u32(bar);
    for (int i = threadIdx.x / kLanes; i < cluster; i += kThreads / kLanes) {
      uint32_t d, m;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(dst), "r"(i));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(at), "r"(i));
      post(d, m, q.a[0].c, q.a[1].c);
      post(d + 16 * kLanes, m, q.a[0].r, q.a[1].r);
      post(d + 32 * kLanes, m, q.h[0], q.h[1]);
    }
  }
  static __device__ __forceinline__ void post(uint32_t dst, uint32_t bar, float2 a, float2 b) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                     dst), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "r"(bar) : "memory");
  }
  static __device__ __forceinline__ bool here(uint64_t* bar, uint32_t parity) {
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
  // Until all of a turn's pieces are here.  (A thread that gives up goes on, so that the block's
  // barriers stay matched, and waits no more.)
  __device__ void wait(int turn) {
    uint64_t* bar = full + (turn & 1);
    const uint32_t parity = (turn >> 1) & 1;
    if (here(bar, parity)) return;
    const uint64_t start = ptx::globaltimer_ns();
    while (!here(bar, parity)) {
      if (ptx::globaltimer_ns() - start >= limit) {
        *error = kErrWait;
        limit = 0;
        return;
      }
    }
  }
  // No block leaves while another may still send to it.
  __device__ void leave() const {
    if (cluster > 1) barrier();
  }
};

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

// A kernel over all channels and sequences, in clusters of p.cluster blocks, behind
// mark_kernel where the batch is packed.
inline cudaError_t launch_tiles(void (*kernel)(ScanParams), const ScanParams& p, size_t smem, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.D + kChannels - 1) / kChannels * (p.q_start ? 1 : p.B) * p.cluster));
  cfg.blockDim = dim3(kThreads);
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
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

int read_grad_device_error(bool clear);   // kda_scan_grad.cu's error word
cudaError_t launch_grad(const ScanParams& p, int x_dtype, int g_dtype, bool wide, cudaStream_t s);

}  // namespace scan
}  // namespace kda
