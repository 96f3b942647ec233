// mla_cache_attn.cu -- absorbed-form latent attention over the 8-bit paged cache (sm_100a).
//
// For a row (new token i of sequence b, head h) over its visible positions t
//   z_t = scale (q_lat . c_t + q_rope . k_t),  c_t = s_t code_t,  k_t = s_t rope_t
//   out = sum_t exp(z_t - m) c_t / sum_t exp(z_t - m),   lse = m + ln sum_t exp(z_t - m)
//
// The codes go into the tensor cores as they lie in the cache (tcgen05
// kind::f8f6f4), with no conversion pass: a tile of 128 positions is the M side
// of both products, the rows are the N side.
//   S^T [128 positions x rows]   = codes [128 x KVL] (K-major)       Q^T
//   O^T [128 channels x rows] += codes^T [128 ch x 128 pos] (M-major) P^T, per 128 channels
// What is not e4m3 is split into e4m3 terms that are exact or nearly so, each
// 16 times finer than the one before: x = x0 + x1 / 16 (+ x2 / 256).  A query
// (scaled by a power of two) in bf16 has 8 significant bits, two terms; fp16 has
// 11, three.  The softmax's weights take as many terms: 2^-9 or 2^-13 of each
// weight, and 2^-20 of the largest, less than the output's own rounding.  The
// terms are more columns of N and are added in fp32 afterwards: at 16 rows the
// products are bound by reading the codes from shared memory (4 KB per
// instruction of 128 x N x 32), so the extra columns cost next to nothing.
//
// A position's scale is a power of two, so the weight that meets the codes is
//   P_t = exp2(z_t log2e + log2 s_t - M),  M the running maximum of the exponents,
// and the sum takes P_t / s_t: the largest P is 1 whatever the scales are.  M
// moves (and O is rescaled in TMEM) only where a row's maximum grew by more than
// 2^2: P carries a factor 2^6, so it stays below e4m3's largest 448 until then.
//
// Work: a row group (R rows of a sequence) times its tiles; all the tiles of a
// call, in order, are cut into equal ranges, one per SM, so a long sequence is
// split over many SMs and short ones share one.  A group cut by a range's end
// leaves fp32 partials and cache_join_kernel adds them in order: the result does
// not depend on timing.
#include <cuda.h>

#include <type_traits>

#include "mla_cache.cuh"
#include "tc_ptx.cuh"

namespace kda {
namespace cache {

__device__ int g_attn_device_error = 0;

namespace {

constexpr int TILE = 128;                  // positions per tile (MMA M)
constexpr int kThreads = 192;              // warps 0-3 softmax, 4 loads, 5 MMA issue
constexpr int kMaxStages = 8;
constexpr int kSmemMax = 232448;           // 227 KB per block
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kBias = 6.f;               // P carries 2^6 ...
constexpr float kSlack = 2.f;              // ... and may outgrow the maximum by 2^2 (2^8 < 448)

// e4m3 terms of a query and of a softmax weight
template <typename T> constexpr int kTerms = std::is_same<T, __nv_bfloat16>::value ? 2 : 3;

template <typename T, int R, int NCH>
struct Cfg {
  static constexpr int NT = kTerms<T>;
  static constexpr int N = NT * R;                       // columns of S and of one O chunk
  static constexpr int O_COLS = NCH * N;
  static constexpr int SBUF = O_COLS + 2 * N <= 512 ? 2 : 1;
  static_assert(O_COLS + SBUF * N <= 512, "TMEM columns");
  static constexpr int CHUNK = TILE * 128;               // bytes of 128 positions x 128 channels
  static constexpr int Q_BYTES = NCH * N * 128;
  static constexpr int QR_BYTES = R * 128;
  static constexpr int P_BYTES = N * 128;
};

// Shared memory besides the stages (4 KB: barriers, rows; 1 KB: alignment), and
// the stages that fit beside it.
constexpr int kFixedBytes = 4096 + 1024;
int stage_bytes(int kvl, int dr) { return (kvl / 128 + (dr ? 1 : 0)) * TILE * 128; }
int fixed_bytes(int kvl, int terms, int R) {
  return kFixedBytes + terms * R * (kvl + 128) + R * 128;
}
int stages(int kvl, int dr, int terms, int R) {
  const int n = (kSmemMax - fixed_bytes(kvl, terms, R)) / stage_bytes(kvl, dr);
  return n < kMaxStages ? n : kMaxStages;
}

// Where a range of tiles starts inside a group; what cache_join_kernel reads.
struct Cut {
  int b, g;        // the group that the range starts in the middle of (b < 0: none)
  int parts;       // ranges that share the group; 0: an earlier cut joins it
  int pad;
};

struct Work {
  float* part;     // [2 ranges][R][KVL] fp32: slot 2 c: group begun before range c; 2 c + 1: left unfinished
  float* lse2;     // [2 ranges][R] log2 of the sum of a part
  Cut* cuts;       // [ranges]
  int stages;
};

// ---------------------------------------------------------------------------
// how the tiles of a call are counted and cut
// ---------------------------------------------------------------------------
// Sequence b as R-row groups.  Groups of one sequence see more and more
// positions; they are counted in pairs (g, groups - 1 - g), which all have about
// as many tiles, so that a place in the count is found by a division.
struct Seq {
  int first, n, off;       // new tokens; token i sits at off + i
  int groups, pair;        // row groups; tiles counted per pair
  int cap;                 // positions that the table holds
};

template <int R>
__device__ __forceinline__ int seen_by(const CacheParams& p, const Seq& s, int row) {
  return max(0, min(s.off + min(row / p.H, s.n - 1) + 1, s.cap));
}
template <int R>
__device__ __forceinline__ int group_tiles(const CacheParams& p, const Seq& s, int g) {
  return max(1, (seen_by<R>(p, s, g * R + R - 1) + TILE - 1) / TILE);
}
template <int R>
__device__ __forceinline__ Seq load_seq(const CacheParams& p, int b) {
  Seq s;
  new_tokens(p, b, s.first, s.n);
  s.off = max(p.lens[b], 0) - s.n;
  s.cap = p.max_pages * p.page_size;
  s.groups = (int)(((int64_t)s.n * p.H + R - 1) / R);
  s.pair = 0;
  if (s.groups == 1) s.pair = group_tiles<R>(p, s, 0);
  // the first pair's sum, and up to two more: the last group may be short, and the
  // tiles are rounded up.  (Where the table ends before the sequence: all may be as long
  // as the last.)
  if (s.groups > 1)
    s.pair = group_tiles<R>(p, s, s.off + s.n > s.cap ? s.groups - 1 : 0) +
             group_tiles<R>(p, s, s.groups - 1) + 2;
  return s;
}
__device__ __forceinline__ int64_t seq_tiles(const Seq& s) {
  return (int64_t)((s.groups + 1) / 2) * s.pair;
}

struct Segment {
  int b, g, t0, t1;        // tiles t0 .. t1 - 1 of group g
  int tiles;               // of the whole group
};

// Walks the segments of the range [u, end): every role runs its own copy.
template <int R>
struct Walk {
  const CacheParams& p;
  Seq s;
  int b;
  int64_t u, end, base;    // base: count at which sequence b starts
  int second_t1;           // pending second group of a pair: its last tile (0: none)
  int second_g, second_t0;
  __device__ Walk(const CacheParams& p_, int b_, int64_t base_, int64_t u_, int64_t end_)
      : p(p_), b(b_), u(u_), end(end_), base(base_), second_t1(0) {
    if (u < end) s = load_seq<R>(p, b);
  }
  __device__ bool next(Segment& seg) {
    if (second_t1 > 0) {
      seg = Segment{b, second_g, second_t0, second_t1, group_tiles<R>(p, s, second_g)};
      second_t1 = 0;
      return true;
    }
    while (u < end) {
      while (u >= base + seq_tiles(s)) {
        base += seq_tiles(s);
        s = load_seq<R>(p, ++b);
      }
      const int64_t r = u - base;
      const int pair = (int)(r / s.pair), q = (int)(r % s.pair);
      const int g1 = pair, g2 = s.groups - 1 - pair;
      const int n1 = group_tiles<R>(p, s, g1), n2 = g2 > g1 ? group_tiles<R>(p, s, g2) : 0;
      const int stop = (int)min((int64_t)s.pair, q + (end - u));
      // the last place of a pair takes whatever is left of it
      const int last = stop == s.pair ? n1 + n2 : min(stop, n1 + n2);
      u += stop - q;
      if (q < n1) {
        seg = Segment{b, g1, q, min(last, n1), n1};
        if (last > n1) {
          second_g = g2;
          second_t0 = 0;
          second_t1 = last - n1;
        }
        return true;
      }
      if (q < last) {
        seg = Segment{b, g2, q - n1, last - n1, n2};
        return true;
      }
    }
    return false;
  }
};

// ---------------------------------------------------------------------------
// PTX used only here
// ---------------------------------------------------------------------------
// D[tmem] = A[smem] B[smem] (+ D): 8-bit operands, fp32 accumulation
__device__ __forceinline__ void mma_f8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Shared-memory descriptor of 128-byte rows with the 128-byte swizzle (eight
// rows = 1024 bytes, consecutive).  K-major operands: rows are M or N; M-major
// ones: rows are K, and the 128 bytes of a row are all of M.
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}
// Instruction descriptors: fp32 accumulator; e4m3 operands, or `fmt` 0 = f16, 1 = bf16
__host__ __device__ constexpr uint32_t idesc(int N, bool a_m_major, uint32_t fmt) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_m_major ? 1u : 0u) << 15) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(TILE >> 4) << 24);
}
// largest of the 32 lanes' values (NaN ignored)
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t warp_max_u32(uint32_t x) {
  return __reduce_max_sync(0xffffffffu, x);
}
// 16 bytes along a 128-byte row: chunk index xor row % 8
__device__ __forceinline__ uint32_t swz(int row, int byte) {
  return (uint32_t)(row * 128 + ((((byte >> 4) ^ row) & 7) << 4) + (byte & 15));
}

// Bounded wait: false once the block gave up (the caller then leaves its loop).
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = ptx::globaltimer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (ptx::mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (ptx::globaltimer_ns() - t0 > kWaitNs) {
      *abort_flag = 1;
      atomicExch(&g_attn_device_error, kErrWait);
      return false;
    }
  }
}

// x = t[0] + t[1] / 16 (+ t[2] / 256), for four values: four codes per term
template <int NT>
__device__ __forceinline__ void split4(const float (&x)[4], uint32_t (&t)[NT]) {
  float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    t[j] = to_e4m3x4(r[0], r[1], r[2], r[3]);
    if (j + 1 < NT) {
      const float2 lo = from_e4m3x2(t[j]), hi = from_e4m3x2(t[j] >> 16);
      r[0] = (r[0] - lo.x) * 16.f;
      r[1] = (r[1] - lo.y) * 16.f;
      r[2] = (r[2] - hi.x) * 16.f;
      r[3] = (r[3] - hi.y) * 16.f;
    }
  }
}
template <int NT>
__device__ __forceinline__ float join(const float* t, int stride) {   // t[0] + t[1] / 16 (+ ...)
  float x = t[(NT - 1) * stride];
#pragma unroll
  for (int j = NT - 2; j >= 0; --j) x = fmaf(x, 1.f / 16.f, t[j * stride]);
  return x;
}

struct Shared {            // at the end of dynamic shared memory
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t s_full[2], s_empty[2], p_full, o_done, q_ready, drain;
  uint32_t tmem;
  int abort_flag;
  int64_t scan[8];
  int64_t base;            // where the range starts: count at which sequence b starts
  int b;
  float q_scale[32];       // per row: 2^e scale log2e
  int seen[32];            // per row: positions that it sees
  float red[2][4][32];     // per warp and row: maxima (two tiles in turn), sums
};
static_assert(sizeof(Shared) <= 4096, "room for barriers and rows");

template <typename T, int R, int NCH>
__global__ void __launch_bounds__(kThreads, 1)
cache_attn_kernel(const CacheParams p, const Work w, const __grid_constant__ CUtensorMap map_codes,
                  const __grid_constant__ CUtensorMap map_rope) {
  using C = Cfg<T, R, NCH>;
  constexpr int NT = C::NT, N = C::N;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_size = (NCH + (p.DR ? 1 : 0)) * C::CHUNK;
  uint8_t* q_s = sm + w.stages * stage_size;
  uint8_t* qr_s = q_s + C::Q_BYTES;
  uint8_t* p_s = qr_s + C::QR_BYTES;
  Shared& sh = *reinterpret_cast<Shared*>(p_s + C::P_BYTES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < w.stages; ++i) {
      ptx::mbar_init(&sh.full[i], 1);
      ptx::mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&sh.s_full[i], 1);
      ptx::mbar_init(&sh.s_empty[i], 128);
    }
    ptx::mbar_init(&sh.p_full, 128);
    ptx::mbar_init(&sh.o_done, 1);
    ptx::mbar_init(&sh.q_ready, 128);
    ptx::mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 5) ptx::tmem_alloc(&sh.tmem, 512);
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();

  // ---- this block's range of the call's tiles
  int64_t u0, u1;
  {
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += seq_tiles(load_seq<R>(p, b));
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sh.scan[warp] = x;
    __syncthreads();
    int64_t before = x - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) before += sh.scan[i];
      total += sh.scan[i];
    }
    const int64_t range = (total + gridDim.x - 1) / gridDim.x;
    u0 = min(total, range * blockIdx.x);
    u1 = min(total, u0 + range);
    if (u0 < u1 && u0 >= before && u0 < before + mine) {
      int b = b0;
      for (;; ++b) {
        const int64_t n = seq_tiles(load_seq<R>(p, b));
        if (u0 < before + n) break;
        before += n;
      }
      sh.b = b;
      sh.base = before;
    }
    // the group that this range starts inside of, for cache_join_kernel
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (tid == 0) {
      Cut cut{-1, 0, 0, 0};
      if (u0 < u1 && blockIdx.x > 0) {
        const Seq s = load_seq<R>(p, sh.b);
        const int64_t r = u0 - sh.base;
        const int pair = (int)(r / s.pair), q = (int)(r % s.pair);
        const int g1 = pair, g2 = s.groups - 1 - pair;
        const int n1 = group_tiles<R>(p, s, g1), n2 = g2 > g1 ? group_tiles<R>(p, s, g2) : 0;
        int64_t start = u0 - q;              // of the group
        int n = 0;
        if (q > 0 && q < n1) {
          cut.b = sh.b; cut.g = g1; n = n1;
        } else if (q > n1 && q < n1 + n2) {
          cut.b = sh.b; cut.g = g2; start += n1; n = n2;
        }
        if (cut.b >= 0 && start >= u0 - range)
          cut.parts = (int)((start + n - 1) / range) - (int)(start / range) + 1;
      }
      w.cuts[blockIdx.x] = cut;
    }
  }
  const uint32_t tmem = sh.tmem;
  const uint32_t tm_s = tmem + C::O_COLS;       // S buffers after the O chunks
  volatile int* ab = &sh.abort_flag;
  Walk<R> walk(p, sh.b, sh.base, u0, u1);
  Segment seg;

  if (warp == 4) {
    // ======== loads: boxes of one page (at most 128 positions) x 128 channels
    int stage = 0, round = 0, issued = 0;
    const int box_rows = min(p.page_size, TILE), boxes = TILE / box_rows;
    bool ok = true;
    while (ok && walk.next(seg)) {
      const int seen = seen_by<R>(p, walk.s, seg.g * R + R - 1);
      if (seen == 0) continue;
      for (int t = seg.t0; t < seg.t1; ++t) {
        const int pos = t * TILE;
        const int nbox = min(boxes, (seen - pos + box_rows - 1) / box_rows);
        int page = p.num_pages;                 // outside: the copy fills in zeros
        if (lane < nbox) {
          const int x = page_of(p, seg.b, pos + lane * box_rows);
          if (x >= 0) page = x;
        }
        if (round > 0 && !wait(&sh.empty[stage], (round - 1) & 1, ab)) { ok = false; break; }
        uint8_t* dst = sm + stage * stage_size;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(&sh.full[stage],
                                     nbox * box_rows * 128 * (NCH + (p.DR ? 1 : 0)));
        }
        __syncwarp();
        if (lane < nbox) {
          const int row = pos & (p.page_size - 1) & ~(box_rows - 1);
          const int at = p.page_size >= TILE ? row : 0;
#pragma unroll
          for (int c = 0; c < NCH; ++c)
            ptx::tma_load_3d(dst + c * C::CHUNK + lane * box_rows * 128, &map_codes, c * 128, at,
                             page, &sh.full[stage]);
          if (p.DR)
            ptx::tma_load_3d(dst + NCH * C::CHUNK + lane * box_rows * 128, &map_rope, 0, at, page,
                             &sh.full[stage]);
        }
        ++issued;
        if (++stage == w.stages) { stage = 0; ++round; }
      }
    }
    if (*ab) {                                  // copies in flight land before the block ends
      for (int i = max(0, issued - w.stages); i < issued; ++i) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(&sh.full[i % w.stages], (i / w.stages) & 1) &&
               ptx::globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    // ======== MMA issue: S of tile i + 1 ahead of O of tile i
    if (lane == 0) {
      constexpr uint32_t id_s = idesc(N, false, 0), id_o = idesc(N, true, 0);
      constexpr uint32_t id_r = idesc(R, false, std::is_same<T, __nv_bfloat16>::value ? 1 : 0);
      const uint64_t dq = sdesc_sw128(ptx::smem_u32(q_s)), dqr = sdesc_sw128(ptx::smem_u32(qr_s));
      const uint64_t dp = sdesc_sw128(ptx::smem_u32(p_s));
      int k = 0;                                // tiles so far
      int stage = 0, round = 0, segs = 0;
      bool ok = true;
      auto issue_o = [&](int i, int st, bool first) {          // O += codes^T P of tile i
        if (!wait(&sh.p_full, i & 1, ab)) return false;
        ptx::tc_fence_after();
        const uint64_t dv = sdesc_sw128(ptx::smem_u32(sm + st * stage_size));
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8_ss(tmem + c * N, dv + ((c * C::CHUNK + kk * 4096) >> 4), dp + ((kk * 32) >> 4),
                      id_o, !(first && kk == 0));
        ptx::tc_commit(&sh.empty[st]);
        ptx::tc_commit(&sh.o_done);
        return true;
      };
      while (ok && walk.next(seg)) {
        if (seen_by<R>(p, walk.s, seg.g * R + R - 1) == 0) continue;
        if (!wait(&sh.q_ready, segs & 1, ab)) break;
        ++segs;
        int prev = 0;
        for (int t = seg.t0; t < seg.t1 && ok; ++t) {
          const int buf = C::SBUF == 2 ? (k & 1) : 0, use = C::SBUF == 2 ? (k >> 1) : k;
          if (!wait(&sh.full[stage], round & 1, ab) ||
              (use > 0 && !wait(&sh.s_empty[buf], (use - 1) & 1, ab))) { ok = false; break; }
          ptx::tc_fence_after();
          const uint32_t st0 = ptx::smem_u32(sm + stage * stage_size);
          const uint64_t dk = sdesc_sw128(st0);
          const uint32_t d = tm_s + buf * N;
#pragma unroll
          for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f8_ss(d, dk + ((c * C::CHUNK + kk * 32) >> 4),
                        dq + ((c * N * 128 + kk * 32) >> 4), id_s, c + kk > 0);
          if (p.DR) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              ptx::mma_f16_ss(d, dk + ((NCH * C::CHUNK + kk * 32) >> 4), dqr + ((kk * 32) >> 4),
                              id_r, 1);
          }
          ptx::tc_commit(&sh.s_full[buf]);
          if (t > seg.t0) ok = issue_o(k - 1, prev, t - 1 == seg.t0);
          prev = stage;
          ++k;
          if (++stage == w.stages) { stage = 0; ++round; }
        }
        if (ok) ok = issue_o(k - 1, prev, seg.t1 - 1 == seg.t0);
      }
      if (*ab) {                                // products in flight end before TMEM is freed
        ptx::tc_commit(&sh.drain);
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(&sh.drain, 0) && ptx::globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
    __syncwarp();
  } else {
    // ======== softmax: thread = position of the tile = TMEM lane
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const int tt = warp * 32 + lane;
    int k = 0;
    bool failed = false;
    while (!failed && walk.next(seg)) {
      const int row0 = seg.g * R, rows = min(R, (int)((int64_t)walk.s.n * p.H - row0));
      const int seen = seen_by<R>(p, walk.s, row0 + R - 1);
      const int seen0 = seen_by<R>(p, walk.s, row0);
      if (seen == 0) {                          // nobody sees anything
        for (int i = tid; i < rows * p.KVL; i += 128) {
          const int row = row0 + i / p.KVL;
          T* o = static_cast<T*>(p.out) + (int64_t)(walk.s.first + row / p.H) * p.o_s[0] +
                 (int64_t)(row % p.H) * p.o_s[1];
          st(o + i % p.KVL, 0.f);
        }
        if (tid < rows && p.lse)
          p.lse[(int64_t)(walk.s.first + (row0 + tid) / p.H) * p.lse_s + (row0 + tid) % p.H] = -INFINITY;
        continue;
      }
      if (tid == 0 && walk.s.off + walk.s.n > walk.s.cap) atomicExch(&g_attn_device_error, kErrOutside);
      // ---- queries: scaled by a power of two, split into e4m3 terms (rows past the end: zeros)
#pragma unroll 1
      for (int r = warp; r < R; r += 4) {
        const int row = row0 + r;
        const bool live = r < rows;
        const int64_t n = walk.s.first + row / p.H, h = row % p.H;
        const T* ql = static_cast<const T*>(p.q_lat) + n * p.ql_s[0] + h * p.ql_s[1];
        float x[NCH][4], y[2] = {0.f, 0.f};     // channels 128 c + 4 lane + i; rope 2 lane + i
        uint32_t amax = 0, rmax = 0;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[c][i] = 0.f;
        if (live) {
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            if (p.vec) {
              ld4(ql + c * 128 + 4 * lane, x[c]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) x[c][i] = ld(ql + c * 128 + 4 * lane + i);
            }
          }
          if (p.DR) {
            const T* qr = static_cast<const T*>(p.q_rope) + n * p.qr_s[0] + h * p.qr_s[1];
            y[0] = ld(qr + 2 * lane);
            y[1] = ld(qr + 2 * lane + 1);
          }
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) amax = max(amax, abs_bits(x[c][i]));
        rmax = max(abs_bits(y[0]), abs_bits(y[1]));
        const int e = scale_exp(warp_max_u32(amax), warp_max_u32(rmax));
        const float inv = pow2i(-e);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[c][i] *= inv;
          uint32_t t[NT];
          split4<NT>(x[c], t);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            *reinterpret_cast<uint32_t*>(q_s + c * N * 128 + swz(j * R + r, 4 * lane)) = t[j];
        }
        if (p.DR) {
          T* d = reinterpret_cast<T*>(qr_s + swz(r, 4 * lane));
          st(d, y[0] * inv);
          st(d + 1, y[1] * inv);
        }
        if (lane == 0) {
          sh.q_scale[r] = pow2i(e) * p.scale * kLog2e;
          sh.seen[r] = live ? seen_by<R>(p, walk.s, row) : seen;
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&sh.q_ready);
      asm volatile("bar.sync 1, 128;" ::: "memory");      // q_scale and seen are written
      // ---- scale of this thread's position, a tile ahead, its page two tiles ahead
      auto page_at = [&](int t) {
        const int pos = t * TILE + tt;
        return t < seg.t1 && pos < seen ? page_of(p, seg.b, pos) : -2;
      };
      auto scale_at = [&](int t, int page) {
        if (page == -2) return 1.f;
        if (page < 0) {
          atomicExch(&g_attn_device_error, kErrOutside);
          return __uint_as_float(0x7fffffffu);
        }
        return p.scales[(int64_t)page * p.scales_s + ((t * TILE + tt) & (p.page_size - 1))];
      };
      float s_next = scale_at(seg.t0, page_at(seg.t0));
      int page_next = page_at(seg.t0 + 1);
      float l[R], m_row = -INFINITY;            // m_row: running maximum of row `lane`
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] = 0.f;
      for (int t = seg.t0; t < seg.t1; ++t, ++k) {
        const float s = s_next;
        s_next = scale_at(t + 1, page_next);
        page_next = page_at(t + 2);
        const int buf = C::SBUF == 2 ? (k & 1) : 0, use = C::SBUF == 2 ? (k >> 1) : k;
        const int pos = t * TILE + tt;
        if (!wait(&sh.s_full[buf], use & 1, ab)) failed = true;
        ptx::tc_fence_after();
        float z[N];
        ptx::tmem_ld<N>(tm_s + buf * N + lane_base, z);
        ptx::tmem_wait_ld();
        ptx::tc_fence_before();
        ptx::mbar_arrive(&sh.s_empty[buf]);
        // positions that nobody sees, or that are NaN as a whole, must not meet
        // a weight of zero: their codes become zeros
        if (pos >= seen || s != s) {
          uint8_t* row = sm + ((k % w.stages) * stage_size) + tt * 128;
#pragma unroll 1
          for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(row + c * C::CHUNK + 16 * i) = make_uint4(0, 0, 0, 0);
        }
        const bool open = t * TILE + TILE <= seen0;       // all rows see the whole tile
        const float ls = log2f(s), rs = s == s ? 1.f / s : 1.f;   // (NaN reaches l through P)
        float a[R], mine = -INFINITY;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          a[r] = fmaf(join<NT>(z + r, R), sh.q_scale[r] * s, ls);
          if (!open && pos >= sh.seen[r]) a[r] = -INFINITY;
          const float mx = warp_max(a[r]);
          if (lane == r) mine = mx;
        }
        if (lane < R) sh.red[k & 1][warp][lane] = mine;
        failed = ptx::bar_red_or(1, 128, failed);
        if (failed) break;
        float alpha = 1.f;
        bool grew = false;
        if (lane < R) {
          const float mx = fmaxf(fmaxf(sh.red[k & 1][0][lane], sh.red[k & 1][1][lane]),
                                 fmaxf(sh.red[k & 1][2][lane], sh.red[k & 1][3][lane]));
          if (mx > m_row + kSlack || (m_row == -INFINITY && mx > -INFINITY)) {
            grew = m_row != -INFINITY;
            alpha = ex2(m_row - mx);
            m_row = mx;
          }
        }
        const float m_use = m_row == -INFINITY ? 0.f : m_row - kBias;
        const bool rescale = __any_sync(0xffffffffu, grew);
        // ---- P of tile k - 1 has been read, O holds it
        if (k > 0 && !wait(&sh.o_done, (k - 1) & 1, ab)) failed = true;
        if (rescale) {
          ptx::tc_fence_after();
          float al[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            al[r] = __shfl_sync(0xffffffffu, alpha, r);
            l[r] *= al[r];
          }
#pragma unroll 1
          for (int c = 0; c < NCH * NT; ++c) {
            float o[R];
            ptx::tmem_ld<R>(tmem + c * R + lane_base, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < R; ++r) o[r] *= al[r];
            ptx::tmem_st<R>(tmem + c * R + lane_base, o);
          }
          ptx::tmem_wait_st();
        }
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          float e4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e4[i] = ex2(a[r + i] - __shfl_sync(0xffffffffu, m_use, r + i));
            l[r + i] = fmaf(e4[i], rs, l[r + i]);
          }
          uint32_t tm[NT];
          split4<NT>(e4, tm);
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              p_s[swz(j * R + r + i, tt)] = (uint8_t)(tm[j] >> (8 * i));
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        ptx::mbar_arrive(&sh.p_full);
      }
      // ---- the segment's result
      if (!failed && !wait(&sh.o_done, (k - 1) & 1, ab)) failed = true;
      ptx::tc_fence_after();
      float mine = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x = l[r];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (lane == r) mine = x;
      }
      // (the other buffer than the last tile's: no warp still reads it)
      if (lane < R) sh.red[k & 1][warp][lane] = mine;
      failed = ptx::bar_red_or(1, 128, failed);
      if (failed) break;
      float total = 0.f;
      if (lane < R)
        total = (sh.red[k & 1][0][lane] + sh.red[k & 1][1][lane]) +
                (sh.red[k & 1][2][lane] + sh.red[k & 1][3][lane]);
      const float inv = total == 0.f ? 0.f : 1.f / total;
      const float lse2 = m_row == -INFINITY && total == 0.f ? -INFINITY
                                                            : m_row - kBias + log2f(total);
      const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
      const int slot = 2 * blockIdx.x + (seg.t0 > 0 ? 0 : 1);
      if (warp == 0 && lane < rows) {
        if (!whole) w.lse2[slot * R + lane] = lse2;
        else if (p.lse)
          p.lse[(int64_t)(walk.s.first + (row0 + lane) / p.H) * p.lse_s + (row0 + lane) % p.H] =
              lse2 * kLn2;
      }
#pragma unroll 1
      for (int c = 0; c < NCH; ++c) {
        float o[N];
        ptx::tmem_ld<N>(tmem + c * N + lane_base, o);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float f = __shfl_sync(0xffffffffu, inv, r);
          const float x = f == 0.f ? 0.f : join<NT>(o + r, R) * f;
          if (r < rows) {
            const int ch = c * 128 + tt;
            if (whole) {
              T* dst = static_cast<T*>(p.out) + (int64_t)(walk.s.first + (row0 + r) / p.H) * p.o_s[0] +
                       (int64_t)((row0 + r) % p.H) * p.o_s[1];
              st(dst + ch, x);
            } else {
              w.part[((int64_t)slot * R + r) * p.KVL + ch] = x;
            }
          }
        }
      }
      // the next segment's queries and row figures come after all warps are done here
      asm volatile("bar.sync 1, 128;" ::: "memory");
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 5) {
    ptx::tmem_relinquish();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a group that several ranges share, in order: one block per
// (range that starts inside a group, row).
template <typename T, int R>
__global__ void __launch_bounds__(128)
cache_join_kernel(const CacheParams p, const Work w) {
  ptx::grid_dep_wait();
  const int c0 = blockIdx.x + 1;
  const Cut cut = w.cuts[c0];
  if (cut.b < 0 || cut.parts == 0) return;
  const Seq s = load_seq<R>(p, cut.b);
  const int r = blockIdx.y, row = cut.g * R + r;
  if (row >= (int64_t)s.n * p.H) return;
  // part 0: what range c0 - 1 left unfinished; part i: what range c0 + i - 1 begins with
  auto slot = [&](int i) { return i == 0 ? 2 * (c0 - 1) + 1 : 2 * (c0 + i - 1); };
  float mx = -INFINITY;
  for (int i = 0; i < cut.parts; ++i) mx = fmaxf(mx, w.lse2[slot(i) * R + r]);
  const float m = mx == -INFINITY ? 0.f : mx;
  const int ch = 4 * threadIdx.x;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, tot = 0.f;
  for (int i = 0; i < cut.parts; ++i) {
    const float f = exp2f(w.lse2[slot(i) * R + r] - m);
    tot += f;
    if (ch < p.KVL) {
      const float4 x = *reinterpret_cast<const float4*>(w.part + ((int64_t)slot(i) * R + r) * p.KVL + ch);
      acc[0] = fmaf(f, x.x, acc[0]);
      acc[1] = fmaf(f, x.y, acc[1]);
      acc[2] = fmaf(f, x.z, acc[2]);
      acc[3] = fmaf(f, x.w, acc[3]);
    }
  }
  const int64_t n = s.first + row / p.H, h = row % p.H;
  const float inv = tot == 0.f ? 0.f : 1.f / tot;
  if (ch < p.KVL) {
    T* o = static_cast<T*>(p.out) + n * p.o_s[0] + h * p.o_s[1] + ch;
#pragma unroll
    for (int i = 0; i < 4; ++i) st(o + i, acc[i] * inv);
  }
  if (threadIdx.x == 0 && p.lse)
    p.lse[n * p.lse_s + h] = tot == 0.f ? -INFINITY : (m + log2f(tot)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int device_sms() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Rows per group: 16 where the sequences of the call have no more rows than that
// on average, or where 32 rows leave no room for the two stages that the order
// of the products needs (fp16, KVL 512 with a rope part); else 32.
int rows_per_group(const CacheParams& p, int terms) {
  if (((int64_t)p.N * p.H + p.B - 1) / p.B <= 16) return 16;
  return stages(p.KVL, p.DR, terms, 32) >= 2 ? 32 : 16;
}

template <typename T, int R, int NCH>
cudaError_t launch(const CacheParams& p, Work w, const CUtensorMap& mc, const CUtensorMap& mr,
                   int ranges, cudaStream_t s) {
  using C = Cfg<T, R, NCH>;
  auto k = cache_attn_kernel<T, R, NCH>;
  w.stages = stages(p.KVL, p.DR, C::NT, R);
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
  if (e != cudaSuccess) return e;
  const size_t smem = fixed_bytes(p.KVL, C::NT, R) + w.stages * stage_bytes(p.KVL, p.DR);
  e = launch_dependent(k, dim3(ranges), kThreads, smem, s, p, w, mc, mr);
  if (e != cudaSuccess) return e;
  return launch_dependent(cache_join_kernel<T, R>, dim3(ranges - 1, R), 128, 0, s, p, w);
}

template <typename T, int R>
cudaError_t launch_r(const CacheParams& p, const Work& w, const CUtensorMap& mc,
                     const CUtensorMap& mr, int ranges, cudaStream_t s) {
  switch (p.KVL) {
    case 128: return launch<T, R, 1>(p, w, mc, mr, ranges, s);
    case 256: return launch<T, R, 2>(p, w, mc, mr, ranges, s);
    case 384: return launch<T, R, 3>(p, w, mc, mr, ranges, s);
    default: return launch<T, R, 4>(p, w, mc, mr, ranges, s);
  }
}

// [num_pages][page_size][width] with 128-byte boxes of one page, 128-byte swizzle
bool encode(CUtensorMap* m, CUtensorMapDataType dt, int elt, void* base, int width,
            const CacheParams& p, const int64_t (&stride)[2]) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return false;
  const int64_t page = p.num_pages > 1 ? stride[0] : stride[1] * p.page_size;
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)p.page_size, (cuuint64_t)p.num_pages};
  const cuuint64_t strides[2] = {(cuuint64_t)(stride[1] * elt), (cuuint64_t)(page * elt)};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / elt), (cuuint32_t)(p.page_size < TILE ? p.page_size : TILE), 1u};
  const cuuint32_t one[3] = {1u, 1u, 1u};
  return enc(m, dt, 3, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

// partials | their log sums | cuts
size_t attention_workspace_bytes(const CacheParams& p) {
  const size_t ranges = device_sms(), R = 32;
  return align256(2 * ranges * R * p.KVL * 4) + align256(2 * ranges * R * 4) +
         align256(ranges * sizeof(Cut));
}

cudaError_t launch_attention(const CacheParams& p, int io_dtype, void* workspace, cudaStream_t s) {
  const int ranges = device_sms();
  const int R = rows_per_group(p, io_dtype == KDA_DTYPE_F16 ? kTerms<__half> : kTerms<__nv_bfloat16>);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Work w{};
  w.part = reinterpret_cast<float*>(ws);
  ws += align256((size_t)2 * ranges * R * p.KVL * 4);
  w.lse2 = reinterpret_cast<float*>(ws);
  ws += align256((size_t)2 * ranges * R * 4);
  w.cuts = reinterpret_cast<Cut*>(ws);
  CUtensorMap mc, mr;
  if (!encode(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.codes, p.KVL, p, p.codes_s))
    return cudaErrorInvalidValue;
  mr = mc;
  if (p.DR && !encode(&mr, io_dtype == KDA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      2, p.rope, p.DR, p, p.rope_s))
    return cudaErrorInvalidValue;
  if (io_dtype == KDA_DTYPE_F16)
    return R == 16 ? launch_r<__half, 16>(p, w, mc, mr, ranges, s)
                   : launch_r<__half, 32>(p, w, mc, mr, ranges, s);
  return R == 16 ? launch_r<__nv_bfloat16, 16>(p, w, mc, mr, ranges, s)
                 : launch_r<__nv_bfloat16, 32>(p, w, mc, mr, ranges, s);
}

int read_attn_device_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_attn_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace cache
}  // namespace kda
