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
// What is not in 8 bits is split into 8-bit terms, each finer than the one before:
// x = x0 + x1 / 16 + ... .  A query (scaled by a power of two) in bf16 has 8
// significant bits, two e4m3 terms hold it; fp16 takes three.  A softmax weight is
// rounded to 11 bits and takes three e5m2 terms, which keep it when it is small.  The terms
// are more columns of N and are added in fp32 afterwards: an instruction of 128 x N x
// 32 spends its time on reading 4 KB of codes from shared memory, so the columns cost
// little (41 cycles at N = 32, 49 at 64, 56 at 96).
//
// A position's scale s_t is a power of two, so the weight that meets the codes is
//   P_t = exp2(z_t log2e + log2 s_t - M),  M the running maximum of the exponents,
// and the sum takes P_t / s_t: P stays in range whatever the scales are.  M moves
// (and O is rescaled in TMEM) only where a row outgrows P's format.
//
// Work: a row group (R rows of a sequence) times its tiles; all the tiles of a
// call, in order, are cut into equal ranges, one per SM, so a long sequence is
// split over many SMs and short ones share one.  A group cut by a range's end
// leaves fp32 partials and cache_join_kernel adds them in order: the result does
// not depend on timing.
//
// Roles: warp 10 walks the block's range and queues its segments (a group's tiles in
// the range); warp 8 loads by TMA into a ring of 16 KB chunks; warps 9 and 11 issue the
// two products, a warp each, because a product that waits for a barrier would hold the
// other one's instructions back (issued from one warp: slower than they execute);
// warps 0-7 do the softmax, half of the rows each four, a position a thread.
//
// Measured (B200, 16 heads, KVL 512, inputs that rotate past L2, join included):
//   one token each for 8 sequences of 32768, bf16     35.6 us, 3.8 TB/s of the cache
//   one token each for 64 sequences of 300 to 8192    36.2 us, 3.3 TB/s
//   512 tokens of one prompt against 8192 positions   215.7 us, 656 TFLOP/s as counted
//     (4 KVL for a row and key), 2.5 times that as executed on the terms
// What bounds it: at 16 rows a tile takes the time of its 64 KB from HBM (1.5 us for
// each SM), and around the tiles stand 7.5 us until the first scores (lengths, page
// numbers, queries, the first tile), 1 to 2 us for a result and 4 us until the join's
// end.  At 32 rows the ring holds 2.5 tiles, less than the chain load -> S -> softmax ->
// O spans (about two tiles' time, 2800 cycles each), and the products' reads of shared
// memory alone take 2200 of them.
#include <cuda.h>

#include <type_traits>

#include "mla_cache.cuh"
#include "mla_cache_ring.cuh"
#include "tc_ptx.cuh"

namespace kda {
namespace cache {

__device__ int g_attn_device_error = 0;

namespace {

constexpr int TILE = 128;                  // positions per tile (MMA M)
constexpr int CHUNK = TILE * 128;          // bytes of 128 positions x 128 bytes
constexpr int kThreads = 384;              // warps 0-7 softmax, 8 loads, 9 S, 10 segments, 11 O
// Registers: the block starts with 384 x 168; the softmax warps take 192 each, the
// others keep 120 (256 x 192 + 128 x 120 = 384 x 168).
constexpr int kSoftmaxRegs = 192, kOtherRegs = 120;

constexpr int kMaxRanges = 256;            // blocks (SMs) that a call's tiles are cut over
constexpr int kSmemMax = 232448;           // 227 KB per block
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kUnset = -3.4e38f;         // maximum of a row that has seen nothing: below any score

// e4m3 terms of a query, each 16 times finer: two hold bf16's 8 bits, three fp16's 11.
// (Values below 2^-12 of the row's largest are off by at most 2^-19 (2^-23) of it: the
// terms' last steps.)
template <typename T> constexpr int kQTerms = std::is_same<T, __nv_bfloat16>::value ? 2 : 3;
// A softmax weight P is rounded to fp16 (11 bits: 2^-11 of itself) and cut into three
// e5m2 terms, each 16 times finer than the one before.  An e5m2 code is an fp16's upper
// byte, so a term is the byte nearest to what is left, and its remainder, of either sign,
// comes next: of 11 bits at most 8 remain, then 4, which three bits hold (they fit whole:
// up to 8 steps).  Nothing of the fp16 value is lost, subnormals included, and no term
// exceeds 2^15.
// P carries 2^BIAS of the row's maximum and may outgrow it by 2^SLACK, to 2^15, before
// the maximum moves.  So a weight holds 11 bits down to 2^-(14 + BIAS) of the largest one,
// and is off by at most 2^-(25 + BIAS) of it below that, while the sum takes it unrounded:
// a crowd of n small weights may lose n 2^-(25 + BIAS) of the largest.  More BIAS costs
// rescales.  (bf16, BIAS 5, 7 and 9, us: 512 tokens on 8192 211, 215, 222; 8 x 32768 34.9,
// 35.4, 36.0.  With 7 a weight of 2^-20 of the largest has all its 11 bits, so that a long
// crowd's part holds to bf16's rounding.)
constexpr int NP = 3;
constexpr uint32_t kE5M2 = 1;
constexpr float kPFiner = 16.f;
template <typename T> constexpr float kBias = std::is_same<T, __nv_bfloat16>::value ? 7.f : 9.f;
constexpr float kPTop = 15.f;             // BIAS + SLACK
__device__ __forceinline__ void split_weights(const float (&x)[4], uint32_t (&t)[NP]) {
  __half2 r[2] = {__floats2half2_rn(x[0], x[1]), __floats2half2_rn(x[2], x[3])};
  const __half2 finer = __float2half2_rn(kPFiner);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = *reinterpret_cast<const uint32_t*>(&r[i]);
      if (j + 1 < NP) {                   // (a NaN may be lost here; the sum keeps it)
        c[i] = (c[i] + 0x00800080u) & 0xff00ff00u;
        r[i] = __hmul2(__hsub2(r[i], *reinterpret_cast<const __half2*>(&c[i])), finer);
      }
    }
    t[j] = __byte_perm(c[0], c[1], 0x7531);
  }
}
constexpr uint32_t kE4M3 = 0;
constexpr float kQFiner = 16.f;

template <typename T, int R, int NCH>
struct Cfg {
  static constexpr int NQ = kQTerms<T>;
  static constexpr int NS = NQ * R, NO = NP * R;         // columns of S and of one O chunk
  static constexpr int SBUF = NCH * NO + 2 * NS <= 512 ? 2 : 1;
  static_assert(NCH * NO + SBUF * NS <= 512, "TMEM columns");
};

// Shared memory besides the ring (barriers and rows; 1 KB: alignment), and the
// chunks that fit beside it, kRingTiles tiles of them at most.  The order of the products
// needs the chunks of two tiles at once.
constexpr int kSharedBytes = 4096;
int fixed_bytes(int kvl, int q_terms, int R) {
  return kSharedBytes + 1024 + q_terms * R * kvl + R * 128 + 2 * NP * R * 128;
}
int tile_chunks(int kvl, int dr) { return kvl / 128 + (dr ? 1 : 0); }
int ring_chunks(int kvl, int dr, int q_terms, int R) {
  const int n = (kSmemMax - fixed_bytes(kvl, q_terms, R)) / CHUNK;
  return min(n, kRingTiles * tile_chunks(kvl, dr));
}

// Where a range of tiles starts inside a group; what cache_join_kernel reads.
struct Cut {
  int parts;       // ranges that share the group that the range starts in the middle of
                   // (0: none, or an earlier cut joins it)
  int row0, rows;  // the group's rows
  int first;       // its sequence's first new token
};

struct Work {
  float* part;     // [2 ranges][R][KVL] fp32: slot 2 c: group begun before range c; 2 c + 1: left unfinished
  float* lse2;     // [2 ranges][R] log2 of the sum of a part
  Cut* cuts;       // [ranges]
  int ring;        // chunks of the ring
  bool whole;      // a group belongs to the range that it starts in: no parts, no join
};

// ---------------------------------------------------------------------------
// how the tiles of a call are counted and cut
// ---------------------------------------------------------------------------
// Sequence b as R-row groups.  A group counts for its tiles and kSetup more: what
// its queries, its first tile's latency and its result cost (3, 4 and 5, us: 64
// sequences of 300 to 8192 tokens 36.9, 36.0, 38.1; prompts of 1 to 1500 tokens 226,
// 225, 221; 4 sequences of 8192 20.3, 19.9, 20.2; all at KVL 512 and 16 heads, the count is
// the same for other widths).  Groups of one sequence see more and
// more positions; they are counted in pairs (g, groups - 1 - g), which all count about
// the same, so that a place in the count is found by a division.
constexpr int kSetup = 4;
struct Seq {
  int first, n, off;       // new tokens; token i sits at off + i
  int groups, pair;        // row groups; count per pair
  int cap;                 // positions that the table holds
};

__device__ __forceinline__ int div_heads(const CacheParams& p, int row) {
  const uint32_t q = __umulhi((uint32_t)row, p.h_mul);      // h_mul = 2^32 / H: short by one at most
  return (int)q + ((uint32_t)row - q * p.H >= (uint32_t)p.H);
}
__device__ __forceinline__ int seen_by(const CacheParams& p, const Seq& s, int row) {
  return max(0, min(s.off + min(div_heads(p, row), s.n - 1) + 1, s.cap));
}
template <int R>
__device__ __forceinline__ int group_tiles(const CacheParams& p, const Seq& s, int g) {
  return max(1, (seen_by(p, s, g * R + R - 1) + TILE - 1) / TILE);
}
template <int R>
__device__ __forceinline__ Seq load_seq(const CacheParams& p, int b) {
  Seq s;
  new_tokens(p, b, s.first, s.n);
  s.off = max(p.lens[b], 0) - s.n;
  s.cap = p.max_pages * p.page_size;
  s.groups = (int)(((int64_t)s.n * p.H + R - 1) / R);
  s.pair = 0;
  if (s.groups == 1) s.pair = kSetup + group_tiles<R>(p, s, 0);
  // the first pair's sum, and up to two more: the last group may be short, and the
  // tiles are rounded up.  (Where the table ends before the sequence: all may be as long
  // as the last.)
  if (s.groups > 1)
    s.pair = 2 * kSetup + 2 + group_tiles<R>(p, s, s.off + s.n > s.cap ? s.groups - 1 : 0) +
             group_tiles<R>(p, s, s.groups - 1);
  return s;
}
__device__ __forceinline__ int64_t seq_tiles(const Seq& s) {
  return (int64_t)((s.groups + 1) / 2) * s.pair;
}

// What lies at count r of a sequence: place q of pair (g1, g2), which has n1 + n2
// tiles (n2 = 0: the middle group, alone).  Group g1 takes the places up to kSetup +
// n1, its tile i place kSetup + i; g2 follows in the same way.
template <int R>
__device__ __forceinline__ void place(const CacheParams& p, const Seq& s, int64_t r, int& g1, int& q,
                                      int& g2, int& n1, int& n2) {
  if (s.groups == 1) {
    g1 = g2 = n2 = 0;
    q = (int)r;
    n1 = s.pair - kSetup;
    return;
  }
  if (r < s.pair) {
    g1 = 0;
    q = (int)r;
  } else if (r <= 0x7fffffff) {
    g1 = (int)((uint32_t)r / (uint32_t)s.pair);
    q = (int)r - g1 * s.pair;
  } else {
    g1 = (int)(r / s.pair);
    q = (int)(r - (int64_t)g1 * s.pair);
  }
  g2 = s.groups - 1 - g1;
  n1 = group_tiles<R>(p, s, g1);
  n2 = g2 > g1 ? group_tiles<R>(p, s, g2) : 0;
}

struct Segment {
  int b, g, t0, t1;        // tiles t0 .. t1 - 1 of group g
  int tiles;               // of the whole group
};

// Walks the segments of the range [u, end).
template <int R>
struct Walk {
  const CacheParams& p;
  Seq s;
  int b;
  int64_t u, end, base;    // base: count at which sequence b starts
  bool whole;              // groups that start in the range, to their end
  Segment second;          // of the pair under way, when there is one (t1 > t0)
  __device__ Walk(const CacheParams& p_, const Seq& s_, int b_, int64_t base_, int64_t u_, int64_t end_,
                  bool whole_)
      : p(p_), s(s_), b(b_), u(u_), end(end_), base(base_), whole(whole_), second{0, 0, 0, 0, 0} {}
  __device__ bool next(Segment& seg) {
    if (second.t1 > second.t0) {
      seg = second;
      second.t1 = second.t0;
      return true;
    }
    while (u < end) {
      while (u >= base + seq_tiles(s)) {
        base += seq_tiles(s);
        s = load_seq<R>(p, ++b);
      }
      int g1, q, g2, n1, n2;
      place<R>(p, s, u - base, g1, q, g2, n1, n2);
      const int end1 = kSetup + n1, all = end1 + (n2 > 0 ? kSetup + n2 : 0);
      int stop = (int)min((int64_t)s.pair, q + (end - u));
      u += stop - q;
      if (whole) {
        second = Segment{b, g2, 0, q <= end1 && end1 < stop ? n2 : 0, n2};
        seg = Segment{b, g1, 0, q == 0 ? n1 : 0, n1};
        if (seg.t1 > 0) return true;
        if (second.t1 > 0) {
          seg = second;
          second.t1 = 0;
          return true;
        }
        continue;
      }
      // the last place of a pair takes whatever is left of it
      stop = stop == s.pair ? all : min(stop, all);
      second = Segment{b, g2, max(0, q - end1 - kSetup), stop - end1 - kSetup, n2};
      seg = Segment{b, g1, max(0, q - kSetup), min(stop, end1) - kSetup, n1};
      if (seg.t1 > seg.t0) return true;
      if (second.t1 > second.t0) {
        seg = second;
        second.t1 = second.t0;
        return true;
      }
    }
    return false;
  }
};

// ---------------------------------------------------------------------------
// PTX used only here
// ---------------------------------------------------------------------------
// The issuing warp runs its loops with all lanes, and each instruction elects one
// lane itself: the operands then stay in uniform registers.  One instruction of 128 x
// 32 x 32 takes 41 cycles this way (49 with N = 64: reading its operands from shared
// memory), 80 or 143 from a branch that one lane takes.
// A shared-memory descriptor is its low word (address and leading offset) and a high
// word that the layout fixes; consecutive operands differ in the low word alone.
// D[tmem] = A[smem] B[smem] (+ D): 8-bit operands, fp32 accumulation
template <uint32_t A_HI, uint32_t B_HI>
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %6};\n\t"
      "elect.sync x|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(A_HI), "n"(B_HI)
      : "memory");
}
// D += A B, 16-bit operands of one type
template <uint32_t A_HI, uint32_t B_HI>
__device__ __forceinline__ void mma_half(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %5};\n\t"
      "elect.sync x|e, 0xffffffff;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(A_HI), "n"(B_HI)
      : "memory");
}
// arrive on `bar` once the warp's products so far have completed
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 x;\n\t"
      "elect.sync x|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          ptx::smem_u32(bar))
      : "memory");
}
// 128-byte rows with the 128-byte swizzle (eight rows = 1024 bytes, consecutive).
// K-major operands: rows are M or N; M-major ones: rows are K, and the 128 bytes of a
// row are all of M.  (High word: stride 1024, version 1, swizzle code 2.)
constexpr uint32_t kSw128Hi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t sw128_lo(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
// no swizzle: core matrices of 8 x 16 bytes, 128 bytes on along K, 2048 along N
constexpr uint32_t kPHi = (TILE * 16 >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t p_lo(uint32_t saddr) { return (saddr >> 4) | ((128 >> 4) << 16); }
// One lane of the warp: bytes to expect on a barrier, and a box of a tensor map.
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 x;\n\t"
      "elect.sync x|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes)
      : "memory");
}
// bytes that a barrier expects and that will not come
__device__ __forceinline__ void give_back(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 x;\n\t"
      "elect.sync x|e, 0xffffffff;\n\t"
      "@e mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                         uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 x;\n\t"
      "elect.sync x|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
// Instruction descriptors: fp32 accumulator; 8-bit formats 0 = e4m3, 1 = e5m2, 16-bit
// ones 0 = f16, 1 = bf16
__host__ __device__ constexpr uint32_t idesc(int N, bool a_m_major, bool b_n_major, uint32_t a_fmt,
                                              uint32_t b_fmt) {
  return (1u << 4) | (a_fmt << 7) | (b_fmt << 10) | ((a_m_major ? 1u : 0u) << 15) |
         ((b_n_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(TILE >> 4) << 24);
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

// Bounded wait: false once the block gave up (the caller then leaves its loop).  A
// try sleeps for at most about a microsecond, so that the limit is some seconds.
constexpr int kTries = 1 << 21;
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(ptx::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < kTries; ++i) {
    if (try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  atomicExch(&g_attn_device_error, kErrWait);
  return false;
}
// the same for what is in flight when the block has given up already
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < kTries && !try_wait(bar, parity); ++i) {
  }
}

// A query's values (times 2^-8; at most 1, so that no term reaches 1.875, the code of
// NaN) as e4m3 terms, x = t[0] + t[1] / 16 (+ t[2] / 256), four at a time.  An e4m3 code
// is the sign and bits 13 .. 7 of the fp16 of the value times 2^-8.
template <int NT>
__device__ __forceinline__ void split_query(const float (&x)[4], uint32_t (&t)[NT]) {
  __half2 r[2] = {__floats2half2_rn(x[0], x[1]), __floats2half2_rn(x[2], x[3])};
  const __half2 finer = __float2half2_rn(kQFiner);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&r[i]) & 0xbf80bf80u;
      if (j + 1 < NT) r[i] = __hmul2(__hsub2(r[i], *reinterpret_cast<const __half2*>(&u)), finer);
      c[i] = ((u >> 7) & 0x007f007fu) | ((u >> 8) & 0x00800080u);
    }
    t[j] = __byte_perm(c[0], c[1], 0x6420);
  }
}
// the sum of a value's terms, each `finer` times finer
template <int NT>
__device__ __forceinline__ float join(const float* t, int stride, float finer) {
  float x = t[(NT - 1) * stride];
#pragma unroll
  for (int j = NT - 2; j >= 0; --j) x = fmaf(x, 1.f / finer, t[j * stride]);
  return x;
}

template <int R>
struct Rows {              // per row of a group
  float q_scale[R];        // 2^e scale log2e
  float m[R];              // running maximum less BIAS
  float alpha[R];          // what its sums and O are rescaled by
  int seen[R];             // positions that it sees
  int64_t out[R], lse[R];  // where its results go
};
// A segment as the other warps get it (t1 = t0: there are no more).
struct Info {
  int b, t0, t1, tiles;    // tiles t0 .. t1 - 1 of a group that has `tiles`
  int row0, rows;          // its rows
  int first, off;          // its sequence's new tokens
  int seen, seen0;         // positions that its last and its first row see
};
constexpr int kQueue = 4;  // segments that are known ahead

template <int R>
struct Shared {            // at the end of dynamic shared memory
  uint64_t full[2 * kStages], freed[2 * kStages];                    // by half tiles
  uint64_t seg_full[kQueue], seg_empty[kQueue];
  uint64_t s_full[2], s_empty[2], p_full[2], q_ready, drain[2];      // tile % 2
  uint32_t tmem;
  int abort_flag;
  int64_t scan[(kThreads + 31) / 32];
  int64_t base;            // where the range starts: count at which sequence b starts
  int b;
  Seq seq;                 // and that sequence
  Info queue[kQueue];
  Rows<R> rows[2];         // of this segment and the next
  float red[8][R / 2];     // per warp and row: maxima, sums
};
static_assert(sizeof(Shared<32>) <= kSharedBytes,
              "room for barriers and rows");

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// sums of v[0 .. N - 1] over the warp: lanes i, i + N, ... get the sum of v[i]
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], int lane) {
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2) {
    const bool up = lane & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
    }
  }
#pragma unroll
  for (int o = N; o < 32; o <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}
// 8 or 16 consecutive TMEM columns of this warp's lanes
template <int N>
__device__ __forceinline__ void tmem_get(uint32_t at, float* v) {
  if constexpr (N == 16) {
    ptx::tmem_ld16(at, v);
  } else {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(at));
  }
}
template <int N>
__device__ __forceinline__ void tmem_put(uint32_t at, const float* v) {
  if constexpr (N == 16) {
    ptx::tmem_st16(at, v);
  } else {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  }
}

template <typename T, int R, int NCH>
__global__ void __launch_bounds__(kThreads, 1)
cache_attn_kernel(const CacheParams p, const Work w, const __grid_constant__ CUtensorMap map_codes,
                  const __grid_constant__ CUtensorMap map_rope) {
  using C = Cfg<T, R, NCH>;
  constexpr float BIAS = kBias<T>;
  constexpr int NQ = C::NQ, NS = C::NS, NO = C::NO;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = sm + w.ring * CHUNK;
  uint8_t* qr_s = q_s + NCH * NS * 128;
  uint8_t* p_s = qr_s + R * 128;                // two buffers
  Shared<R>& sh = *reinterpret_cast<Shared<R>*>(p_s + 2 * NO * 128);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int ring = w.ring, tile_chunks = NCH + (p.DR ? 1 : 0);
  constexpr int HC = (NCH + 1) / 2;             // code chunks of a tile's first half
  const int half = tile_chunks - NCH + HC;      // chunks of it

  if (tid == 0) {
    for (int i = 0; i < 2 * kStages; ++i) {
      ptx::mbar_init(&sh.full[i], 1);
      ptx::mbar_init(&sh.freed[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&sh.s_full[i], 1);
      ptx::mbar_init(&sh.s_empty[i], 256);
      ptx::mbar_init(&sh.p_full[i], 256);
    }
    for (int i = 0; i < kQueue; ++i) {
      ptx::mbar_init(&sh.seg_full[i], 1);
      ptx::mbar_init(&sh.seg_empty[i], 3 + 256);
    }
    ptx::mbar_init(&sh.q_ready, 256);
    ptx::mbar_init(&sh.drain[0], 1);
    ptx::mbar_init(&sh.drain[1], 1);
    sh.abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 9) ptx::tmem_alloc(&sh.tmem, 512);
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();

  // ---- this block's range of the call's tiles
  int64_t u0, u1, range_tiles;
  {
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t mine = 0;
    Seq s{};
    for (int b = b0; b < b1; ++b) {
      s = load_seq<R>(p, b);
      mine += seq_tiles(s);
    }
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
    const int64_t range = total <= 0x7fffffff
                              ? ((uint32_t)total + gridDim.x - 1) / gridDim.x
                              : (total + gridDim.x - 1) / gridDim.x;
    u0 = min(total, range * blockIdx.x);
    u1 = min(total, u0 + range);
    if (u0 < u1 && u0 >= before && u0 < before + mine) {
      int b = b0;
      if (per > 1) {
        for (;; ++b) {
          s = load_seq<R>(p, b);
          if (u0 < before + seq_tiles(s)) break;
          before += seq_tiles(s);
        }
      }
      sh.b = b;
      sh.base = before;
      sh.seq = s;
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    range_tiles = range;
  }
  const uint32_t tmem = sh.tmem;
  const uint32_t tm_s = tmem + NCH * NO;        // S buffers after the O chunks
  volatile int* ab = &sh.abort_flag;
  // the next segment from the queue, copied out; 0: there are no more, -1: given up
  int taken = 0;
  auto take = [&](Info& sg, bool one_arrives) {
    const int i = taken % kQueue;
    if (!wait(&sh.seg_full[i], (taken / kQueue) & 1, ab)) return -1;
    sg = sh.queue[i];
    if (one_arrives) {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.seg_empty[i]);
    } else {
      ptx::mbar_arrive(&sh.seg_empty[i]);
    }
    ++taken;
    return sg.t1 > sg.t0 ? 1 : 0;
  };

  const auto uniform = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 10) {
      // ======== segments: a queue of them for the other warps; groups that see nothing
      // get their zeros here, and so do the rows of no sequence
      const auto empty_row = [&](int64_t n, int64_t h) {
        T* o = static_cast<T*>(p.out) + n * p.o_s[0] + h * p.o_s[1];
        for (int c = lane; c < p.KVL; c += 32) st(o + c, 0.f);
        if (lane == 0 && p.lse) p.lse[n * p.lse_s + h] = -INFINITY;
      };
      Walk<R> walk(p, sh.seq, sh.b, sh.base, u0, u1, w.whole);
      for (int i = 0;;) {
        Segment seg;
        const bool have = walk.next(seg);
        Info info{};
        if (have) {
          const int row0 = seg.g * R;
          info = Info{seg.b, seg.t0, seg.t1, seg.tiles, row0,
                      (int)min((int64_t)R, (int64_t)walk.s.n * p.H - row0), walk.s.first, walk.s.off,
                      seen_by(p, walk.s, row0 + R - 1), seen_by(p, walk.s, row0)};
          if (lane == 0 && walk.s.off + walk.s.n > walk.s.cap)
            atomicExch(&g_attn_device_error, kErrOutside);
          if (info.seen == 0) {
            for (int r = 0; r < info.rows; ++r) {
              const int tok = div_heads(p, row0 + r);
              empty_row(info.first + tok, row0 + r - tok * p.H);
            }
            continue;
          }
        }
        if (i >= kQueue && !wait(&sh.seg_empty[i % kQueue], (i / kQueue - 1) & 1, ab)) break;
        if (lane == 0) {
          sh.queue[i % kQueue] = info;
          ptx::mbar_arrive(&sh.seg_full[i % kQueue]);
        }
        if (!have) break;
        ++i;
      }
      // ---- the group that this range starts inside of, for cache_join_kernel
      Cut cut{0, 0, 0, 0};
      int cut_g = -1;
      if (u0 < u1 && blockIdx.x > 0 && !w.whole) {
        int g1, q, g2, n1, n2;
        place<R>(p, sh.seq, u0 - sh.base, g1, q, g2, n1, n2);
        int64_t start = u0 - q + kSetup;         // where the group's first tile counts
        int n = 0;
        if (q > kSetup && q < kSetup + n1) {
          cut_g = g1; n = n1;
        } else if (n2 > 0 && q > 2 * kSetup + n1 && q < 2 * kSetup + n1 + n2) {
          cut_g = g2; start += kSetup + n1; n = n2;
        }
        if (cut_g >= 0 && start >= u0 - range_tiles) {
          cut = Cut{(int)((start + n - 1) / range_tiles) - (int)(start / range_tiles) + 1, cut_g * R,
                    (int)min((int64_t)R, (int64_t)sh.seq.n * p.H - cut_g * R), sh.seq.first};
        }
      }
      if (lane == 0 && !w.whole) w.cuts[blockIdx.x] = cut;
      // ---- new tokens before the first sequence's and after the last one's (a batch that
      // is padded to a fixed N)
      if (p.q_start != nullptr || p.B == 0) {
        const int lo = p.B > 0 ? min(max(p.q_start[0], 0), p.N) : 0;
        const int hi = p.B > 0 ? max(min(p.q_start[p.B], p.N), lo) : 0;
        for (int r = blockIdx.x; r < (lo + p.N - hi) * p.H; r += gridDim.x) {
          const int tok = div_heads(p, r);
          empty_row(tok < lo ? tok : hi + tok - lo, r - tok * p.H);
        }
      }
      __syncwarp();
    } else if (warp == 8) {
      // ======== loads: boxes of one page (at most 128 positions) x 128 bytes into a
      // ring of 16 KB chunks; a tile is its rope chunk, then its code chunks, in two halves
      // that land and are freed apart.  (A look at a barrier takes some 300 cycles while
      // the products read shared memory: one for each chunk was too many, one for a whole
      // tile keeps the chunks waiting for one another.)
      const Ring places(ring, tile_chunks, half);
      const int box_rows = min(p.page_size, TILE), boxes = TILE / box_rows;
      const uint32_t sm0 = ptx::smem_u32(sm);
      int k = 0, slot = 0, freed = -1;            // freed: half tiles known to be
      bool ok = true;
      Info seg;
      while (ok && uniform(take(seg, true)) > 0) {
        const int t1 = uniform(seg.t1), seen = uniform(seg.seen);
        // lane i: page of box i of a tile
        auto page_of_box = [&](int t) {
          const int pos = t * TILE + lane * box_rows, i = pos >> p.page_shift;
          int x = -1;
          if (lane < boxes && t < t1 && pos < seen && i < p.max_pages)
            x = p.table[(int64_t)seg.b * p.table_s + i];
          return x;
        };
        int page_next = page_of_box(seg.t0);
        for (int t = uniform(seg.t0); t < t1 && ok; ++t, ++k) {
          // outside the pool: the copy fills in zeros
          const int page = (uint32_t)page_next < (uint32_t)p.num_pages ? page_next : p.num_pages;
          page_next = page_of_box(t + 1);
          const int pos = t * TILE, nbox = min(boxes, (seen - pos + box_rows - 1) / box_rows);
          const int at = p.page_size > TILE ? pos & (p.page_size - 1) : 0;
          const uint32_t bar = ptx::smem_u32(&sh.full[half_barrier(2 * k)]);
          expect_bytes(bar, nbox * box_rows * 128 * half);
          expect_bytes(bar + 8, nbox * box_rows * 128 * (tile_chunks - half));
          for (int c = 0; c < tile_chunks; ++c) {
            const int need = places.held_by(k, c);
            if (need > freed) {
              if (!wait(&sh.freed[half_barrier(need)], half_parity(need), ab)) {
                for (int h = 0; h < 2; ++h) give_back(bar + 8 * h, nbox * box_rows * 128 * places.missing(c, h));
                ok = false;
                break;
              }
              freed = need;
            }
            const int code = c - (tile_chunks - NCH);
            const CUtensorMap* map = code < 0 ? &map_rope : &map_codes;
            for (int i = 0; i < nbox; ++i)
              load_box(sm0 + slot * CHUNK + i * box_rows * 128, map, max(code, 0) * 128, at,
                       __shfl_sync(0xffffffffu, page, i), bar + 8 * (c >= half));
            if (++slot == ring) slot = 0;
          }
        }
      }
      if (*ab) {                                  // copies in flight land before the block ends
        for (int i = first_in_flight(k); i < 2 * k; ++i) drain(&sh.full[half_barrier(i)], half_parity(i));
      }
      __syncwarp();
    } else if (warp == 9) {
      // ======== S^T = codes Q^T, a tile or two ahead of the softmax.  (Two warps issue the
      // two products: one warp issues more slowly than the products execute, and would
      // hold back the scores of a tile behind the wait for another's weights.)
      constexpr uint32_t kHalf = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t id_s = idesc(NS, false, false, kE4M3, kE4M3);
      constexpr uint32_t id_r = idesc(R, false, false, kHalf, kHalf);
      const uint32_t dq = sw128_lo(ptx::smem_u32(q_s)), dqr = sw128_lo(ptx::smem_u32(qr_s));
      const uint32_t dk0 = sw128_lo(ptx::smem_u32(sm)), ts = (uint32_t)uniform((int)tm_s);
      int k = 0, segs = 0, slot = 0;
      bool ok = true;
      Info seg;
      while (ok && uniform(take(seg, true)) > 0) {
        const int tiles = uniform(seg.t1 - seg.t0);
        if (!wait(&sh.q_ready, segs & 1, ab)) break;
        ++segs;
        for (int t = 0; t < tiles; ++t, ++k) {
          const int before = k - C::SBUF;         // the tile whose scores were here
          if (before >= 0 && !wait(&sh.s_empty[before & 1], (before >> 1) & 1, ab)) { ok = false; break; }
          const uint32_t d = ts + (C::SBUF == 2 ? (k & 1) * NS : 0);
          const int rope_slot = slot;
          if (p.DR && ++slot == ring) slot = 0;
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            if (c == 0 || c == HC) {
              if (!wait(&sh.full[half_barrier(2 * k) + (c == HC)], half_parity(2 * k), ab)) { ok = false; break; }
              ptx::tc_fence_after();
            }
            const uint32_t dk = dk0 + slot * (CHUNK >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f8<kSw128Hi, kSw128Hi>(d, dk + ((kk * 32) >> 4), dq + ((c * NS * 128 + kk * 32) >> 4), id_s,
                                         c + kk > 0);
            if (++slot == ring) slot = 0;
          }
          if (!ok) break;
          if (p.DR) {
            const uint32_t dk = dk0 + rope_slot * (CHUNK >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_half<kSw128Hi, kSw128Hi>(d, dk + ((kk * 32) >> 4), dqr + ((kk * 32) >> 4), id_r);
          }
          commit(&sh.s_full[k & 1]);
        }
      }
      if (*ab) {                                  // products in flight end before TMEM is freed
        commit(&sh.drain[0]);
        drain(&sh.drain[0], 0);
      }
      __syncwarp();
    } else if (warp == 11) {
      // ======== O^T += codes^T P^T
      constexpr uint32_t id_o = idesc(NO, true, true, kE4M3, kE5M2);
      const uint32_t dp = p_lo(ptx::smem_u32(p_s)), dk0 = sw128_lo(ptx::smem_u32(sm));
      const uint32_t to = (uint32_t)uniform((int)tmem);
      int k = 0, slot = 0;
      bool ok = true;
      Info seg;
      while (ok && uniform(take(seg, true)) > 0) {
        const int tiles = uniform(seg.t1 - seg.t0);
        for (int t = 0; t < tiles; ++t, ++k) {
          const int par = k & 1;
          if (!wait(&sh.p_full[par], (k >> 1) & 1, ab)) { ok = false; break; }
          ptx::tc_fence_after();
          if (p.DR && ++slot == ring) slot = 0;
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            const uint32_t dv = dk0 + slot * (CHUNK >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f8<kSw128Hi, kPHi>(to + c * NO, dv + ((kk * 4096) >> 4),
                                     dp + ((par * NO * 128 + kk * 512) >> 4), id_o, t > 0 || kk > 0);
            if (++slot == ring) slot = 0;
            if (c == HC - 1) commit(&sh.freed[half_barrier(2 * k)]);
          }
          commit(&sh.freed[half_barrier(2 * k + 1)]);
        }
      }
      if (*ab) {
        commit(&sh.drain[1]);
        drain(&sh.drain[1], 0);
      }
      __syncwarp();
    }
  } else {
    // ======== softmax: two groups of four warps have half of the rows each; thread =
    // position of the tile = TMEM lane
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    constexpr int HR = R / 2;                   // rows of a group
    const int wg = warp >> 2, rb = wg * HR;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int tt = tid & 127;
    int k = 0;
    bool failed = false;
    auto o_done = [&](int i) {                  // the products have read tile i
      return wait(&sh.freed[half_barrier(2 * i + 1)], half_parity(2 * i + 1), ab);
    };

    // ---- a segment's loads: the queries, the pages of this thread's first two positions
    constexpr int RW = R / 8;                   // rows of a warp: warp + 8 i
    uint2 raw[RW][NCH];                         // channels 128 c + 4 lane + j
    uint32_t raw_r[RW];                         // rope 2 lane + j
    // (a table entry as it is, so that nothing waits for it here; kNoPage: not needed)
    constexpr int kNoPage = -0x7fffffff;
    auto page_at = [&](const Info& sg, int t) {
      const int pos = t * TILE + tt, i = pos >> p.page_shift;
      int x = kNoPage;
      if (t < sg.t1 && pos < sg.seen) x = i < p.max_pages ? p.table[(int64_t)sg.b * p.table_s + i] : -1;
      return x;
    };
    int page_first = kNoPage, page_second = kNoPage;
    auto fetch = [&](const Info& sg) {
      const T *ql[RW], *qr[RW];
#pragma unroll
      for (int i = 0; i < RW; ++i) {            // (rows past the end: the last one's)
        const int row = sg.row0 + min(warp + 8 * i, sg.rows - 1), tok = div_heads(p, row);
        const int64_t n = sg.first + tok, h = row - tok * p.H;
        ql[i] = static_cast<const T*>(p.q_lat) + n * p.ql_s[0] + h * p.ql_s[1] + 4 * lane;
        qr[i] = static_cast<const T*>(p.q_rope) + n * p.qr_s[0] + h * p.qr_s[1] + 2 * lane;
        raw_r[i] = 0;
      }
      if (p.vec) {
#pragma unroll
        for (int i = 0; i < RW; ++i) {
#pragma unroll
          for (int c = 0; c < NCH; ++c) raw[i][c] = *reinterpret_cast<const uint2*>(ql[i] + c * 128);
          if (p.DR) raw_r[i] = *reinterpret_cast<const uint32_t*>(qr[i]);
        }
      } else {
        const auto bits = [](const T* q) { return (uint32_t)*reinterpret_cast<const uint16_t*>(q); };
#pragma unroll
        for (int i = 0; i < RW; ++i) {
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            const T* q = ql[i] + c * 128;
            raw[i][c] = make_uint2(bits(q) | bits(q + 1) << 16, bits(q + 2) | bits(q + 3) << 16);
          }
          if (p.DR) raw_r[i] = bits(qr[i]) | bits(qr[i] + 1) << 16;
        }
      }
      page_first = page_at(sg, sg.t0);
      page_second = page_at(sg, sg.t0 + 1);
    };
    // ---- its queries, scaled by a power of two and split into e4m3 terms (rows past
    // the end: zeros), and its rows' figures
    auto write_queries = [&](const Info& sg, Rows<R>& rw) {
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        const int r = warp + 8 * i;
        const bool live = r < sg.rows;
        float x[NCH][4], y[2];
        uint32_t amax = 0;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const T* v = reinterpret_cast<const T*>(&raw[i][c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[c][j] = live ? ld(v + j) : 0.f;
            amax = max(amax, abs_bits(x[c][j]));
          }
        }
        const T* v = reinterpret_cast<const T*>(&raw_r[i]);
        y[0] = live ? ld(v) : 0.f;
        y[1] = live ? ld(v + 1) : 0.f;
        const uint32_t rmax = max(abs_bits(y[0]), abs_bits(y[1]));
        const int e = scale_exp(warp_max_u32(amax), p.DR ? warp_max_u32(rmax) : 0);
        // half of what scale_exp allows: at most 224
        const float inv = 0.5f * pow2i(-e), inv8 = inv * (1.f / 256.f);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[c][j] *= inv8;
          uint32_t term[NQ];
          split_query<NQ>(x[c], term);
#pragma unroll
          for (int j = 0; j < NQ; ++j)
            *reinterpret_cast<uint32_t*>(q_s + c * NS * 128 + swz(j * R + r, 4 * lane)) = term[j];
        }
        if (p.DR) {
          T* d = reinterpret_cast<T*>(qr_s + swz(r, 4 * lane));
          st(d, y[0] * inv);
          st(d + 1, y[1] * inv);
        }
        if (lane == 0) {
          const int row = sg.row0 + min(r, sg.rows - 1), tok = div_heads(p, row);
          const int64_t n = sg.first + tok, h = row - tok * p.H;
          rw.q_scale[r] = 2.f * pow2i(e) * p.scale * kLog2e;
          rw.seen[r] = live ? max(0, min(sg.off + tok + 1, sg.seen)) : sg.seen;
          rw.m[r] = kUnset;
          rw.out[r] = n * p.o_s[0] + h * p.o_s[1];
          rw.lse[r] = n * p.lse_s + h;
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&sh.q_ready);
    };
    auto scale_at = [&](int t, int page) {
      if (page == kNoPage) return 1.f;
      if ((uint32_t)page >= (uint32_t)p.num_pages) {
        atomicExch(&g_attn_device_error, kErrOutside);
        return __uint_as_float(0x7fffffffu);
      }
      return p.scales[(int64_t)page * p.scales_s + ((t * TILE + tt) & (p.page_size - 1))];
    };

    // Each round: the next segment's loads, this segment's tiles, the next one's queries
    // (so that its scores are under way meanwhile), this one's result.
    Info seg, nseg;
    bool have = false;
    float s_first = 1.f;
    for (int si = 1;; ++si) {
      const int took = take(nseg, false);
      const bool have_next = took > 0;
      if (took < 0) failed = true;
      float s_next = s_first;
      int page_next = page_second;
      if (have_next) fetch(nseg);
      Rows<R>& rw = sh.rows[si & 1];
      const float *q_scale = rw.q_scale + rb, *m = rw.m + rb, *alpha = rw.alpha + rb;
      const int* sees = rw.seen + rb;
      float l[HR];
      if (have) {
        float ls_next = log2f(s_next), rs_next = s_next == s_next ? __frcp_rn(s_next) : 1.f;
#pragma unroll
        for (int r = 0; r < HR; ++r) l[r] = 0.f;
        ptx::tc_fence_before();
        bar_sync(3, 256);                         // the rows' figures are written, O has been read
        for (int t = seg.t0; t < seg.t1; ++t, ++k) {
          const int par = k & 1;
          const bool start = t == seg.t0;
          // log2 of the position's scale and its reciprocal (a NaN scale: NaN reaches
          // the sum through P, where the row sees the position)
          const float s = s_next, ls = ls_next, rs = rs_next;
          s_next = scale_at(t + 1, page_next);
          page_next = page_at(seg, t + 2);
          const int pos = t * TILE + tt;
          if (!wait(&sh.s_full[par], (k >> 1) & 1, ab)) failed = true;
          ptx::tc_fence_after();
          float a[HR];
          {
            float z[NQ * HR];
            const uint32_t at = tm_s + (C::SBUF == 2 ? par * NS : 0) + rb + lane_base;
#pragma unroll
            for (int j = 0; j < NQ; ++j) tmem_get<HR>(at + j * R, z + HR * j);
            ptx::tmem_wait_ld();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&sh.s_empty[par]);
#pragma unroll
            for (int r = 0; r < HR; ++r) a[r] = fmaf(join<NQ>(z + r, HR, kQFiner), q_scale[r] * s, ls);
          }
          if (t * TILE + TILE > seg.seen0) {      // some row does not see the whole tile
#pragma unroll
            for (int r = 0; r < HR; ++r)
              if (pos >= sees[r]) a[r] = -INFINITY;
          }
          // positions that nobody sees, or that are NaN as a whole, must not meet
          // a weight of zero: their codes become zeros
          if (wg == 0 && (pos >= seg.seen || s != s)) {
            int at = (int)(((int64_t)k * tile_chunks + tile_chunks - NCH) % ring);
#pragma unroll 1
            for (int c = 0; c < NCH; ++c) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(sm + at * CHUNK + tt * 128 + 16 * i) = make_uint4(0, 0, 0, 0);
              if (++at == ring) at = 0;
            }
          }
          float top = -INFINITY;
#pragma unroll
          for (int r = 0; r < HR; ++r) top = fmaxf(top, a[r] - m[r]);
          if (ptx::bar_red_or(1 + wg, 128, failed || top > kPTop)) {
            // a row outgrew P's range (or has its first position): new maxima, and O
            // follows once the products so far are in it
            if (*ab) failed = true;
#pragma unroll
            for (int r = 0; r < HR; ++r) {
              const float mx = warp_max(a[r]);
              if (lane == 0) sh.red[warp][r] = mx;
            }
            failed = ptx::bar_red_or(1 + wg, 128, failed);
            if (failed) break;
            if (tt < HR) {
              const float* red = &sh.red[4 * wg][tt];
              const float mx = fmaxf(fmaxf(red[0], red[HR]), fmaxf(red[2 * HR], red[3 * HR]));
              const float old = m[tt];
              const bool up = mx - old > kPTop;
              rw.alpha[rb + tt] = up ? ex2(old - (mx - BIAS)) : 1.f;
              if (up) rw.m[rb + tt] = mx - BIAS;
            }
            bar_sync(1 + wg, 128);
            if (!start) {
              if (!o_done(k - 1)) failed = true;
              ptx::tc_fence_after();
              float al[HR];
#pragma unroll
              for (int r = 0; r < HR; ++r) {
                al[r] = alpha[r];
                l[r] *= al[r];
              }
#pragma unroll 1
              for (int c = 0; c < NCH; ++c) {
                const uint32_t at = tmem + c * NO + rb + lane_base;
                float o[NP * HR];
#pragma unroll
                for (int j = 0; j < NP; ++j) tmem_get<HR>(at + j * R, o + HR * j);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < NP * HR; ++i) o[i] *= al[i % HR];
#pragma unroll
                for (int j = 0; j < NP; ++j) tmem_put<HR>(at + j * R, o + HR * j);
              }
              ptx::tmem_wait_st();
              ptx::tc_fence_before();
            }
          }
          // ---- P, once the buffer's last products have read it
          if (k > 1 && !o_done(k - 2)) failed = true;
          // (16 rows of a position are 16 bytes, 8 rows one half of them)
          uint8_t* pt = p_s + par * NO * 128 + tt * 16 + (HR == 8 ? wg * 8 : wg * (TILE * 16));
          uint32_t term[NP][HR / 4];
#pragma unroll
          for (int q = 0; q < HR / 4; ++q) {
            float e4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              e4[i] = ex2(a[4 * q + i] - m[4 * q + i]);
              l[4 * q + i] = fmaf(e4[i], rs, l[4 * q + i]);
            }
            uint32_t u[NP];
            split_weights(e4, u);
#pragma unroll
            for (int j = 0; j < NP; ++j) term[j][q] = u[j];
          }
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            uint8_t* d = pt + j * (R / 16) * (TILE * 16);
            if constexpr (HR == 16)
              *reinterpret_cast<uint4*>(d) = make_uint4(term[j][0], term[j][1], term[j][2], term[j][3]);
            else
              *reinterpret_cast<uint2*>(d) = make_uint2(term[j][0], term[j][1]);
          }
          ptx::fence_proxy_async_smem();
          ptx::mbar_arrive(&sh.p_full[par]);
          ls_next = log2f(s_next);
          rs_next = s_next == s_next ? __frcp_rn(s_next) : 1.f;
        }
      }
      failed = ptx::bar_red_or(3, 256, failed);  // the scores have all been read
      if (failed) break;
      if (have_next) {
        s_first = scale_at(nseg.t0, page_first);
        write_queries(nseg, sh.rows[(si + 1) & 1]);
      }
      if (have) {
        // ---- the segment's result
        const float sum = warp_sums<HR>(l, lane);
        if (lane < HR) sh.red[warp][lane] = sum;
        if (!failed && !o_done(k - 1)) failed = true;
        ptx::tc_fence_after();
        failed = ptx::bar_red_or(3, 256, failed);
        if (failed) break;
        const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
        const int slot = 2 * blockIdx.x + (seg.t0 > 0 ? 0 : 1);
        float inv = 0.f;                          // of row rb + lane
        if (lane < HR) {
          const float* red = &sh.red[4 * wg][lane];
          const float total = (red[0] + red[HR]) + (red[2 * HR] + red[3 * HR]);
          inv = total == 0.f ? 0.f : 1.f / total;
          if ((warp & 3) == 0 && rb + lane < seg.rows) {
            const float lse2 = total == 0.f ? -INFINITY : m[lane] + log2f(total);
            if (!whole) w.lse2[slot * R + rb + lane] = lse2;
            else if (p.lse) p.lse[rw.lse[rb + lane]] = lse2 * kLn2;
          }
        }
        const bool odd = lane & 1;
        float f[HR];
        T* dst[HR / 2];                           // neighbouring lanes swap a row each: four bytes a store
#pragma unroll
        for (int r = 0; r < HR; ++r) f[r] = __shfl_sync(0xffffffffu, inv, r);
#pragma unroll
        for (int r = 0; r < HR; r += 2)
          dst[r / 2] = static_cast<T*>(p.out) + rw.out[rb + r + odd] + (tt & ~1);
#pragma unroll 1
        for (int c = 0; c < NCH; ++c) {           // 128 channels of this group's rows
          float o[NP * HR];
#pragma unroll
          for (int j = 0; j < NP; ++j) tmem_get<HR>(tmem + c * NO + j * R + rb + lane_base, o + HR * j);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int r = 0; r < HR; ++r) o[r] = join<NP>(o + r, HR, kPFiner) * f[r];
          if (whole) {
#pragma unroll
            for (int r = 0; r < HR; r += 2) {
              const float other = __shfl_xor_sync(0xffffffffu, odd ? o[r] : o[r + 1], 1);
              T pair[2];
              st(pair, odd ? other : o[r]);
              st(pair + 1, odd ? o[r + 1] : other);
              if (rb + r + odd < seg.rows) {
                T* d = dst[r / 2] + c * 128;
                if (p.out_vec) {
                  *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(pair);
                } else {
                  d[0] = pair[0];
                  d[1] = pair[1];
                }
              }
            }
          } else {
            float* part = w.part + ((int64_t)slot * R + rb) * p.KVL + c * 128 + tt;
#pragma unroll
            for (int r = 0; r < HR; ++r)
              if (rb + r < seg.rows) part[r * p.KVL] = o[r];
          }
        }
      }
      if (!have_next) break;
      seg = nseg;
      have = true;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 9) {
    ptx::tmem_relinquish();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a group that several ranges share, in order: one block per
// (range that starts inside a group, row).  Two halves of the block take every second
// part each, eight loads in flight; every warp works the weights out for itself.  Bound
// by latency: the launch, a cut, the parts' sums, then the parts, one after the other;
// 3 us with 19 parts of 16 rows of 512.
constexpr int kJoinThreads = 256;

template <typename T, int R>
__global__ void __launch_bounds__(kJoinThreads)
cache_join_kernel(const CacheParams p, const Work w) {
  __shared__ float4 half[128];
  ptx::grid_dep_wait();
  const int c0 = blockIdx.x + 1, r = blockIdx.y;
  const Cut cut = w.cuts[c0];
  const int parts = cut.parts;
  if (parts == 0 || r >= cut.rows) return;
  const int tid = threadIdx.x, lane = tid & 31;
  // part 0: what range c0 - 1 left unfinished; part i: what range c0 + i - 1 begins with
  auto slot = [&](int i) { return (int64_t)(i == 0 ? 2 * (c0 - 1) + 1 : 2 * (c0 + i - 1)) * R + r; };
  const int ch = 4 * (tid & 127), h0 = tid >> 7;
  const bool live = ch < p.KVL;
  float4 x[8];
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (live && h0 + 2 * u < parts)
      x[u] = *reinterpret_cast<const float4*>(w.part + slot(h0 + 2 * u) * p.KVL + ch);
  float mx = -INFINITY;
  for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, w.lse2[slot(i)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float m = mx == -INFINITY ? 0.f : mx;
  float tot = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < parts; i0 += 32) {     // lane i: the weight of part i0 + i
    const float weight = i0 + lane < parts ? exp2f(w.lse2[slot(i0 + lane)] - m) : 0.f;
    tot += weight;
#pragma unroll
    for (int j0 = 0; j0 < 32; j0 += 16) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = i0 + j0 + h0 + 2 * u;
        const float f = __shfl_sync(0xffffffffu, weight, j0 + h0 + 2 * u);
        if (live && j < parts) {
          acc.x = fmaf(f, x[u].x, acc.x);
          acc.y = fmaf(f, x[u].y, acc.y);
          acc.z = fmaf(f, x[u].z, acc.z);
          acc.w = fmaf(f, x[u].w, acc.w);
          if (j + 16 < parts) x[u] = *reinterpret_cast<const float4*>(w.part + slot(j + 16) * p.KVL + ch);
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
  if (h0 == 1) half[tid & 127] = acc;
  __syncthreads();
  const int row = cut.row0 + r, tok = div_heads(p, row);
  const int64_t n = cut.first + tok, h = row - tok * p.H;
  const float inv = tot == 0.f ? 0.f : 1.f / tot;
  if (h0 == 0 && live) {
    const float4 b = half[tid];
    T* o = static_cast<T*>(p.out) + n * p.o_s[0] + h * p.o_s[1] + ch;
    st(o, (acc.x + b.x) * inv);
    st(o + 1, (acc.y + b.y) * inv);
    st(o + 2, (acc.z + b.z) * inv);
    st(o + 3, (acc.w + b.w) * inv);
  }
  if (tid == 0 && p.lse)
    p.lse[n * p.lse_s + h] = tot == 0.f ? -INFINITY : (m + log2f(tot)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int device_sms() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 1 ? min(n, kMaxRanges) : 2;
}
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

int q_terms(int io_dtype) {
  return io_dtype == KDA_DTYPE_F16 ? kQTerms<__half> : kQTerms<__nv_bfloat16>;
}

// Contexts that a block goes through about as fast as it would join parts of them stay
// whole: no workspace and no second launch.  Up to 4 tiles (one token for each of B
// sequences of 512, 16 heads, KVL 512; whole and split, us): B = 1 11.7 and 11.8, B = 16
// 12.3 and 13.7; at 768 14.5 and 11.9, 15.1 and 14.8.  Up to 8 tiles where 64 groups or
// more occupy the SMs anyhow: B = 64 at 1024 19.0 and 23.5, at 2048 30.6 and 28.5.  (Not
// swept at other widths.)
bool whole_groups(const CacheParams& p, int R) {
  const int64_t groups = max((int64_t)min(p.B, p.N), (int64_t)p.N * p.H / R);
  return (int64_t)p.max_pages * p.page_size <= (groups >= 64 ? 8 : 4) * TILE;
}

// Rows per group: 16 where the sequences of the call have no more rows than that on
// average, or where 32 rows leave too small a ring; else 32.  (16 sequences of 4096, 16
// and 32 rows a group, us: 16 rows a sequence 18.5 and 22.9, 32 rows 25.0 and 25.6, 48
// rows 37.0 and 32.9; 128 tokens of one prompt 64.9 and 50.0; KVL 512, other widths were not
// swept.)
int rows_per_group(const CacheParams& p, int q_terms) {
  if ((int64_t)p.N * p.H <= (int64_t)p.B * 16) return 16;
  return ring_chunks(p.KVL, p.DR, q_terms, 32) >= 2 * tile_chunks(p.KVL, p.DR) ? 32 : 16;
}

template <typename T, int R, int NCH>
cudaError_t launch(const CacheParams& p, Work w, const CUtensorMap& mc, const CUtensorMap& mr,
                   int ranges, cudaStream_t s) {
  using C = Cfg<T, R, NCH>;
  auto k = cache_attn_kernel<T, R, NCH>;
  w.ring = ring_chunks(p.KVL, p.DR, C::NQ, R);
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
  if (e != cudaSuccess) return e;
  const size_t smem = fixed_bytes(p.KVL, C::NQ, R) + w.ring * CHUNK;
  e = launch_dependent(k, dim3(ranges), kThreads, smem, s, p, w, mc, mr);
  if (e != cudaSuccess || w.whole) return e;
  return launch_dependent(cache_join_kernel<T, R>, dim3(ranges - 1, R), kJoinThreads, 0, s, p, w);
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
size_t attention_workspace_bytes(const CacheParams& p, int io_dtype) {
  const size_t ranges = device_sms(), R = rows_per_group(p, q_terms(io_dtype));
  if (whole_groups(p, (int)R)) return 0;
  return align256(2 * ranges * R * p.KVL * 4) + align256(2 * ranges * R * 4) +
         align256(ranges * sizeof(Cut));
}

cudaError_t launch_attention(const CacheParams& p, int io_dtype, void* workspace, cudaStream_t s) {
  const int ranges = device_sms();
  const int R = rows_per_group(p, q_terms(io_dtype));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Work w{};
  w.whole = whole_groups(p, R);
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
