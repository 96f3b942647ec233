// kda_scan.cuh -- gated linear recurrence: parameters, and the arithmetic of its decays.
//
// A decay a = exp(g) close to one is held as a - 1: rounding a itself to 24 bits
// would be off by up to 2^-25 per token, always to the same side for a steady g, which a
// state that remembers n tokens adds up to n 2^-25.  One register holds either form,
// told apart by its sign bit:
//   sign set    a = 1 + r,  r in (-1, -0]
//   sign clear  a = r
// so that a h is h + r h or r h, one rounding more than a product.
#pragma once

#include "kda_internal.cuh"

namespace kda {
namespace scan {

constexpr int kErrSlot = 8;       // device error word: a step's slot past the pool
constexpr int kTile = 64;         // tokens between two checkpoints of the state

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
  // step
  const int* slots; int num_states; bool scatter;
};

// exp(g) in the form above.  From -1/4 to 0: g (1 + g/2! + ... + g^6/7!), the series of
// exp(g) - 1, whose first term left out is 2^-29 of the sum.
__device__ __forceinline__ float decay(float g) {
  float p = fmaf(g, 1.f / 5040.f, 1.f / 720.f);
  p = fmaf(p, g, 1.f / 120.f);
  p = fmaf(p, g, 1.f / 24.f);
  p = fmaf(p, g, 1.f / 6.f);
  p = fmaf(p, g, 0.5f);
  p = fmaf(p, g, 1.f);
  const float near = __uint_as_float(__float_as_uint(g * p) | 0x80000000u);
  return g <= 0.f && g > -0.25f ? near : expf(g);
}
__device__ __forceinline__ bool is_near(float r) { return __float_as_int(r) < 0; }
// a h + b
__device__ __forceinline__ float apply(float r, float h, float b) {
  return fmaf(r, h, is_near(r) ? h + b : b);
}
// a v
__device__ __forceinline__ float times(float r, float v) {
  return is_near(r) ? fmaf(r, v, v) : r * v;
}
// 1 - a
__device__ __forceinline__ float rest(float r) { return is_near(r) ? -r : 1.f - r; }

// Rows of sequence b of a packed batch, inside 0 .. T whatever q_start holds.
__device__ __forceinline__ void owned_rows(const ScanParams& p, int b, int& first, int& last) {
  first = min(max(p.q_start[b], 0), p.T);
  last = min(max(p.q_start[b + 1], first), p.T);
}

}  // namespace scan
}  // namespace kda
