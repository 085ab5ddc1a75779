// Rotary positions with several axes: what the rotation of given rows and the mxfp4 append share.
//
// Eight lanes hold a row of 128 channels: lane l the channels 8 l .. 8 l + 7 (x[0..7]) and 64 + 8 l .. (x[8..15]), two
// loads of 16 bytes (fp32: four) that are whole 128-byte lines for the eight.  Both channels of a pair are then in one
// lane, whether pairs are (j, j + 64) or (2 j, 2 j + 1), and so is a quantizer's block of 32 in four lanes.
// Sines and cosines of a token are computed once for all of its heads, into LDS.
#pragma once

#include "ffa_mi355x.h"
#include "mxfp4.h"

namespace ffa {

constexpr long kMostWorkgroups = (1l << 24) - 1;  // workgroups of 256 threads in a dimension: fewer than 2^32 threads
enum { kTurnNone = 0, kTurnHalf = 1, kTurnAdjacent = 2 };

struct RopeParams {
  const ffa_rope_pair *pairs;
  const void *positions;  // nullptr: the token's position in its sequence
  long pos_axis, pos_batch;
  int positions64, axes, inverse;
};

// cos and sin of 2 pi r, |r| <= 1/2, each within 2^-40 before its rounding to fp32: the remainder from the next quarter turn
// (|x| <= pi / 4) by the Taylor sums, whose first terms left out are x^15 / 15! < 2^-45 and x^16 / 16! < 2^-49.
__device__ __forceinline__ float2 cos_sin_turns(double r) {
  const double k = rint(4.0 * r), x = (r - 0.25 * k) * 6.283185307179586476925287, y = x * x;
  double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;
  s = fma(s, y, -1.0 / 39916800.0);
  s = fma(s, y, 1.0 / 362880.0);
  s = fma(s, y, -1.0 / 5040.0);
  s = fma(s, y, 1.0 / 120.0);
  s = fma(s, y, -1.0 / 6.0);
  s = fma(s * y, x, x);
  c = fma(c, y, 1.0 / 479001600.0);
  c = fma(c, y, -1.0 / 3628800.0);
  c = fma(c, y, 1.0 / 40320.0);
  c = fma(c, y, -1.0 / 720.0);
  c = fma(c, y, 1.0 / 24.0);
  c = fma(c, y, -0.5);
  c = fma(c, y, 1.0);
  const int q = (int)k & 3;
  const float fc = (float)c, fs = (float)s, a = q & 1 ? fs : fc, b = q & 1 ? fc : fs;  // (c, s) (-s, c) (-c, -s) (s, -c)
  return make_float2(q == 1 || q == 2 ? -a : a, q & 2 ? -b : b);
}

// cos and sin of pair j of token t of sequence b (own: its position there).  All of it in 64 bits up to the one rounding: at
// position 2^20 the product in turns is off by 2^-33, where 32 bits would be by 2^-4.
__device__ __forceinline__ float2 rope_angle(const RopeParams &p, int j, int b, int t, long own) {
  const ffa_rope_pair pr = p.pairs[j];
  long pos = own;
  if (p.positions) {
    const long axis = (unsigned long)pr.axis < (unsigned long)p.axes ? pr.axis : 0;
    const long at = axis * p.pos_axis + b * p.pos_batch + t;
    pos = p.positions64 ? ((const int64_t *)p.positions)[at] : ((const int32_t *)p.positions)[at];
  }
  const double a = (double)pos * pr.turns;
  const float2 f = cos_sin_turns(a - rint(a));
  return make_float2(f.x, p.inverse ? -f.y : f.y);
}

// x of lane l turned by the token's cos and sin cs[64].  Two products and their sum, each rounded: a fused sum would keep
// one of the products exact, and the codes of what is quantized next would depend on which.  It takes no longer.
__device__ __forceinline__ void turn_pair(float2 f, float &a, float &b) {
#pragma clang fp contract(off)
  const float ac = a * f.x, bs = b * f.y, bc = b * f.x, as = a * f.y;
  a = ac - bs;
  b = bc + as;
}
template <int TURN>
__device__ __forceinline__ void rope_turn(const float2 *cs, int l, float *x) {
  if constexpr (TURN == kTurnHalf) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn_pair(cs[8 * l + i], x[i], x[8 + i]);
  } else if constexpr (TURN == kTurnAdjacent) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) turn_pair(cs[32 * h + 4 * l + i], x[8 * h + 2 * i], x[8 * h + 2 * i + 1]);
  }
}

// N (4 or 8) values to elements `at` .. of p, of type DT.  NT: not kept in the caches, as nothing reads them soon (a 16K
// prompt's append 95 -> 93 us, read-backs 132 -> 124; but its V's values, 8 bytes a lane, so 89 -> 94)
template <int DT, int N, bool NT = true>
__device__ __forceinline__ void store_values(void *p, size_t at, const float *x) {
  typedef uint32_t Words __attribute__((ext_vector_type(DT != 2 && N == 4 ? 2 : 4)));
  constexpr int kPer = DT == 2 ? 1 : 2, kWords = DT != 2 && N == 4 ? 2 : 4;  // values a word, words a store
  Words *d = (Words *)((uint8_t *)p + at * (DT == 2 ? 4 : 2));
#pragma unroll
  for (int i = 0; i < N / (kPer * kWords); ++i) {
    Words w;
#pragma unroll
    for (int e = 0; e < kWords; ++e) {
      const float *y = x + (i * kWords + e) * kPer;
      w[e] = DT == 2 ? __float_as_uint(y[0]) : (DT == 1 ? pk_bf16_bits(y[0], y[kPer - 1]) : pk_f16_bits(y[0], y[kPer - 1]));
    }
    if constexpr (NT) __builtin_nontemporal_store(w, d + i);
    else d[i] = w;
  }
}

// lane l's sixteen channels of the row at element `at`
template <int DT>
struct Row16 {
  Raw8<DT> a, b;
};
template <int DT>
__device__ __forceinline__ Row16<DT> load_row(const void *p, long at, int l) {
  return Row16<DT>{load8<DT>(p, (size_t)(at + 8 * l)), load8<DT>(p, (size_t)(at + 64 + 8 * l))};
}
template <int DT>
__device__ __forceinline__ void row_values(const Row16<DT> &r, float *x) {
  raw8_to_f32<DT>(r.a, x);
  raw8_to_f32<DT>(r.b, x + 8);
}
template <int DT>
__device__ __forceinline__ void store_row(void *p, long at, int l, const float *x) {
  store_values<DT, 8>(p, (size_t)(at + 8 * l), x);
  store_values<DT, 8>(p, (size_t)(at + 64 + 8 * l), x + 8);
}

}  // namespace ffa
