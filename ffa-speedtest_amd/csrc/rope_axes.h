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

enum { kTurnNone = 0, kTurnHalf = 1, kTurnAdjacent = 2 };

struct RopeParams {
  const ffa_rope_pair *pairs;
  const void *positions;  // nullptr: the token's position in its sequence
  long pos_axis, pos_batch;
  int positions64, axes, inverse;
};

// cos and sin of pair j of token t of sequence b (own: its position there).  The product in turns, in 64 bits: at
// position 2^20 it is off by 2^-33 turns, where 32 bits would be by 2^-4; then the remainder in 32.
__device__ __forceinline__ float2 rope_angle(const RopeParams &p, int j, int b, int t, long own) {
  const ffa_rope_pair pr = p.pairs[j];
  long pos = own;
  if (p.positions) {
    const long axis = (unsigned long)pr.axis < (unsigned long)p.axes ? pr.axis : 0;
    const long at = axis * p.pos_axis + b * p.pos_batch + t;
    pos = p.positions64 ? ((const int64_t *)p.positions)[at] : ((const int32_t *)p.positions)[at];
  }
  const double a = (double)pos * pr.turns;
  float s, c;
  sincospif(2.f * (float)(a - rint(a)), &s, &c);
  return make_float2(c, p.inverse ? -s : s);
}

// x of lane l turned by the token's cos and sin cs[64]
template <int TURN>
__device__ __forceinline__ void rope_turn(const float2 *cs, int l, float *x) {
  if constexpr (TURN == kTurnHalf) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = cs[8 * l + i];
      const float a = x[i], b = x[8 + i];
      x[i] = __builtin_fmaf(a, f.x, -b * f.y);
      x[8 + i] = __builtin_fmaf(b, f.x, a * f.y);
    }
  } else if constexpr (TURN == kTurnAdjacent) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = cs[32 * h + 4 * l + i];
        const float a = x[8 * h + 2 * i], b = x[8 * h + 2 * i + 1];
        x[8 * h + 2 * i] = __builtin_fmaf(a, f.x, -b * f.y);
        x[8 * h + 2 * i + 1] = __builtin_fmaf(b, f.x, a * f.y);
      }
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
