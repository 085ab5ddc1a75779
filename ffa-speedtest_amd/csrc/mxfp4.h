// The MXFP4 format of the cache that holds keys and values in 4 bits: e2m1 codes and one power of two per 32 channels
// of a token, value = level * 2^(byte - 127).  The byte is kept in 105 .. 140 (2^-22 .. 2^13): every value is then exact
// in fp16 and bf16 (0.5 * 2^-22 is an fp16 subnormal, 6 * 2^13 = 49152), so that neither reading the cache back nor the
// matrix operands round.  255 stands for a block with an infinity or NaN in it; its codes are 0 and its values NaN.
//
// A (page, KV head) block of 64 tokens, in the order of the matrix operands (paged_attend.h):
//   K codes   [4 tiles tau][4 blocks kc][16 rows m][16 bytes]     token 4 m + tau, channels 32 kc + (0..31)
//   V codes   [4 i][4 g][16 n][2 h][8 bytes]                      channel 32 i + 16 h + n, tokens 16 g + (0..15)
//   scales    [4 blocks of 32 channels][64 tokens], K and V
// A byte holds two channels of a token (K) or two tokens of a channel (V), the first in its low half.
#pragma once

#include "decode_common.h"

namespace ffa {

constexpr int kMxLow = 105, kMxHigh = 140, kMxNan = 255;
constexpr int kMxCodes = 4096, kMxScales = 256;  // bytes of a (page, KV head) block

// byte offset of channels 8 j .. 8 j + 7 of token t among the K codes
__host__ __device__ constexpr uint32_t mx_k_off(int t, int j) {
  return (uint32_t)(((t & 3) * 64 + (j >> 2) * 16 + (t >> 2)) * 16 + (j & 3) * 4);
}
// byte offset of channel c, tokens t and t ^ 1, among the V codes
__host__ __device__ constexpr uint32_t mx_v_off(int c, int t) {
  return (uint32_t)(((c >> 5) * 64 + (t >> 4) * 16 + (c & 15)) * 16 + ((c >> 4) & 1) * 8 + ((t & 15) >> 1));
}

// The scale's byte for a block whose largest magnitude has the bits `top`: the smallest power of two of which it is at
// most seven (six is the largest level: what saturates is off by at most half a step).
__device__ __forceinline__ int mx_scale(uint32_t top) {
  const int e = (int)((top + 0x1fffffu) >> 23) - 2;  // mantissas above 1.75 carry
  return top >= 0x7f800000u ? kMxNan : min(max(e, kMxLow), kMxHigh);
}
__device__ __forceinline__ float mx_factor(int byte) { return __uint_as_float((uint32_t)byte << 23); }  // 255: an infinity
__device__ __forceinline__ float mx_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// Eight values to codes, the first in the lowest nibble: to nearest, ties to the even code, saturating
__device__ __forceinline__ uint32_t mx_codes8(const float *x, int byte) {
  const float s = mx_factor(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return byte == kMxNan ? 0u : w;
}
// Eight codes to values, times s
__device__ __forceinline__ void mx_values8(uint32_t w, float s, float *x) {
  const f32x2 c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3)};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = c[i >> 1][i & 1] * s;
}
// Eight codes to an fp16 operand, times the power of two s (a NaN where s is an infinity)
__device__ __forceinline__ f16x8 mx_operand(uint32_t w, float s) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1),
           c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// the same with a factor for each of the eight besides: fp16 pairs, normal numbers, as are the eight times s; products within fp16
__device__ __forceinline__ f16x8 mx_operand(uint32_t w, float s, const f16x2 *f) {
  const f16x8 x = mx_operand(w, s);
  const f16x2 a = f16x2{x[0], x[1]} * f[0], b = f16x2{x[2], x[3]} * f[1], c = f16x2{x[4], x[5]} * f[2], d = f16x2{x[6], x[7]} * f[3];
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// the same with the factors given as bytes of `s`
__device__ __forceinline__ f16x8 mx_operand(uint32_t w, uint2 s) {
  float x[8];
  mx_values8(w, 1.f, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= mx_factor(((i < 4 ? s.x : s.y) >> (8 * (i & 3))) & 0xffu);
  const u32x4 o = {pk_f16_bits(x[0], x[1]), pk_f16_bits(x[2], x[3]), pk_f16_bits(x[4], x[5]), pk_f16_bits(x[6], x[7])};
  return __builtin_bit_cast(f16x8, o);
}

}  // namespace ffa
