// Exact attention of L query tokens per sequence over the paged quantized caches, and the same for groups of
// sequences that share leading pages.
//
// Row (b, i, h) is query token i of sequence b at head h.  It sees the keys t < lim = len_b - qlen_b + i + 1 and
//   out = sum_t p_t v_t / sum_t p_t,   p_t = 2^(s_t - m),   s_t = scale log2(e) q . k_t,   m + 8 <= max s_t <= m + 15,
// one pass over the pages with a running m; k = code * scale + zero + residual (2-bit), level * scale + residual
// (nvfp4, nf4) in fp32, rounded once to the fp16 matrix operand.  Partial results (m, sum p, sum p v) of page ranges
// are fp32 and joined by q's row afterwards; a call whose rows each have one range writes the output directly.
//
// The pools' order is the order of the matrix operands: with S^T = K Q^T (16x16x32 f16), the A operand of tile tau
// (tokens 4 m + tau, m = 0..15) is what lane (kc, m) loads, and the four tiles' results in lane (g, n) are the 16
// consecutive tokens 16 g .. 16 g + 15 of query row n: with O^T = V^T P^T those are the B operand, V^T's blocks the A
// operand, and each lane's results belong to its own row n again, whose m and sum it holds.  No value of S, P or O
// changes lanes.
#pragma once

#include "decode_common.h"
#include "ffa_mi355x.h"
#include "routes.h"

#include <type_traits>

namespace ffa {

enum { kFmtQ2 = 0, kFmtNvfp4 = 1, kFmtNf4 = 2 };
constexpr float kNoMax = -1e30f;  // m of a row that has seen no key: below every score, and 2^(x - m) stays defined
constexpr float kLeast = 0x1p-126f;  // least factor of a joined sum: an infinity times it stays one (times 0: NaN)
// m lies kHead log2 units below the largest score when it is set, and may lag it by kStale more: p <= 2^15 fits the fp16
// operand, whose steps of 2^-24 below 2^-14 are then at most 2^-32 of the largest weight.  (With kHead 0 they were up to
// 2^-24 of it and smaller weights were lost: of 3300 tokens of 2^-25.7 each, 5.87e-5 together, 5.1e-5 came out.)
constexpr float kHead = 8.f, kStale = 7.f;

struct AttendParams {
  const void *q;
  const uint8_t *k;
  const uint8_t *ks;
  const uint8_t *kz;
  const uint8_t *kr;
  const uint8_t *v;
  const int32_t *bt;
  const int32_t *seq_lens, *q_lens;
  const int32_t *group_start, *group_pages, *seq_group;
  void *out;
  float *part_ml, *part_o;  // [rows][nslots][2], [rows][nslots][128]
  int bt_stride, num_pages, ngroups;
  int B, T, L, HQ, HKV, G;
  int q_bf16, out_bf16;
  float scale2;
  int nslots;  // partials per row, 0: one page range per row, written to out
  // sets of a launch: z < nshared are groups over their shared pages, then (from b = 0) sequences over their own
  int nshared;
  int shared_slots, shared_ppw, own_slots;
  int shared_blocks, shared_wgs;  // of the launch of both kinds
};

__device__ __forceinline__ int seq_len_of(const AttendParams &p, int b) {
  return p.seq_lens ? min(max(p.seq_lens[b], 0), p.T) : p.T;
}
// pages of sequence b that its group shares (0 without groups)
__device__ __forceinline__ int shared_pages_of(const AttendParams &p, int b) {
  if (p.ngroups == 0) return 0;
  const int g = p.seq_group[b];
  return (unsigned)g < (unsigned)p.ngroups ? min(max(p.group_pages[g], 0), p.bt_stride) : 0;
}
// pages per range of a sequence with so many own pages: its ranges divide them (a call's T may be far above its length),
// a page for each of four waves at least
__device__ __forceinline__ int own_range(const AttendParams &p, int pages) {
  return max((pages + 4 * p.own_slots - 1) / (4 * p.own_slots), 1) * 4;
}
// keys that query token i of sequence b sees: positions below this
__device__ __forceinline__ int row_limit(const AttendParams &p, int b, int i) {
  const int len = seq_len_of(p, b);
  const int ql = p.q_lens ? min(max(p.q_lens[b], 0), p.L) : p.L;
  return i < ql ? max(len - ql + i + 1, 0) : 0;
}

// The rows and pages of a workgroup: sequences b0 .. b0 + n - 1 (a group's, over the shared pages; or one, over its
// own), pages [p0, p1) of the block-table row of b0; the slot of the partials.
struct AttendSet {
  int b0, n, p0, p1, slot;
};
// the range `split` of set z, and the slot of its partials
__device__ __forceinline__ AttendSet attend_set(const AttendParams &p, int z, int split) {
  AttendSet s;
  int ppw;
  if (z < p.nshared) {
    s.b0 = min(max(p.group_start[z], 0), p.B);
    s.n = max(min(p.group_start[z + 1], p.B) - s.b0, 0);
    s.p0 = 0;
    s.p1 = min(max(p.group_pages[z], 0), p.bt_stride);
    ppw = p.shared_ppw;
    s.slot = split;
  } else {
    s.b0 = z - p.nshared;
    s.n = 1;
    s.p0 = shared_pages_of(p, s.b0);
    s.p1 = (seq_len_of(p, s.b0) + kPage - 1) / kPage;
    ppw = own_range(p, s.p1 - s.p0);
    s.slot = p.shared_slots + split;
  }
  s.p0 += split * ppw;
  s.p1 = min(s.p0 + ppw, s.p1);
  return s;
}

// ---------------------------------------------------------------------------
// K of one (page, KV head): what lane (kc, m) loads, and its operands
// ---------------------------------------------------------------------------
// 16 bytes of a page that one workgroup reads once (non-temporal: 16 x 8K-64K tokens 394 -> 354 us; not the codes', whose
// hint cost 1-3 %)
__device__ __forceinline__ uint4 load_once(const uint4 *p) {
  const u32x4 w = __builtin_nontemporal_load((const u32x4 *)p);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int FMT, int RES>
struct KRaw {
  uint4 code[FMT == kFmtQ2 ? 2 : 4];
  uint4 res[RES == kResNone ? 1 : 8];
  uint16_t s[4], z[FMT == kFmtQ2 ? 4 : 1];
};

template <int FMT, int RES>
__device__ __forceinline__ void load_k(const AttendParams &p, size_t blk, int lane, KRaw<FMT, RES> &r) {
  const int kc = lane >> 4, m = lane & 15;
  if constexpr (FMT == kFmtQ2) {
    const uint4 *c = (const uint4 *)(p.k + blk * 2048);
    r.code[0] = c[lane];
    r.code[1] = c[64 + lane];
    const uint16_t *s = (const uint16_t *)(p.ks + blk * 512), *z = (const uint16_t *)(p.kz + blk * 512);
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      const int at = (((tau >> 1) * 4 + kc) * 4 + (m >> 2)) * 8 + 4 * (tau & 1) + (m & 3);
      r.s[tau] = s[at];
      r.z[tau] = z[at];
    }
  } else {
    const uint4 *c = (const uint4 *)(p.k + blk * 4096);
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      r.code[tau] = c[64 * tau + lane];
      if constexpr (FMT == kFmtNvfp4) r.s[tau] = ((const uint16_t *)(p.ks + blk * 512))[(4 * m + tau) * 4 + kc];
      else r.s[tau] = ((const uint16_t *)(p.ks + blk * 256))[(4 * m + tau) * 2 + (kc >> 1)];
    }
  }
  if constexpr (RES != kResNone) {
    const uint4 *c = (const uint4 *)(p.kr + blk * 8192);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.res[i] = load_once(c + 64 * i + lane);
  }
}

template <bool E4M3, bool HI>
__device__ __forceinline__ f32x2 fp8_pair(uint32_t w) {
  if constexpr (E4M3) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, 1.0f, HI);
  else return __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w, 1.0f, HI);
}

// Two operands: channels 32 kc + 16 h + (0..7) and + (8..15) of a token, in fp32 arithmetic with one rounding.
// q2: c0 holds the 16 codes; 4-bit: c0 and c1 8 codes each.  s: the scale of these channels, z the zero point (q2).
template <int FMT, int RES>
__device__ __forceinline__ void k_half(uint32_t c0, uint32_t c1, float s, float z, uint4 rw, const float2 *nf4, f16x8 *op) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float k[8];
    f32x2 res[4];
    if constexpr (RES != kResNone) {
      const uint32_t lo = e ? rw.z : rw.x, hi = e ? rw.w : rw.y;
      res[0] = fp8_pair<RES == kResE4M3, false>(lo);
      res[1] = fp8_pair<RES == kResE4M3, true>(lo);
      res[2] = fp8_pair<RES == kResE4M3, false>(hi);
      res[3] = fp8_pair<RES == kResE4M3, true>(hi);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) res[i] = f32x2{0.f, 0.f};
    }
    if constexpr (FMT == kFmtQ2) {
      // a 2-bit code as a nibble is the e2m1 value c / 2: the conversion with scale 2 gives codes 4 i, 4 i + 2 of
      // byte i, and of the word shifted by one code 4 i + 1, 4 i + 3
      const uint32_t a = c0 & 0x33333333u, b = (c0 >> 2) & 0x33333333u;
      f32x2 a0, a1, b0, b1;
      if (e) {
        a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 2.0f, 2);
        a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 2.0f, 3);
        b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 2.0f, 2);
        b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 2.0f, 3);
      } else {
        a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 2.0f, 0);
        a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 2.0f, 1);
        b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 2.0f, 0);
        b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 2.0f, 1);
      }
      const float c[8] = {a0[0], b0[0], a0[1], b0[1], a1[0], b1[0], a1[1], b1[1]};
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = __builtin_fmaf(c[i], s, z) + res[i >> 1][i & 1];
    } else if constexpr (FMT == kFmtNvfp4) {
      const uint32_t w = e ? c1 : c0;
      const f32x2 c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3)};
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = __builtin_fmaf(c[i >> 1][i & 1], s, res[i >> 1][i & 1]);
    } else {
      const uint32_t w = e ? c1 : c0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 c = nf4[(w >> (8 * i)) & 0xffu];
        k[2 * i] = __builtin_fmaf(c.x, s, res[i][0]);
        k[2 * i + 1] = __builtin_fmaf(c.y, s, res[i][1]);
      }
    }
    const u32x4 w = {pk_f16_bits(k[0], k[1]), pk_f16_bits(k[2], k[3]), pk_f16_bits(k[4], k[5]), pk_f16_bits(k[6], k[7])};
    op[e] = __builtin_bit_cast(f16x8, w);
  }
}

// Operands e = 0..3 of tile tau: channels 32 kc + 8 e + (0..7) of token 4 m + tau
template <int FMT, int RES>
__device__ __forceinline__ void k_operands(const KRaw<FMT, RES> &r, int tau, const float2 *nf4, f16x8 *op) {
  float s[2], z = 0.f;
  if constexpr (FMT == kFmtNvfp4) {
    const f32x2 w = fp8_pair<true, false>(r.s[tau]);
    s[0] = w[0];
    s[1] = w[1];
  } else {
    s[0] = s[1] = f16_bits_to_f32(r.s[tau]);
    if constexpr (FMT == kFmtQ2) z = f16_bits_to_f32(r.z[tau]);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t c0, c1 = 0;
    if constexpr (FMT == kFmtQ2) {
      const uint4 c = r.code[tau >> 1];
      c0 = h ? (tau & 1 ? c.w : c.y) : (tau & 1 ? c.z : c.x);
    } else {
      c0 = h ? r.code[tau].z : r.code[tau].x;
      c1 = h ? r.code[tau].w : r.code[tau].y;
    }
    k_half<FMT, RES>(c0, c1, s[h], z, r.res[RES == kResNone ? 0 : 2 * tau + h], nf4, op + 2 * h);
  }
}

// ---------------------------------------------------------------------------
// q of one row tile as the B operands, each row divided by a power of two that brings its largest element into
// [1, 2): every bf16 row fits fp16 that way (elements below 2^-14 of the row's largest lose bits that its scores,
// rounded at 2^-24 of the sum, do not hold).  cs: the row's factor back to log2-scaled scores.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load_q(const AttendParams &p, size_t row, bool ok, int kc, f16x8 *op, float &cs) {
  float x[32];
  const uint4 *src = (const uint4 *)((const uint16_t *)p.q + row * kD + 32 * kc);
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint4 w = ok ? src[e] : make_uint4(0, 0, 0, 0);
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[8 * e + 2 * i] = p.q_bf16 ? __uint_as_float(ww[i] << 16) : f16_bits_to_f32(ww[i] & 0xffffu);
      x[8 * e + 2 * i + 1] = p.q_bf16 ? __uint_as_float(ww[i] & 0xffff0000u) : f16_bits_to_f32(ww[i] >> 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[8 * e + i]));
  }
  top = xor_max(top, 16);
  top = xor_max(top, 32);
  int ex = (int)((__float_as_uint(top) >> 23) & 0xffu);  // 0: all zero or tiny; 255: an infinity
  ex = ex == 255 ? 127 : min(max(ex, 1), 253);
  float f = __uint_as_float((uint32_t)(254 - ex) << 23);
  cs = p.scale2 * __uint_as_float((uint32_t)ex << 23);
  if (cs < 0.f) f = -f;  // a negative scale: into q, so that the largest product is the largest score
  cs = fmaxf(fabsf(cs), 1e-37f);  // above 0: a hidden key's product of -inf stays -inf
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pk_f16_bits(x[8 * e + 2 * i] * f, x[8 * e + 2 * i + 1] * f);
    op[e] = __builtin_bit_cast(f16x8, w);
  }
}

// V words (8 tokens of a column) with infinities and NaN taken out; `bad` becomes non-zero where there were any.
// A product with them would give 0 * inf, a NaN, to the rows that do not see them; add_not_finite puts them back.
__device__ __forceinline__ u32x4 finite8(u32x4 w, uint32_t &bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = ((w[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;  // top bit of a half: all exponent bits set
    bad |= x;
    w[i] &= ~((x >> 15) * 0xffffu);
  }
  return w;
}

// infinities and NaN of V at tokens that the lane's row sees, into its columns 16 u + 4 g + (0..3): whatever the
// weight (above zero), they make the result what they are
template <int VT>
__device__ __forceinline__ void add_not_finite(const uint8_t *v, int g, int nvis, f32x4 *o) {
#pragma unroll 1
  for (int t = 0; t < nvis && t < kPage; ++t)
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = ((const uint16_t *)v)[vt_off(16 * u + 4 * g + e, t)];
        const float x = VT == kVBF16 ? round_to(bf16_bits_to_f32(w), 0) : f16_bits_to_f32(w);
        if (!(fabsf(x) < INFINITY)) o[u][e] += x;
      }
}

// The sums o of a row tile after its pages pa, pa + step, .. below pe.  A page that all rows of a workgroup see is
// multiplied as it is: an infinity of V comes out as one, or as NaN where the weight rounds to 0 or a later maximum
// scales the sum by 0.  A column that is not finite becomes the sum of the infinities and NaN that the row sees in it,
// if there are any: whatever its weights, the rows beside it and the order of the pages were.  `rows`: lanes of a row.
template <int VT, class BlockOf>
__device__ __forceinline__ void settle_not_finite(const AttendParams &p, BlockOf block_of, int pa, int pe, int step, int lane,
                                                  bool rows, int lim, f32x4 *o) {
  float any = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) any = __builtin_fmaf(o[u][e], 0.f, any);  // NaN, or 0
  if (__ballot(rows && any != 0.f) == 0) return;
  f32x4 sum[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) sum[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int pg = pa; pg < pe; pg += step) {
    const uint8_t *v = p.v + block_of(pg) * (kD * kPage * 2);
    uint32_t bad = 0;
#pragma unroll 1
    for (int i = 0; i < 16; i += 4)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        finite8(__builtin_bit_cast(u32x4, VTraits<VT>::operand(((const u32x4 *)v)[64 * (i + j) + lane])), bad);
    if (__ballot(bad != 0) != 0) add_not_finite<VT>(v, lane >> 4, lim - pg * kPage, sum);
  }
#pragma unroll
  for (int u = 0; u < 8; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(fabsf(o[u][e]) < INFINITY) && sum[u][e] != 0.f) o[u][e] = sum[u][e];
}

// ---------------------------------------------------------------------------
// The softmax step of one row tile over one page: scores to P operands, m and l of lane (g, n)'s row n
// (l: the lane's own tokens only, summed over g at the end).  MASK: only the page's first nvis tokens count.  Returns
// whether a maximum of the wave moved; alpha is then the factor of the row's O so far (1 where its m stands).
// ---------------------------------------------------------------------------
template <bool MASK>
__device__ __forceinline__ bool softmax_step(f32x4 *S, float cs, int nvis, int g, float &m, float &l, float &alpha,
                                             f16x8 *P) {
  float x[16];
  float top = -INFINITY;
#pragma unroll
  for (int tau = 0; tau < 4; ++tau)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 4 * i + tau;
      x[k] = S[tau][i];
      if (!MASK || 16 * g + k < nvis) top = fmaxf(top, x[k]);
    }
  top *= cs;
  // m may lag: most pages need no exchange between the row's four lanes and leave O as it is
  const bool moved = __ballot(top > m + (kHead + kStale)) != 0;
  alpha = 1.f;
  if (moved) {
    top = xor_max(top, 16);
    top = xor_max(top, 32);
    const float mn = fmaxf(m, top - kHead);
    alpha = exp2_hw(m - mn);
    m = mn;
    l *= alpha;
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = (!MASK || 16 * g + k < nvis) ? exp2_hw(__builtin_fmaf(x[k], cs, -m)) : 0.f;
  float sum = 0.f;  // of the weights as they are multiplied: their rounding then leaves a weighted mean of the same values
#pragma unroll
  for (int kap = 0; kap < 2; ++kap) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pk_f16_bits(x[8 * kap + 2 * i], x[8 * kap + 2 * i + 1]);
    P[kap] = __builtin_bit_cast(f16x8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (float)P[kap][i];
  }
  l += sum;
  return moved;
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// a partial (or, without slots, the output) of columns c0 .. c0 + 3 of one row
__device__ __forceinline__ void store_row4(const AttendParams &p, size_t row, int slot, int c0, f32x4 o, float m, float l,
                                           bool sees) {
  if (p.nslots == 0) {
    const f32x4 y = sees ? o * (1.f / l) : f32x4{0.f, 0.f, 0.f, 0.f};
    *(uint2 *)((uint16_t *)p.out + row * kD + c0) =
        p.out_bf16 ? make_uint2(pk_bf16_bits(y[0], y[1]), pk_bf16_bits(y[2], y[3]))
                   : make_uint2(pk_f16_bits(y[0], y[1]), pk_f16_bits(y[2], y[3]));
    return;
  }
  const size_t at = row * p.nslots + slot;
  *(f32x4 *)(p.part_o + at * kD + c0) = o;
  if (c0 == 0) *(float2 *)(p.part_ml + 2 * at) = make_float2(m, l);
}

// ---------------------------------------------------------------------------
// Few rows (up to 16 NT of a KV head and set per workgroup): each of the W waves takes every Wth page of the range
// with all rows, its operands straight from memory; the waves' results are joined in LDS.
// ---------------------------------------------------------------------------
template <int FMT, int NT, int W>
struct FewLds {
  float m[W][16 * NT], l[W][16 * NT];
  float o[W][16][kD + 4];
  float2 nf4[FMT == kFmtNf4 ? 256 : 1];
};
template <int FMT, int RES, int VT, int NT, int W>
__device__ __forceinline__ void few_rows(const AttendParams &p, int split, int hkv, int rb, int z, FewLds<FMT, NT, W> &s) {
  typedef VTraits<VT> VTr;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const AttendSet set = attend_set(p, z, split);
  const int LG = p.L * p.G, R = set.n * LG, r0 = rb * 16 * NT;
  if (r0 >= R) return;
  const int pa = set.p0, pe = set.p1;
  if (pa >= pe && p.nslots != 0) return;
  if constexpr (FMT == kFmtNf4) {
    if (threadIdx.x < 256) s.nf4[threadIdx.x] = make_float2(kNF4Levels[threadIdx.x & 15], kNF4Levels[threadIdx.x >> 4]);
    __syncthreads();
  }

  const int32_t *bt = p.bt + (size_t)set.b0 * p.bt_stride;
  KRaw<FMT, RES> kr;
  u32x4 V[16];
  size_t blk = 0;
  auto block_of = [&](int pg) {
    int id = bt[pg];
    id = __builtin_amdgcn_readfirstlane((unsigned)id < (unsigned)p.num_pages ? id : 0);
    return (size_t)id * p.HKV + hkv;
  };
  auto load_page = [&](int pg) {
    blk = block_of(pg);
    load_k<FMT, RES>(p, blk, lane, kr);
    const uint4 *vp = (const uint4 *)(p.v + blk * (kD * kPage * 2));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint4 w = load_once(vp + 64 * i + lane);
      V[i] = u32x4{w.x, w.y, w.z, w.w};
    }
  };
  f16x8 Q[NT][4];
  float cs[NT], m[NT], l[NT];
  int lim[NT];
  int lo = 0x7fffffff, hi = 0;
  f32x4 O[NT][8];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + n;
    const bool ok = r < R;
    const int bi = ok ? r / LG : 0, j = ok ? r - bi * LG : 0, i = j / p.G;
    const size_t row = ((size_t)(set.b0 + bi) * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
    load_q(p, row, ok, g, Q[t], cs[t]);
    lim[t] = ok ? row_limit(p, set.b0 + bi, i) : 0x7fffffff;  // rows past the last are computed, and not stored
    lo = min(lo, lim[t]);
    hi = max(hi, ok ? lim[t] : 0);
    m[t] = kNoMax;
    l[t] = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) O[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    lo = min(lo, __shfl_xor(lo, d));
    hi = max(hi, __shfl_xor(hi, d));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);

  const int last = min(pe, (hi + kPage - 1) / kPage);  // no row sees a later page
  for (int pg = pa + wv; pg < last; pg += W) {
    const int t0 = pg * kPage;
    load_page(pg);
    f32x4 S[NT][4];
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      f16x8 K[4];
      k_operands<FMT, RES>(kr, tau, s.nf4, K);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) a = mfma16(K[e], Q[t][e], a);
        S[t][tau] = a;
      }
    }
    const bool full = lo >= t0 + kPage;  // every row sees the whole page
    f16x8 P[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float alpha;
      const bool moved = full ? softmax_step<false>(S[t], cs[t], 64, g, m[t], l[t], alpha, P[t])
                              : softmax_step<true>(S[t], cs[t], lim[t] - t0, g, m[t], l[t], alpha, P[t]);
      if (moved)
#pragma unroll
        for (int u = 0; u < 8; ++u) O[t][u] *= alpha;
    }
    uint32_t bad = 0;
    if (!full) {
      u32x4 keep[2];
      partial_page_masks(g, hi - t0, keep);  // slots that no row sees are not data
#pragma unroll
      for (int i = 0; i < 16; ++i)
        V[i] = finite8(__builtin_bit_cast(u32x4, VTr::operand(V[i] & keep[i & 1])), bad);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int kap = 0; kap < 2; ++kap) {
        const f16x8 a = full ? VTr::operand(V[2 * u + kap]) : __builtin_bit_cast(f16x8, V[2 * u + kap]);
#pragma unroll
        for (int t = 0; t < NT; ++t) O[t][u] = mfma16(a, P[t][kap], O[t][u]);
      }
    if (__ballot(bad != 0) != 0)
#pragma unroll
      for (int t = 0; t < NT; ++t) add_not_finite<VT>(p.v + blk * (kD * kPage * 2), g, lim[t] - t0, O[t]);
  }

#pragma unroll
  for (int t = 0; t < NT; ++t)
    settle_not_finite<VT>(p, block_of, pa + wv, last, W, lane, r0 + 16 * t + n < R, lim[t], O[t]);

  // join the waves
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] = xor_sum(l[t], 16);
    l[t] = xor_sum(l[t], 32);
    if (g == 0) {
      s.m[wv][16 * t + n] = m[t];
      s.l[wv][16 * t + n] = l[t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float M = kNoMax;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, s.m[w][16 * t + n]);
    const float f = fmaxf(exp2_hw(m[t] - M), kLeast);
#pragma unroll
    for (int u = 0; u < 8; ++u) *(f32x4 *)&s.o[wv][n][16 * u + 4 * g] = O[t][u] * f;
    __syncthreads();
    constexpr int C = 32 / W;  // columns per thread
    const int rr = threadIdx.x / (kD / C), c0 = C * (threadIdx.x % (kD / C));
    const int r = r0 + 16 * t + rr;
    if (r < R) {
      float mm = kNoMax, ll = 0.f, o[C] = {};
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s.m[w][16 * t + rr]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        ll += s.l[w][16 * t + rr] * exp2_hw(s.m[w][16 * t + rr] - mm);
#pragma unroll
        for (int e = 0; e < C; ++e) o[e] += s.o[w][rr][c0 + e];
      }
      const int bi = r / LG, j = r - bi * LG, i = j / p.G, b = set.b0 + bi;
      const size_t row = ((size_t)b * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
      const bool sees = row_limit(p, b, i) > 0;
#pragma unroll
      for (int e = 0; e < C; e += 4)
        store_row4(p, row, set.slot, c0 + e, f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]}, mm, ll, sees);
    }
    __syncthreads();
  }
}

template <int FMT, int RES, int VT, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void paged_attend_kernel(const AttendParams p) {
  __shared__ FewLds<FMT, NT, 4> s;
  few_rows<FMT, RES, VT, NT, 4>(p, blockIdx.x, blockIdx.y % p.HKV, blockIdx.y / p.HKV, blockIdx.z, s);
}

// ---------------------------------------------------------------------------
// Many rows: 16 NT rows to each of the W waves.  The workgroup dequantizes a page once, as operands in LDS (K: wave w
// takes 8 / W of the eight (tile, half of the channels) units; V comes as it lies in the pool), and every wave reads
// them for its rows.  Two pages are in flight: while a wave exponentiates page j and multiplies it with V, it computes
// the scores of page j + 1, dequantizes its share of page j + 2 and has page j + 3's bytes under way, so that matrix
// and vector instructions have independent work at any time, with one barrier a page.
// ---------------------------------------------------------------------------
template <int FMT>
struct KUnit {  // one unit's bytes of lane (kc, m): token 4 m + tau, channels 32 kc + 16 h + (0..15)
  uint32_t c0, c1;
  uint16_t s, z;
  uint4 res;
};
template <int FMT, int RES>
__device__ __forceinline__ void load_unit(const AttendParams &p, size_t blk, int unit, int lane, KUnit<FMT> &r) {
  const int kc = lane >> 4, m = lane & 15, tau = unit >> 1, h = unit & 1;
  if constexpr (FMT == kFmtQ2) {
    r.c0 = *(const uint32_t *)(p.k + blk * 2048 + (((tau >> 1) * 64 + lane) * 2 + (tau & 1)) * 8 + 4 * h);
    const int at = (((tau >> 1) * 4 + kc) * 4 + (m >> 2)) * 8 + 4 * (tau & 1) + (m & 3);
    r.s = ((const uint16_t *)(p.ks + blk * 512))[at];
    r.z = ((const uint16_t *)(p.kz + blk * 512))[at];
  } else {
    const uint2 c = *(const uint2 *)(p.k + blk * 4096 + (tau * 64 + lane) * 16 + 8 * h);
    r.c0 = c.x;
    r.c1 = c.y;
    if constexpr (FMT == kFmtNvfp4) r.s = (p.ks + blk * 512)[(4 * m + tau) * 8 + 2 * kc + h];
    else r.s = ((const uint16_t *)(p.ks + blk * 256))[(4 * m + tau) * 2 + (kc >> 1)];
  }
  if constexpr (RES != kResNone) r.res = ((const uint4 *)(p.kr + blk * 8192))[64 * unit + lane];
}
template <int FMT, int RES>
__device__ __forceinline__ void unit_to_lds(const KUnit<FMT> &r, int unit, int lane, const float2 *nf4, u32x4 *dst) {
  const float s = FMT == kFmtNvfp4 ? fp8_pair<true, false>(r.s)[0] : f16_bits_to_f32(r.s);
  const float z = FMT == kFmtQ2 ? f16_bits_to_f32(r.z) : 0.f;
  f16x8 op[2];
  k_half<FMT, RES>(r.c0, r.c1, s, z, r.res, nf4, op);
  dst[(2 * unit) * 64 + lane] = __builtin_bit_cast(u32x4, op[0]);
  dst[(2 * unit + 1) * 64 + lane] = __builtin_bit_cast(u32x4, op[1]);
}

template <int FMT, int W>
struct ManyLds {
  u32x4 k[2][16 * 64], v[2][16 * 64];
  float2 nf4[FMT == kFmtNf4 ? 256 : 1];
  int hi[W], lo[W], bad;
};
template <int FMT, int RES, int VT, int NT, int W>
__device__ __forceinline__ void many_rows(const AttendParams &p, int split, int hkv, int nth, int z, ManyLds<FMT, W> &s) {
  constexpr int kUnits = 8 / W, kVPieces = 16 / W;  // of a page, per wave
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const AttendSet set = attend_set(p, z, split);
  // the set's row tiles over as few workgroups as hold them, evenly, and a workgroup's over its waves in turn
  const int LG = p.L * p.G, R = set.n * LG, tiles = (R + 15) / 16, blocks = (tiles + W * NT - 1) / (W * NT);
  if (nth >= blocks) return;
  const int per = (tiles + blocks - 1) / blocks;
  // the set's nth workgroup: of one sequence's rows the last first, which see the most keys of a causal chunk; those
  // past its q_lens, which see none, behind them
  int rb = nth;
  if (set.n == 1) {
    const int ql = p.q_lens ? min(max(p.q_lens[set.b0], 0), p.L) : p.L;
    const int live = ((ql * p.G + 15) / 16 + per - 1) / per;
    if (nth < live) rb = live - 1 - nth;
  }
  const int tile0 = rb * per + wv, tile_end = min((rb + 1) * per, tiles);
  const int pa = set.p0;
  int pe = set.p1;
  if (pa >= pe && p.nslots != 0) return;

  const int last = max(set.p1 - 1, pa);  // in the table also where the range is empty
  const int32_t *bt = p.bt + (size_t)set.b0 * p.bt_stride;
  auto block_of = [&](int pg) {  // pages past the range repeat its last one: loaded, never used
    int id = bt[min(pg, last)];
    id = __builtin_amdgcn_readfirstlane((unsigned)id < (unsigned)p.num_pages ? id : 0);
    return (size_t)id * p.HKV + hkv;
  };
  KUnit<FMT> raw[kUnits];
  auto load_raw = [&](size_t blk, KUnit<FMT> *r) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) load_unit<FMT, RES>(p, blk, wv * kUnits + i, lane, r[i]);
  };
  auto raw_to_lds = [&](int buf, const KUnit<FMT> *r) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) unit_to_lds<FMT, RES>(r[i], wv * kUnits + i, lane, s.nf4, s.k[buf]);
  };
  // V: straight into LDS; a bf16 pool's, which becomes the fp16 operand, through registers a page earlier
  u32x4 vraw[VT == kVF16 ? 1 : kVPieces];
  auto fetch_v = [&](size_t blk) {
    if constexpr (VT != kVF16) {
      const u32x4 *src = (const u32x4 *)(p.v + blk * (kD * kPage * 2));
#pragma unroll
      for (int i = 0; i < kVPieces; ++i) vraw[i] = src[(wv * kVPieces + i) * 64 + lane];
    }
  };
  auto store_v = [&](size_t blk, int buf) {
    const u32x4 *src = (const u32x4 *)(p.v + blk * (kD * kPage * 2));
#pragma unroll
    for (int i = 0; i < kVPieces; ++i) {
      const int at = (wv * kVPieces + i) * 64;
      if constexpr (VT == kVF16)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src + at + lane),
                                         (__attribute__((address_space(3))) void *)(&s.v[buf][at]), 16, 0, 0);
      else
        s.v[buf][at + lane] = __builtin_bit_cast(u32x4, VTraits<VT>::operand(vraw[i]));
    }
  };
  // the first pages' bytes are under way while q and the rows' limits are read
  size_t b0 = block_of(pa), b1 = block_of(pa + 1), b2 = block_of(pa + 2);
  KUnit<FMT> raw0[kUnits];
  load_raw(b0, raw0);
  load_raw(b1, raw);
  fetch_v(b0);
  if constexpr (VT == kVF16) store_v(b0, 0);

  f16x8 Q[NT][4];
  float cs[NT], m[NT];
  int lim[NT], lo = 0x7fffffff, hi = 0;
  f32x4 O[NT][8], Ls[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = 16 * (tile0 + W * t) + n;
    const bool ok = tile0 + W * t < tile_end && r < R;
    const int bi = ok ? r / LG : 0, j = ok ? r - bi * LG : 0, i = j / p.G;
    const size_t row = ((size_t)(set.b0 + bi) * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
    load_q(p, row, ok, g, Q[t], cs[t]);
    lim[t] = ok ? row_limit(p, set.b0 + bi, i) : 0x7fffffff;
    lo = min(lo, lim[t]);
    hi = max(hi, ok ? lim[t] : 0);
    m[t] = kNoMax;
    Ls[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 8; ++u) O[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    lo = min(lo, __shfl_xor(lo, d));
    hi = max(hi, __shfl_xor(hi, d));
  }
  if (lane == 0) {
    s.lo[wv] = lo;
    s.hi[wv] = hi;
  }
  if constexpr (FMT == kFmtNf4)
    if (threadIdx.x < 256) s.nf4[threadIdx.x] = make_float2(kNF4Levels[threadIdx.x & 15], kNF4Levels[threadIdx.x >> 4]);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) {
    lo = min(lo, s.lo[w]);
    hi = max(hi, s.hi[w]);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);  // every row of the workgroup sees the keys below lo, none those from hi on
  hi = __builtin_amdgcn_readfirstlane(hi);
  pe = min(pe, (hi + kPage - 1) / kPage);

  f32x4 S[NT][4];
  auto scores = [&](int buf, auto na) {
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      f16x8 K[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) K[e] = __builtin_bit_cast(f16x8, s.k[buf][(4 * tau + e) * 64 + lane]);
#pragma unroll
      for (int t = 0; t < na(); ++t) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) a = mfma16(K[e], Q[t][e], a);
        S[t][tau] = a;
      }
    }
  };
  const f16x8 one = {1, 1, 1, 1, 1, 1, 1, 1};
  auto weights = [&](int t, f16x8 *P) {  // of S[t], against m[t]; their sum by a product with ones
    float x[16];
#pragma unroll
    for (int tau = 0; tau < 4; ++tau)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * i + tau] = exp2_hw(__builtin_fmaf(S[t][tau][i], cs[t], -m[t]));
#pragma unroll
    for (int kap = 0; kap < 2; ++kap) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pk_f16_bits(x[8 * kap + 2 * i], x[8 * kap + 2 * i + 1]);
      P[kap] = __builtin_bit_cast(f16x8, w);
      Ls[t] = mfma16(one, P[kap], Ls[t]);
    }
  };

  // a wave's part of page pg with its first `na` tiles: softmax and P.V of the page, scores of the next one
  auto page = [&](int t0, int cur, bool full, size_t blk, auto na) {
    if (!full) {
#pragma unroll
      for (int t = 0; t < na(); ++t)
#pragma unroll
        for (int tau = 0; tau < 4; ++tau)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t0 + 16 * g + 4 * i + tau >= lim[t]) S[t][tau][i] = -INFINITY;
    }
    float top[NT];
    bool lag = false;
#pragma unroll
    for (int t = 0; t < na(); ++t) {
      float x = S[t][0][0];
#pragma unroll
      for (int k = 1; k < 16; ++k) x = fmaxf(x, S[t][k >> 2][k & 3]);
      top[t] = x * cs[t];
      lag |= top[t] > m[t] + (kHead + kStale);
    }
    if (__ballot(lag) != 0) {
#pragma unroll
      for (int t = 0; t < na(); ++t) {
        const float mn = fmaxf(m[t], xor_max(xor_max(top[t], 16), 32) - kHead);
        const float alpha = exp2_hw(m[t] - mn);
        m[t] = mn;
        Ls[t] *= alpha;
#pragma unroll
        for (int u = 0; u < 8; ++u) O[t][u] *= alpha;
      }
    }
    f16x8 P[NT][2];
#pragma unroll
    for (int t = 0; t < na(); ++t) weights(t, P[t]);
    scores(cur ^ 1, na);
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int kap = 0; kap < 2; ++kap) {
        const f16x8 a = __builtin_bit_cast(f16x8, s.v[cur][(2 * u + kap) * 64 + lane]);
#pragma unroll
        for (int t = 0; t < na(); ++t) O[t][u] = mfma16(a, P[t][kap], O[t][u]);
      }
    if (!full && s.bad)
#pragma unroll
      for (int t = 0; t < na(); ++t) add_not_finite<VT>(p.v + blk * (kD * kPage * 2), g, lim[t] - t0, O[t]);
  };
  constexpr std::integral_constant<int, NT> kAll = {};
  constexpr std::integral_constant<int, 1> kOne = {};
  const bool any = tile0 < tile_end, all = tile0 + W * (NT - 1) < tile_end;

  auto page_barrier = [&]() {  // loads into LDS are counted with the others, and no barrier waits for those
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
  };
  if (pa < pe) {
    if constexpr (VT != kVF16) store_v(b0, 0);
    fetch_v(b1);
    raw_to_lds(0, raw0);
    raw_to_lds(1, raw);
    load_raw(b2, raw);
    page_barrier();
    scores(0, kAll);
    __syncthreads();
  }
  auto pages = [&](auto na) {
    for (int pg = pa, cur = 0; pg < pe; ++pg, cur ^= 1) {
      const size_t b3 = block_of(pg + 3);
      store_v(b1, cur ^ 1);
      fetch_v(b2);
      raw_to_lds(cur, raw);
      load_raw(b3, raw);
      const int t0 = pg * kPage;
      const bool full = lo >= t0 + kPage;
      if (!full) {  // the last pages of a sequence or chunk
        if (threadIdx.x == 0) s.bad = 0;
        u32x4 keep[2];
        uint32_t bad = 0;
        partial_page_masks(g, hi - t0, keep);  // slots that no row sees are not data
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kVPieces; ++i) {
          const int at = (wv * kVPieces + i) * 64 + lane;
          s.v[cur][at] = finite8(s.v[cur][at] & keep[(wv * kVPieces + i) & 1], bad);
        }
        if (bad) s.bad = 1;
        __syncthreads();
      }
      if constexpr (na() > 0) page(t0, cur, full, b0, na);
      b0 = b1;
      b1 = b2;
      b2 = b3;
      page_barrier();
    }
  };
  // Each wave runs the loop of its tiles.  The loops meet in the same barriers: pa, pe and the pages that are not full are
  // the workgroup's.  (Both tiles' code for a wave with one, and tiles in order: 192 rows 64.7 -> 59.4 us, 320 100 -> 89.)
  if (all) pages(kAll);
  else if (any) pages(kOne);
  else pages(std::integral_constant<int, 0>());

#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (tile0 + W * t < tile_end)
      settle_not_finite<VT>(p, block_of, pa, pe, 1, lane, 16 * (tile0 + W * t) + n < R, lim[t], O[t]);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = 16 * (tile0 + W * t) + n;
    if (tile0 + W * t >= tile_end || r >= R) continue;
    const int bi = r / LG, j = r - bi * LG, i = j / p.G;
    const size_t row = ((size_t)(set.b0 + bi) * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
#pragma unroll
    for (int u = 0; u < 8; ++u) store_row4(p, row, set.slot, 16 * u + 4 * g, O[t][u], m[t], Ls[t][0], lim[t] > 0);
  }
}

template <int FMT, int RES, int VT, int NT, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) void paged_attend_wide_kernel(
    const AttendParams p) {
  __shared__ ManyLds<FMT, W> s;
  // KV head fastest (a head's workgroups, which read the same pages, on one XCD where heads are a multiple of 8), a set
  // after the other (interleaved, batches of prompts took 0.85 to 1.3 of the time: 4 x 512 tokens 33 -> 28 us, 8 ragged
  // ones of up to 2048 180 -> 226)
  many_rows<FMT, RES, VT, NT, W>(p, blockIdx.y, blockIdx.x % p.HKV, blockIdx.x / p.HKV, blockIdx.z, s);
}

// Shared pages for many rows (256 a workgroup) and own pages for few (up to 16 NT), one launch: the first kind is
// bound by its instructions, the second by memory, so they run side by side.  The first gets fewer workgroups than CUs;
// the others, dispatched after it, pass through the CUs that are left.
template <int FMT, int RES, int VT, int NT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void paged_attend_both_kernel(const AttendParams p) {
  __shared__ union Lds {
    FewLds<FMT, NT, 8> few;
    ManyLds<FMT, 8> many;
    __device__ Lds() {}
  } s;
  int x = blockIdx.x;
  if (x < p.shared_wgs) {
    const int hkv = x % p.HKV, y = x / p.HKV, w = y / p.shared_blocks;
    many_rows<FMT, RES, VT, 2, 8>(p, w % p.shared_slots, hkv, y % p.shared_blocks, w / p.shared_slots, s.many);
  } else {
    x -= p.shared_wgs;
    const int split = x % p.own_slots, y = x / p.own_slots;
    few_rows<FMT, RES, VT, NT, 8>(p, split, y % p.HKV, 0, p.nshared + y / p.HKV, s.few);
  }
}

// One launch over `sets` sets (own < 0), or one of both kinds: shared pages by 256 rows a workgroup, own pages by the
// kernel for few rows of kind `own`.
struct AttendLaunch {
  int kind, slots, blocks, sets, own;
  int res, vdt;  // FFA_DT_*
  hipStream_t st;
};

template <int FMT, int RES, int VT>
static void launch_types(const AttendParams &p, const AttendLaunch &a) {
  if (a.own >= 0) {
    const dim3 grid((unsigned)(p.shared_wgs + (long)p.B * p.HKV * p.own_slots));
    if (a.own == kRows16) hipLaunchKernelGGL((paged_attend_both_kernel<FMT, RES, VT, 1>), grid, dim3(512), 0, a.st, p);
    else hipLaunchKernelGGL((paged_attend_both_kernel<FMT, RES, VT, 2>), grid, dim3(512), 0, a.st, p);
    return;
  }
  const dim3 few((unsigned)a.slots, (unsigned)(p.HKV * a.blocks), (unsigned)a.sets);
  const dim3 wide((unsigned)(p.HKV * a.blocks), (unsigned)a.slots, (unsigned)a.sets);
  switch (a.kind) {
    case kRows16: hipLaunchKernelGGL((paged_attend_kernel<FMT, RES, VT, 1>), few, dim3(256), 0, a.st, p); break;
    case kRows32: hipLaunchKernelGGL((paged_attend_kernel<FMT, RES, VT, 2>), few, dim3(256), 0, a.st, p); break;
    case kRows64: hipLaunchKernelGGL((paged_attend_wide_kernel<FMT, RES, VT, 1, 4>), wide, dim3(256), 0, a.st, p); break;
    case kRows128: hipLaunchKernelGGL((paged_attend_wide_kernel<FMT, RES, VT, 2, 4>), wide, dim3(256), 0, a.st, p); break;
    default: hipLaunchKernelGGL((paged_attend_wide_kernel<FMT, RES, VT, 2, 8>), wide, dim3(512), 0, a.st, p);
  }
}
template <int FMT>
static void launch_format(const AttendParams &p, const AttendLaunch &a) {
  const bool bf = a.vdt == FFA_DT_BF16;
  if (a.res == FFA_DT_FP8_E4M3) bf ? launch_types<FMT, kResE4M3, kVBF16>(p, a) : launch_types<FMT, kResE4M3, kVF16>(p, a);
  else if (a.res == FFA_DT_FP8_E5M2) bf ? launch_types<FMT, kResE5M2, kVBF16>(p, a) : launch_types<FMT, kResE5M2, kVF16>(p, a);
  else bf ? launch_types<FMT, kResNone, kVBF16>(p, a) : launch_types<FMT, kResNone, kVF16>(p, a);
}
// the formats' builds, one source each
void attend_q2(const AttendParams &p, const AttendLaunch &a);
void attend_nvfp4(const AttendParams &p, const AttendLaunch &a);
void attend_nf4(const AttendParams &p, const AttendLaunch &a);

}  // namespace ffa
