// Exact attention over mxfp4 pages (keys and values in 4 bits): the kernel for few rows, the one for the most, and the
// builds of paged_attend.h between them.
//
// Few rows (16 sequences of 8K-64K, 32 + 8 heads: 122 us, 5.8 TB/s; five drafted tokens of 8: 78 us, 4.0) are bound by
// the pages' bytes (136 a token and head) only while the vector unit keeps up: the bytes of a 16-bit cache's token bring
// four tokens to convert.  K's codes become the fp16 operand by one conversion a pair, which applies the block's power of
// two.  V's powers of two belong to tokens, of which a V^T operand holds eight: its codes are converted times 2^-8 and
// multiplied, in pairs, by fp16 numbers 2^(e + 8), made of four scale bytes at a time.  With e within -22 .. 7 those are normal
// numbers; pages with others (blocks beyond 896, blocks of NaN) or with keys that some row does not see are put off to the end of
// a run of 64 and take V through fp32, with NaN taken out and given to the rows that see it.  Either way each operand is the
// value held, exactly, and blocks of zeros (2^-22) stay among the usual ones.  (With the powers of two in the weights' operand,
// relative to the largest so far, which took 1-7 % less time, a token of no weight whose V was 2^24 times the others' took 4 % of the
// result below fp16's steps, one of 2^28 nearly all of it.)  The weights' sum is a product with ones, of the weights as they
// are rounded.
// (The block-scaled matrix instruction on the codes themselves needs neither conversion, but it sums the products of a
// group of channels on a common 14-bit grid: 256 + 2^-6 = 256 there, where sums in 32 bits keep 2^-15.)
#include "paged_attend.h"

namespace ffa {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// One (page, KV head) as lane (g, n) takes it: K, and V with its scales.  Each half is loaded for the next page as soon
// as this page's is used.  (The pages that need care are a loop of their own: as a branch of this one they cost it 30
// registers, whose spills, waited for in order behind the next page's loads, took 1.4 times as long with two row tiles.)
struct MxKeys {
  u32x4 code[4];
  uint32_t scale;  // tokens 4 n + (0..3), block g
};
struct MxValues {
  u32x4 code[4], scale[4];  // block cb, tokens 16 g + (0..15)
  uint32_t every;           // block g, tokens 4 n + (0..3): each scale of the page in one lane
};
__device__ __forceinline__ void load_keys(const AttendParams &p, size_t blk, int lane, MxKeys &r) {
  r.scale = ((const uint32_t *)(p.ks + blk * kMxScales))[lane];
#pragma unroll
  for (int i = 0; i < 4; ++i) r.code[i] = __builtin_nontemporal_load((const u32x4 *)(p.k + blk * kMxCodes) + 64 * i + lane);
}
__device__ __forceinline__ void load_values(const AttendParams &p, size_t blk, int lane, MxValues &r) {
  const uint8_t *vs = p.vs + blk * kMxScales;
  r.every = ((const uint32_t *)vs)[lane];
#pragma unroll
  for (int i = 0; i < 4; ++i) r.scale[i] = ((const u32x4 *)vs)[4 * i + (lane >> 4)];
#pragma unroll
  for (int i = 0; i < 4; ++i) r.code[i] = __builtin_nontemporal_load((const u32x4 *)(p.v + blk * kMxCodes) + 64 * i + lane);
}

// With two row tiles a page's registers are short: the wave's pages then come through LDS, two ahead of use and in no
// registers (with V's powers of two in the weights still, five drafted tokens of 8 sequences 88 -> 74 us, of 2 35 -> 29; with one
// tile, 120.9 -> 121.6, one token after 2000 12.6 -> 14.5).  The copies are buffer loads, for whose data the compiler waits
// nowhere: the waits below are all there are.
// (Global loads into LDS make each wait of the kernel one for every load under way, those of the next page too: 77 us for 74.)
struct MxSlot {
  u32x4 k[4][64], v[4][64];
  uint32_t ks[64], vs[64];
};
constexpr int kSlotLoads = 10;
typedef __attribute__((address_space(3))) void *LdsTo;
__device__ __forceinline__ void copy_256(const uint8_t *from, int lane, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(from, 256), (LdsTo)to, 4, 4 * lane, 0, 0, 0);
}
__device__ __forceinline__ void copy_1k(const uint8_t *from, int lane, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(from, 1024), (LdsTo)to, 16, 16 * lane, 0, 0, kNonTemporal);
}
__device__ __forceinline__ void copy_page(const AttendParams &p, size_t blk, int lane, MxSlot &s) {
  // what was read from the slot has arrived before anything is copied there
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  copy_256(p.ks + blk * kMxScales, lane, s.ks);
  copy_256(p.vs + blk * kMxScales, lane, s.vs);
#pragma unroll
  for (int i = 0; i < 4; ++i) copy_1k(p.k + blk * kMxCodes + 1024 * i, lane, s.k[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) copy_1k(p.v + blk * kMxCodes + 1024 * i, lane, s.v[i]);
  asm volatile("" ::: "memory");
}
// the oldest page's copies have arrived: those of at most one other may be under way
__device__ __forceinline__ void await_page() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | kSlotLoads);  // vmcnt
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void read_keys(const MxSlot &s, int lane, MxKeys &K, uint32_t &every) {
  K.scale = s.ks[lane];
  every = s.vs[lane];
#pragma unroll
  for (int i = 0; i < 4; ++i) K.code[i] = s.k[i][lane];
}
__device__ __forceinline__ void read_values(const MxSlot &s, int lane, MxValues &V) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    V.scale[i] = ((const u32x4 *)s.vs)[4 * i + (lane >> 4)];
    V.code[i] = s.v[i][lane];
  }
}

// The largest of the first 16 lanes' x (lane n: row n's), wave-uniform
__device__ __forceinline__ int row16_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor8, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor4, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor2, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor1, 0xF, 0xF, false));
  return __builtin_amdgcn_readfirstlane(x);
}

template <int NT, int W>
union MxLds {
  FewLds<kFmtMxfp4, NT, W> join;
  MxSlot slot[NT == 2 ? W : 1][NT == 2 ? 2 : 1];
  __device__ MxLds() {}
};

template <int NT, int W>
__device__ __forceinline__ void few_rows_mx(const AttendParams &p, int split, int hkv, int rb, int z, MxLds<NT, W> &s) {
  constexpr bool kRing = NT == 2;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const AttendSet set = p.even ? even_set(p, split) : attend_set(p, z, split);
  const int LG = p.L * p.G, R = set.n * LG, r0 = rb * 16 * NT;
  if (r0 >= R) return;
  const int pa = set.p0, pe = set.p1;
  if (pa >= pe && p.nslots != 0) return;

  const int32_t *bt = p.bt + (size_t)set.b0 * p.bt_stride;
  auto page_id = [&](int pg) { return bt[max(min(pg, pe - 1), pa)]; };  // past the range its last page: loaded, never used
  auto block = [&](int id) {
    id = __builtin_amdgcn_readfirstlane((unsigned)id < (unsigned)p.num_pages ? id : 0);
    return (size_t)id * p.HKV + hkv;
  };
  MxKeys K;
  MxValues V;
  int id = 0;
  if (pa < pe) {
    const int id0 = page_id(pa + wv), id1 = page_id(pa + wv + W);
    if constexpr (kRing) {
      id = page_id(pa + wv + 2 * W);
      copy_page(p, block(id0), lane, s.slot[wv][0]);
      copy_page(p, block(id1), lane, s.slot[wv][1]);
    } else {
      id = id1;
      const size_t blk = block(id0);
      load_keys(p, blk, lane, K);
      load_values(p, blk, lane, V);
    }
  }

  f16x8 Q[NT][4];
  float cs[NT], m[NT];
  int lim[NT];
  int lo = 0x7fffffff, hi = 0;
  f32x4 O[NT][8], Ls[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + n;
    const bool ok = r < R;
    const int bi = ok ? r / LG : 0, j = ok ? r - bi * LG : 0, i = j / p.G;
    const size_t row = ((size_t)(set.b0 + bi) * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
    lim[t] = ok ? row_limit(p, set.b0 + bi, i) : 0x7fffffff;  // rows past the last are computed, and not stored
    // rows that see nothing are zeros whatever is computed (of zeros, so that the others' maxima move without regard to them):
    // with them, a padded batch would put every page off (five drafted tokens of 8 sequences, some padded, 239 us)
    load_q(p, row, ok && lim[t] > 0, g, Q[t], cs[t]);
    lo = min(lo, lim[t] > 0 ? lim[t] : 0x7fffffff);
    hi = max(hi, ok ? lim[t] : 0);
    m[t] = kNoMax;
    Ls[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 8; ++u) O[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  lo = -row16_max(-lo);
  hi = row16_max(hi);

  const f16x8 one = {1, 1, 1, 1, 1, 1, 1, 1};
  f32x4 S[NT][4];
  auto scores = [&]() {
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      const float ks = mx_factor((K.scale >> (8 * tau)) & 0xffu);
      f16x8 op[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) op[e] = mx_operand(K.code[tau][e], ks);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) a = mfma16(op[e], Q[t][e], a);
        S[t][tau] = a;
      }
    }
  };
  u32x4 w16[NT][2];  // the weights, tokens 16 g + 8 kap + (0..7)
  auto weights = [&]() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = S[t][0][0];
#pragma unroll
      for (int k = 1; k < 16; ++k) top = fmaxf(top, S[t][k >> 2][k & 3]);
      top *= cs[t];
      if (__ballot(top > m[t] + (kHead + kStale)) != 0) [[unlikely]] {
        const float mn = fmaxf(m[t], xor_max(xor_max(top, 16), 32) - kHead), alpha = exp2_hw(m[t] - mn);
        m[t] = mn;
        Ls[t] *= alpha;
#pragma unroll
        for (int u = 0; u < 8; ++u) O[t][u] *= alpha;
      }
#pragma unroll
      for (int k = 0; k < 16; k += 2) {  // tokens 16 g + k, + 1
        const float a = exp2_hw(__builtin_fmaf(S[t][k & 3][k >> 2], cs[t], -m[t]));
        const float b = exp2_hw(__builtin_fmaf(S[t][(k + 1) & 3][k >> 2], cs[t], -m[t]));
        w16[t][k >> 3][(k >> 1) & 3] = pk_f16_bits(a, b);
      }
#pragma unroll
      for (int kap = 0; kap < 2; ++kap) Ls[t] = mfma16(one, __builtin_bit_cast(f16x8, w16[t][kap]), Ls[t]);
    }
  };
  // whether all of the page's powers of two are within 2^-22 .. 2^7
  auto usual = [&]() {
    const u16x2 low = {kMxLow, kMxLow};
    const u16x2 a = __builtin_bit_cast(u16x2, V.every & 0x00ff00ffu) - low, b = __builtin_bit_cast(u16x2, (V.every >> 8) & 0x00ff00ffu) - low;
    const u16x2 off = __builtin_elementwise_max(a, b);  // those below are far above
    return __ballot(max((int)off[0], (int)off[1]) > 29) == 0;
  };

  const int last = min(pe, (hi + kPage - 1) / kPage);  // no row sees a later page
  // 64 pages of the wave at a time: the usual ones that every row sees whole, then the others
#pragma unroll 1
  for (int p0 = pa + wv; p0 < last; p0 += 64 * W) {
    uint64_t others = 0;
#pragma unroll 1
    for (int i = 0, pg = p0; i < 64 && pg < last; ++i, pg += W) {
      size_t next = 0;
      auto find_next = [&]() {
        next = block(id);
        id = page_id(pg + (kRing ? 3 : 2) * W);
      };
      if constexpr (!kRing) find_next();
      MxSlot &slot = s.slot[kRing ? wv : 0][kRing ? i & 1 : 0];
      if constexpr (kRing) {
        await_page();
        read_keys(slot, lane, K, V.every);
      }
      if (lo < (pg + 1) * kPage || !usual()) [[unlikely]] {
        others |= 1ull << i;
        if constexpr (kRing) {
          find_next();
          copy_page(p, next, lane, slot);
        } else {
          load_keys(p, next, lane, K);
          load_values(p, next, lane, V);
        }
        continue;
      }
      scores();
      if constexpr (!kRing) load_keys(p, next, lane, K);
      weights();
      if constexpr (kRing) {
        read_values(slot, lane, V);
        find_next();  // (before the copies: await_page counts those alone)
        copy_page(p, next, lane, slot);
      }
#pragma unroll
      for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int kap = 0; kap < 2; ++kap) {
          f16x2 f[4];  // 2^(e + 8) of tokens 16 g + 8 kap + 2 i, + 1
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = (V.scale[cb][2 * kap + i] - 0x68686868u) << 2;  // the upper bytes of four
            f[2 * i] = bits_f16x2(__builtin_amdgcn_perm(0, x, 0x010c000cu));
            f[2 * i + 1] = bits_f16x2(__builtin_amdgcn_perm(0, x, 0x030c020cu));
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f16x8 a = mx_operand(V.code[cb][2 * h + kap], 0x1p-8f, f);
#pragma unroll
            for (int t = 0; t < NT; ++t) O[t][2 * cb + h] = mfma16(a, __builtin_bit_cast(f16x8, w16[t][kap]), O[t][2 * cb + h]);
          }
        }
      if constexpr (!kRing) load_values(p, next, lane, V);
    }
    if (others == 0) [[likely]] continue;
#pragma unroll 1
    for (; others != 0; others &= others - 1) {
      const int pg = p0 + W * __builtin_ctzll(others), t0 = pg * kPage;
      const size_t blk = block(page_id(pg));
      load_keys(p, blk, lane, K);
      load_values(p, blk, lane, V);
      scores();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int tau = 0; tau < 4; ++tau)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t0 + 16 * g + 4 * i + tau >= lim[t]) S[t][tau][i] = -INFINITY;
      weights();
      u32x4 keep[2];
      uint32_t bad = 0;
      partial_page_masks(g, hi - t0, keep);  // slots that no row sees are not data
#pragma unroll
      for (int cb = 0; cb < 4; ++cb)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int kap = 0; kap < 2; ++kap) {
            const uint2 vs = make_uint2(V.scale[cb][2 * kap], V.scale[cb][2 * kap + 1]);
            const u32x4 v = __builtin_bit_cast(u32x4, mx_operand(V.code[cb][2 * h + kap], vs)) & keep[kap];
            const f16x8 a = __builtin_bit_cast(f16x8, finite8(v, bad));
#pragma unroll
            for (int t = 0; t < NT; ++t) O[t][2 * cb + h] = mfma16(a, __builtin_bit_cast(f16x8, w16[t][kap]), O[t][2 * cb + h]);
          }
      if (__ballot(bad != 0) != 0)
#pragma unroll
        for (int t = 0; t < NT; ++t) add_nan_blocks(p.vs + blk * kMxScales, lim[t] - t0, O[t]);
    }
    if (!kRing && p0 + 64 * W < last) {
      load_keys(p, block(page_id(p0 + 64 * W)), lane, K);
      load_values(p, block(page_id(p0 + 64 * W)), lane, V);
    }
  }
  float l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) l[t] = g == 0 ? Ls[t][0] : 0.f;  // join_waves sums over g
  if constexpr (kRing) {  // the waves' copies, used or not, have arrived: their place is the join's
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
  }
  join_waves<NT, W>(p, set, hkv, r0, m, l, O, s.join);
}

// ---------------------------------------------------------------------------
// Many rows: 256 a workgroup, 32 to each of its eight waves; a page is dequantized once, as operands in LDS.
//
// A product (16x16x32) takes 16.4 cycles of its SIMD; two vector instructions, or one exponential, cost nothing beside it in
// the same wave, each further one 4 cycles, and two waves of a SIMD of which one multiplies while the other adds gain less
// (1.2 times the serial rate).  So every product has vector work of another page beside it.  A turn j of the loop is eight
// steps of eight products, with the operands of the next step under way from LDS:
//   steps 0-3   O += V_(j-1) P_(j-1)     beside the first quarter of page j's weights and the wave's share of the pages to
//                                        come: K_(j+2) and V_(j+1) from registers into LDS, then the next ones' loads
//   steps 4-7   S_(j+1) = K_(j+1) Q      beside the other quarters: step 4 + tau takes S_(j+1)'s tile tau into the registers
//                                        of S_j's, whose weights are done a step before
// A weight's word holds two tokens of one tile, so V's operands are in that order in LDS: of a lane's sixteen tokens 0, 4,
// 8, 12, 1, 5, ... .  Maxima are powers of two, so that weights not yet multiplied scale without a rounding of
// their own when one moves (but below fp16's normal numbers, by steps of 2^-24 beside weights of 2^8 and more).
//
// 2048 rows of 32 heads over 16K keys of 8: 450 us at the clock that holds (534 in the first launches), 1.15 PFLOP/s of products
// where a large library product in fp16 reaches 1.17 (a page at a time, scores, weights and values one after the other: 485; two
// groups of waves half a page apart: 461; 32x32x16 products, six instructions beside each: 491; 64 rows a wave, half of the LDS
// reads: 558).  The matrix cores are busy 49 % of the cycles, vector issue 55 %.
// ---------------------------------------------------------------------------
struct WideLds {
  u32x4 k[2][16 * 64], v[3][16 * 64];
  int hi[8], lo[8], nan[3][8];
};

// V's operand KAP of 16 columns' tokens 0 .. 15 (codes w, scale bytes s) in the weights' order
template <int KAP>
__device__ __forceinline__ u32x4 wide_values(uint2 w, uint4 s) {
  const uint32_t x = __builtin_amdgcn_perm(w.y, w.x, 0x05040100u), y = __builtin_amdgcn_perm(w.y, w.x, 0x07060302u);
  // pairs of tokens (t, t + 4): byte 0 of even (0, 4), 1 (2, 6), 2 (8, 12), 3 (10, 14); odd: one more each
  const uint32_t even = (x & 0x0f0f0f0fu) | ((y & 0x0f0f0f0fu) << 4), odd = ((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u);
  const f32x2 c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(even, 1.f, KAP), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(even, 1.f, KAP + 2),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(odd, 1.f, KAP), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(odd, 1.f, KAP + 2)};
  const uint32_t sw[4] = {s.x, s.y, s.z, s.w};
  u32x4 op;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int tau = 2 * KAP + (q >> 1), i = 2 * (q & 1);  // tokens 4 i + tau, 4 (i + 1) + tau
    op[q] = pk_f16_bits(c[q][0] * mx_factor((sw[i] >> (8 * tau)) & 0xffu), c[q][1] * mx_factor((sw[i + 1] >> (8 * tau)) & 0xffu));
  }
  return op;
}

__device__ __forceinline__ void many_rows_mx(const AttendParams &p, int split, int hkv, int nth, int z, WideLds &s) {
  constexpr int NT = 2, W = 8;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const AttendSet set = p.even ? even_set(p, split) : attend_set(p, z, split);
  const int LG = p.L * p.G, R = set.n * LG, tiles = (R + 15) / 16, blocks = (tiles + W * NT - 1) / (W * NT);
  if (nth >= blocks) return;
  const int per = (tiles + blocks - 1) / blocks;
  int rb = nth;  // as in many_rows: the rows with the most keys first
  if (set.n == 1) {
    const int ql = p.q_lens ? min(max(p.q_lens[set.b0], 0), p.L) : p.L;
    const int live = ((ql * p.G + 15) / 16 + per - 1) / per;
    if (nth < live) rb = live - 1 - nth;
  }
  const int tile0 = rb * per + wv, tile_end = min((rb + 1) * per, tiles);
  const int pa = set.p0;
  int pe = set.p1;
  if (pa >= pe && p.nslots != 0) return;

  const int32_t *bt = p.bt + (size_t)set.b0 * p.bt_stride;
  const int end = max(set.p1 - 1, pa);  // in the table also where the range is empty
  auto page_id = [&](int j) { return bt[min(pa + j, end)]; };  // page j of the range; past it its last one: loaded, never used
  auto block = [&](int id) {
    id = __builtin_amdgcn_readfirstlane((unsigned)id < (unsigned)p.num_pages ? id : 0);
    return (size_t)id * p.HKV + hkv;
  };
  // a wave's eighths of a page: K's tile wv / 2, half wv % 2 of each block; V's columns 16 wv .. 16 wv + 15
  KUnit<kFmtMxfp4> kraw;
  uint2 vcode;
  uint4 vscale;
  auto load_k = [&](size_t blk) { load_unit<kFmtMxfp4, kResNone>(p, blk, wv, lane, kraw); };
  auto load_v = [&](size_t blk) {
    vcode = *(const uint2 *)(p.v + blk * kMxCodes + ((wv >> 1) * 64 + lane) * 16 + (wv & 1) * 8);
    vscale = *(const uint4 *)(p.vs + blk * kMxScales + (wv >> 1) * kPage + 16 * g);
  };
  auto store_k = [&](int slot) { unit_to_lds<kFmtMxfp4, kResNone>(kraw, wv, lane, nullptr, s.k[slot]); };
  int id1 = page_id(1), id2 = page_id(2), id3 = page_id(3);  // of the next loads' pages, read turns before
  {
    const size_t blk = block(page_id(0));
    load_k(blk);
    load_v(blk);
  }

  f16x8 Q[NT][4];
  float cs[NT], m[NT];
  int lim[NT], lo = 0x7fffffff, hi = 0;
  f32x4 O[NT][8], Ls[NT], S[NT][4];
  u32x4 P[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = 16 * (tile0 + W * t) + n;
    const bool ok = tile0 + W * t < tile_end && r < R;
    const int bi = ok ? r / LG : 0, j = ok ? r - bi * LG : 0, i = j / p.G;
    const size_t row = ((size_t)(set.b0 + bi) * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
    lim[t] = ok ? row_limit(p, set.b0 + bi, i) : 0x7fffffff;
    load_q(p, row, ok && lim[t] > 0, g, Q[t], cs[t]);  // as in few_rows_mx
    lo = min(lo, lim[t] > 0 ? lim[t] : 0x7fffffff);
    hi = max(hi, ok ? lim[t] : 0);
    m[t] = kNoMax;
    Ls[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 8; ++u) O[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    P[t][0] = P[t][1] = u32x4{0, 0, 0, 0};
  }
  lo = -row16_max(-lo);
  hi = row16_max(hi);
  if (lane == 0) {
    s.lo[wv] = lo;
    s.hi[wv] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) {
    lo = min(lo, s.lo[w]);
    hi = max(hi, s.hi[w]);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);  // every row of the workgroup sees the keys below lo, none those from hi on
  hi = __builtin_amdgcn_readfirstlane(hi);
  pe = min(pe, (hi + kPage - 1) / kPage);
  const int pages = max(pe - pa, 0);
  auto whole = [&](int j) { return lo >= (pa + j + 1) * kPage; };  // every row sees page j whole

  // V's share of page j into LDS
  uint32_t bad = 0;
  auto store_v = [&](int j, int slot, auto kap, auto masked) {
    u32x4 w = wide_values<kap()>(vcode, vscale);
    if (masked() && !whole(j)) {
      const int nvs = hi - (pa + j) * kPage - 16 * g;  // slots that no row sees are not data
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int t = 8 * (q & 1) + 2 * kap() + (q >> 1);
        w[q] &= (t < nvs ? 0xffffu : 0u) | (t + 4 < nvs ? 0xffff0000u : 0u);
      }
      w = finite8(w, bad);
      if constexpr (kap() == 1) {
        const int any = __ballot(bad != 0) != 0;
        if (lane == 0) s.nan[slot][wv] = any;
        bad = 0;
      }
    }
    s.v[slot][(2 * wv + kap()) * 64 + lane] = w;
  };
  constexpr std::integral_constant<int, 0> kLow = {};
  constexpr std::integral_constant<int, 1> kHigh = {};
  f16x8 op[2][4];
  auto fetch = [&](int into, const u32x4 *from, int step) {
#pragma unroll
    for (int e = 0; e < 4; ++e) op[into][e] = __builtin_bit_cast(f16x8, from[(4 * step + e) * 64 + lane]);
  };
  const f16x8 one = {1, 1, 1, 1, 1, 1, 1, 1};
  auto score_step = [&](int tau, const f16x8 *K, auto na) {
#pragma unroll
    for (int t = 0; t < na(); ++t) S[t][tau] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t = 0; t < na(); ++t) S[t][tau] = mfma16(K[e], Q[t][e], S[t][tau]);
  };
  auto value_step = [&](int i, const f16x8 *V, auto na) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t = 0; t < na(); ++t)
        O[t][2 * i + (e >> 1)] = mfma16(V[e], __builtin_bit_cast(f16x8, P[t][e & 1]), O[t][2 * i + (e >> 1)]);
  };
  auto sum_step = [&](auto na) {
#pragma unroll
    for (int t = 0; t < na(); ++t)
#pragma unroll
      for (int kap = 0; kap < 2; ++kap) Ls[t] = mfma16(one, __builtin_bit_cast(f16x8, P[t][kap]), Ls[t]);
  };
  auto weight = [&](int t, int tau, int h) {  // tokens 16 g + 4 i + tau, i = 2 h, 2 h + 1
    return pk_f16_bits(exp2_hw(__builtin_fmaf(S[t][tau][2 * h], cs[t], -m[t])), exp2_hw(__builtin_fmaf(S[t][tau][2 * h + 1], cs[t], -m[t])));
  };
  auto nan_step = [&](int j, int slot, auto na) {  // after page j's values, where it is not whole
    int any = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) any |= s.nan[slot][w];
    if (any) {
      const uint8_t *vs = p.vs + block(page_id(j)) * kMxScales;
#pragma unroll
      for (int t = 0; t < na(); ++t) add_nan_blocks(vs, lim[t] - (pa + j) * kPage, O[t]);
    }
  };

  // The scheduling groups of a step: the next one's four LDS reads, then a product and up to three or four vector
  // instructions in turn (left to the compiler, with one barrier a step: 464 us; two or three of them: 452)
  auto turn = [&](int j, int v0, int v1, int v2, auto na, auto masked) {  // V_(j-1) lies in slot v0, V_(j+1) goes to v2
    if (masked() && !whole(j)) {
      const int t0 = (pa + j) * kPage;
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
    if (__ballot(lag) != 0) [[unlikely]] {
#pragma unroll
      for (int t = 0; t < na(); ++t) {
        const float mn = fmaxf(m[t], floorf(xor_max(xor_max(top[t], 16), 32) - kHead));
        const float alpha = exp2_hw(m[t] - mn);
        m[t] = mn;
        Ls[t] *= alpha;
#pragma unroll
        for (int u = 0; u < 8; ++u) O[t][u] *= alpha;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const f16x2 w = bits_f16x2(P[t][k >> 2][k & 3]);
          P[t][k >> 2][k & 3] = pk_f16_bits((float)w[0] * alpha, (float)w[1] * alpha);
        }
      }
    }
    uint32_t first[NT][2];
    const u32x4 *kp = s.k[(j + 1) & 1], *vp = s.v[v0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!masked()) __builtin_amdgcn_sched_barrier(0);
      fetch((i + 1) & 1, i < 3 ? vp : kp, i < 3 ? i + 1 : 0);
      value_step(i, op[i & 1], na);
      if (i == 0)
#pragma unroll
        for (int t = 0; t < na(); ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) first[t][h] = weight(t, 0, h);
      if (i == 1) store_k(j & 1);
      if (i == 2) store_v(j + 1, v2, kLow, masked);
      if (i == 3) {
        store_v(j + 1, v2, kHigh, masked);
        sum_step(na);
        load_k(block(id3));
        load_v(block(id2));
        id2 = id3;
        id3 = page_id(j + 4);
      }
      if (!masked()) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x402, 4, 0);
        }
      }
    }
    if (masked() && j > 0 && !whole(j - 1)) nan_step(j - 1, v0, na);
#pragma unroll
    for (int t = 0; t < na(); ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) P[t][0][h] = first[t][h];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!masked()) __builtin_amdgcn_sched_barrier(0);
      if (i < 3) fetch((i + 1) & 1, kp, i + 1);
      else fetch(0, s.v[v1], 0);
      if (i < 3)
#pragma unroll
        for (int t = 0; t < na(); ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) P[t][(i + 1) >> 1][2 * ((i + 1) & 1) + h] = weight(t, i + 1, h);
      score_step(i, op[i & 1], na);
      if (!masked()) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x402, 3, 0);
        }
      }
    }
    __syncthreads();
  };
  auto run = [&](auto na) {
    if (pages == 0) return;
    // K_0, K_1 and V_0 into LDS, and zeros in V_(-1)'s place; scores of page 0
    store_k(0);
    store_v(0, 0, kLow, std::true_type());
    store_v(0, 0, kHigh, std::true_type());
    s.v[2][(2 * wv) * 64 + lane] = s.v[2][(2 * wv + 1) * 64 + lane] = u32x4{0, 0, 0, 0};
    load_k(block(id1));
    load_v(block(id1));
    store_k(1);
    load_k(block(id2));
    __syncthreads();
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      fetch(tau & 1, s.k[0], tau);
      score_step(tau, op[tau & 1], na);
    }
    fetch(0, s.v[2], 0);
    __syncthreads();
    int v0 = 2, v1 = 0, v2 = 1;  // slots of V_(j-1), V_j, V_(j+1)
    const int fast = min(max((lo >> 6) - pa - 1, 0), pages);  // turns of whole pages: up to j + 1
    int j = 0;
    auto rotate = [&]() {
      const int x = v0;
      v0 = v1;
      v1 = v2;
      v2 = x;
    };
    if constexpr (na() == NT)
      for (; j < fast; ++j) {
        turn(j, v0, v1, v2, na, std::false_type());
        rotate();
      }
    for (; j < pages; ++j) {
      turn(j, v0, v1, v2, na, std::true_type());
      rotate();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // the last page's values
      if (i < 3) fetch((i + 1) & 1, s.v[v0], i + 1);
      value_step(i, op[i & 1], na);
    }
    sum_step(na);
    if (!whole(pages - 1)) nan_step(pages - 1, v0, na);
  };
  if (tile0 + W * (NT - 1) < tile_end) run(std::integral_constant<int, NT>());
  else if (tile0 < tile_end) run(std::integral_constant<int, 1>());
  else run(std::integral_constant<int, 0>());

#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = 16 * (tile0 + W * t) + n;
    if (tile0 + W * t >= tile_end || r >= R) continue;
    const int bi = r / LG, j = r - bi * LG, i = j / p.G;
    const size_t row = p.even ? even_row(p, set.slot, hkv, r) : ((size_t)(set.b0 + bi) * p.L + i) * p.HQ + hkv * p.G + (j - i * p.G);
#pragma unroll
    for (int u = 0; u < 8; ++u) store_row4(p, row, set.slot, 16 * u + 4 * g, O[t][u], m[t], Ls[t][0], lim[t] > 0);
  }
}

__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void mxfp4_attend_wide_kernel(const AttendParams p) {
  __shared__ WideLds s;
  many_rows_mx(p, blockIdx.y, blockIdx.x % p.HKV, blockIdx.x / p.HKV, blockIdx.z, s);  // order as paged_attend_wide_kernel's
}

// Ranges are the few-row grid's fast order, but where about as many of them may be none as not: a CU then got two while another
// got none (one token of 32 sequences of 3000, 34 -> 28 us; of 3 of 9000, where few are none, 15.4 -> 16.3).
__host__ __device__ __forceinline__ bool ranges_last(const AttendParams &p) { return p.even != 0 && p.even <= 2 * p.B; }

template <int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void mxfp4_attend_kernel(const AttendParams p) {
  __shared__ MxLds<NT, 4> s;
  const int split = ranges_last(p) ? blockIdx.y : blockIdx.x, u = ranges_last(p) ? blockIdx.x : blockIdx.y;
  few_rows_mx<NT, 4>(p, split, u % p.HKV, u / p.HKV, blockIdx.z, s);
}

// Shared pages for many rows and own pages for few in one launch, as paged_attend_both_kernel
template <int NT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void mxfp4_attend_both_kernel(const AttendParams p) {
  __shared__ union Lds {
    MxLds<NT, 8> few;
    WideLds many;
    __device__ Lds() {}
  } s;
  int x = blockIdx.x;
  if (x < p.shared_wgs) {
    const int hkv = x % p.HKV, y = x / p.HKV, w = y / p.shared_blocks;
    many_rows_mx(p, w % p.shared_slots, hkv, y % p.shared_blocks, w / p.shared_slots, s.many);
  } else {
    x -= p.shared_wgs;
    const int split = x % p.own_slots, y = x / p.own_slots;
    few_rows_mx<NT, 8>(p, split, y % p.HKV, 0, p.nshared + y / p.HKV, s.few);
  }
}

void attend_mxfp4(const AttendParams &p, const AttendLaunch &a) {
  if (a.own >= 0) {
    const dim3 grid((unsigned)(p.shared_wgs + (long)p.B * p.HKV * p.own_slots));
    if (a.own == kRows16) hipLaunchKernelGGL(mxfp4_attend_both_kernel<1>, grid, dim3(512), 0, a.st, p);
    else hipLaunchKernelGGL(mxfp4_attend_both_kernel<2>, grid, dim3(512), 0, a.st, p);
    return;
  }
  const unsigned slots = (unsigned)a.slots, units = (unsigned)(p.HKV * a.blocks);
  const dim3 wide(units, slots, (unsigned)a.sets), few = ranges_last(p) ? wide : dim3(slots, units, (unsigned)a.sets);
  switch (a.kind) {
    case kRows16: hipLaunchKernelGGL(mxfp4_attend_kernel<1>, few, dim3(256), 0, a.st, p); break;
    case kRows32: hipLaunchKernelGGL(mxfp4_attend_kernel<2>, few, dim3(256), 0, a.st, p); break;
    case kRows64: hipLaunchKernelGGL((paged_attend_wide_kernel<kFmtMxfp4, kResNone, kVMxfp4, 1, 4>), wide, dim3(256), 0, a.st, p); break;
    case kRows128: hipLaunchKernelGGL((paged_attend_wide_kernel<kFmtMxfp4, kResNone, kVMxfp4, 2, 4>), wide, dim3(256), 0, a.st, p); break;
    default: hipLaunchKernelGGL(mxfp4_attend_wide_kernel, wide, dim3(512), 0, a.st, p);
  }
}

}  // namespace ffa
