// Exact attention over mxfp4 pages (keys and values in 4 bits): the kernel for few rows, and the builds of paged_attend.h
// for many.
//
// Few rows are bound by the pages' bytes (136 a token and head) only while the vector unit keeps up: the bytes of a
// 16-bit cache's token bring four tokens to convert.  K's codes become the fp16 operand by one conversion a pair, which
// applies the block's power of two.  V's powers of two belong to tokens, of which a V^T operand holds eight, so they
// multiply the weights: for each block of 32 columns the weights' operand is w_t 2^(e_t - R), R the largest e so far, and
// V's codes are converted as they are.  In a page that every row sees whole, and whose e lie within 14 of R, that is a
// packed product of fp16 pairs, exact; other pages, put off to the end of a run of 64, take it in fp32, with what a row does
// not see left out.  A NaN block thereby reaches the rows that see it and no other.  The weights' sum is a product with ones, of the weights as
// they are rounded.
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
// registers (five drafted tokens of 8 sequences 88 -> 79 us, of 2 35 -> 29; with one tile, which memory bounds, 121 -> 125).
// What is read from there goes by the instruction itself: the compiler makes every read of LDS it knows of wait for all
// copies under way.
struct MxSlot {
  u32x4 k[4][64], v[4][64];
  uint32_t ks[64], vs[64];
};
constexpr int kSlotLoads = 10;
__device__ __forceinline__ void copy_page(const AttendParams &p, size_t blk, int lane, MxSlot &s) {
  typedef const __attribute__((address_space(1))) void *From;
  typedef __attribute__((address_space(3))) void *To;
  __builtin_amdgcn_global_load_lds((From)(p.ks + blk * kMxScales + 4 * lane), (To)s.ks, 4, 0, 0);
  __builtin_amdgcn_global_load_lds((From)(p.vs + blk * kMxScales + 4 * lane), (To)s.vs, 4, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    __builtin_amdgcn_global_load_lds((From)(p.k + blk * kMxCodes + 1024 * i + 16 * lane), (To)s.k[i], 16, 0, kNonTemporal);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    __builtin_amdgcn_global_load_lds((From)(p.v + blk * kMxCodes + 1024 * i + 16 * lane), (To)s.v[i], 16, 0, kNonTemporal);
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
__device__ __forceinline__ void read_keys(const MxSlot &s, int lane, MxKeys &K, uint32_t &every) {
  const uint32_t a = lds_address(&s) + 16 * lane, b = lds_address(&s) + 8192 + 4 * lane;
  asm volatile(
      "ds_read_b32 %4, %7\n ds_read_b32 %5, %7 offset:256\n ds_read_b128 %0, %6\n ds_read_b128 %1, %6 offset:1024\n"
      " ds_read_b128 %2, %6 offset:2048\n ds_read_b128 %3, %6 offset:3072\n s_waitcnt lgkmcnt(0)"
      : "=&v"(K.code[0]), "=&v"(K.code[1]), "=&v"(K.code[2]), "=&v"(K.code[3]), "=&v"(K.scale), "=&v"(every)
      : "v"(a), "v"(b)
      : "memory");
}
__device__ __forceinline__ void read_values(const MxSlot &s, int lane, MxValues &V) {
  const uint32_t a = lds_address(&s) + 4096 + 16 * lane, b = lds_address(&s) + 8448 + 16 * (lane >> 4);
  asm volatile(
      "ds_read_b128 %4, %9\n ds_read_b128 %5, %9 offset:64\n ds_read_b128 %6, %9 offset:128\n ds_read_b128 %7, %9 offset:192\n"
      " ds_read_b128 %0, %8\n ds_read_b128 %1, %8 offset:1024\n ds_read_b128 %2, %8 offset:2048\n ds_read_b128 %3, %8 offset:3072\n"
      " s_waitcnt lgkmcnt(0)"
      : "=&v"(V.code[0]), "=&v"(V.code[1]), "=&v"(V.code[2]), "=&v"(V.code[3]), "=&v"(V.scale[0]), "=&v"(V.scale[1]),
        "=&v"(V.scale[2]), "=&v"(V.scale[3])
      : "v"(a), "v"(b)
      : "memory");
}

// The largest of the first 16 lanes' x (lane n: row n's), wave-uniform
__device__ __forceinline__ int row16_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor8, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor4, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor2, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kRowRor1, 0xF, 0xF, false));
  return __builtin_amdgcn_readfirstlane(x);
}

// The largest scale byte of a page's first `tokens` tokens (NaN blocks apart), wave-uniform
__device__ __forceinline__ int page_scale(uint32_t every, int lane, int tokens) {
  int best = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int byte = (every >> (8 * j)) & 0xffu;
    if (byte != kMxNan && 4 * (lane & 15) + j < tokens) best = max(best, byte);
  }
  return __builtin_amdgcn_readfirstlane((int)wave_max((float)best));
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
  AttendSet set;
  if (p.even) {
    const EvenRange e = even_find(p, split, -1);
    if (e.b >= p.B) return;
    set = AttendSet{e.b, 1, e.split * e.ppw, min((e.split + 1) * e.ppw, pages_of(p, e.b)), split};
  } else {
    set = attend_set(p, z, split);
  }
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
    const size_t blk = block(page_id(pa + wv));
    id = page_id(pa + wv + W);
    if constexpr (kRing) {
      copy_page(p, blk, lane, s.slot[wv][0]);
      copy_page(p, block(id), lane, s.slot[wv][1]);
      id = page_id(pa + wv + 2 * W);
    } else {
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
    load_q(p, row, ok, g, Q[t], cs[t]);
    lim[t] = ok ? row_limit(p, set.b0 + bi, i) : 0x7fffffff;  // rows past the last are computed, and not stored
    lo = min(lo, lim[t]);
    hi = max(hi, ok ? lim[t] : 0);
    m[t] = kNoMax;
    Ls[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 8; ++u) O[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  lo = -row16_max(-lo);
  hi = row16_max(hi);

  const f16x8 one = {1, 1, 1, 1, 1, 1, 1, 1};
  int vtop = kMxLow;  // R + 127
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
  // R up to the page's largest scale; whether all of its scales then lie within 14 below R
  auto scales = [&](int t0) {
    const u16x2 a = __builtin_bit_cast(u16x2, V.every & 0x00ff00ffu), b = __builtin_bit_cast(u16x2, (V.every >> 8) & 0x00ff00ffu);
    const u16x2 most = __builtin_elementwise_max(a, b), least = __builtin_elementwise_min(a, b);
    const int up = max((int)most[0], (int)most[1]), low = min((int)least[0], (int)least[1]);
    if (__ballot(up > vtop) != 0) [[unlikely]] {
      const int now = max(vtop, page_scale(V.every, lane, hi - t0));
      const float f = now - vtop > 126 ? 0.f : mx_factor(127 + vtop - now);
      vtop = now;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 8; ++u) O[t][u] *= f;
    }
    return __ballot(up > vtop || low < vtop - 14) == 0;
  };
  auto values = [&](int cb, const f16x8 (*P)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int kap = 0; kap < 2; ++kap) {
        const f16x8 a = mx_operand(V.code[cb][2 * h + kap], 1.0f);
#pragma unroll
        for (int t = 0; t < NT; ++t) O[t][2 * cb + h] = mfma16(a, P[t][kap], O[t][2 * cb + h]);
      }
  };

  const int last = min(pe, (hi + kPage - 1) / kPage);  // no row sees a later page
  // 64 pages of the wave at a time: those that every row sees whole and whose scales lie together, then the others
#pragma unroll 1
  for (int p0 = pa + wv; p0 < last; p0 += 64 * W) {
    uint64_t others = 0;
#pragma unroll 1
    for (int i = 0, pg = p0; i < 64 && pg < last; ++i, pg += W) {
      const size_t next = block(id);
      id = page_id(pg + (kRing ? 3 : 2) * W);
      MxSlot &slot = s.slot[kRing ? wv : 0][kRing ? i & 1 : 0];
      if constexpr (kRing) {
        __builtin_amdgcn_s_waitcnt(0x0f70 | kSlotLoads);  // vmcnt: the next page's copies may be under way
        read_keys(slot, lane, K, V.every);
      }
      if (lo < (pg + 1) * kPage || !scales(pg * kPage)) [[unlikely]] {
        others |= 1ull << i;
        if constexpr (kRing) {
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
        copy_page(p, next, lane, slot);  // its last page is read
      }
      const uint32_t base = (uint32_t)(vtop - 15) * 0x01010101u;
#pragma unroll
      for (int cb = 0; cb < 4; ++cb) {
        f16x8 P[NT][2];
#pragma unroll
        for (int kap = 0; kap < 2; ++kap)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // four bytes 127 + e to the upper bytes of the fp16 numbers 2^(e - R)
            const uint32_t x = (V.scale[cb][2 * kap + j] - base) << 2;
            const f16x2 f[2] = {bits_f16x2(__builtin_amdgcn_perm(0, x, 0x010c000cu)), bits_f16x2(__builtin_amdgcn_perm(0, x, 0x030c020cu))};
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const f16x2 y = bits_f16x2(w16[t][kap][2 * j + e]) * f[e];
                P[t][kap][4 * j + 2 * e] = y[0];
                P[t][kap][4 * j + 2 * e + 1] = y[1];
              }
          }
        values(cb, P);
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
      scales(t0);
      scores();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int tau = 0; tau < 4; ++tau)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t0 + 16 * g + 4 * i + tau >= lim[t]) S[t][tau][i] = -INFINITY;
      weights();
#pragma unroll
      for (int cb = 0; cb < 4; ++cb) {
        f16x8 P[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int byte = (V.scale[cb][k >> 2] >> (8 * (k & 3))) & 0xffu;
            // byte - vtop <= 0 for what a row sees, but for NaN blocks
            const float f = byte == kMxNan ? NAN : mx_factor(max(127 + min(byte - vtop, 0), 0));
            const float w = (float)__builtin_bit_cast(f16x8, w16[t][k >> 3])[k & 7];
            P[t][k >> 3][k & 7] = (_Float16)(t0 + 16 * g + k < lim[t] ? w * f : 0.f);
          }
        values(cb, P);
      }
    }
    if (!kRing && p0 + 64 * W < last) {
      load_keys(p, block(page_id(p0 + 64 * W)), lane, K);
      load_values(p, block(page_id(p0 + 64 * W)), lane, V);
    }
  }
  float l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] = g == 0 ? Ls[t][0] : 0.f;  // join_waves sums over g
#pragma unroll
    for (int u = 0; u < 8; ++u) O[t][u] *= mx_factor(vtop);
  }
  if constexpr (kRing) {  // the waves' copies, used or not, have arrived: their place is the join's
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
  }
  join_waves<NT, W>(p, set, hkv, r0, m, l, O, s.join);
}

template <int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void mxfp4_attend_kernel(const AttendParams p) {
  __shared__ MxLds<NT, 4> s;
  few_rows_mx<NT, 4>(p, blockIdx.x, blockIdx.y % p.HKV, blockIdx.y / p.HKV, blockIdx.z, s);
}

// Shared pages for many rows and own pages for few in one launch, as paged_attend_both_kernel
template <int NT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void mxfp4_attend_both_kernel(const AttendParams p) {
  __shared__ union Lds {
    MxLds<NT, 8> few;
    ManyLds<kFmtMxfp4, 8> many;
    __device__ Lds() {}
  } s;
  int x = blockIdx.x;
  if (x < p.shared_wgs) {
    const int hkv = x % p.HKV, y = x / p.HKV, w = y / p.shared_blocks;
    many_rows<kFmtMxfp4, kResNone, kVMxfp4, 2, 8>(p, w % p.shared_slots, hkv, y % p.shared_blocks, w / p.shared_slots, s.many);
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
  const dim3 few((unsigned)a.slots, (unsigned)(p.HKV * a.blocks), (unsigned)a.sets);
  const dim3 wide((unsigned)(p.HKV * a.blocks), (unsigned)a.slots, (unsigned)a.sets);
  switch (a.kind) {
    case kRows16: hipLaunchKernelGGL(mxfp4_attend_kernel<1>, few, dim3(256), 0, a.st, p); break;
    case kRows32: hipLaunchKernelGGL(mxfp4_attend_kernel<2>, few, dim3(256), 0, a.st, p); break;
    case kRows64: hipLaunchKernelGGL((paged_attend_wide_kernel<kFmtMxfp4, kResNone, kVMxfp4, 1, 4>), wide, dim3(256), 0, a.st, p); break;
    case kRows128: hipLaunchKernelGGL((paged_attend_wide_kernel<kFmtMxfp4, kResNone, kVMxfp4, 2, 4>), wide, dim3(256), 0, a.st, p); break;
    default: hipLaunchKernelGGL((paged_attend_wide_kernel<kFmtMxfp4, kResNone, kVMxfp4, 2, 8>), wide, dim3(512), 0, a.st, p);
  }
}

}  // namespace ffa
