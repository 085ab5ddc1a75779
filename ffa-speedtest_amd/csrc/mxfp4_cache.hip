// The mxfp4 pages: append (with or without rotary positions, with or without the held values), and read-back.
//
// Bound by bytes: k, v and q are read once; codes and scales (136 bytes a token and head), the turned q and the values
// are written once.  The two appends differ in how a token's V nibble, which shares its byte with the next token's, is
// written.
//   tiles   a workgroup takes a page of a sequence (64 tokens); each of its waves, one after the other, 32 tokens of a
//           head's K (or q), or 16 of its V: eight tokens' codes of a column are a word in one lane, which trades its
//           words for whole 16-byte pieces in LDS, so that every store of a wave is 1 KB.
//   tokens  eight lanes take two tokens of a head that share bytes, whichever of them are new, and write the bytes one by
//           one: a decode step's rows in one round.
// mx_by_tiles says which takes a call.
#include "rope_axes.h"
#include "routes.h"

extern "C" int ffa_set_error_internal(int code, const char *msg);

namespace ffa {

struct MxAppendParams {
  RopeParams rope;
  const void *k, *v, *q;
  long k_batch, k_token, k_head, v_batch, v_token, v_head, q_batch, q_token, q_head;
  int B, T, HKV, HQ;
  const int32_t *pos, *bt;
  int bt_stride, num_pages;
  uint8_t *kp, *ks, *vp, *vs;
  void *q_out, *k_values, *v_values;
  int tiles;  // pages, or pairs of positions, that the new tokens of a sequence can touch
};

// the larger of x and those of the lanes that differ from this one in the low two bits, then in the third
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));  // lanes 1 0 3 2
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));  // 2 3 0 1
}
__device__ __forceinline__ uint32_t oct_max(uint32_t x) {
  x = quad_max(x);
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, false));  // 7 6 .. 0
}
// |x| as bits: ordered as the magnitudes are, infinities and NaN above all
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
template <int N>
__device__ __forceinline__ uint32_t top_magnitude(const float *x) {
  uint32_t top = magnitude(x[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) top = max(top, magnitude(x[i]));
  return top;
}
// a value's factor: a NaN, not an infinity, for the block of NaN
__device__ __forceinline__ float value_factor(int byte) { return byte == kMxNan ? NAN : mx_factor(byte); }

// K of one token and head in eight lanes: codes and scales of both halves of the lane's row
struct MxRow {
  uint32_t code[2];
  int byte[2];
};
__device__ __forceinline__ MxRow quantize_row(const float *x) {
  MxRow r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    r.byte[h] = mx_scale(quad_max(top_magnitude<8>(x + 8 * h)));
    r.code[h] = mx_codes8(x + 8 * h, r.byte[h]);
  }
  return r;
}
__device__ __forceinline__ void held_row(const MxRow &r, float *x) {
#pragma unroll
  for (int h = 0; h < 2; ++h) mx_values8(r.code[h], value_factor(r.byte[h]), x + 8 * h);
}

// ---------------------------------------------------------------------------
// by tiles of 64 tokens
// ---------------------------------------------------------------------------
constexpr int kAnglePitch = 66;  // a token's angles in LDS, 16 bytes apart from a power of two: eight tokens' meet in few banks
struct MxTile {
  int b, page, n0, lo, hi;  // slots [lo, hi) of the page are new tokens n0 + slot; page -1: nothing is written
};

template <int DT, int TURN>
__device__ __forceinline__ void tile_k(const MxAppendParams &p, const MxTile &tl, int h, int half, const float2 (*cs)[kAnglePitch]) {
  const int lane = threadIdx.x & 63, l = lane & 7, m = 8 * half + (lane >> 3);
  Row16<DT> w[4];
#pragma unroll
  for (int tau = 0; tau < 4; ++tau) {  // tokens past the sequence's repeat its last one
    const int t = min(max(4 * m + tau, tl.lo), tl.hi - 1);
    w[tau] = load_row<DT>(p.k, tl.b * p.k_batch + (long)(tl.n0 + t) * p.k_token + h * p.k_head, l);
  }
  const size_t blk = (size_t)tl.page * p.HKV + h;
  uint32_t sc[2] = {0, 0};
#pragma unroll
  for (int tau = 0; tau < 4; ++tau) {
    const int t = 4 * m + tau;
    const bool ok = t >= tl.lo && t < tl.hi;
    float x[16];
    row_values<DT>(w[tau], x);
    if constexpr (TURN != kTurnNone) rope_turn<TURN>(cs[t], l, x);
    const MxRow r = quantize_row(x);
    if (ok && tl.page >= 0) {
      *(uint32_t *)(p.kp + blk * kMxCodes + mx_k_off(t, l)) = r.code[0];
      *(uint32_t *)(p.kp + blk * kMxCodes + mx_k_off(t, l + 8)) = r.code[1];
    }
    sc[0] |= (uint32_t)r.byte[0] << (8 * tau);
    sc[1] |= (uint32_t)r.byte[1] << (8 * tau);
    if (p.k_values && ok) {
      held_row(r, x);
      store_row<DT>(p.k_values, (((long)tl.b * p.T + tl.n0 + t) * p.HKV + h) * kD, l, x);
    }
  }
  if ((l & 3) != 0 || tl.page < 0) return;
  uint8_t *s = p.ks + blk * kMxScales + (l >> 2) * kPage + 4 * m;
  if (4 * m >= tl.lo && 4 * m + 4 <= tl.hi) {
    *(uint32_t *)s = sc[0];
    *(uint32_t *)(s + 2 * kPage) = sc[1];
  } else {
#pragma unroll
    for (int tau = 0; tau < 4; ++tau)
      if (4 * m + tau >= tl.lo && 4 * m + tau < tl.hi) {
        s[tau] = (uint8_t)(sc[0] >> (8 * tau));
        s[2 * kPage + tau] = (uint8_t)(sc[1] >> (8 * tau));
      }
  }
}

template <int DT, int TURN>
__device__ __forceinline__ void tile_q(const MxAppendParams &p, const MxTile &tl, int h, int half, const float2 (*cs)[kAnglePitch]) {
  const int lane = threadIdx.x & 63, l = lane & 7;
  Row16<DT> w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = min(max(32 * half + 8 * i + (lane >> 3), tl.lo), tl.hi - 1);
    w[i] = load_row<DT>(p.q, tl.b * p.q_batch + (long)(tl.n0 + t) * p.q_token + h * p.q_head, l);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 32 * half + 8 * i + (lane >> 3);
    if (t < tl.lo || t >= tl.hi) continue;
    float x[16];
    row_values<DT>(w[i], x);
    rope_turn<TURN>(cs[t], l, x);
    store_row<DT>(p.q_out, (((long)tl.b * p.T + tl.n0 + t) * p.HQ + h) * kD, l, x);
  }
}

// V: lane (o, c) takes tokens 16 g + 8 o + (0..7), channels 4 c + (0..3).  lds: 1 KB of the wave's own.
template <int DT>
__device__ __forceinline__ void tile_v(const MxAppendParams &p, const MxTile &tl, int h, int g, uint32_t *lds) {
  const int lane = threadIdx.x & 63, o = lane >> 5, c = lane & 31, t0 = 16 * g + 8 * o;
  typedef typename std::conditional<DT == 2, uint4, uint2>::type Raw4;
  Raw4 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = min(max(t0 + i, tl.lo), tl.hi - 1);
    const long at = tl.b * p.v_batch + (long)(tl.n0 + t) * p.v_token + h * p.v_head + 4 * c;
    w[i] = *(const Raw4 *)((const uint8_t *)p.v + at * (DT == 2 ? 4 : 2));
  }
  float x[8][4];
  int byte[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == 2) {
      x[i][0] = __uint_as_float(w[i].x);
      x[i][1] = __uint_as_float(w[i].y);
      x[i][2] = __uint_as_float(w[i].z);
      x[i][3] = __uint_as_float(w[i].w);
    } else {
      const uint32_t a[2] = {w[i].x, w[i].y};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[i][2 * e] = DT == 1 ? __uint_as_float(a[e] << 16) : f16_bits_to_f32(a[e] & 0xffffu);
        x[i][2 * e + 1] = DT == 1 ? __uint_as_float(a[e] & 0xffff0000u) : f16_bits_to_f32(a[e] >> 16);
      }
    }
    byte[i] = mx_scale(oct_max(top_magnitude<4>(x[i])));
    const float f = mx_inverse(byte[i]);  // a power of two: exact
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = byte[i] == kMxNan ? 0.f : x[i][e] * f;
  }
  uint32_t code[4];  // of channel 4 c + e, eight tokens
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y[8] = {x[0][e], x[1][e], x[2][e], x[3][e], x[4][e], x[5][e], x[6][e], x[7][e]};
    code[e] = mx_codes8(y, 127);
  }
  if (p.v_values) {
    float y[4][8];
#pragma unroll
    for (int e = 0; e < 4; ++e) mx_values8(code[e], 1.f, y[e]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (t0 + i < tl.lo || t0 + i >= tl.hi) continue;
      const float f = value_factor(byte[i]);
      const float held[4] = {y[0][i] * f, y[1][i] * f, y[2][i] * f, y[3][i] * f};
      store_values<DT, 4, false>(p.v_values, (((size_t)tl.b * p.T + tl.n0 + t0 + i) * p.HKV + h) * kD + 4 * c, held);
    }
  }
  if (tl.page < 0) return;
  const size_t blk = (size_t)tl.page * p.HKV + h;
#pragma unroll
  for (int e = 0; e < 4; ++e) lds[((c >> 3) * 16 + 4 * (c & 3) + e) * 4 + ((c >> 2) & 1) * 2 + o] = code[e];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  u32x4 out = ((const u32x4 *)lds)[lane];  // piece (lane >> 4, lane & 15): words (h, o)
  u32x4 *dst = (u32x4 *)(p.vp + blk * kMxCodes) + ((lane >> 4) * 64 + g * 16 + (lane & 15));
  uint8_t *s = p.vs + blk * kMxScales + (c >> 3) * kPage + t0;
  if (16 * g >= tl.lo && 16 * g + 16 <= tl.hi) {
    *dst = out;
    if ((c & 7) == 0) {
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a |= (uint32_t)byte[i] << (8 * i);
        b |= (uint32_t)byte[4 + i] << (8 * i);
      }
      *(uint2 *)s = make_uint2(a, b);
    }
  } else {  // older tokens' nibbles, and those not yet written, stay
    uint32_t keep[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      keep[k] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = 16 * g + 8 * k + i;
        if (t < tl.lo || t >= tl.hi) keep[k] |= 0xfu << (4 * i);
      }
    }
    if ((keep[0] & keep[1]) != 0xffffffffu) {
      const u32x4 old = *dst;
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = (old[k] & keep[k & 1]) | (out[k] & ~keep[k & 1]);
      *dst = out;
    }
    if ((c & 7) == 0)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t0 + i >= tl.lo && t0 + i < tl.hi) s[i] = (uint8_t)byte[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's next unit writes lds again
}

template <int DT, int TURN>
__global__ __launch_bounds__(256) void mxfp4_append_tiles_kernel(const MxAppendParams p) {
  __shared__ float2 cs[TURN == kTurnNone ? 1 : 64][kAnglePitch];
  __shared__ u32x4 words[4][64];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  MxTile tl;
  tl.b = blockIdx.x / p.tiles;
  const int pos = p.pos[tl.b], P0 = ((pos >> 6) + (int)(blockIdx.x % p.tiles)) * kPage;
  tl.n0 = P0 - pos;
  tl.lo = max(-tl.n0, 0);
  tl.hi = min(kPage, p.T - tl.n0);
  if (tl.lo >= tl.hi) return;
  tl.page = append_page(p.bt, p.bt_stride, p.num_pages, tl.b, P0);
  uint32_t *lds = (uint32_t *)words[wv];
  int part = blockIdx.y, parts = gridDim.y;
  if (TURN != kTurnNone && p.v && parts >= 3) {
    // V, which does not turn, by the first workgroup alone, beside the others' angles
    if (part == 0) {
      for (int u = wv; u < 4 * p.HKV; u += 4) tile_v<DT>(p, tl, u >> 2, u & 3, lds);
      return;
    }
    --part;
    --parts;
  }
  const bool v = p.v && parts == (int)gridDim.y;
  if constexpr (TURN != kTurnNone) {
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
      const int t = i >> 6;
      if (t >= tl.lo && t < tl.hi) cs[t][i & 63] = rope_angle(p.rope, i & 63, tl.b, tl.n0 + t, (long)P0 + t);
    }
    __syncthreads();
  }
  // units: two a head of K, four of V, two of q, the waves of the tile's workgroups in turn; q, which only turns, last (a 16K
  // prompt's append 4 % less)
  const int nk = 2 * p.HKV, kv = nk + (v ? 4 * p.HKV : 0), units = kv + (TURN == kTurnNone ? 0 : 2 * p.HQ);
  for (int u = part * 4 + wv; u < units; u += 4 * parts) {
    if (u < nk) {
      tile_k<DT, TURN>(p, tl, u >> 1, u & 1, cs);
    } else if (u < kv) {
      tile_v<DT>(p, tl, (u - nk) >> 2, (u - nk) & 3, lds);
    } else {
      if constexpr (TURN != kTurnNone) tile_q<DT, TURN>(p, tl, (u - kv) >> 1, (u - kv) & 1, cs);
    }
  }
}

// ---------------------------------------------------------------------------
// by pairs of positions
// ---------------------------------------------------------------------------
template <int DT, int TURN>
__global__ __launch_bounds__(256) void mxfp4_append_tokens_kernel(const MxAppendParams p) {
  __shared__ float2 cs[TURN == kTurnNone ? 1 : 2][64];
  const int b = blockIdx.x / p.tiles, l = threadIdx.x & 7;
  const int pos = p.pos[b], P0 = (pos & ~1) + 2 * (int)(blockIdx.x % p.tiles);
  const int n0 = P0 - pos;  // of position P0 among the new tokens
  const bool is[2] = {n0 >= 0 && n0 < p.T, n0 + 1 < p.T};  // n0 >= -1
  if (!is[0] && !is[1]) return;
  const int nq = TURN == kTurnNone ? 0 : p.HQ, units = nq + p.HKV + (p.v ? p.HKV : 0);
  const int u = blockIdx.y * 32 + (threadIdx.x >> 3);
  const int kind = u < nq ? 0 : (u < nq + p.HKV ? 1 : 2), h = u - (kind == 0 ? 0 : (kind == 1 ? nq : nq + p.HKV));
  Row16<DT> w[2];
  if (u < units) {
    const void *x = kind == 0 ? p.q : (kind == 1 ? p.k : p.v);
    const long batch = kind == 0 ? p.q_batch : (kind == 1 ? p.k_batch : p.v_batch);
    const long token = kind == 0 ? p.q_token : (kind == 1 ? p.k_token : p.v_token);
    const long head = kind == 0 ? p.q_head : (kind == 1 ? p.k_head : p.v_head);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (is[i]) w[i] = load_row<DT>(x, b * batch + (long)(n0 + i) * token + h * head, l);
  }
  if constexpr (TURN != kTurnNone) {
    const int i = threadIdx.x >> 6;
    if (i < 2 && is[i]) cs[i][threadIdx.x & 63] = rope_angle(p.rope, threadIdx.x & 63, b, n0 + i, (long)P0 + i);
    __syncthreads();
  }
  if (u >= units) return;
  const int page = append_page(p.bt, p.bt_stride, p.num_pages, b, P0);  // P0 + 1 is of the same page
  const size_t blk = (size_t)page * p.HKV + h;
  if (kind != 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!is[i]) continue;
      float x[16];
      row_values<DT>(w[i], x);
      if constexpr (TURN != kTurnNone) rope_turn<TURN>(cs[i], l, x);
      if (kind == 0) {
        store_row<DT>(p.q_out, (((long)b * p.T + n0 + i) * p.HQ + h) * kD, l, x);
        continue;
      }
      const int t = (P0 + i) & 63;
      const MxRow r = quantize_row(x);
      if (page >= 0) {
        *(uint32_t *)(p.kp + blk * kMxCodes + mx_k_off(t, l)) = r.code[0];
        *(uint32_t *)(p.kp + blk * kMxCodes + mx_k_off(t, l + 8)) = r.code[1];
        if ((l & 3) == 0) {
          uint8_t *s = p.ks + blk * kMxScales + (l >> 2) * kPage + t;
          s[0] = (uint8_t)r.byte[0];
          s[2 * kPage] = (uint8_t)r.byte[1];
        }
      }
      if (p.k_values) {
        held_row(r, x);
        store_row<DT>(p.k_values, (((long)b * p.T + n0 + i) * p.HKV + h) * kD, l, x);
      }
    }
    return;
  }
  const int t = P0 & 63;
  MxRow r[2] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (is[i]) {
      float x[16];
      row_values<DT>(w[i], x);
      r[i] = quantize_row(x);
      if (p.v_values) {
        held_row(r[i], x);
        store_row<DT>(p.v_values, (((long)b * p.T + n0 + i) * p.HKV + h) * kD, l, x);
      }
    }
  if (page < 0) return;
  uint8_t *c = p.vp + blk * kMxCodes;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    uint8_t old[8];
    if (!is[0] || !is[1])
#pragma unroll
      for (int i = 0; i < 8; ++i) old[i] = c[mx_v_off(64 * hf + 8 * l + i, t)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = (r[0].code[hf] >> (4 * i)) & 15u, up = (r[1].code[hf] >> (4 * i)) & 15u;
      c[mx_v_off(64 * hf + 8 * l + i, t)] =
          (uint8_t)(is[0] && is[1] ? lo | up << 4 : (is[0] ? (old[i] & 0xf0u) | lo : (old[i] & 0x0fu) | up << 4));
    }
    if ((l & 3) == 0) {
      uint8_t *s = p.vs + blk * kMxScales + (2 * hf + (l >> 2)) * kPage + t;
      if (is[0]) s[0] = (uint8_t)r[0].byte[hf];
      if (is[1]) s[1] = (uint8_t)r[1].byte[hf];
    }
  }
}

template <int DT, int TURN>
static void launch_append(MxAppendParams &p, hipStream_t st) {
  const int units = (TURN == kTurnNone ? 0 : p.HQ) + p.HKV + (p.v ? p.HKV : 0);
  if (mx_by_tiles(p.B, p.T, units, TURN != kTurnNone)) {
    p.tiles = page_tiles(p.T);
    const long x = (long)p.B * p.tiles, n = (2l * (units - (p.v ? p.HKV : 0)) + (p.v ? 4l * p.HKV : 0) + 3) / 4;
    hipLaunchKernelGGL((mxfp4_append_tiles_kernel<DT, TURN>), dim3((unsigned)x, (unsigned)mx_tile_splits(x, n, device_cus())), dim3(256), 0, st,
                       p);
  } else {
    p.tiles = p.T / 2 + 1;
    hipLaunchKernelGGL((mxfp4_append_tokens_kernel<DT, TURN>), dim3((unsigned)((long)p.B * p.tiles), (unsigned)((units + 31) / 32)),
                       dim3(256), 0, st, p);
  }
}
template <int DT>
static void launch_append(MxAppendParams &p, int turn, hipStream_t st) {
  if (turn == kTurnHalf) launch_append<DT, kTurnHalf>(p, st);
  else if (turn == kTurnAdjacent) launch_append<DT, kTurnAdjacent>(p, st);
  else launch_append<DT, kTurnNone>(p, st);
}

// ---------------------------------------------------------------------------
// read-back: a wave takes 32 tokens of a head's K, or 16 of its V, as the tiles' append does
// ---------------------------------------------------------------------------
struct MxReadParams {
  const uint8_t *kp, *ks, *vp, *vs;
  const int32_t *bt, *lens;
  int bt_stride, num_pages, T, HKV, tiles;
  void *k, *v;
};
template <int DT>
__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const MxReadParams p) {
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x / p.tiles, pg = blockIdx.x % p.tiles, u = blockIdx.y * 4 + wv;
  if (u >= 6 * p.HKV) return;
  const int len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T, n = len - pg * kPage;  // of the page's tokens
  int id = p.bt[(size_t)b * p.bt_stride + pg];
  id = (unsigned)id < (unsigned)p.num_pages ? id : 0;
  const long row0 = (long)b * p.T + pg * kPage;
  if (u < 2 * p.HKV) {
    const int h = u >> 1, l = lane & 7, m = 8 * (u & 1) + (lane >> 3);
    const size_t blk = (size_t)id * p.HKV + h;
    uint32_t c[4][2], s[2] = {0, 0};
    if (n > 0) {
#pragma unroll
      for (int tau = 0; tau < 4; ++tau) {
        c[tau][0] = *(const uint32_t *)(p.kp + blk * kMxCodes + mx_k_off(4 * m + tau, l));
        c[tau][1] = *(const uint32_t *)(p.kp + blk * kMxCodes + mx_k_off(4 * m + tau, l + 8));
      }
      s[0] = *(const uint32_t *)(p.ks + blk * kMxScales + (l >> 2) * kPage + 4 * m);
      s[1] = *(const uint32_t *)(p.ks + blk * kMxScales + (2 + (l >> 2)) * kPage + 4 * m);
    }
#pragma unroll
    for (int tau = 0; tau < 4; ++tau) {
      const int t = 4 * m + tau;
      float x[16] = {};
      if (t < n) {
        const MxRow r = {{c[tau][0], c[tau][1]}, {(int)((s[0] >> (8 * tau)) & 0xffu), (int)((s[1] >> (8 * tau)) & 0xffu)}};
        held_row(r, x);
      }
      store_row<DT>(p.k, ((row0 + t) * p.HKV + h) * kD, l, x);
    }
    return;
  }
  const int h = (u - 2 * p.HKV) >> 2, g = (u - 2 * p.HKV) & 3, o = lane >> 5, cq = lane & 31, t0 = 16 * g + 8 * o;
  const size_t blk = (size_t)id * p.HKV + h;
  uint32_t c[4];
  uint2 s = make_uint2(0, 0);
  if (n > 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = *(const uint32_t *)(p.vp + blk * kMxCodes + mx_v_off(4 * cq + e, t0));
    s = *(const uint2 *)(p.vs + blk * kMxScales + (cq >> 3) * kPage + t0);
  }
  float y[4][8];
#pragma unroll
  for (int e = 0; e < 4; ++e) mx_values8(n > 0 ? c[e] : 0u, 1.f, y[e]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = value_factor(((i < 4 ? s.x : s.y) >> (8 * (i & 3))) & 0xffu);
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = t0 + i < n ? y[e][i] * f : 0.f;
    store_values<DT, 4>(p.v, ((size_t)(row0 + t0 + i) * p.HKV + h) * kD + 4 * cq, x);
  }
}

}  // namespace ffa

#define FFA_BAD(msg) return ffa_set_error_internal(FFA_E_INVALID, msg)
#define FFA_NO(msg) return ffa_set_error_internal(FFA_E_UNSUPPORTED, msg)

extern "C" int ffa_mxfp4_append(const ffa_mxfp4_append_args *a, void *stream) {
  using namespace ffa;
  if (!a) FFA_BAD("null args");
  if (a->dtype != FFA_DT_F16 && a->dtype != FFA_DT_BF16 && a->dtype != FFA_DT_F32) FFA_BAD("rows must be fp16, bf16 or fp32");
  if (a->B <= 0 || a->T <= 0 || a->HKV <= 0 || a->HQ < 0) FFA_BAD("bad dims");
  if (a->bt_stride <= 0 || a->num_pages <= 0) FFA_BAD("empty block table or pool");
  if (!a->k || !a->pos || !a->block_table || !a->k_pages || !a->k_scale || (a->v && (!a->v_pages || !a->v_scale)))
    FFA_BAD("null pointer");
  if (a->HQ > 0 && (!a->q || !a->q_out || !a->pairs)) FFA_BAD("q is turned: it needs q_out and pairs");
  if (a->pairs && a->positions && a->axes <= 0) FFA_BAD("positions need an axis");
  if (!a->v && a->v_values) FFA_BAD("v_values without v");
  const int es = a->dtype == FFA_DT_F32 ? 4 : 2;
  const unsigned long off = (unsigned long)(a->k_batch | a->k_token | a->k_head | (a->v ? a->v_batch | a->v_token | a->v_head : 0) |
                                            (a->HQ ? a->q_batch | a->q_token | a->q_head : 0)) * es;
  const uintptr_t al = (uintptr_t)a->k | (uintptr_t)a->v | (a->HQ ? (uintptr_t)a->q | (uintptr_t)a->q_out : 0) |
                       (uintptr_t)a->k_values | (uintptr_t)a->v_values | (uintptr_t)a->k_pages | (uintptr_t)a->k_scale |
                       (uintptr_t)a->v_pages | (uintptr_t)a->v_scale;
  if ((off | al) & 15) FFA_BAD("rows and pools must start at multiples of 16 bytes");
  const long wgs = (long)a->B * (mx_by_tiles(a->B, a->T, a->HQ + (a->v ? 2 : 1) * a->HKV, a->pairs) ? page_tiles(a->T) : a->T / 2 + 1);
  if (a->T > 1 << 30 || a->HKV > 1 << 16 || a->HQ > 1 << 20 || wgs > kMostWorkgroups) FFA_NO("more workgroups than a grid holds");
  MxAppendParams p = {};
  p.rope = RopeParams{a->pairs, a->positions, a->pos_axis, a->pos_batch, a->positions64, a->axes, 0};
  p.k = a->k;
  p.v = a->v;
  p.q = a->q;
  p.k_batch = a->k_batch;
  p.k_token = a->k_token;
  p.k_head = a->k_head;
  p.v_batch = a->v_batch;
  p.v_token = a->v_token;
  p.v_head = a->v_head;
  p.q_batch = a->q_batch;
  p.q_token = a->q_token;
  p.q_head = a->q_head;
  p.B = a->B;
  p.T = a->T;
  p.HKV = a->HKV;
  p.HQ = a->HQ;
  p.pos = a->pos;
  p.bt = a->block_table;
  p.bt_stride = a->bt_stride;
  p.num_pages = a->num_pages;
  p.kp = a->k_pages;
  p.ks = a->k_scale;
  p.vp = a->v_pages;
  p.vs = a->v_scale;
  p.q_out = a->q_out;
  p.k_values = a->k_values;
  p.v_values = a->v_values;
  const int turn = a->pairs ? (a->adjacent ? kTurnAdjacent : kTurnHalf) : kTurnNone;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == FFA_DT_F32) launch_append<2>(p, turn, st);
  else if (a->dtype == FFA_DT_BF16) launch_append<1>(p, turn, st);
  else launch_append<0>(p, turn, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FFA_OK : ffa_set_error_internal(FFA_E_LAUNCH, hipGetErrorString(e));
}

extern "C" int ffa_mxfp4_dequant(const uint8_t *k_pages, const uint8_t *k_scale, const uint8_t *v_pages, const uint8_t *v_scale,
                                 const int32_t *block_table, int bt_stride, int num_pages, const int32_t *seq_lens, int B, int T,
                                 int HKV, void *k_out, void *v_out, int out_dtype, void *stream) {
  using namespace ffa;
  if (B <= 0 || T <= 0 || HKV <= 0 || T % kPage) FFA_BAD("bad dims (T is a multiple of 64)");
  if (bt_stride <= 0 || num_pages <= 0 || (long)bt_stride * kPage < T) FFA_BAD("block table has fewer than T/64 columns");
  if (!k_pages || !k_scale || !v_pages || !v_scale || !block_table || !k_out || !v_out) FFA_BAD("null pointer");
  if (out_dtype != FFA_DT_F16 && out_dtype != FFA_DT_BF16 && out_dtype != FFA_DT_F32) FFA_BAD("out dtype must be fp16, bf16 or fp32");
  const uintptr_t al = (uintptr_t)k_pages | (uintptr_t)k_scale | (uintptr_t)v_pages | (uintptr_t)v_scale | (uintptr_t)k_out |
                       (uintptr_t)v_out;
  if (al & 15) FFA_BAD("outputs and pools must be multiples of 16 bytes");
  if (HKV > 32768 || (long)B * (T / kPage) > kMostWorkgroups) FFA_NO("more workgroups than a grid holds");
  MxReadParams p = {k_pages, k_scale, v_pages, v_scale, block_table, seq_lens, bt_stride, num_pages, T, HKV, T / kPage, k_out, v_out};
  const dim3 grid((unsigned)((long)B * p.tiles), (unsigned)((6 * HKV + 3) / 4));
  const hipStream_t st = (hipStream_t)stream;
  if (out_dtype == FFA_DT_F32) hipLaunchKernelGGL(mxfp4_dequant_kernel<2>, grid, dim3(256), 0, st, p);
  else if (out_dtype == FFA_DT_BF16) hipLaunchKernelGGL(mxfp4_dequant_kernel<1>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(mxfp4_dequant_kernel<0>, grid, dim3(256), 0, st, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FFA_OK : ffa_set_error_internal(FFA_E_LAUNCH, hipGetErrorString(e));
}
