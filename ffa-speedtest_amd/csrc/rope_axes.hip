// Rotary positions with several axes on given queries and keys, and their gradient (the rotation back).
//
// Bound by the rows' bytes, read once and written once: a token's 64 sines and cosines (64-bit angles, some 60
// instructions each) are computed once for all of its heads.  A workgroup of 256 threads takes `tokens` tokens and
// their rows, 32 at a time; calls of few tokens are one token and up to 32 rows a workgroup.
#include "rope_axes.h"
#include "routes.h"

extern "C" int ffa_set_error_internal(int code, const char *msg);

namespace ffa {

struct RopeRows {
  const void *x;
  void *out;
  long batch, token, head, out_batch, out_token, out_head;
};
struct RopeAxesParams {
  RopeParams rope;
  RopeRows q, k;
  int B, T, HQ, HKV, tokens;
};

constexpr int kRopeTokens = 16;  // of a workgroup, at most

template <int DT, int TURN>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeAxesParams p) {
  __shared__ float2 cs[kRopeTokens][64];
  const long n0 = (long)blockIdx.x * p.tokens, all = (long)p.B * p.T;
  const int count = (int)min((long)p.tokens, all - n0);
  const int H = p.HQ + p.HKV, rows = count * H, per = (rows + gridDim.y - 1) / gridDim.y;
  const int first = blockIdx.y * per, end = min(first + per, rows);
  const int l = threadIdx.x & 7;
  constexpr int kRows = 2;  // under way at a time
  for (int i = threadIdx.x; i < count * 64; i += 256) {
    const long n = n0 + (i >> 6);
    const int b = (int)(n / p.T), t = (int)(n - (long)b * p.T);
    cs[i >> 6][i & 63] = rope_angle(p.rope, i & 63, b, t, t);
  }
  __syncthreads();
  for (int r0 = first + (threadIdx.x >> 3); r0 < end; r0 += 32 * kRows) {
    Row16<DT> w[kRows];
    void *out[kRows];
    long at[kRows];
    int tok[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = min(r0 + 32 * i, end - 1);
      tok[i] = r / H;
      const int h = r - tok[i] * H;
      const long n = n0 + tok[i];
      const int b = (int)(n / p.T), t = (int)(n - (long)b * p.T);
      const bool q = h < p.HQ;
      const RopeRows &x = q ? p.q : p.k;
      const int hh = q ? h : h - p.HQ;
      w[i] = load_row<DT>(x.x, b * x.batch + t * x.token + hh * x.head, l);
      out[i] = x.out;
      at[i] = b * x.out_batch + t * x.out_token + hh * x.out_head;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (r0 + 32 * i >= end) break;
      float x[16];
      row_values<DT>(w[i], x);
      rope_turn<TURN>(cs[tok[i]], l, x);
      store_row<DT>(out[i], at[i], l, x);
    }
  }
}

template <int DT>
static void launch_rope(const RopeAxesParams &p, bool adjacent, dim3 grid, hipStream_t st) {
  if (adjacent) hipLaunchKernelGGL((rope_axes_kernel<DT, kTurnAdjacent>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((rope_axes_kernel<DT, kTurnHalf>), grid, dim3(256), 0, st, p);
}

}  // namespace ffa

#define FFA_BAD(msg) return ffa_set_error_internal(FFA_E_INVALID, msg)
#define FFA_NO(msg) return ffa_set_error_internal(FFA_E_UNSUPPORTED, msg)
extern "C" int ffa_rope_axes(const ffa_rope_axes_args *a, void *stream) {
  using namespace ffa;
  if (!a) FFA_BAD("null args");
  if (a->dtype != FFA_DT_F16 && a->dtype != FFA_DT_BF16 && a->dtype != FFA_DT_F32) FFA_BAD("rows must be fp16, bf16 or fp32");
  if (a->B <= 0 || a->T <= 0 || a->HQ <= 0 || a->HKV < 0) FFA_BAD("bad dims");
  if (!a->q || !a->q_out || !a->pairs || !a->positions || (a->HKV > 0 && (!a->k || !a->k_out))) FFA_BAD("null pointer");
  if (a->axes <= 0) FFA_BAD("positions need an axis");
  const int H = a->HQ + a->HKV;
  if (H < 0 || H > 1 << 20) FFA_NO("more than 2^20 heads");
  const long all = (long)a->B * a->T;
  const int es = a->dtype == FFA_DT_F32 ? 4 : 2;
  const unsigned long off =
      (unsigned long)(a->q_batch | a->q_token | a->q_head | a->q_out_batch | a->q_out_token | a->q_out_head |
                      (a->HKV ? a->k_batch | a->k_token | a->k_head | a->k_out_batch | a->k_out_token | a->k_out_head : 0)) * es;
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->q_out | (a->HKV ? (uintptr_t)a->k | (uintptr_t)a->k_out : 0);
  if ((off | al) & 15) FFA_BAD("rows must start at multiples of 16 bytes");
  RopeAxesParams p = {};
  p.rope = RopeParams{a->pairs, a->positions, a->pos_axis, a->pos_batch, a->positions64, a->axes, a->inverse};
  p.q = RopeRows{a->q, a->q_out, a->q_batch, a->q_token, a->q_head, a->q_out_batch, a->q_out_token, a->q_out_head};
  p.k = RopeRows{a->k, a->k_out, a->k_batch, a->k_token, a->k_head, a->k_out_batch, a->k_out_token, a->k_out_head};
  p.B = a->B;
  p.T = a->T;
  p.HQ = a->HQ;
  p.HKV = a->HKV;
  p.tokens = rope_tokens(all, kRopeTokens);
  const long tiles = (all + p.tokens - 1) / p.tokens;
  if (tiles > kMostWorkgroups) FFA_NO("more than 2^28 tokens");
  const dim3 grid((unsigned)tiles, (unsigned)rope_splits(tiles, (long)p.tokens * H));
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == FFA_DT_F32) launch_rope<2>(p, a->adjacent, grid, st);
  else if (a->dtype == FFA_DT_BF16) launch_rope<1>(p, a->adjacent, grid, st);
  else launch_rope<0>(p, a->adjacent, grid, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FFA_OK : ffa_set_error_internal(FFA_E_LAUNCH, hipGetErrorString(e));
}
