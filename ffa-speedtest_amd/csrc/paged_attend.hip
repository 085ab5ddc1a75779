// Exact attention over the paged caches (paged_attend.h): the join of the partials, the launch plan and the C entry.
#include "paged_attend.h"

extern "C" int ffa_set_error_internal(int code, const char *msg);

namespace ffa {

// ---------------------------------------------------------------------------
// Join of the partials: WPR waves per row (4, or 1 where rows are many: a workgroup then takes four of them), each
// with four slots' loads under way at a time
// ---------------------------------------------------------------------------
template <int WPR>
__global__ __launch_bounds__(256) void paged_attend_join_kernel(const AttendParams p, int rows) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int row = WPR == 4 ? blockIdx.x : 4 * blockIdx.x + wv;
  if (row >= rows) return;  // (whole workgroups only where waves meet)
  const int i = (row / p.HQ) % p.L, b = row / (p.HQ * p.L);
  const bool sees = row_limit(p, b, i) > 0;
  const int sp = shared_pages_of(p, b), own = max((seq_len_of(p, b) + kPage - 1) / kPage - sp, 0);
  const int na = p.shared_slots ? min((sp + p.shared_ppw - 1) / p.shared_ppw, p.shared_slots) : 0;
  int nb = 0;
  if (p.own_slots) {
    const int per = own_range(p, own);
    nb = min((own + per - 1) / per, p.own_slots);
  }
  const float2 *ml = (const float2 *)p.part_ml + (size_t)row * p.nslots;
  const float *po = p.part_o + (size_t)row * p.nslots * kD;
  float m = kNoMax, l = 0.f;
  float2 o = make_float2(0.f, 0.f);
  const int slots = sees ? na + nb : 0;
  for (int s0 = WPR == 4 ? wv : 0; s0 < slots; s0 += 4 * WPR) {
    float2 x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = min(s0 + WPR * k, slots - 1), slot = s < na ? s : p.shared_slots + s - na;
      x[k] = ml[slot];
      y[k] = *(const float2 *)(po + (size_t)slot * kD + 2 * lane);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < 4; ++k) mn = fmaxf(mn, x[k].x);
    const float fo = fmaxf(exp2_hw(m - mn), kLeast);
    m = mn;
    l *= fo;
    o.x *= fo;
    o.y *= fo;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (s0 + WPR * k < slots) {
        const float f = fmaxf(exp2_hw(x[k].x - mn), kLeast);
        l += x[k].y * f;
        o.x += y[k].x * f;
        o.y += y[k].y * f;
      }
  }
  if constexpr (WPR == 4) {
    __shared__ float s_m[4], s_l[4];
    __shared__ float s_o[4][kD];
    if (lane == 0) {
      s_m[wv] = m;
      s_l[wv] = l;
    }
    *(float2 *)&s_o[wv][2 * lane] = o;
    __syncthreads();
    if (wv != 0) return;
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    l = o.x = o.y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = fmaxf(exp2_hw(s_m[w] - m), kLeast);
      l += s_l[w] * f;
      o.x += s_o[w][2 * lane] * f;
      o.y += s_o[w][2 * lane + 1] * f;
    }
  }
  const float inv = 1.f / l, x = sees ? o.x * inv : 0.f, y = sees ? o.y * inv : 0.f;
  ((uint32_t *)p.out)[(size_t)row * (kD / 2) + lane] = p.out_bf16 ? pk_bf16_bits(x, y) : pk_f16_bits(x, y);
}

// Launch plan of a call: page ranges of the shared and of the own pages
struct AttendPlan {
  int shared_slots, shared_ppw, own_slots, nslots;
  int shared_kind, shared_blocks, own_kind, own_blocks;
  bool both;  // one launch of 256-row workgroups over shared pages and of few-row ones over own pages
};

static AttendPlan attend_plan(const ffa_paged_attend_args *a, int cus) {
  AttendPlan pl = {};
  if (cus <= 0) cus = 256;
  const long LG = (long)a->L * (a->HQ / a->HKV);
  long units = 0, rows = 0;
  int most = 0, least = a->ngroups > 0 ? a->group_pages_host[0] : 0;  // shared pages
  for (int g = 0; g < a->ngroups; ++g) {
    const long n = a->group_start_host[g + 1] - a->group_start_host[g];
    const int gp = a->group_pages_host[g];
    if (gp > 0 && n * LG > rows) rows = n * LG;
    if (gp > most) most = gp;
    if (gp < least) least = gp;
  }
  const int own = (a->T + kPage - 1) / kPage - least;
  const long heads = (long)a->B * a->HKV;
  pl.own_kind = attend_own_kind(LG, heads, own, cus);
  pl.own_blocks = (int)attend_blocks(LG, pl.own_kind);
  if (own > 0) {
    int ppw;  // of the longest sequence
    page_ranges((long)own * heads * pl.own_blocks, own, attend_resident(pl.own_kind, cus), ppw, pl.own_slots);
    if (attend_one_range(LG, heads, own, cus)) pl.own_slots = 1;
  }
  if (most > 0) {
    pl.shared_kind = attend_kind(rows);
    pl.shared_blocks = (int)attend_blocks(rows, pl.shared_kind);
    for (int g = 0; g < a->ngroups; ++g) {
      const long n = a->group_start_host[g + 1] - a->group_start_host[g];
      units += (long)a->group_pages_host[g] * a->HKV * attend_blocks(n * LG, pl.shared_kind);
    }
    long want = attend_resident(pl.shared_kind, cus);
    pl.both = attend_both(pl.shared_kind, pl.own_kind, a->own_pages_host, a->B) && own > 0 &&
              heads * pl.own_slots < 1l << 30;
    if (pl.both) want = attend_shared_wgs(units, a->own_pages_host * a->HKV, cus);
    page_ranges(units, most, want, pl.shared_ppw, pl.shared_slots);
    pl.both = pl.both && (long)a->HKV * pl.shared_blocks * pl.shared_slots * a->ngroups < 1l << 30;
  }
  pl.nslots = pl.shared_slots + pl.own_slots;
  if (pl.shared_slots == 0 && pl.own_slots <= 1) {  // one range: no partials
    pl.own_slots = 1;
    pl.nslots = 0;
  }
  return pl;
}

static int attend_check(const ffa_paged_attend_args *a) {
#define FFA_BAD(msg) return ffa_set_error_internal(FFA_E_INVALID, msg)
#define FFA_NO(msg) return ffa_set_error_internal(FFA_E_UNSUPPORTED, msg)
  if (!a) FFA_BAD("null args");
  if (a->B <= 0 || a->T <= 0 || a->L <= 0 || a->HQ <= 0 || a->HKV <= 0) FFA_BAD("bad dims");
  if (a->HQ % a->HKV) FFA_BAD("HQ must be a multiple of HKV");
  if (a->B > 65535 || a->HKV > 65535) FFA_NO("B and HKV are grid dimensions");
  if (a->T > 1 << 30) FFA_NO("T above 2^30 tokens");
  if (!(a->q_dtype == FFA_DT_F16 || a->q_dtype == FFA_DT_BF16)) FFA_BAD("q must be fp16 or bf16");
  if (!(a->v_dtype == FFA_DT_F16 || a->v_dtype == FFA_DT_BF16)) FFA_BAD("v dtype");
  if (a->format < FFA_PAGES_Q2 || a->format > FFA_PAGES_NF4) FFA_BAD("page format");
  if (!(a->res_dtype == FFA_DT_FP8_E4M3 || a->res_dtype == FFA_DT_FP8_E5M2 || a->res_dtype == FFA_DT_NONE))
    FFA_BAD("residual dtype must be fp8 or none");
  if (a->bt_stride <= 0 || a->num_pages <= 0) FFA_BAD("empty block table or pool");
  if ((long)a->bt_stride * kPage < a->T) FFA_BAD("block table has fewer than ceil(T/64) columns");
  if (!a->q || !a->k || !a->k_scale || !a->v || !a->block_table || !a->out) FFA_BAD("null pointer");
  if (a->format == FFA_PAGES_Q2 && !a->k_zero) FFA_BAD("2-bit pages need k_zero");
  if (a->res_dtype != FFA_DT_NONE && !a->k_residual) FFA_BAD("null residual");
  if ((long)a->B * a->L * a->HQ > 1l << 30) FFA_NO("more than 2^30 query rows");
  if (a->ngroups < 0 || a->ngroups > a->B) FFA_BAD("ngroups must be within [0, B]");
  if (a->ngroups > 0) {
    if (!a->group_start || !a->group_pages || !a->seq_group || !a->group_start_host || !a->group_pages_host)
      FFA_BAD("groups need their arrays");
    if (a->group_start_host[0] != 0 || a->group_start_host[a->ngroups] != a->B) FFA_BAD("groups must cover the batch");
    for (int g = 0; g < a->ngroups; ++g) {
      if (a->group_start_host[g + 1] <= a->group_start_host[g]) FFA_BAD("a group without sequences");
      if (a->group_pages_host[g] < 0 || a->group_pages_host[g] > a->bt_stride) FFA_BAD("shared pages exceed the block table");
    }
  }
  const uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out |
                       (uintptr_t)a->k_residual | (uintptr_t)a->k_scale | (uintptr_t)a->k_zero;
  if (al & 15) FFA_BAD("q, out and the pools must be multiples of 16 bytes");
  return FFA_OK;
}

}  // namespace ffa

extern "C" size_t ffa_paged_attend_scratch(const ffa_paged_attend_args *a) {
  using namespace ffa;
  if (attend_check(a) != FFA_OK) return 0;
  return (size_t)a->B * a->L * a->HQ * attend_plan(a, device_cus()).nslots * (kD + 2) * sizeof(float);
}

extern "C" int ffa_paged_attend(const ffa_paged_attend_args *a, void *stream) {
  using namespace ffa;
  const int bad = attend_check(a);
  if (bad != FFA_OK) return bad;
  const AttendPlan pl = attend_plan(a, device_cus());
  const size_t rows = (size_t)a->B * a->L * a->HQ;
  if (a->scratch_bytes < rows * pl.nslots * (kD + 2) * sizeof(float) || (pl.nslots && !a->scratch))
    FFA_BAD("scratch below ffa_paged_attend_scratch()");
  if ((uintptr_t)a->scratch & 15) FFA_BAD("scratch must be a multiple of 16 bytes");
  AttendParams p = {};
  p.q = a->q;
  p.k = a->k;
  p.ks = (const uint8_t *)a->k_scale;
  p.kz = (const uint8_t *)a->k_zero;
  p.kr = a->k_residual;
  p.v = (const uint8_t *)a->v;
  p.bt = a->block_table;
  p.seq_lens = a->seq_lens;
  p.q_lens = a->q_lens;
  p.group_start = a->group_start;
  p.group_pages = a->group_pages;
  p.seq_group = a->seq_group;
  p.out = a->out;
  p.part_o = (float *)a->scratch;
  p.part_ml = p.part_o + rows * pl.nslots * kD;
  p.bt_stride = a->bt_stride;
  p.num_pages = a->num_pages;
  p.ngroups = a->ngroups;
  p.B = a->B;
  p.T = a->T;
  p.L = a->L;
  p.HQ = a->HQ;
  p.HKV = a->HKV;
  p.G = a->HQ / a->HKV;
  p.q_bf16 = p.out_bf16 = a->q_dtype == FFA_DT_BF16;
  p.scale2 = a->scale * kLog2e;
  p.nslots = pl.nslots;
  p.shared_slots = pl.shared_slots;
  p.shared_ppw = pl.shared_ppw;
  p.own_slots = pl.own_slots;
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](int kind, int slots, int blocks, int sets, int own) {
    const AttendLaunch l = {kind, slots, blocks, sets, own, a->res_dtype, a->v_dtype, st};
    (a->format == FFA_PAGES_Q2 ? attend_q2 : (a->format == FFA_PAGES_NVFP4 ? attend_nvfp4 : attend_nf4))(p, l);
  };
  if (pl.both) {
    p.nshared = a->ngroups;
    p.shared_blocks = pl.shared_blocks;
    p.shared_wgs = a->HKV * pl.shared_blocks * pl.shared_slots * a->ngroups;
    launch(pl.shared_kind, pl.shared_slots, pl.shared_blocks, a->ngroups, pl.own_kind);
  } else if (pl.shared_slots > 0 && pl.own_slots > 0 && pl.shared_kind == pl.own_kind && a->ngroups + a->B <= 65535) {
    p.nshared = a->ngroups;  // both in the grid of one kernel
    launch(pl.own_kind, pl.shared_slots > pl.own_slots ? pl.shared_slots : pl.own_slots,
           pl.shared_blocks > pl.own_blocks ? pl.shared_blocks : pl.own_blocks, a->ngroups + a->B, -1);
  } else {
    if (pl.shared_slots > 0) {
      p.nshared = a->ngroups;
      launch(pl.shared_kind, pl.shared_slots, pl.shared_blocks, a->ngroups, -1);
    }
    p.nshared = 0;
    if (pl.own_slots > 0) launch(pl.own_kind, pl.own_slots, pl.own_blocks, a->B, -1);
  }
  if (pl.nslots > 0 && !join_by_wave((long)rows))
    hipLaunchKernelGGL(paged_attend_join_kernel<4>, dim3((unsigned)rows), dim3(256), 0, st, p, (int)rows);
  else if (pl.nslots > 0)
    hipLaunchKernelGGL(paged_attend_join_kernel<1>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p, (int)rows);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FFA_OK : ffa_set_error_internal(FFA_E_LAUNCH, hipGetErrorString(e));
}
#undef FFA_BAD
#undef FFA_NO
