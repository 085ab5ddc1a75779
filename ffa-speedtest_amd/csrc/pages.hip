// Management of the pages of one or several caches that share page ids: copy, fork, extend, free, compact.
//
// refs[P] counts the block-table rows that hold each page; a page is free while its count is 0.  New pages are the
// lowest free ids, given in (row, column) order, so that every result is a function of the counts and tables alone
// (one workgroup ranks the free pages; counts are changed by integer atomics, whose order does not show).
//
// What bounds these calls is the copying, 2 x the bytes of the pages (a 2-bit page of 8 KV heads: 221 KB a layer);
// for a few pages it is the two launches.  All pools of all layers are copied by one launch: its workgroups walk
// (page pair, 16 KB piece of a pool's page), wide loads of a piece before its stores.
#include "ffa_common.h"
#include "ffa_mi355x.h"
#include "routes.h"

extern "C" int ffa_set_error_internal(int code, const char *msg);

namespace ffa {

int device_cus();

constexpr int kPageTokens = 64;
constexpr int kMaxPools = 128;      // pools of one launch (kernel arguments); more take several
constexpr uint32_t kPiece = 16384;  // bytes of a pool's page copied by a workgroup at a time
constexpr int kMaxTables = 8;
enum { kErrFull = 1, kErrRow = 2, kErrPage = 4 };

struct PoolSet {
  uint8_t *ptr[kMaxPools];
  uint32_t bytes[kMaxPools];       // of one page
  uint32_t piece0[kMaxPools + 1];  // pieces of the pools before this one
  int npools, num_pages;
};

// piece c of the pools' pages src -> dst
__device__ __forceinline__ void copy_piece(const PoolSet &s, uint32_t c, int src, int dst) {
  int lo = 0, hi = s.npools - 1;  // the pool whose pieces hold c
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.piece0[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  const size_t bytes = s.bytes[lo];
  const uint32_t off = (c - s.piece0[lo]) * kPiece;
  const uint32_t n = min((uint32_t)bytes - off, kPiece);
  const uint8_t *from = s.ptr[lo] + (size_t)src * bytes + off;
  uint8_t *to = s.ptr[lo] + (size_t)dst * bytes + off;
  const uint32_t at = 16 * threadIdx.x;
  if (n == kPiece) {
    u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *(const u32x4 *)(from + at + 4096 * i);
    // stores non-temporal, loads not (siblings copy the same page): fork of 64 children in 8 layers 55 -> 47 us,
    // compaction of 1024 pages of 4 layers 119 -> 96 (loads alone 89, but fork 55; both 107)
#pragma unroll
    for (int i = 0; i < 4; ++i) __builtin_nontemporal_store(w[i], (u32x4 *)(to + at + 4096 * i));
  } else {
    for (uint32_t x = at; x < n; x += 4096) *(uint4 *)(to + x) = *(const uint4 *)(from + x);
  }
}

__global__ __launch_bounds__(256) void pages_copy_kernel(const PoolSet s, const int32_t *src, const int32_t *dst,
                                                         int n) {
  const uint32_t pieces = s.piece0[s.npools];
  const uint64_t total = (uint64_t)n * pieces;
  for (uint64_t x = blockIdx.x; x < total; x += gridDim.x) {
    const int i = (int)(x / pieces);
    const int a = src[i], b = dst[i];
    if ((unsigned)a < (unsigned)s.num_pages && (unsigned)b < (unsigned)s.num_pages) copy_piece(s, (uint32_t)(x - (uint64_t)i * pieces), a, b);
  }
}

// ---------------------------------------------------------------------------
// Ranks over one workgroup of 1024 threads
// ---------------------------------------------------------------------------
// sum of x over the threads before this one; total: over all.  Every thread calls it.
__device__ __forceinline__ int block_rank(int x, int &total) {
  __shared__ int s_wave[16];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 63) s_wave[wv] = sum;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wv ? s_wave[w] : 0;
    total += s_wave[w];
  }
  __syncthreads();
  return before + sum - x;
}

struct AllocArgs {
  int32_t *refs, *table;  // table: rows that get pages (the children's, or the sequences')
  const int32_t *parent_table, *seq_lens, *parents;
  int32_t *scratch;  // [0] error bits, [1] pages needed, [2 ..] ids
  int32_t *errors;
  int P, rows, cols, B, tokens;  // tokens < 0: fork
  int checked;                   // fork: pages_fork_check_kernel left a word per row in scratch[2 ..]
};

// pages that row r gets: `cnt` from column `first` on.  Returns false for a row that cannot be served (before any page is
// given out; afterwards counts have grown, and only `first` and `cnt` are read).
__device__ __forceinline__ bool row_need(const AllocArgs &a, int r, int &first, int &cnt) {
  first = cnt = 0;
  if (a.tokens < 0) {
    const int par = a.parents[r];
    if ((unsigned)par >= (unsigned)a.B) return false;
    const int len = a.seq_lens[par];
    if (len < 0 || len > a.cols * kPageTokens) return false;
    first = len / kPageTokens;
    cnt = len % kPageTokens ? 1 : 0;
    if (cnt == 0) return true;
    const int id = a.parent_table[(size_t)par * a.cols + first];
    return (unsigned)id < (unsigned)a.P && a.refs[id] > 0;
  }
  const int len = a.seq_lens[r];
  if (len < 0 || (long)len + a.tokens > (long)a.cols * kPageTokens) return false;
  first = (len + kPageTokens - 1) / kPageTokens;
  cnt = (len + a.tokens + kPageTokens - 1) / kPageTokens - first;
  if (len % kPageTokens == 0) return true;
  const int id = a.table[(size_t)r * a.cols + len / kPageTokens];  // the partial page, which the new tokens fill first
  return (unsigned)id < (unsigned)a.P && a.refs[id] > 0;
}

// Fork: whether the parent of row r holds its whole pages t, t + n, ..: inside the pool, counts above 0 (a free one could
// be given out as another's new page).  Rows that row_need refuses pass.
__device__ __forceinline__ bool whole_pages_held(const AllocArgs &a, int r, int t, int n) {
  const int par = a.parents[r];
  if ((unsigned)par >= (unsigned)a.B) return true;
  const int len = a.seq_lens[par];
  if (len < 0 || len > a.cols * kPageTokens) return true;
  const int32_t *from = a.parent_table + (size_t)par * a.cols;
  const int full = len / kPageTokens;
  int ok = 1;
#pragma unroll 4
  for (int j = t; j < full; j += n) {
    const int id = from[j], in = (unsigned)id < (unsigned)a.P;
    ok &= in & (a.refs[in ? id : 0] > 0);
  }
  return ok;
}

// the same by a workgroup per row (fork_check_apart)
__global__ __launch_bounds__(256) void pages_fork_check_kernel(const AllocArgs a) {
  const int bad = __syncthreads_or(!whole_pages_held(a, blockIdx.x, threadIdx.x, 256));
  if (threadIdx.x == 0) a.scratch[2 + blockIdx.x] = bad;
}

__global__ __launch_bounds__(1024) void pages_alloc_kernel(const AllocArgs a) {
  int need = 0, bad = 0, page = 0;
  if (a.tokens < 0 && !a.checked)
    for (int r = threadIdx.x >> 6; r < a.rows; r += 16) page |= !whole_pages_held(a, r, threadIdx.x & 63, 64);
  for (int base = 0; base < a.rows; base += 1024) {
    const int r = base + threadIdx.x;
    int first = 0, cnt = 0, sum;
    if (r < a.rows && !row_need(a, r, first, cnt)) bad = 1;
    if (r < a.rows && a.checked) page |= a.scratch[2 + r];
    block_rank(cnt, sum);
    need += sum;
  }
  bad = __syncthreads_or(bad);
  page = __syncthreads_or(page);  // behind every read of the rows' words: the ids go over them
  // the lowest free pages, in order: 16 counts a thread and step
  int found = 0;
  for (int base = 0; base < a.P && found < need; base += 16 * 1024) {
    const int p0 = base + 16 * (int)threadIdx.x;
    uint32_t free = 0;
    if (p0 + 16 <= a.P) {
      int4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *(const int4 *)(a.refs + p0 + 4 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        free |= (uint32_t)((w[i].x == 0) | (w[i].y == 0) << 1 | (w[i].z == 0) << 2 | (w[i].w == 0) << 3) << (4 * i);
    } else {
      for (int i = 0; i < 16 && p0 + i < a.P; ++i) free |= (uint32_t)(a.refs[p0 + i] == 0) << i;
    }
    int sum;
    int rank = found + block_rank(__builtin_popcount(free), sum);
    for (; free && rank < need; ++rank, free &= free - 1) a.scratch[2 + rank] = p0 + __builtin_ctz(free);
    found += sum;
  }
  __syncthreads();
  const int err = (bad ? kErrRow : 0) | (found < need ? kErrFull : 0) | (page ? kErrPage : 0);
  if (threadIdx.x == 0) {
    a.scratch[0] = err;
    a.scratch[1] = need;
    if (err) atomicOr(a.errors, err);
  }
  if (err) return;
  int given = 0;
  for (int base = 0; base < a.rows; base += 1024) {
    const int r = base + threadIdx.x;
    int first = 0, cnt = 0, sum;
    if (r < a.rows) row_need(a, r, first, cnt);
    const int at = given + block_rank(cnt, sum);
    for (int j = 0; j < cnt; ++j) {
      const int id = a.scratch[2 + at + j];
      a.table[(size_t)r * a.cols + first + j] = id;
      a.refs[id] = 1;
    }
    given += sum;
  }
}

// Fork: workgroup (0, child) writes the child's row and counts the pages it shares; the others copy the pieces of its
// partial page.  Where the allocation found an error every child's row is empty (-1) and nothing else changes.
__global__ __launch_bounds__(256) void pages_fork_kernel(const PoolSet s, const AllocArgs a, int tables) {
  const int r = blockIdx.y, par = a.parents[r];
  const bool ok = a.scratch[0] == 0;
  const int len = ok ? a.seq_lens[par] : 0, full = len / kPageTokens, part = len % kPageTokens ? 1 : 0;
  int32_t *row = a.table + (size_t)r * a.cols;
  const int32_t *from = a.parent_table + (size_t)(ok ? par : 0) * a.cols;
  if (tables) {
    if (blockIdx.x == 0) {
      for (int j = threadIdx.x; j < a.cols; j += 256) {
        if (part && j == full) continue;  // the new page's column
        int id = -1;
        if (j < full) {
          id = from[j];
          if ((unsigned)id < (unsigned)a.P) atomicAdd(&a.refs[id], 1);
        }
        row[j] = id;
      }
      return;
    }
  }
  if (!ok || !part) return;
  const int src = from[full], dst = row[full];
  const uint32_t pieces = s.piece0[s.npools];
  for (uint32_t c = blockIdx.x - (tables ? 1 : 0); c < pieces; c += gridDim.x - (tables ? 1 : 0)) copy_piece(s, c, src, dst);
}

// counts of the pages that the rows hold, plus or minus one for each time that a row holds it
__global__ __launch_bounds__(256) void pages_count_kernel(int32_t *refs, int P, const int32_t *table, int cols,
                                                          const int32_t *seq_lens, int step, int32_t *call, int32_t *errors) {
  const int r = blockIdx.y;
  const int len = seq_lens[r];
  const int n = (int)min((long)cols, ((long)max(len, 0) + kPageTokens - 1) / kPageTokens);
  bool bad = len < 0 || (long)len > (long)cols * kPageTokens;
  for (int j = blockIdx.x * 256 + threadIdx.x; j < n; j += 256 * gridDim.x) {
    const int id = table[(size_t)r * cols + j];
    if ((unsigned)id >= (unsigned)P) {
      bad = true;
    } else if (step > 0) {
      atomicAdd(&refs[id], 1);
    } else {
      // a page that is free already stays free: the step is taken back (no step that finds a count above 0 can follow
      // one that did not, so the result does not depend on their order)
      if (atomicSub(&refs[id], 1) <= 0) {
        atomicAdd(&refs[id], 1);
        bad = true;
      }
    }
  }
  if (bad) {
    atomicOr(errors, kErrPage);
    atomicOr(call, kErrPage);
  }
}

// ---------------------------------------------------------------------------
// Compaction: with n pages held, the i-th held page from id n on moves to the i-th free page below n.
// scratch: [0] moves, [1] n, src [P/2 + 1], dst [P/2 + 1], to [P] (for ids from n on: the page's new id or -1)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void pages_compact_plan_kernel(int32_t *refs, int P, int32_t *scratch) {
  int32_t *src = scratch + 2, *dst = src + P / 2 + 1, *to = dst + P / 2 + 1;
  auto held16 = [&](int p0) {
    uint32_t m = 0;
    if (p0 + 16 <= P) {
      int4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *(const int4 *)(refs + p0 + 4 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m |= (uint32_t)((w[i].x > 0) | (w[i].y > 0) << 1 | (w[i].z > 0) << 2 | (w[i].w > 0) << 3) << (4 * i);
    } else {
      for (int i = 0; i < 16 && p0 + i < P; ++i) m |= (uint32_t)(refs[p0 + i] > 0) << i;
    }
    return m;
  };
  int n = 0;
  for (int base = 0; base < P; base += 16 * 1024) {
    int sum;
    block_rank(__builtin_popcount(held16(base + 16 * (int)threadIdx.x)), sum);
    n += sum;
  }
  int holes = 0, moves = 0;
  for (int base = 0; base < P; base += 16 * 1024) {
    const int p0 = base + 16 * (int)threadIdx.x;
    const uint32_t held = held16(p0);
    const int below = min(max(n - p0, 0), 16), in = min(max(P - p0, 0), 16);
    const uint32_t low = (1u << below) - 1u, all = (1u << in) - 1u;
    uint32_t hole = ~held & low & all, move = held & ~low;
    int sum;
    int rank = holes + block_rank(__builtin_popcount(hole), sum);
    holes += sum;
    for (; hole; hole &= hole - 1, ++rank) dst[rank] = p0 + __builtin_ctz(hole);
    rank = moves + block_rank(__builtin_popcount(move), sum);
    moves += sum;
    for (; move; move &= move - 1, ++rank) src[rank] = p0 + __builtin_ctz(move);
    for (int i = below; i < in; ++i) to[p0 + i] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += 1024) {
    const int a = src[i], b = dst[i];
    to[a] = b;
    refs[b] = refs[a];
    refs[a] = 0;
  }
  if (threadIdx.x == 0) {
    scratch[0] = moves;
    scratch[1] = n;
  }
}

struct TableSet {
  int32_t *ptr[kMaxTables];
  size_t entries[kMaxTables];
  int n;
};
__global__ __launch_bounds__(256) void pages_compact_kernel(const PoolSet s, const TableSet tables, const int32_t *scratch) {
  const int P = s.num_pages, moves = scratch[0], n = scratch[1];
  const int32_t *src = scratch + 2, *dst = src + P / 2 + 1, *to = dst + P / 2 + 1;
  for (int t = 0; t < tables.n; ++t)
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < tables.entries[t]; i += (size_t)gridDim.x * 256) {
      const int id = tables.ptr[t][i];
      if (id >= n && id < P) {
        const int now = to[id];
        if (now >= 0) tables.ptr[t][i] = now;
      }
    }
  const uint32_t pieces = s.piece0[s.npools];
  const uint64_t total = (uint64_t)moves * pieces;
  for (uint64_t x = blockIdx.x; x < total; x += gridDim.x) {
    const int i = (int)(x / pieces);
    copy_piece(s, (uint32_t)(x - (uint64_t)i * pieces), src[i], dst[i]);
  }
}

}  // namespace ffa

#define FFA_BAD(msg) return ffa_set_error_internal(FFA_E_INVALID, msg)
#define FFA_NO(msg) return ffa_set_error_internal(FFA_E_UNSUPPORTED, msg)

static int pages_check(const ffa_pages *pg) {
  if (!pg) FFA_BAD("null pages");
  if (pg->npools <= 0 || !pg->pools || !pg->page_bytes) FFA_BAD("no pools");
  if (pg->num_pages <= 0) FFA_BAD("empty pool");
  if (pg->num_pages > 1 << 28) FFA_NO("more than 2^28 pages");
  if (!pg->refs || ((uintptr_t)pg->refs & 15)) FFA_BAD("refs must be a multiple of 16 bytes");
  for (int i = 0; i < pg->npools; ++i) {
    if (!pg->pools[i] || ((uintptr_t)pg->pools[i] & 15)) FFA_BAD("pools must be multiples of 16 bytes");
    if (pg->page_bytes[i] == 0 || pg->page_bytes[i] % 16) FFA_BAD("a page's bytes must be a multiple of 16");
    if (pg->page_bytes[i] >= (size_t)1 << 31) FFA_NO("pages of 2 GiB");
  }
  return FFA_OK;
}

// pools [i0, i0 + kMaxPools) of the caller's list
static ffa::PoolSet pool_set(const ffa_pages *pg, int i0) {
  ffa::PoolSet s = {};
  s.npools = pg->npools - i0 < ffa::kMaxPools ? pg->npools - i0 : ffa::kMaxPools;
  s.num_pages = pg->num_pages;
  uint32_t at = 0;
  for (int i = 0; i < s.npools; ++i) {
    s.ptr[i] = (uint8_t *)pg->pools[i0 + i];
    s.bytes[i] = (uint32_t)pg->page_bytes[i0 + i];
    s.piece0[i] = at;
    at += (s.bytes[i] + ffa::kPiece - 1) / ffa::kPiece;
  }
  s.piece0[s.npools] = at;
  return s;
}
// workgroups that copy n pages of a set: each walks its share (64 a CU: compaction 96 -> 85 us against 8 a CU)
static unsigned copy_grid(const ffa::PoolSet &s, long n) {
  const int cus = ffa::device_cus();
  const long all = n * (long)s.piece0[s.npools], most = 64l * (cus > 0 ? cus : 256);
  return (unsigned)(all < 1 ? 1 : (all < most ? all : most));
}
static int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FFA_OK : ffa_set_error_internal(FFA_E_LAUNCH, hipGetErrorString(e));
}

extern "C" int ffa_pages_copy(const ffa_pages *pg, const int32_t *src, const int32_t *dst, int n, void *stream) {
  const int bad = pages_check(pg);
  if (bad != FFA_OK) return bad;
  if (n < 0 || (n && (!src || !dst))) FFA_BAD("page lists");
  if (n == 0) return FFA_OK;
  for (int i = 0; i < pg->npools; i += ffa::kMaxPools) {
    const ffa::PoolSet s = pool_set(pg, i);
    hipLaunchKernelGGL(ffa::pages_copy_kernel, dim3(copy_grid(s, n)), dim3(256), 0, (hipStream_t)stream, s, src, dst, n);
  }
  return launched();
}

extern "C" size_t ffa_pages_alloc_scratch(int rows, int tokens) {
  if (rows <= 0 || tokens < 0) return 0;
  return 2 + (size_t)rows * (((size_t)tokens + 63) / 64 + 1);
}

static int table_check(const void *table, int cols, int rows, const void *seq_lens, const void *errors) {
  if (!table || !seq_lens || !errors) FFA_BAD("null pointer");
  if (cols <= 0 || rows <= 0) FFA_BAD("empty block table");
  if (cols > 1 << 24) FFA_NO("more than 2^24 columns");
  if (rows > 65535) FFA_NO("rows are a grid dimension");
  return FFA_OK;
}

extern "C" int ffa_pages_fork(const ffa_pages *pg, const int32_t *block_table, int bt_stride, int B,
                              const int32_t *seq_lens, const int32_t *parents, int children, int32_t *child_table,
                              int32_t *scratch, int32_t *errors, void *stream) {
  int bad = pages_check(pg);
  if (bad != FFA_OK) return bad;
  bad = table_check(block_table, bt_stride, children, seq_lens, errors);
  if (bad != FFA_OK) return bad;
  if (B <= 0 || !parents || !child_table || !scratch) FFA_BAD("fork needs parents, a table for the children and scratch");
  if (child_table == block_table) FFA_BAD("the children's table cannot be the parents'");
  const int checked = ffa::fork_check_apart(children, bt_stride);
  const ffa::AllocArgs a = {pg->refs, child_table, block_table, seq_lens, parents, scratch, errors,
                            pg->num_pages, children, bt_stride, B, -1, checked};
  if (checked)
    hipLaunchKernelGGL(ffa::pages_fork_check_kernel, dim3((unsigned)children), dim3(256), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(ffa::pages_alloc_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
  for (int i = 0; i < pg->npools; i += ffa::kMaxPools) {
    const ffa::PoolSet s = pool_set(pg, i);
    const int tables = i == 0;
    const unsigned per = (copy_grid(s, children) + children - 1) / children;
    hipLaunchKernelGGL(ffa::pages_fork_kernel, dim3(per + tables, (unsigned)children), dim3(256), 0,
                       (hipStream_t)stream, s, a, tables);
  }
  return launched();
}

extern "C" int ffa_pages_extend(const ffa_pages *pg, int32_t *block_table, int bt_stride, int rows,
                                const int32_t *seq_lens, int tokens, int32_t *scratch, int32_t *errors, void *stream) {
  int bad = pages_check(pg);
  if (bad != FFA_OK) return bad;
  bad = table_check(block_table, bt_stride, rows, seq_lens, errors);
  if (bad != FFA_OK) return bad;
  if (tokens < 0 || !scratch) FFA_BAD("extend needs a number of tokens and scratch");
  if (ffa_pages_alloc_scratch(rows, tokens) > (size_t)1 << 30) FFA_NO("more than 2^30 pages in a call");
  const ffa::AllocArgs a = {pg->refs, block_table, nullptr, seq_lens, nullptr, scratch, errors,
                            pg->num_pages, rows, bt_stride, rows, tokens, 0};
  hipLaunchKernelGGL(ffa::pages_alloc_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
  return launched();
}

extern "C" int ffa_pages_count(const ffa_pages *pg, const int32_t *block_table, int bt_stride, int rows,
                               const int32_t *seq_lens, int step, int32_t *call_errors, int32_t *errors, void *stream) {
  int bad = pages_check(pg);
  if (bad != FFA_OK) return bad;
  bad = table_check(block_table, bt_stride, rows, seq_lens, errors);
  if (bad != FFA_OK) return bad;
  if ((step != 1 && step != -1) || !call_errors) FFA_BAD("step must be 1 or -1");
  const int gx = (bt_stride + 1023) / 1024;
  hipLaunchKernelGGL(ffa::pages_count_kernel, dim3((unsigned)(gx < 64 ? gx : 64), (unsigned)rows), dim3(256), 0,
                     (hipStream_t)stream, pg->refs, pg->num_pages, block_table, bt_stride, seq_lens, step, call_errors, errors);
  return launched();
}

extern "C" size_t ffa_pages_compact_scratch(int num_pages) {
  return num_pages <= 0 ? 0 : 2 + 2 * ((size_t)num_pages / 2 + 1) + num_pages;
}

extern "C" int ffa_pages_compact(const ffa_pages *pg, int32_t *const *tables, const size_t *table_entries, int ntables,
                                 int32_t *scratch, void *stream) {
  const int bad = pages_check(pg);
  if (bad != FFA_OK) return bad;
  if (ntables < 0 || (ntables && (!tables || !table_entries)) || !scratch) FFA_BAD("tables and scratch");
  if (ntables > ffa::kMaxTables) FFA_NO("more than 8 tables");
  ffa::TableSet ts = {};
  ts.n = ntables;
  for (int t = 0; t < ntables; ++t) {
    if (!tables[t] && table_entries[t]) FFA_BAD("null table");
    ts.ptr[t] = tables[t];
    ts.entries[t] = table_entries[t];
  }
  hipLaunchKernelGGL(ffa::pages_compact_plan_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, pg->refs,
                     pg->num_pages, scratch);
  for (int i = 0; i < pg->npools; i += ffa::kMaxPools) {
    const ffa::PoolSet s = pool_set(pg, i);
    hipLaunchKernelGGL(ffa::pages_compact_kernel, dim3(copy_grid(s, pg->num_pages / 2 + 1)), dim3(256), 0,
                       (hipStream_t)stream, s, ts, scratch);
    ts.n = 0;  // the tables once
  }
  return launched();
}
#undef FFA_BAD
#undef FFA_NO
