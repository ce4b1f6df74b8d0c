// bk_pages.cu -- a cache in pages: copying, forking, growing, freeing and compacting (bkPages in bunker_cuda.h has the rules).
//
// No counterpart in the reference (one contiguous buffer of 128 rows, src/emitters.ts:202).  Each call is one or two launches: a plan by
// one CTA, which owns the order in which free pages are given out, then the copies by the whole GPU.  Everything is integer and
// independent of the order in which threads run, so results are reproducible to the bit.
#include <string.h>

#include <algorithm>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

constexpr int kPlanThreads = 1024;   // also the longest list
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;         // 16-byte vectors that a lane has on the way: a warp moves 4 KB at a time, 256 KB an SM

struct Pool {
  uint8_t* base;
  unsigned long long plane_bytes, page_bytes;
  int *ref, *table, *lens;
  int n_planes, n_pages, heads, page_rows, row_bytes, n_seqs, max_pages;
};

// rows below 2^31
BK_DEVINL int pages_of(unsigned int rows, int page_rows) { return (int)((rows + (unsigned int)page_rows - 1) / (unsigned int)page_rows); }

// inclusive sum over the block
BK_DEVINL long long block_scan(long long v, long long* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long w = warp_sums[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += o;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += warp_sums[warp - 1];
  __syncthreads();   // warp_sums may be used again
  return v;
}

// Whether entry i of a list of n names a sequence that an earlier entry has not named.  Every thread looks at as many entries, four a load and
// without a way out of the loop: one that ends early, an entry a load, took 11 us of a call with 64 entries.
BK_DEVINL bool first_entry(const int* list, int n, int i) {
  const int s = list[i];
  bool again = false;
#pragma unroll 4
  for (int j = 0; j < n; j += 4) {   // (entries behind the list are -1)
    const int4 v = *reinterpret_cast<const int4*>(list + j);
    again |= (v.x == s && j < i) | (v.y == s && j + 1 < i) | (v.z == s && j + 2 < i) | (v.w == s && j + 3 < i);
  }
  return !again;
}

// The lowest-numbered free pages, at most `want`, in ascending order into fresh[]; returns how many there are.  All threads call.
BK_DEVINL int find_free(const Pool& p, long long want, int* fresh, long long* warp_sums, int* total_s) {
  int found = 0;
  for (int p0 = 0; p0 < p.n_pages && found < want; p0 += kPlanThreads * 4) {
    const int at = p0 + (int)threadIdx.x * 4;
    int r[4];
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = at + e < p.n_pages ? __ldcg(p.ref + at + e) : 1;
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) n += r[e] == 0;
    const int upto = (int)block_scan(n, warp_sums);
    int k = found + upto - n;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (r[e] == 0) {
        if (k < want) fresh[k] = at + e;
        k++;
      }
    if (threadIdx.x == kPlanThreads - 1) *total_s = upto;
    __syncthreads();
    found += *total_s;
    __syncthreads();
  }
  return (int)min((long long)found, want);
}

// The first launch of each call waits before it lets the next one start: a launch behind the call may read, before its own wait, what a launch
// before the call wrote (weights, settled caches).

struct ForkPlan {   // of one fork, in the scratch buffer
  int src, dst, rows, fresh;   // rows: -1 = not served; fresh: page of the partial rows, -1 = none
};

// One CTA: which forks are served, and the fresh page of each.  A thread per fork; the free pages come from one pass over the counts, which ends when
// enough are found.  Bound: latency of that chain.
__global__ void __launch_bounds__(kPlanThreads) pages_fork_plan_kernel(const Pool p, const int* src, const int* dst, int n, int* ok, ForkPlan* plan, int* fresh) {
  __shared__ long long warp_sums[32];
  __shared__ __align__(16) int dst_s[kPlanThreads];
  __shared__ int total_s;
  __shared__ long long want_s;
  bk_pdl_wait();
  bk_pdl_trigger();
  const int i = threadIdx.x;
  const int s = i < n ? src[i] : -1, d = i < n ? dst[i] : -1;
  dst_s[i] = d;
  __syncthreads();
  int rows = -1;
  if (i < n && s >= 0 && s < p.n_seqs && d >= 0 && d < p.n_seqs && s != d) {
    const int held = __ldcg(p.lens + s), there = __ldcg(p.lens + d);
    if (first_entry(dst_s, n, i) && there == 0 && held <= p.max_pages * p.page_rows) rows = held;
  }
  const int need = rows > 0 && rows % p.page_rows ? 1 : 0;
  const long long upto = block_scan(need, warp_sums);
  if (i == kPlanThreads - 1) want_s = upto;
  __syncthreads();
  const int have = find_free(p, want_s, fresh, warp_sums, &total_s);
  __syncthreads();   // fresh[] is visible to the block
  if (i < n) {
    const bool served = rows >= 0 && (need == 0 || upto <= have);
    plan[i] = ForkPlan{s, d, served ? rows : -1, served && need ? fresh[upto - 1] : -1};
    if (ok) ok[i] = served;
  }
}

// 16-byte vectors v0, v0 + 32, ... of a run of n vectors, up to 4 KB of them at a time.
BK_DEVINL void copy_vecs(uint4* dst, const uint4* src, int n, int lane) {
  uint4 v[kCopyVecs];
#pragma unroll
  for (int e = 0; e < kCopyVecs; e++)
    if (lane + 32 * e < n) v[e] = __ldcg(src + lane + 32 * e);   // (several forks read one page)
#pragma unroll
  for (int e = 0; e < kCopyVecs; e++)
    if (lane + 32 * e < n) __stcs(dst + lane + 32 * e, v[e]);
}

// Forks: table and counts of the child, filled rows of its partial last page.  grid (x, fork).  Bound: memory for many rows, else latency; 64 forks of
// 8 parents, up to 2 MB of rows each, with the calls that free and grow: 27 us, 72 MB.  A parent's rows come from L2 after the first child has read them.
__global__ void __launch_bounds__(kCopyThreads) pages_fork_kernel(const Pool p, const ForkPlan* plan) {
  bk_pdl_trigger();
  bk_pdl_wait();
  const ForkPlan f = plan[blockIdx.y];
  if (f.rows < 0) return;
  const int whole = f.rows / p.page_rows, part = f.rows % p.page_rows;
  const int* from = p.table + (size_t)f.src * p.max_pages;
  if (blockIdx.x == 0) {
    int* to = p.table + (size_t)f.dst * p.max_pages;
    for (int j = threadIdx.x; j < whole; j += kCopyThreads) {
      const int page = from[j];
      to[j] = page;
      if (page >= 0 && page < p.n_pages) atomicAdd(p.ref + page, 1);
    }
    if (threadIdx.x == 0) {
      if (f.fresh >= 0) {
        to[whole] = f.fresh;
        p.ref[f.fresh] = 1;
      }
      p.lens[f.dst] = f.rows;
    }
  }
  if (f.fresh < 0) return;
  const int old = from[whole];
  if (old < 0 || old >= p.n_pages) return;
  const int vecs = (int)((long long)part * p.row_bytes / 16), pieces = (vecs + 32 * kCopyVecs - 1) / (32 * kCopyVecs);
  const long long items = (long long)p.n_planes * p.heads * pieces;
  const int lane = threadIdx.x & 31;
  for (long long it = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); it < items; it += (long long)gridDim.x * (kCopyThreads / 32)) {
    const int piece = (int)(it % pieces), run = (int)(it / pieces), head = run % p.heads, plane = run / p.heads;
    uint8_t* at = p.base + plane * p.plane_bytes + (size_t)head * p.page_rows * p.row_bytes + (size_t)piece * (32 * kCopyVecs * 16);
    copy_vecs(reinterpret_cast<uint4*>(at + f.fresh * p.page_bytes), reinterpret_cast<const uint4*>(at + old * p.page_bytes),
              vecs - piece * 32 * kCopyVecs, lane);
  }
}

// One CTA: room for more rows.  A thread per sequence, a warp per sequence for its new entries.  Bound: latency.
__global__ void __launch_bounds__(kPlanThreads) pages_grow_kernel(const Pool p, const int* seqs, const int* add, int n, int* ok, int* fresh) {
  __shared__ long long warp_sums[32], upto_s[kPlanThreads];
  __shared__ __align__(16) int list_s[kPlanThreads];
  __shared__ int need_s[kPlanThreads], before_s[kPlanThreads], total_s;
  __shared__ long long want_s;
  bk_pdl_wait();
  bk_pdl_trigger();
  const int i = threadIdx.x;
  const int s = i < n ? seqs[i] : -1;
  const int more = i < n ? add[i] : -1;
  list_s[i] = s;
  __syncthreads();
  long long rows = -1;
  int len = 0, need = 0;
  if (i < n && s >= 0 && s < p.n_seqs && more >= 0) {
    len = __ldcg(p.lens + s);
    rows = (long long)len + more;
    if (!first_entry(list_s, n, i) || len < 0 || rows > p.max_pages * p.page_rows) rows = -1;
    else need = pages_of((unsigned int)rows, p.page_rows) - pages_of(len, p.page_rows);
  }
  const long long upto = block_scan(need, warp_sums);
  if (i == kPlanThreads - 1) want_s = upto;
  __syncthreads();
  const int have = find_free(p, min(want_s, (long long)p.n_pages), fresh, warp_sums, &total_s);
  const bool served = rows >= 0 && (need == 0 || upto <= have);
  need_s[i] = served ? need : 0;
  before_s[i] = len > 0 ? pages_of(len, p.page_rows) : 0;
  upto_s[i] = upto;
  if (served) p.lens[s] = (int)rows;
  if (i < n && ok) ok[i] = served;
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < n; r += kPlanThreads / 32)
    for (int j = threadIdx.x & 31; j < need_s[r]; j += 32) {
      const int page = fresh[upto_s[r] - need_s[r] + j];
      p.table[(size_t)list_s[r] * p.max_pages + before_s[r] + j] = page;
      p.ref[page] = 1;
    }
}

// One CTA per entry of the list.  Counts go down by atomics, whose order does not show.  Bound: latency.
__global__ void __launch_bounds__(kCopyThreads) pages_free_kernel(const Pool p, const int* seqs) {
  bk_pdl_wait();
  bk_pdl_trigger();
  const int i = blockIdx.x, s = seqs[i];
  if (s < 0 || s >= p.n_seqs) return;
  bool again = false;
  for (int j = threadIdx.x; j < i; j += kCopyThreads) again = again || seqs[j] == s;
  if (__syncthreads_or(again)) return;
  const int len = p.lens[s];
  __syncthreads();
  if (len <= 0) return;
  const int n = min(pages_of(len, p.page_rows), p.max_pages);
  int* t = p.table + (size_t)s * p.max_pages;
  for (int j = threadIdx.x; j < n; j += kCopyThreads) {
    const int page = t[j];
    if (page >= 0 && page < p.n_pages && atomicSub(p.ref + page, 1) <= 0) atomicAdd(p.ref + page, 1);   // (a count is never negative)
    t[j] = -1;
  }
  if (threadIdx.x == 0) p.lens[s] = 0;
}

// One CTA: where each used page goes, by running sums of the pages that leave and the places that are free.  Bound: latency, of a block scan for every
// 1,024 pages; 6 us with the copies for 64 pages.  moves[0] = how many move, then their old places, then (at n_pages + 1) their new ones.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const Pool p, int* ref_out, int* map, int* used_out, int* moves) {
  __shared__ long long warp_sums[32];
  __shared__ int total_s[2];
  bk_pdl_wait();
  bk_pdl_trigger();
  int mine = 0;
  for (int q = threadIdx.x; q < p.n_pages; q += kPlanThreads) mine += p.ref[q] > 0;
  const long long upto = block_scan(mine, warp_sums);
  if (threadIdx.x == kPlanThreads - 1) total_s[0] = (int)upto;
  __syncthreads();
  const int used = total_s[0];
  __syncthreads();
  int *old_s = moves + 1, *new_s = moves + 1 + p.n_pages;
  int n_old = 0, n_new = 0;
  for (int p0 = 0; p0 < p.n_pages; p0 += kPlanThreads) {
    const int q = p0 + (int)threadIdx.x;
    const int r = q < p.n_pages ? p.ref[q] : 0;
    const bool in = q < p.n_pages, leaves = in && r > 0 && q >= used, takes = in && r <= 0 && q < used;
    // both ranks in one sum: blocks on the boundary have pages of both kinds
    const long long both = block_scan((leaves ? 1ll : 0ll) + (takes ? 1ll << 32 : 0ll), warp_sums);
    if (leaves) old_s[n_old + (int)(both & 0xffffffffll) - 1] = q;
    if (takes) new_s[n_new + (int)(both >> 32) - 1] = q;
    if (in) {
      map[q] = r > 0 && q < used ? q : -1;
      ref_out[q] = q < used && r > 0 ? r : leaves ? r : 0;   // (a leaving page's count is taken to its new place below)
    }
    if (threadIdx.x == kPlanThreads - 1) {
      total_s[0] = (int)(both & 0xffffffffll);
      total_s[1] = (int)(both >> 32);
    }
    __syncthreads();
    n_old += total_s[0];
    n_new += total_s[1];
    __syncthreads();
  }
  for (int k = threadIdx.x; k < n_old; k += kPlanThreads) {
    const int a = old_s[k], b = new_s[k];
    map[a] = b;
    ref_out[b] = ref_out[a];
    ref_out[a] = 0;
  }
  if (threadIdx.x == 0) {
    moves[0] = n_old;
    *used_out = used;
  }
}

// Whole pages: pair i is src[i] of `from`, dst[i] of `to`.  n_dev: the number of pairs lies on the device.  The tables of a compaction
// are rewritten beside the copies.  Bound: memory.  500 pages of 64 rows, 2 heads, 12 planes (786 MB read and written): 128 us, 6.15 TB/s, 0.94 of a
// plain copy of the device; 490 of 2,048 such pages moved by a compaction: 126 to 132 us.  Whole warps on 4 KB pieces, eight CTAs an SM: no page is too
// small or too large for an even spread.
struct CopyJob {
  const int *src, *dst, *n_dev;
  int n;
  const int *table_in, *map;   // map != 0: table_out[j] = map[table_in[j]]
  int* table_out;
  long long table_n;
};
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const Pool from, const Pool to, const CopyJob job) {
  bk_pdl_wait();
  bk_pdl_trigger();
  if (job.map)
    for (long long j = (long long)blockIdx.x * kCopyThreads + threadIdx.x; j < job.table_n; j += (long long)gridDim.x * kCopyThreads) {
      const int page = job.table_in[j];
      job.table_out[j] = page >= 0 && page < from.n_pages ? job.map[page] : -1;
    }
  const int n = job.n_dev ? __ldcg(job.n_dev) : job.n;
  const unsigned int vecs = (unsigned int)(from.page_bytes / 16), pieces = (vecs + 32 * kCopyVecs - 1) / (32 * kCopyVecs);
  const long long items = (long long)n * from.n_planes * pieces;
  const int lane = threadIdx.x & 31;
  for (long long it = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); it < items; it += (long long)gridDim.x * (kCopyThreads / 32)) {
    const long long run = it / pieces;
    const unsigned int piece = (unsigned int)(it - run * pieces);
    const int i = (int)(run / from.n_planes), plane = (int)(run - (long long)i * from.n_planes);
    const int a = __ldg(job.src + i), b = __ldg(job.dst + i);
    if (a < 0 || a >= from.n_pages || b < 0 || b >= to.n_pages) continue;
    const size_t off = (size_t)piece * (32 * kCopyVecs * 16);
    copy_vecs(reinterpret_cast<uint4*>(to.base + plane * to.plane_bytes + b * to.page_bytes + off),
              reinterpret_cast<const uint4*>(from.base + plane * from.plane_bytes + a * from.page_bytes + off), (int)(vecs - piece * 32 * kCopyVecs), lane);
  }
}

int32_t read_pool(const bkPages* a, const char* what, Pool* out) {
  BK_ARG(a != nullptr, "%s: the pool is null", what);
  BK_ARG(a->n_planes > 0 && a->n_pages > 0 && a->heads > 0 && a->page_rows > 0 && a->row_bytes > 0 && a->row_bytes % 16 == 0 && a->n_seqs > 0 && a->max_pages > 0,
         "%s: n_planes=%d n_pages=%d heads=%d page_rows=%d row_bytes=%d n_seqs=%d max_pages=%d (all positive, row_bytes a multiple of 16)", what, a->n_planes,
         a->n_pages, a->heads, a->page_rows, a->row_bytes, a->n_seqs, a->max_pages);
  const unsigned long long row = (unsigned long long)a->heads * a->page_rows;   // below 2^62
  BK_ARG(row < (1ull << 31) && row * a->row_bytes < (1ull << 31), "%s: a page of %d x %d x %d bytes (below 2 GB)", what, a->heads, a->page_rows, a->row_bytes);
  BK_ARG(a->n_pages <= (1 << 30), "%s: %d pages", what, a->n_pages);
  BK_ARG((long long)a->max_pages * a->page_rows < (1ll << 31), "%s: %d pages of %d rows a sequence (below 2^31 rows)", what, a->max_pages, a->page_rows);
  const unsigned long long page = row * a->row_bytes;
  BK_ARG(a->plane_bytes % 16 == 0 && a->plane_bytes / page >= (unsigned long long)a->n_pages, "%s: plane_bytes=%llu for %d pages of %llu bytes", what,
         (unsigned long long)a->plane_bytes, a->n_pages, page);
  BK_ARG(a->base && (a->base & 15) == 0, "%s: base must be non-null and 16-byte aligned", what);
  BK_ARG(a->ref && a->table && a->lens && ((a->ref | a->table | a->lens) & 3) == 0, "%s: ref, table and lens must be non-null int32 arrays", what);
  BK_ARG(a->scratch && (a->scratch & 15) == 0 && a->scratch_bytes >= bkPagesScratchBytes(a->n_pages, a->n_seqs), "%s: scratch of %llu bytes, %llu needed, 16-byte aligned",
         what, (unsigned long long)a->scratch_bytes, (unsigned long long)bkPagesScratchBytes(a->n_pages, a->n_seqs));
  *out = Pool{bk_ptr<uint8_t>(a->base), a->plane_bytes, page, bk_ptr<int>(a->ref), bk_ptr<int>(a->table), bk_ptr<int>(a->lens), a->n_planes, a->n_pages,
              a->heads, a->page_rows, a->row_bytes, a->n_seqs, a->max_pages};
  return BK_OK;
}
int32_t check_list(const char* what, int32_t n, uint64_t a, uint64_t b) {
  BK_ARG(n >= 0 && n <= BK_PAGES_MAX_LIST, "%s: a list of %d entries (0 to %d)", what, n, BK_PAGES_MAX_LIST);
  BK_ARG(n == 0 || (a && b && ((a | b) & 3) == 0), "%s: lists must be non-null int32 arrays", what);
  return BK_OK;
}

// CTAs for `items` warps' worth of copying, at most eight an SM
int copy_ctas(long long items) { return (int)std::max<long long>(1, std::min<long long>((items + kCopyThreads / 32 - 1) / (kCopyThreads / 32), 8ll * bk_ctx().sm_count)); }

#define TRY(expr)            \
  do {                       \
    int32_t _rc = (expr);    \
    if (_rc) return _rc;     \
  } while (0)

}  // namespace

extern "C" {

uint64_t bkPagesScratchBytes(int32_t n_pages, int32_t n_seqs) {
  (void)n_seqs;   // (lists are bounded)
  if (n_pages <= 0) return 0;
  // plans of forks, then free pages or the moves of a compaction
  return ((uint64_t)BK_PAGES_MAX_LIST * sizeof(ForkPlan) + ((uint64_t)n_pages * 2 + 4) * 4 + 15) / 16 * 16;
}

int32_t bkPagesCopy(const bkPages* from, const bkPages* to, uint64_t src, uint64_t dst, int32_t n) {
  BK_REQUIRE_INIT();
  Pool a, b;
  TRY(read_pool(from, "bkPagesCopy", &a));
  TRY(read_pool(to, "bkPagesCopy", &b));
  TRY(check_list("bkPagesCopy", n, src, dst));
  BK_ARG(a.n_planes == b.n_planes && a.heads == b.heads && a.page_rows == b.page_rows && a.row_bytes == b.row_bytes,
         "bkPagesCopy: the pools differ in planes or page shape (%d x %d x %d x %d and %d x %d x %d x %d)", a.n_planes, a.heads, a.page_rows, a.row_bytes, b.n_planes,
         b.heads, b.page_rows, b.row_bytes);
  if (n == 0) return BK_OK;
  CopyJob job;
  memset(&job, 0, sizeof(job));
  job.src = bk_ptr<int>(src); job.dst = bk_ptr<int>(dst); job.n = n;
  const long long items = (long long)n * a.n_planes * (((long long)a.page_bytes / 16 + 32 * kCopyVecs - 1) / (32 * kCopyVecs));
  BK_CUDA(bk_launch_pdl(pages_copy_kernel, dim3(copy_ctas(items)), dim3(kCopyThreads), 0, a, b, job));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

int32_t bkPagesFork(const bkPages* pool, uint64_t src, uint64_t dst, int32_t n, uint64_t ok) {
  BK_REQUIRE_INIT();
  Pool p;
  TRY(read_pool(pool, "bkPagesFork", &p));
  TRY(check_list("bkPagesFork", n, src, dst));
  BK_ARG((ok & 3) == 0, "bkPagesFork: ok must be an int32 array");
  if (n == 0) return BK_OK;
  ForkPlan* plan = bk_ptr<ForkPlan>(pool->scratch);
  int* fresh = reinterpret_cast<int*>(plan + BK_PAGES_MAX_LIST);
  BK_CUDA(bk_launch_pdl(pages_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, p, bk_ptr<int>(src), bk_ptr<int>(dst), n, bk_ptr<int>(ok), plan, fresh));
  BK_CHECK_LAUNCH();
  const long long items = (long long)p.n_planes * p.heads * (((long long)p.page_rows * p.row_bytes / 16 + 32 * kCopyVecs - 1) / (32 * kCopyVecs));   // of a full page
  const int x = (int)std::min<long long>(copy_ctas(items), std::max(1, 8 * bk_ctx().sm_count / n));
  BK_CUDA(bk_launch_pdl(pages_fork_kernel, dim3(x, n), dim3(kCopyThreads), 0, p, plan));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

int32_t bkPagesGrow(const bkPages* pool, uint64_t seqs, uint64_t add, int32_t n, uint64_t ok) {
  BK_REQUIRE_INIT();
  Pool p;
  TRY(read_pool(pool, "bkPagesGrow", &p));
  TRY(check_list("bkPagesGrow", n, seqs, add));
  BK_ARG((ok & 3) == 0, "bkPagesGrow: ok must be an int32 array");
  if (n == 0) return BK_OK;
  int* fresh = reinterpret_cast<int*>(bk_ptr<ForkPlan>(pool->scratch) + BK_PAGES_MAX_LIST);
  BK_CUDA(bk_launch_pdl(pages_grow_kernel, dim3(1), dim3(kPlanThreads), 0, p, bk_ptr<int>(seqs), bk_ptr<int>(add), n, bk_ptr<int>(ok), fresh));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

int32_t bkPagesFree(const bkPages* pool, uint64_t seqs, int32_t n) {
  BK_REQUIRE_INIT();
  Pool p;
  TRY(read_pool(pool, "bkPagesFree", &p));
  TRY(check_list("bkPagesFree", n, seqs, seqs));
  if (n == 0) return BK_OK;
  BK_CUDA(bk_launch_pdl(pages_free_kernel, dim3(n), dim3(kCopyThreads), 0, p, bk_ptr<int>(seqs)));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

int32_t bkPagesCompact(const bkPages* pool, uint64_t table_out, uint64_t ref_out, uint64_t map, uint64_t used) {
  BK_REQUIRE_INIT();
  Pool p;
  TRY(read_pool(pool, "bkPagesCompact", &p));
  BK_ARG(table_out && ref_out && map && used && ((table_out | ref_out | map | used) & 3) == 0, "bkPagesCompact: table_out, ref_out, map and used must be non-null int32 arrays");
  int* moves = reinterpret_cast<int*>(bk_ptr<ForkPlan>(pool->scratch) + BK_PAGES_MAX_LIST);
  BK_CUDA(bk_launch_pdl(pages_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, p, bk_ptr<int>(ref_out), bk_ptr<int>(map), bk_ptr<int>(used), moves));
  BK_CHECK_LAUNCH();
  CopyJob job;
  memset(&job, 0, sizeof(job));
  job.src = moves + 1; job.dst = moves + 1 + p.n_pages; job.n_dev = moves;
  job.table_in = p.table; job.map = bk_ptr<int>(map); job.table_out = bk_ptr<int>(table_out); job.table_n = (long long)p.n_seqs * p.max_pages;
  const long long items = (long long)(p.n_pages + 1) / 2 * p.n_planes * (((long long)p.page_bytes / 16 + 32 * kCopyVecs - 1) / (32 * kCopyVecs));
  BK_CUDA(bk_launch_pdl(pages_copy_kernel, dim3(copy_ctas(items)), dim3(kCopyThreads), 0, p, p, job));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

}  // extern "C"
