// bk_pages.cu -- a cache in pages: copying, forking, growing, freeing and compacting, maps of a step, and which drafted rows stay (bkPages in bunker_cuda.h
// has the rules).
//
// No counterpart in the reference (one contiguous buffer of 128 rows, src/emitters.ts:202).  Each call that gives out or moves pages is one or two launches: a plan by
// one CTA, which owns the order in which free pages are given out, then the copies by the whole GPU.  Everything is integer and
// independent of the order in which threads run, so results are reproducible to the bit.
#include <string.h>

#include <algorithm>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

constexpr int kPlanThreads = 1024;   // also the longest list
constexpr int kCopyThreads = 256;
constexpr int kMaxNodes = 1024;      // of a drafted tree
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

// ---- drafted trees ---------------------------------------------------------------------

struct BatchParams {
  const int *seqs, *n_new, *parent, *ok;
  int *table, *lens, *pos, *slot, *count;
  uint32_t* mask;
  int n, T, words;
};

// Maps of a batch: a CTA row per sequence, its CTAs share the table; the nodes are the first one's, a thread each.  A node's ancestors have lower numbers, so a walk up
// the tree writes the words of its mask from the last to the first, each once.  Bound: latency, of a chain of loads (list, length, table) and the walk; a call of one sequence 5.0 us, of
// 256 with tables of 2,048 pages and trees of up to 64 nodes 5.2: the host's launch.
__global__ void __launch_bounds__(kCopyThreads) pages_batch_kernel(const Pool p, const BatchParams a) {
  __shared__ int parent_s[kMaxNodes];
  bk_pdl_wait();
  bk_pdl_trigger();
  const int i = blockIdx.x, s = a.seqs[i];
  int len = s >= 0 && s < p.n_seqs ? __ldcg(p.lens + s) : 0;
  if (len < 0 || len > p.max_pages * p.page_rows) len = 0;
  const int held = pages_of(len, p.page_rows);
  const int* from = p.table + (size_t)max(s, 0) * p.max_pages;
  if (a.table) {
    int* to = a.table + (size_t)i * p.max_pages;
    for (int j = blockIdx.y * kCopyThreads + threadIdx.x; j < p.max_pages; j += gridDim.y * kCopyThreads) to[j] = j < held ? __ldcg(from + j) : -1;
  }
  if (blockIdx.y) return;
  if (a.lens && threadIdx.x == 0) a.lens[i] = len;
  int n = a.n_new ? max(0, min(a.n_new[i], a.T)) : a.T;
  if (a.ok && a.ok[i] == 0) n = 0;
  const int base = len - n;
  if (base < 0) n = 0;
  __syncthreads();   // (count may be what n_new or ok was read from)
  if (a.count && threadIdx.x == 0) a.count[i] = n;
  if (!a.pos && !a.slot && !a.mask) return;
  if (a.parent) {
    for (int t = threadIdx.x; t < n; t += kCopyThreads) parent_s[t] = a.parent[(size_t)t * a.n + i];
    __syncthreads();
  }
  for (int t = threadIdx.x; t < a.T; t += kCopyThreads) {
    const size_t e = (size_t)t * a.n + i;
    uint32_t* words = a.mask ? a.mask + e * a.words : nullptr;
    int w = a.words - 1, depth = -1;
    if (t < n) {
      uint32_t bits = 0;
      int top = w;   // the last word that a bit can be in
      if (words)
        for (; top > t >> 5; top--) words[top] = 0;
      else
        top = t >> 5;
      w = top;
      for (int u = t; u >= 0;) {
        if (u >> 5 != w) {
          if (words) {
            words[w] = bits;
            for (w--; w > u >> 5; w--) words[w] = 0;
          }
          w = u >> 5;
          bits = 0;
        }
        bits |= 1u << (u & 31);
        depth++;
        const int up = a.parent ? parent_s[u] : u - 1;
        u = up < u ? up : -1;
      }
      if (words) words[w] = bits;
      w--;
    }
    if (words)
      for (; w >= 0; w--) words[w] = 0;
    if (a.pos) a.pos[e] = t < n ? base + depth : -1;
    if (a.slot) {
      int slot = -1;
      if (t < n) {
        const int row = base + t, page = __ldcg(from + row / p.page_rows);
        if (page >= 0 && page < p.n_pages) slot = page * p.page_rows + row % p.page_rows;
      }
      a.slot[e] = slot;
    }
  }
}

struct CommitParams {
  const int *seqs, *n_new, *parent, *token, *target;
  int *path, *n_path, *next, *ok, *history, *hist_len;
  int n, T, history_ld, values;
};

// A cluster of CTAs per sequence.  Each finds the path for itself: every node that the model agrees with tells its parent, the lowest child stays, and one thread follows
// the children.  Then the CTAs' warps move rows: a warp has 512 bytes of a row of one head and plane, of all rows that move, which it takes in order (row i of the
// tree is written after it was read, since a path's node i has a number of at least i).  What the others still read (table, counts, lengths) is changed by the
// first CTA behind the cluster's barrier; other sequences read none of it, for pages of a tree belong to one sequence alone.  Bound: latency of the chain list, length,
// pages, counts, rows; the tree is asked for ahead of it and the pages are kept (with the call that makes room: one sequence 9.0 us; 64 of up to 64 nodes, 32 planes of 4 heads, 11.7 MB: 15.2 us, with the tree
// and pages read where they are needed 17.8, with a CTA a sequence 25).
__global__ void __launch_bounds__(kCopyThreads) pages_commit_kernel(const Pool p, const CommitParams a) {
  __shared__ int child_s[kMaxNodes], path_s[kMaxNodes], target_s[kMaxNodes], page_s[kMaxNodes + 1], n_s, refused_s;
  constexpr int kEach = kMaxNodes / kCopyThreads;
  const int tid = threadIdx.x, rank = blockIdx.x, ranks = gridDim.x, i = blockIdx.y;   // (a cluster is a row of the grid)
  bk_pdl_wait();
  bk_pdl_trigger();
  const int s = a.seqs[i], n = a.n_new ? a.n_new[i] : a.T;
  int parent[kEach], token[kEach];
#pragma unroll
  for (int k = 0; k < kEach; k++) {
    const int t = tid + k * kCopyThreads;
    if (t >= a.T) break;
    parent[k] = a.parent[(size_t)t * a.n + i];
    token[k] = a.token[(size_t)t * a.n + i];
    const int target = a.target[(size_t)t * a.n + i];
    // (-inf: the best of what a grammar left, which is nothing)
    target_s[t] = a.values && a.target[(size_t)(a.T + t) * a.n + i] == (int)0xff800000u ? -1 : target;
    child_s[t] = kMaxNodes;
  }
  bool bad = false;
  for (int j = tid; j < i; j += kCopyThreads) bad |= a.seqs[j] == s;
  const bool named = s >= 0 && s < p.n_seqs && n >= 1 && n <= a.T;
  const int len = named ? __ldcg(p.lens + s) : 0, base = len - n, first_page = max(base, 0) / p.page_rows;
  const int said = named && a.history ? __ldcg(a.hist_len + s) : 0;
  bool good = named && base >= 0 && len <= p.max_pages * p.page_rows;
  int* table = p.table + (size_t)max(s, 0) * p.max_pages;
  if (good)   // pages of the tree's rows: this sequence's alone
    for (int j = first_page + tid; j < pages_of(len, p.page_rows); j += kCopyThreads) {
      const int page = __ldcg(table + j);
      page_s[j - first_page] = page;
      bad |= page < 0 || page >= p.n_pages || __ldcg(p.ref + page) != 1;
    }
  good = !__syncthreads_or(bad) && good;   // (of the whole CTA)
#pragma unroll
  for (int k = 0; k < kEach; k++) {
    const int t = tid + k * kCopyThreads;
    if (t >= a.T) break;
    if (good && t >= 1 && t < n && parent[k] >= 0 && parent[k] < t && token[k] >= 0 && token[k] == target_s[parent[k]]) atomicMin(child_s + parent[k], t);
  }
  __syncthreads();
  if (tid == 0) {
    int m = 0;
    if (good)
      for (int t = 0; t < kMaxNodes; t = child_s[t]) path_s[m++] = t;
    n_s = m;
    refused_s = a.history && (said < 0 || said > a.history_ld - m);
  }
  __syncthreads();
  good = good && !refused_s;
  const int m = good ? n_s : 0;
  if (rank == 0) {
    if (a.path)
      for (int t = tid; t < a.T; t += kCopyThreads) a.path[(size_t)t * a.n + i] = t < m ? path_s[t] : -1;
    if (tid == 0) {
      if (a.n_path) a.n_path[i] = m;
      if (a.next) a.next[i] = good ? target_s[path_s[m - 1]] : -1;
      if (a.ok) a.ok[i] = good;
    }
  }
  if (!good) return;   // (of the whole cluster: its CTAs have read the same)
  // the rows that move: from the first whose place is another
  int first = 0;
  while (first < m && path_s[first] == first) first++;
  if (first < m) {
    const int lane = tid & 31, chunks = (p.row_bytes / 16 + 31) / 32;
    const long long items = (long long)p.n_planes * p.heads * chunks;
    for (long long it = rank * (kCopyThreads / 32) + (tid >> 5); it < items; it += (long long)ranks * (kCopyThreads / 32)) {
      const int chunk = (int)(it % chunks), run = (int)(it / chunks), head = run % p.heads, plane = run / p.heads, vec = chunk * 32 + lane;
      uint8_t* at = p.base + plane * p.plane_bytes + (size_t)head * p.page_rows * p.row_bytes + (size_t)vec * 16;
      auto row_at = [&](int t) {
        const int row = base + t, page = row / p.page_rows;
        return reinterpret_cast<uint4*>(at + page_s[page - first_page] * p.page_bytes + (size_t)(row - page * p.page_rows) * p.row_bytes);
      };
      if (vec < p.row_bytes / 16)
        for (int k = first; k < m; k += kCopyVecs) {
          uint4 v[kCopyVecs];
#pragma unroll
          for (int e = 0; e < kCopyVecs; e++)
            if (k + e < m) v[e] = *row_at(path_s[k + e]);
#pragma unroll
          for (int e = 0; e < kCopyVecs; e++)
            if (k + e < m) *row_at(k + e) = v[e];
        }
    }
  }
  if (ranks > 1) {
    asm volatile("barrier.cluster.arrive;" ::: "memory");
    asm volatile("barrier.cluster.wait;" ::: "memory");
  } else {
    __syncthreads();
  }
  if (rank) return;
  for (int j = pages_of(base + m, p.page_rows) + tid; j < pages_of(len, p.page_rows); j += kCopyThreads) {
    p.ref[page_s[j - first_page]] = 0;
    table[j] = -1;
  }
  if (a.history) {
    int* to = a.history + (size_t)s * a.history_ld + said;
    for (int t = tid; t < m; t += kCopyThreads) to[t] = a.token[(size_t)path_s[t] * a.n + i];
    if (tid == 0) a.hist_len[s] = said + m;
  }
  if (tid == 0) p.lens[s] = base + m;
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

// bytes of device memory, none where at is 0
struct Span {
  uint64_t at, bytes;
};
bool overlap(const Span& a, const Span& b) { return a.at && b.at && a.at < b.at + b.bytes && b.at < a.at + a.bytes; }
// whether they are part of what a pool holds: its lists and pages (not what lies between planes)
bool in_pool(const bkPages& pool, const Pool& p, const Span& a) {
  if (overlap(a, {pool.lens, 4ull * p.n_seqs}) || overlap(a, {pool.table, 4ull * p.n_seqs * p.max_pages}) || overlap(a, {pool.ref, 4ull * p.n_pages})) return true;
  const unsigned long long plane = p.n_pages * p.page_bytes;
  for (int i = 0; i < p.n_planes; i++)
    if (overlap(a, {pool.base + i * p.plane_bytes, plane})) return true;
  return false;
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

int32_t bkPagesBatch(const bkPages* pool, const bkPagesBatchArgs* args) {
  BK_REQUIRE_INIT();
  Pool p;
  TRY(read_pool(pool, "bkPagesBatch", &p));
  BK_ARG(args != nullptr, "bkPagesBatch: args is null");
  const bkPagesBatchArgs& a = *args;
  TRY(check_list("bkPagesBatch", a.n, a.seqs, a.seqs));
  BK_ARG(a.T >= 1 && a.T <= kMaxNodes, "bkPagesBatch: T=%d (1 to %d)", a.T, kMaxNodes);
  BK_ARG(((a.n_new | a.parent | a.table | a.lens | a.pos | a.slot | a.mask | a.ok | a.count) & 3) == 0, "bkPagesBatch: all arrays are of 32-bit words");
  BK_ARG(!a.mask || a.mask_words >= (a.T + 31) / 32, "bkPagesBatch: mask_words=%d for %d nodes", a.mask_words, a.T);
  BK_ARG(!a.slot || (long long)p.n_pages * p.page_rows < (1ll << 31), "bkPagesBatch: %d pages of %d rows: a slot has 31 bits", p.n_pages, p.page_rows);
  if (a.n == 0) return BK_OK;
  // a sequence's CTAs read while the first writes
  const uint64_t list = 4ull * a.n, nodes = list * a.T;
  const Span read[] = {{a.seqs, list}, {a.parent, nodes}, {a.n_new, list}, {a.ok, list}};
  const Span write[] = {{a.count, list}, {a.table, list * p.max_pages}, {a.lens, list}, {a.pos, nodes}, {a.slot, nodes}, {a.mask, a.mask ? nodes * a.mask_words : 0}};
  for (int i = 0; i < 6; i++) {
    bool apart = !in_pool(*pool, p, write[i]);
    for (int j = 0; j < 4; j++) apart = apart && (!overlap(write[i], read[j]) || (i == 0 && j >= 2 && write[i].at == read[j].at));
    BK_ARG(apart, "bkPagesBatch: results must lie apart from what the call reads (count alone may be the array of n_new or ok)");
  }
  const BatchParams b = {bk_ptr<int>(a.seqs), bk_ptr<int>(a.n_new), bk_ptr<int>(a.parent), bk_ptr<int>(a.ok), bk_ptr<int>(a.table), bk_ptr<int>(a.lens), bk_ptr<int>(a.pos),
                         bk_ptr<int>(a.slot), bk_ptr<int>(a.count), bk_ptr<uint32_t>(a.mask), a.n, a.T, a.mask_words};
  // CTAs a sequence: 1,024 entries of its table each, no more than fill the GPU twice
  const int y = a.table ? std::max(1, std::min((p.max_pages + 4 * kCopyThreads - 1) / (4 * kCopyThreads), 2 * bk_ctx().sm_count / a.n)) : 1;
  BK_CUDA(bk_launch_pdl(pages_batch_kernel, dim3(a.n, y), dim3(kCopyThreads), 0, p, b));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

int32_t bkPagesCommit(const bkPages* pool, const bkPagesCommitArgs* args) {
  BK_REQUIRE_INIT();
  Pool p;
  TRY(read_pool(pool, "bkPagesCommit", &p));
  BK_ARG(args != nullptr, "bkPagesCommit: args is null");
  const bkPagesCommitArgs& a = *args;
  TRY(check_list("bkPagesCommit", a.n, a.seqs, a.seqs));
  BK_ARG(a.T >= 1 && a.T <= kMaxNodes, "bkPagesCommit: T=%d (1 to %d)", a.T, kMaxNodes);
  BK_ARG(a.n == 0 || (a.parent && a.token && a.target), "bkPagesCommit: parent, token and target must be non-null int32 arrays");
  BK_ARG(((a.n_new | a.parent | a.token | a.target | a.path | a.n_path | a.next | a.ok | a.history | a.hist_len) & 3) == 0, "bkPagesCommit: all arrays are of int32");
  BK_ARG(a.values == 0 || a.values == 1, "bkPagesCommit: values=%d (0 or 1)", a.values);
  BK_ARG((a.history != 0) == (a.hist_len != 0) && (!a.history || a.history_ld > 0), "bkPagesCommit: history and hist_len go together (history_ld=%d)", a.history_ld);
  if (a.n == 0) return BK_OK;
  // a cluster's CTAs, and those of other sequences, read while the first writes
  const uint64_t list = 4ull * a.n, nodes = list * a.T;
  const Span read[] = {{a.seqs, list}, {a.n_new, list}, {a.parent, nodes}, {a.token, nodes}, {a.target, nodes * (1 + a.values)}};
  const Span histories[] = {{a.history, 4ull * p.n_seqs * a.history_ld}, {a.hist_len, 4ull * p.n_seqs}};
  auto apart = [&](const Span& w) {
    for (const Span& r : read)
      if (overlap(w, r)) return false;
    return !in_pool(*pool, p, w);
  };
  for (const Span& w : {Span{a.path, nodes}, Span{a.n_path, list}, Span{a.next, list}, Span{a.ok, list}})
    BK_ARG(apart(w) && !overlap(w, histories[0]) && !overlap(w, histories[1]), "bkPagesCommit: path, n_path, next and ok must lie apart from what the call reads");
  BK_ARG(apart(histories[0]) && apart(histories[1]) && !overlap(histories[0], histories[1]), "bkPagesCommit: history and hist_len must lie apart from the other arrays");
  const CommitParams c = {bk_ptr<int>(a.seqs), bk_ptr<int>(a.n_new), bk_ptr<int>(a.parent), bk_ptr<int>(a.token), bk_ptr<int>(a.target), bk_ptr<int>(a.path), bk_ptr<int>(a.n_path),
                          bk_ptr<int>(a.next), bk_ptr<int>(a.ok), bk_ptr<int>(a.history), bk_ptr<int>(a.hist_len), a.n, a.T, a.history_ld, a.values};
  // CTAs a sequence: as many as its warps have runs of rows for, at most 8 (a cluster) and four an SM
  const long long items = (long long)p.n_planes * p.heads * ((p.row_bytes / 16 + 31) / 32);
  int ranks = 1;
  while (ranks < 8 && ranks * (kCopyThreads / 32) < items && (long long)2 * ranks * a.n <= 4 * bk_ctx().sm_count) ranks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, a.n);
  cfg.blockDim = dim3(kCopyThreads);
  cfg.stream = bk_ctx().stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  BK_CUDA(cudaLaunchKernelEx(&cfg, pages_commit_kernel, p, c));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

}  // extern "C"
