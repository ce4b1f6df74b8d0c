// bk_paged_attn.cu -- attention of many sequences over pages of keys and values (bkPagedAttn in bunker_cuda.h has the rules).
//
// o[r] = sum over keys j <= row of r of 2^(S[r][j] - m[r]) v[j] / sum of the same without v, S = q k^T scale log2(e).  Three launches: queries and new
// rows (with the plan of the next), tiles of rows and keys, the pieces' results together.  Each hides little of the one before: a tile CTA takes all of an
// SM's shared memory.  One sequence of 300 rows, 16 heads on 2: 16 us, nearly all of it the three launches' latency; 32 sequences behind 8,192
// common rows: 30 us; 64 behind 32,768, 24 heads on 4: 96 us, 114 where the power limit sets the clock for long: 0.33 and 0.28 of the bf16 rate by
// the operations that the result needs, half of it again in operations done; 32 sequences of 8,192 rows that share nothing: 98 us, 5.5 TB/s.
//
// bkTreeAttn is the same for drafted trees (TREE): a row sees the keys before its sequence's tree and those of its nodes whose bits are set.  Trees bring many rows to a
// sequence, so its work is shared out by a plan of its own (plan_trees), over tokens that are there.  A step of 128 rows and 64 keys takes 1,900 cycles (HD 256; 1,755 for HD 128), 600 of them
// exponentials (512 of the unit's), 1,536 (768) of the tensor cores beside them: both groups of rows wait for the same tile.  Four groups, groups that take turns at tiles, and the next
// tile's scores asked for ahead of the wait for this one's probabilities were no faster.
//
// No counterpart in the reference (one contiguous cache of 128 rows, src/emitters.ts:188-226).
#include <math.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "bk_common.cuh"
#include "bk_internal.h"
#include "bk_ring.h"

namespace {

struct PagedParams {
  const uint16_t *qg, *k, *v, *gate, *q_norm_w, *k_norm_w;
  const float *cos_t, *sin_t;
  uint16_t *k_pages, *v_pages;
  const int *table, *lens, *n_new;
  uint16_t* out;
  uint16_t* q;        // ready q [Hkv][B][T][Hq / Hkv][HD] in the scratch buffer: the rows of a job lie together
  int B, T, Hq, Hkv, rot_half, n_pages, page_rows, max_pages, max_rows, fused;   // max_rows: what a sequence can have
  float scale, eps;
};

// What a call for trees (bkTreeAttn) has besides.  Its rows see the keys before the tree and the nodes whose bits are set; where new rows go and
// where their rotation stands is given.
struct TreeParams {
  const int *pos, *slot;
  const uint32_t* mask;   // [T * B][words]
  int words, max_pos;
  int each;               // heads that a warp makes ready
  // In the scratch buffer, made by the first launch.  Ready queries and rows of jobs are those of tokens that are there, one sequence's behind the other's (with more
  // than kCompact sequences: T for each).
  int* first;             // [B + 1]: where a sequence's tokens begin; how many there are
  int* token;             // [B * T]: t * B + b of each (up to kCompact sequences)
  int* place;             // [T * B]: which of them a row is, -1: not there, or it sees nothing
  int4* team;             // see plan_trees
};
constexpr int kCompact = 1024;
struct NoTree {};
template <bool TREE>
struct Params : PagedParams, std::conditional<TREE, TreeParams, NoTree>::type {};

// row of its sequence at which token t of sequence b stands, -1 where it is not there
BK_DEVINL int row_of(const Params<false>& p, int b, int t) {
  const int n = p.n_new ? min(p.n_new[b], p.T) : p.T;
  const long long at = (long long)p.lens[b] - n + t;
  return t < n && at >= 0 && at < p.max_rows ? (int)at : -1;
}
// the tree of sequence b: its nodes (0: none is there), and the row of the first, which is the number of keys that all of them see
struct Tree {
  int n, base;
};
BK_DEVINL Tree tree_of(const Params<true>& p, int b) {
  Tree r;
  r.n = p.n_new ? max(0, min(p.n_new[b], p.T)) : p.T;
  const int len = p.lens[b];
  r.base = len - r.n;
  if (len < r.n || len > p.max_rows) r.n = r.base = 0;
  return r;
}
// word i of the nodes that a row sees, of n; all ones before the first
BK_DEVINL uint32_t node_word(const uint32_t* bits, int n, int i) {
  if (i < 0) return 0xffffffffu;
  const int left = n - 32 * i;
  return left <= 0 ? 0u : __ldg(bits + i) & (left >= 32 ? 0xffffffffu : (1u << left) - 1u);
}
// Which of the keys key, key + 1, ... key + 31 a row sees: bit for bit.  Those before the tree, and nodes whose bits are set.
BK_DEVINL uint32_t seen_keys(const uint32_t* bits, const Tree& r, int key) {
  const int o = key - r.base;
  if (o <= -32) return 0xffffffffu;
  const int i = o >> 5;
  return __funnelshift_r(node_word(bits, r.n, i), node_word(bits, r.n, i + 1), o & 31);
}
// The same in two steps: the words as they lie in memory, asked for a tile ahead, and what they say.
BK_DEVINL uint2 ask_seen(const uint32_t* bits, const Tree& r, int key) {
  const int i = (key - r.base) >> 5;
  uint2 w = make_uint2(0, 0);
  if (i >= 0 && 32 * i < r.n) w.x = __ldg(bits + i);
  if (i >= -1 && 32 * (i + 1) < r.n) w.y = __ldg(bits + i + 1);
  return w;
}
BK_DEVINL uint32_t tell_seen(uint2 w, const Tree& r, int key) {
  const int o = key - r.base, i = o >> 5;
  if (o <= -32) return 0xffffffffu;
  auto part = [&](uint32_t v, int j) {
    const int left = r.n - 32 * j;
    return j < 0 ? 0xffffffffu : left >= 32 ? v : left > 0 ? v & ((1u << left) - 1u) : 0u;
  };
  return __funnelshift_r(part(w.x, i), part(w.y, i + 1), o & 31);
}

template <int PER>
BK_DEVINL void load_bf16(const uint16_t* src, float (&y)[PER]) {
#pragma unroll
  for (int e = 0; e < PER; e += 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(src + e);
    y[e] = __uint_as_float(v.x << 16); y[e + 1] = __uint_as_float(v.x & 0xffff0000u);
    y[e + 2] = __uint_as_float(v.y << 16); y[e + 3] = __uint_as_float(v.y & 0xffff0000u);
  }
}

// ---- who does what -----------------------------------------------------------------
// A job is a tile of up to 128 rows (token, query head) of one KV head and the keys they attend to: the common keys [0, P) once for the
// rows of all sequences, then for each sequence its own keys [P, end).  The jobs, in tiles of 64 keys and kOverhead more for each job, are laid
// out in one line and cut into equal pieces, one per CTA, so that a long prefix and many short sequences keep every SM busy until the end.
// Where common keys have several row tiles, all of those are cut at the same keys, one range a CTA, and the line is for the other CTAs: the row tiles
// of a KV head then read the same keys at the same time, once from memory (in one line they read them at times that hang on the cuts: 64
// sequences, 24 heads on 4, 32,768 common rows 100 to 118 us by the overhead that the line counts with, so 97).
// The plan is made on the device (lengths are there), by one CTA of the first launch.  (Every CTA of the second making it for itself, in shared memory
// and without records, starts later than that one, since an SM has no room for it beside a CTA of the first: 29.2 to 32.6 us, 22.4 to 25.8.)
constexpr int kTile = 64;       // keys of a step
constexpr int kRows = 128;      // rows of a job: the lanes of tensor memory
constexpr int kOverhead = 3;    // what a job's start and end cost, in steps

struct Layout {                 // of the scratch buffer, and the numbers of jobs
  int P;                        // common keys: whole pages
  int mt_p, mt_s;               // row tiles of a KV head: of all sequences together, of one sequence
  int n_p, n_s;                 // jobs over common keys, over a sequence's own
  int rows_s;                   // rows of a partial result of the latter
  int ctas;
  size_t q, jobs, pieces, ml_p, ml_s, o_p, o_s, bytes;   // byte offsets
};

__host__ __device__ inline size_t round16(size_t n) { return (n + 15) / 16 * 16; }

inline Layout make_layout(int B, int T, int Hq, int Hkv, int HD, int prefix_rows, int page_rows, int ctas) {
  Layout L;
  const int G = Hq / Hkv;
  L.P = prefix_rows / page_rows * page_rows;
  L.mt_p = (B * T * G + kRows - 1) / kRows;
  L.mt_s = (T * G + kRows - 1) / kRows;
  L.n_p = L.P ? Hkv * L.mt_p : 0;
  L.n_s = B * Hkv * L.mt_s;
  L.rows_s = std::min(T * G, kRows);
  L.ctas = ctas;
  size_t at = round16((size_t)B * T * Hq * HD * 2);
  L.q = 0;
  L.jobs = at;
  at += (size_t)(L.n_p + L.n_s + 1) * 16;
  L.pieces = at;
  at += (size_t)ctas * 32;
  // partial results: on the line a job and a CTA that has a piece of it meet in slot job + CTA, which no other pair has; off it the slot is the CTA
  const size_t slots_p = L.n_p ? L.n_p + ctas : 0, slots_s = L.n_s + ctas;
  L.ml_p = at;
  at += slots_p * kRows * 16;
  L.ml_s = at;
  at += slots_s * L.rows_s * 16;
  L.o_p = at;
  at += slots_p * kRows * HD * 4;
  L.o_s = at;
  at += slots_s * L.rows_s * HD * 4;
  L.bytes = at;
  return L;
}

template <bool TREE>
struct TileParams {
  Params<TREE> g;
  Layout L;
  uint8_t* scratch;
  int* status;
  int box_rows;   // rows of a page that one copy takes: min(page_rows, kTile)
  int q_rows[2];  // rows of queries that a job takes: over a sequence's own keys, over the common ones
  CUtensorMap k_map, v_map, q_map[2];
};

// job j: its KV head, row tile, sequence (-1: all) and where its keys begin
struct Job {
  int seq, kvh, mt, key0;
};
BK_DEVINL Job job_of(const PagedParams& p, const Layout& L, int j) {
  Job q;
  if (j < L.n_p) {
    q.seq = -1;
    q.kvh = j / L.mt_p;
    q.mt = j - q.kvh * L.mt_p;
    q.key0 = 0;
    return q;
  }
  const int i = j - L.n_p, bk = i / L.mt_s;
  q.mt = i - bk * L.mt_s;
  q.seq = bk / p.Hkv;
  q.kvh = bk - q.seq * p.Hkv;
  q.key0 = L.P;
  return q;
}
// the end of its keys: behind the row of the last of the tile's tokens that is there
BK_DEVINL int keys_end(const Params<false>& p, const Layout& L, const Job& q) {
  if (q.seq < 0) return L.P;
  const int G = p.Hq / p.Hkv, n = p.n_new ? min(p.n_new[q.seq], p.T) : p.T, last = min(n, (min(p.T * G, (q.mt + 1) * kRows) - 1) / G + 1) - 1;
  for (int t = last; t >= 0 && t >= q.mt * kRows / G; t--) {   // (one turn but for tokens past max_len)
    const int at = row_of(p, q.seq, t);
    if (at >= 0) return max(L.P, at + 1);
  }
  return L.P;
}

// What the first launch leaves for the others.  jobs[j] = {start on the line, end of the keys, slot of its first partial result, their number and
// (<< 16) the distance of their slots}; pieces[2c] = {start and end of CTA c's piece of the line, first job in it, job over common keys or -1},
// pieces[2c + 1] = {.x and .y of the first job in the line, the range of tiles over common keys}.
BK_DEVINL int4* jobs_of(const Layout& L, uint8_t* scratch) { return reinterpret_cast<int4*>(scratch + L.jobs); }
BK_DEVINL int4* pieces_of(const Layout& L, uint8_t* scratch) { return reinterpret_cast<int4*>(scratch + L.pieces); }
BK_DEVINL int tiles_of(const Layout& L, int j, int key1) { return (key1 - (j < L.n_p ? 0 : L.P) + kTile - 1) / kTile; }
// the tiles of a job that starts at s and has n tiles which lie in units [u0, u1): [t0, t1)
BK_DEVINL void piece_of(int s, int n, int u0, int u1, int* t0, int* t1, int overhead = kOverhead) {
  *t0 = max(0, min(n, u0 - s - overhead));
  *t1 = max(0, min(n, u1 - s - overhead));
}

// one CTA
constexpr int kPrepThreads = 256, kPlanned = 1024;   // jobs whose starts fit in shared memory
// SMEM: no more than kPlanned jobs, whose lines are worked on in shared memory; otherwise in the records themselves.  What it takes is on every
// call's way: a chain of loads from L2 costs 0.6 us a link.
template <bool SMEM>
BK_DEVINL void plan_jobs(const Params<false>& p, const Layout& L, uint8_t* scratch) {
  __shared__ int warp_s[kPrepThreads / 32][2], starts_s[SMEM ? kPlanned + 1 : 1], ends_s[SMEM ? kPlanned : 1], bounds_s[kPrepThreads + 1];
  int4* jobs = jobs_of(L, scratch);
  int4* pieces = pieces_of(L, scratch);
  const int n = L.n_p + L.n_s, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles_p = (L.P + kTile - 1) / kTile, all_ctas = min(L.ctas, kPrepThreads);
  const bool apart = L.mt_p > 1 && L.n_p > 0 && L.n_p <= all_ctas / 2 && L.n_p * tiles_p >= all_ctas;   // common keys apart from the line
  if (SMEM) {
    for (int j = threadIdx.x; j < n; j += kPrepThreads) ends_s[j] = keys_end(p, L, job_of(p, L, j));
    __syncthreads();
  }
  auto units_of = [&](int j, int end, int* tiles) {
    *tiles = apart && j < L.n_p ? 0 : tiles_of(L, j, end);
    return *tiles ? *tiles + kOverhead : 0;
  };
  // a thread has `per` jobs in a row
  const int per = (n + kPrepThreads - 1) / kPrepThreads, j0 = threadIdx.x * per, j1 = min(n, j0 + per);
  int mine = 0, tiles_mine = 0;
  for (int j = j0; j < j1; j++) {
    const int end = SMEM ? ends_s[j] : keys_end(p, L, job_of(p, L, j));
    int tiles;
    const int units = units_of(j, end, &tiles);
    if (SMEM) starts_s[j] = mine;
    else *reinterpret_cast<int2*>(jobs + j) = make_int2(mine, end);   // .x: within the thread, for now
    mine += units;
    tiles_mine += tiles;
  }
  int v = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  const int sum = __reduce_add_sync(0xffffffffu, tiles_mine);
  if (lane == 31) {
    warp_s[warp][0] = v;
    warp_s[warp][1] = sum;
  }
  __syncthreads();
  int before = v - mine, units = 0, tiles_all = 0;
#pragma unroll
  for (int w = 0; w < kPrepThreads / 32; w++) {
    if (w < warp) before += warp_s[w][0];
    units += warp_s[w][0];
    tiles_all += warp_s[w][1];
  }
  for (int j = j0; j < j1; j++) {
    if (SMEM) starts_s[j] += before;
    else jobs[j].x += before;
  }
  if (threadIdx.x == 0) {
    if (SMEM) starts_s[n] = units;
    else jobs[n].x = units;
  }
  // ranges of a job over common keys: so many that the longest range and the line's pieces come out equal, as far as whole numbers let them
  int ranges = 0;
  if (apart) {
    unsigned int best = 0xffffffffu;
    for (int r = lane + 1; r <= min(all_ctas / L.n_p, tiles_p); r += 32) {
      const int others = all_ctas - L.n_p * r;
      const float cost = fmaxf((float)((tiles_p + r - 1) / r), units ? others ? __fdividef((float)units, (float)others) : 4e6f : 0.0f);
      best = min(best, (unsigned int)fminf(cost * 4.0f, 4e6f) << 8 | r);   // (r below 256)
    }
    ranges = __reduce_min_sync(0xffffffffu, best) & 255;
  }
  const int c0 = L.n_p * ranges, C = max(c0 + 1, min(all_ctas, c0 + tiles_all));   // the line's CTAs: from c0 on, no more than there are tiles (a short piece may be a job's start alone)
  for (int c = threadIdx.x; c <= C; c += kPrepThreads) {
    // (a quotient that is no whole number is at least 1 / C away from one, so the double below it is too)
    const int share = units < (1 << 23) ? (int)((unsigned int)units * (unsigned int)max(0, c - c0) / (unsigned int)(C - c0)) : (int)((double)units * (c - c0) / (C - c0));
    bounds_s[c] = c <= c0 ? 0 : share;
  }
  __syncthreads();
  auto start = [&](int j) { return SMEM ? starts_s[j] : jobs[j].x; };
  for (int c = threadIdx.x; c < L.ctas; c += kPrepThreads) {
    const int u0 = c < C ? bounds_s[c] : 0, u1 = c < C ? bounds_s[c + 1] : 0;
    int lo = 0, hi = n;   // the last job that starts at u0 or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= u0) lo = mid;
      else hi = mid;
    }
    // CTA c < c0: range r of job (KV head, row tile), the row tiles next to one another
    int job = -1, t0 = 0, t1 = 0;
    if (c < c0) {
      const int group = c / L.mt_p, kvh = group / ranges, r = group - kvh * ranges;
      job = kvh * L.mt_p + c - group * L.mt_p;
      t0 = tiles_p * r / ranges;
      t1 = tiles_p * (r + 1) / ranges;
    }
    pieces[2 * c] = make_int4(u0, u1, lo, job);
    pieces[2 * c + 1] = make_int4(start(lo), SMEM ? ends_s[lo] : jobs[lo].y, t0, t1);
  }
  auto cta_at = [&](int unit) {   // the CTA that has it
    int lo = c0, hi = C;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bounds_s[mid] <= unit) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  for (int j = threadIdx.x; j < n; j += kPrepThreads) {
    const int s = start(j), s1 = start(j + 1);
    int2 slots = make_int2(0, 0);
    if (apart && j < L.n_p) {
      const int kvh = j / L.mt_p;
      slots = make_int2(kvh * ranges * L.mt_p + j - kvh * L.mt_p, ranges | L.mt_p << 16);
    } else if (s1 > s) {
      const int first = cta_at(s + kOverhead);
      slots = make_int2((j < L.n_p ? j : j - L.n_p) + first, (cta_at(s1 - 1) - first + 1) | 1 << 16);
    }
    if (SMEM) jobs[j] = make_int4(s, ends_s[j], slots.x, slots.y);
    else *reinterpret_cast<int2*>(&jobs[j].z) = slots;
  }
  if (SMEM && threadIdx.x == 0) jobs[n] = make_int4(units, 0, 0, 0);
}

// ---- who does what, for trees --------------------------------------------------------------
// A tree has many rows to a sequence, so most jobs are several row tiles over the same keys.  CTAs come in teams, each of which takes one row tile of the same keys at the
// same time, so that the keys are read from memory once: a sequence's m row tiles (the common keys' too) are cut into as few teams of up to kTeam tiles as there can be, of
// equal width but for one tile.  Teams of one width are jobs on a line of their own, which is cut into equal pieces for the line's share of the CTAs; shares are the
// smallest longest piece.  (32 sequences of up to 16,384 rows and 64 nodes, 24 heads on 4, with the merge that the calls had then: teams of one 578 us, of up to two 543, three 520, four 527,
// six 539; 16 behind 8,192 common rows, 16 on 2: 77, 69, 63, 63, 61.)  Only row tiles and tokens that are there have a place; with all of T for each sequence, half of
// them there, the first took 704 us on one line.  It takes 450 to 480 now in a loop, where the power limit sets the clock (984 W, 1,395 MHz); one call at
// a time, at 1,965 MHz, 410: queries and plan 29, tiles 329, merge 37 (each alone), the rest between them.
constexpr int kTeam = 4;
// What a job's start and end cost, in steps: its queries and masks, the tile at its end whose rows are not seen by all, and the partial result, 4,500 cycles for 128 rows of 256.
// (In us, at 3, 4, 5, 6 steps.  HD 256: one sequence of 16,384 rows and 64 nodes, 24 heads on 4: 82, 70, 65, 65; the same with 188: 151, 157, 130, 131; 16 behind 8,192 common rows,
// 16 nodes, 16 on 2: 45.6, 44.2, 44.2, 44.2; 64 of 2,000 and one, 24 on 4: 58.8, 59.1, 59.9, 60.0.
// HD 128, at 2, 3, 4, 5 steps, 24 on 4: 4 of up to 4,300 and 100: 61.2, 60.4, 61.6, 64.2; 64 of 2,000 and one 46.4, 44.2, 44.5, 45.1; 64 of 4 behind 1,000 31.5, 31.9, 33.0, 33.6; 32 of 32 and up to 500
// 49.8, 49.7, 48.5, 48.4; 16 of up to 8,192 and 64 110, 109, 109, 109; 16 behind 8,192 common rows, 16 nodes, 16 on 2 40.1, 37.0, 37.0, 37.6.)
__host__ __device__ constexpr int tree_overhead(int HD) { return HD == 256 ? 5 : 3; }
// Team job i: {start on its line, job of its first row tile, end of its keys, slot of its first row tile's partial result for team 0}; the slots of a team job's pieces
// are kTeam-wide steps: slot + w * team + rank, which no two pieces share since i + team grows from piece to piece of a line.  jobs[j] = {.., .., first slot, number and
// distance of slots}; pieces[2c] = {start and end of CTA c's piece of its line, first team job in it, end of the line's team jobs}, pieces[2c + 1] = {w * team + rank, rank}.
struct Teams {   // of m row tiles: `wide` teams of w + 1, `all - wide` of w
  int all, wide, w;
  BK_DEVINL explicit Teams(int m) {
    all = (m + kTeam - 1) / kTeam;
    w = all ? m / all : 0;
    wide = m - all * w;
  }
  BK_DEVINL int of_width(int v) const { return v == w ? all - wide : v == w + 1 ? wide : 0; }
};
// floor((n t - less) / of)
BK_DEVINL int share_of(int n, int t, int of, int less = 0) {
  const unsigned long long x = (unsigned long long)n * t - less;
  return x >> 32 ? (int)(x / of) : (int)((unsigned int)x / (unsigned int)of);
}
// one CTA
template <int HD>
BK_DEVINL void plan_trees(const Params<true>& p, const Layout& L, uint8_t* scratch) {
  __shared__ int sum_s[2 * kTeam][kPrepThreads / 32], total_s[2 * kTeam];
  __shared__ int teams_s[kTeam + 1], common_s[kTeam + 1], start_s[kPlanned];   // start_s: of the team jobs, as far as they fit
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = p.Hq / p.Hkv;
  int4* jobs = jobs_of(L, scratch);
  int4* pieces = pieces_of(L, scratch);
  // exclusive sums over the block of n values a thread; the totals in total_s
  auto scan = [&](int* v, int n) {
    int up[2 * kTeam];
#pragma unroll
    for (int k = 0; k < 2 * kTeam; k++) {
      if (k >= n) break;
      up[k] = v[k];
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, up[k], off);
        if (lane >= off) up[k] += o;
      }
      if (lane == 31) sum_s[k][warp] = up[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2 * kTeam; k++) {
      if (k >= n) break;
      int before = up[k] - v[k], all = 0;
#pragma unroll
      for (int w = 0; w < kPrepThreads / 32; w++) {
        if (w < warp) before += sum_s[k][w];
        all += sum_s[k][w];
      }
      v[k] = before;
      if (tid == 0) total_s[k] = all;
    }
    __syncthreads();
  };
  // where each sequence's tokens begin
  const bool compact = p.B <= kCompact;
  int tokens = p.B * p.T;
  if (compact) {
    constexpr int kEach = kCompact / kPrepThreads;
    int n[kEach], at[1] = {0};
    const int per = (p.B + kPrepThreads - 1) / kPrepThreads;
#pragma unroll
    for (int k = 0; k < kEach; k++) {
      const int b = tid * per + k;
      n[k] = k < per && b < p.B ? tree_of(p, b).n : 0;
      at[0] += n[k];
    }
    scan(at, 1);
    tokens = total_s[0];
#pragma unroll
    for (int k = 0; k < kEach; k++) {
      const int b = tid * per + k;
      if (k < per && b < p.B) p.first[b] = at[0];
      at[0] += n[k];
    }
    if (tid == 0) p.first[p.B] = tokens;
    __syncthreads();   // (total_s is used again)
  }
  // groups: the common keys of each KV head, then (sequence, KV head)
  const int commons = L.n_p ? p.Hkv : 0, groups = commons + p.B * p.Hkv, per = (groups + kPrepThreads - 1) / kPrepThreads, g0 = min(groups, tid * per), g1 = min(groups, g0 + per);
  const Teams common((int)(((long long)tokens * G + kRows - 1) / kRows));
  const int common_tiles = tokens ? (L.P + kTile - 1) / kTile : 0;
  auto group_of = [&](int g, Teams* teams, int* tiles, int* end) {
    if (g < commons) {
      *teams = common;
      *tiles = common_tiles;
      *end = L.P;
      return;
    }
    const Tree r = tree_of(p, (g - commons) / p.Hkv);
    *teams = Teams((r.n * G + kRows - 1) / kRows);
    *end = max(L.P, r.base + r.n);
    *tiles = r.n ? (*end - L.P + kTile - 1) / kTile : 0;
  };
  int v[2 * kTeam];   // of each width: team jobs, units
#pragma unroll
  for (int k = 0; k < 2 * kTeam; k++) v[k] = 0;
  Teams teams(0);
  int tiles, end;
  for (int g = g0; g < g1; g++) {
    group_of(g, &teams, &tiles, &end);
    if (tiles == 0) continue;
#pragma unroll
    for (int k = 0; k < kTeam; k++) {
      const int n = teams.of_width(k + 1);
      v[k] += n;
      v[kTeam + k] += n * (tiles + tree_overhead(HD));
    }
  }
  scan(v, 2 * kTeam);
  // shares: the smallest piece X for which the teams that it takes fit; one of 32 candidates between the mean and what surely fits
  if (warp == 0) {
    const int all_ctas = L.ctas;
    float work = 0.0f;
#pragma unroll
    for (int k = 0; k < kTeam; k++) work += (float)(k + 1) * (float)total_s[kTeam + k];
    const float lo = work / (float)all_ctas, hi = all_ctas > kTeam * (kTeam + 1) / 2 ? work / (float)(all_ctas - kTeam * (kTeam + 1) / 2) : 2.0f * work;
    const float X = fmaxf(1.0f, lo + (hi - lo) * (float)(lane + 1) * (1.01f / 32.0f));
    int take[kTeam], sum = 0;
#pragma unroll
    for (int k = 0; k < kTeam; k++) {
      const int units = total_s[kTeam + k];
      take[k] = units ? max(1, (int)ceilf((float)units / X)) : 0;
      sum += (k + 1) * take[k];
    }
    const uint32_t fits = __ballot_sync(0xffffffffu, sum <= all_ctas);
    const int best = fits ? __ffs(fits) - 1 : 31;
#pragma unroll
    for (int k = 0; k < kTeam; k++) {
      take[k] = __shfl_sync(0xffffffffu, take[k], best);
      if (!fits) take[k] = total_s[kTeam + k] ? 1 : 0;
      if (lane == 0) teams_s[k + 1] = take[k];
    }
    if (lane <= kTeam) common_s[lane] = lane && common_tiles ? commons * common.of_width(lane) : 0;   // team jobs over common keys, at a line's front
  }
  __syncthreads();
  // records of team jobs, of their row tiles and of the CTAs whose pieces begin in them
  int list0[kTeam], slot_p[kTeam], slot_s[kTeam], cta0[kTeam];
  {
    int a = 0, b = 0, c = 0, d = 0;
#pragma unroll
    for (int k = 0; k < kTeam; k++) {
      list0[k] = a;
      slot_p[k] = b;
      slot_s[k] = c;
      cta0[k] = d;
      a += total_s[k];
      b += (common_s[k + 1] + teams_s[k + 1]) * (k + 1);
      c += (total_s[k] - common_s[k + 1] + teams_s[k + 1]) * (k + 1);
      d += teams_s[k + 1] * (k + 1);
    }
  }
  for (int g = g0; g < g1; g++) {
    group_of(g, &teams, &tiles, &end);
    const bool is_common = g < commons;
    const int j0 = is_common ? g * L.mt_p : L.n_p + (g - commons) * L.mt_s, row_tiles = is_common ? L.mt_p : L.mt_s;
    int mt = 0;
    for (int i = 0; tiles && i < teams.all; i++) {
      const int w = i < teams.wide ? teams.w + 1 : teams.w;
#pragma unroll
      for (int k = 0; k < kTeam; k++)   // (registers, not indexes)
        if (w == k + 1) {
          const int at = v[k]++, start = v[kTeam + k], len = tiles + tree_overhead(HD), units = total_s[kTeam + k], K = teams_s[k + 1];
          v[kTeam + k] += len;
          const int slot = is_common ? slot_p[k] + at * w : slot_s[k] + (at - common_s[k + 1]) * w;
          p.team[list0[k] + at] = make_int4(start, j0 + mt, end, slot);
          // team t has units [units t / K, units (t + 1) / K): unit u is team ((u + 1) K - 1) / units's
          auto team_at = [&](int u) { return share_of(K, u + 1, units, 1); };
          const int t0 = team_at(start + tree_overhead(HD)), t1 = team_at(start + len - 1);
          for (int r = 0; r < w; r++) jobs[j0 + mt + r] = make_int4(0, 0, slot + t0 * w + r, (t1 - t0 + 1) | w << 16);
          if (list0[k] + at < kPlanned) start_s[list0[k] + at] = start;
        }
      mt += w;
    }
    for (; mt < row_tiles; mt++) jobs[j0 + mt] = make_int4(0, 0, 0, 0);
  }
  __syncthreads();
  for (int cta = tid; cta < L.ctas; cta += kPrepThreads) {
    int4 piece = make_int4(0, 0, 0, 0), more = make_int4(0, 0, 0, 0);   // (without work)
#pragma unroll
    for (int k = 0; k < kTeam; k++) {
      const int K = teams_s[k + 1], c = cta - cta0[k], t = c / (k + 1);
      if (c < 0 || t >= K) continue;
      const int u0 = share_of(total_s[kTeam + k], t, K), u1 = share_of(total_s[kTeam + k], t + 1, K);
      int lo = list0[k], hi = list0[k] + total_s[k];   // the last that starts at u0 or before
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, start = mid < kPlanned ? start_s[mid] : p.team[mid].x;
        if (start <= u0) lo = mid;
        else hi = mid;
      }
      piece = make_int4(u0, u1, lo, list0[k] + total_s[k]);
      more = make_int4(c, c - t * (k + 1), 0, 0);
    }
    pieces[2 * cta] = piece;
    pieces[2 * cta + 1] = more;
  }
}

// row i of a job's tile -> token row e and query head of its group; false past the last
BK_DEVINL bool row_at(const PagedParams& p, const Job& q, int i, int* b, int* t, int* g) {
  const int G = p.Hq / p.Hkv, r = q.mt * kRows + i;
  if (q.seq >= 0) {
    *b = q.seq;
    *t = r / G;
    *g = r - *t * G;
    return r < p.T * G;
  }
  const int bt = r / G;
  *g = r - bt * G;
  *b = bt / p.T;
  *t = bt - *b * p.T;
  return r < p.B * p.T * G;
}

template <int PER>
BK_DEVINL void store_bf16(uint16_t* dst, const float (&x)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; i += 4) *reinterpret_cast<uint2*>(dst + i) = make_uint2(bk_f32x2_to_bf16x2(x[i], x[i + 1]), bk_f32x2_to_bf16x2(x[i + 2], x[i + 3]));
}
// One warp per (token row, head): y = x / sqrt(mean(x^2) + eps) (1 + w), then the rotation of pairs (d, d + rot_half), in f32; q heads to the scratch
// buffer, k and v heads into their page, rounded to bf16: operands of the tensor cores (q's rounding is what the result's error is made of, 0.0024 of
// its norm against 0.0017 for exact arithmetic rounded once).  The first CTA lays out the work of the next launch.  Bound: latency, 5 us for 32
// sequences and 7 for 64 of 24 heads, most of it that CTA's.  Trees: a warp takes up to eight heads of a token one after the other, once there are more than the GPU holds, with what
// they share in registers (2,048 tokens of 28 heads: 42 us a warp for each, so 28; caches cold).
template <int HD, bool TREE>
__global__ void __launch_bounds__(kPrepThreads, TREE ? 3 : 0) paged_prepare_kernel(const Params<TREE> p, const Layout L, uint8_t* scratch) {
  constexpr int PER = HD / 32;
  __shared__ float y_s[kPrepThreads / 32][HD];
  // The wait comes first: a launch behind this call may read, before its own wait, what a launch before this call wrote (weights, settled caches).
  bk_pdl_wait();
  bk_pdl_trigger();
  if (blockIdx.x == 0) {   // (first: it takes longest)
    if constexpr (TREE) plan_trees<HD>(p, L, scratch);
    else if (L.n_p + L.n_s <= kPlanned) plan_jobs<true>(p, L, scratch);
    else plan_jobs<false>(p, L, scratch);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = p.Hq + (p.k ? p.Hkv : 0);
  const int item = (blockIdx.x - 1) * (kPrepThreads / 32) + warp;
  if constexpr (TREE) {   // p.each heads of a token
    const int turns = (heads + p.each - 1) / p.each;
    if (item >= p.T * p.B * turns) return;
    const int e = item / turns, h0 = (item - e * turns) * p.each, h1 = min(heads, h0 + p.each), t = e / p.B, b = e - t * p.B, G = p.Hq / p.Hkv;
    float x[PER];
    auto load = [&](int h) {
      load_bf16((h < p.Hq ? p.qg + ((size_t)e * p.Hq + h) * (p.fused ? 2 : 1) * HD : p.k + ((size_t)e * p.Hkv + h - p.Hq) * HD) + lane * PER, x);
    };
    load(h0);   // (does not wait for what follows)
    const Tree tree = tree_of(p, b);
    const int at = p.fused ? p.pos[e] : 0;
    const bool here = t < tree.n && at >= 0 && (!p.fused || at < p.max_pos);
    int place = b * p.T + t;   // of the token among the ready queries
    if (h0 < p.Hq && p.B <= kCompact) {
      place = 0;
      for (int i = lane; i < b; i += 32) place += tree_of(p, i).n;
      place = __reduce_add_sync(0xffffffffu, place) + t;
    }
    if (h0 == 0) {
      bool sees = here && tree.base > 0;
      if (here && tree.base == 0)
        for (int i = lane; i < (tree.n + 31) / 32; i += 32) sees = sees || node_word(p.mask + (size_t)e * p.words, tree.n, i);
      sees = __any_sync(0xffffffffu, sees);
      if (lane == 0) {
        p.place[e] = sees ? place : -1;
        if (t < tree.n && p.B <= kCompact) p.token[place] = e;
      }
    }
    if (!here) return;
    const int slot = h1 > p.Hq ? p.slot[e] : -1, page = slot >= 0 ? slot / p.page_rows : -1, row_in = slot - page * p.page_rows;
    // what all heads of the token share: norm weights, and of each dim the cosine, the signed sine and the place of the other one of its pair
    float w[PER], c[PER], sn[PER];
    int other[PER];
    auto weights = [&](const uint16_t* from) { load_bf16(from + lane * PER, w); };
    if (p.fused) {
      const float *cr = p.cos_t + (size_t)at * p.rot_half, *sr = p.sin_t + (size_t)at * p.rot_half;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int d = lane * PER + i, half = p.rot_half;
        other[i] = d < half ? d + half : d < 2 * half ? d - half : -1;
        c[i] = other[i] >= 0 ? cr[min(d, other[i])] : 1.0f;
        sn[i] = other[i] < 0 ? 0.0f : d < half ? -sr[d] : sr[d - half];
      }
      weights(h0 < p.Hq ? p.q_norm_w : p.k_norm_w);
    }
    for (int h = h0; h < h1; h++) {
      float y[PER];
#pragma unroll
      for (int i = 0; i < PER; i++) y[i] = x[i];
      if (h + 1 < h1) load(h + 1);
      uint16_t* dst;
      if (h < p.Hq) {
        const int head = h / G;
        dst = p.q + ((size_t)head * p.B * p.T + place) * G * HD + (size_t)(h - head * G) * HD;
      } else {
        if (page < 0 || page >= p.n_pages) break;
        const size_t row = (((size_t)page * p.Hkv + h - p.Hq) * p.page_rows + row_in) * HD;
        dst = p.k_pages + row;
#pragma unroll
        for (int i = 0; i < PER; i += 4)
          *reinterpret_cast<uint2*>(p.v_pages + row + lane * PER + i) = *reinterpret_cast<const uint2*>(p.v + ((size_t)e * p.Hkv + h - p.Hq) * HD + lane * PER + i);
        if (p.fused && h == p.Hq) weights(p.k_norm_w);
      }
      if (p.fused) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) sum = fmaf(y[i], y[i], sum);
        const float rstd = bk_rcp_sqrt(__fadd_rn(__fdiv_rn(bk_warp_sum(sum), (float)HD), p.eps));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PER; i++) y_s[warp][lane * PER + i] = y[i] = __fmul_rn(__fmul_rn(y[i], rstd), __fadd_rn(1.0f, w[i]));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PER; i++)
          if (other[i] >= 0) y[i] = __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(y_s[warp][other[i]], sn[i]));
      }
      store_bf16(dst + lane * PER, y);
    }
    return;
  } else {
  if (item >= p.T * p.B * heads) return;
  const int e = item / heads, h = item - e * heads, t = e / p.B, b = e - t * p.B;
  const bool is_q = h < p.Hq;
  const int kvh = h - p.Hq, G = p.Hq / p.Hkv;
  // what does not wait for the token's row first
  const uint16_t* src = is_q ? p.qg + ((size_t)e * p.Hq + h) * (p.fused ? 2 : 1) * HD : p.k + ((size_t)e * p.Hkv + kvh) * HD;
  float x[PER], w[PER];
  uint2 v[PER / 4];
  load_bf16(src + lane * PER, x);
  if (p.fused) load_bf16((is_q ? p.q_norm_w : p.k_norm_w) + lane * PER, w);
  if (!is_q) {
#pragma unroll
    for (int i = 0; i < PER / 4; i++) v[i] = *reinterpret_cast<const uint2*>(p.v + ((size_t)e * p.Hkv + kvh) * HD + lane * PER + 4 * i);
  }
  const int at = row_of(p, b, t);
  if (at < 0) return;
  uint16_t* dst;
  if (is_q) {
    const int head = h / G;
    dst = p.q + (((size_t)head * p.B + b) * p.T + t) * G * HD + (size_t)(h - head * G) * HD;
  } else {
    const int page = p.table[(size_t)b * p.max_pages + at / p.page_rows];
    if (page < 0 || page >= p.n_pages) return;
    const size_t row = (((size_t)page * p.Hkv + kvh) * p.page_rows + at % p.page_rows) * HD;
    dst = p.k_pages + row;
#pragma unroll
    for (int i = 0; i < PER / 4; i++) *reinterpret_cast<uint2*>(p.v_pages + row + lane * PER + 4 * i) = v[i];
  }
  if (p.fused) {
    const float *cr = p.cos_t + (size_t)at * p.rot_half, *sr = p.sin_t + (size_t)at * p.rot_half;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) sum = fmaf(x[i], x[i], sum);
    const float rstd = bk_rcp_sqrt(__fadd_rn(__fdiv_rn(bk_warp_sum(sum), (float)HD), p.eps));
#pragma unroll
    for (int i = 0; i < PER; i++) y_s[warp][lane * PER + i] = __fmul_rn(__fmul_rn(x[i], rstd), __fadd_rn(1.0f, w[i]));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int d = lane * PER + i;
      const float y = y_s[warp][d];
      if (d < p.rot_half) x[i] = __fsub_rn(__fmul_rn(y, cr[d]), __fmul_rn(y_s[warp][d + p.rot_half], sr[d]));
      else if (d < 2 * p.rot_half) x[i] = __fadd_rn(__fmul_rn(y, cr[d - p.rot_half]), __fmul_rn(y_s[warp][d - p.rot_half], sr[d - p.rot_half]));
      else x[i] = y;
    }
  }
  store_bf16(dst + lane * PER, x);
  }
}

// ---- tensor memory and its instructions ------------------------------------------------
#define BK_R32(F, v, o) F(v[o]), F(v[o + 1]), F(v[o + 2]), F(v[o + 3]), F(v[o + 4]), F(v[o + 5]), F(v[o + 6]), F(v[o + 7]), F(v[o + 8]), F(v[o + 9]), F(v[o + 10]), \
    F(v[o + 11]), F(v[o + 12]), F(v[o + 13]), F(v[o + 14]), F(v[o + 15]), F(v[o + 16]), F(v[o + 17]), F(v[o + 18]), F(v[o + 19]), F(v[o + 20]), F(v[o + 21]), F(v[o + 22]), \
    F(v[o + 23]), F(v[o + 24]), F(v[o + 25]), F(v[o + 26]), F(v[o + 27]), F(v[o + 28]), F(v[o + 29]), F(v[o + 30]), F(v[o + 31])
#define BK_OUT(x) "=r"(x)
#define BK_IN(x) "r"(x)
// 32 or 16 columns of the calling lane's row.  The wait is part of it, so that no use of a register can come before.
BK_DEVINL void tmem_ld32(uint32_t at, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : BK_R32(BK_OUT, v, 0)
      : "r"(at)
      : "memory");
}
BK_DEVINL void tmem_st32(uint32_t at, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      BK_R32(BK_IN, v, 0)
      : "memory");
}
BK_DEVINL void tmem_st16(uint32_t at, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
BK_DEVINL void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
BK_DEVINL void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
BK_DEVINL void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
BK_DEVINL void tc_commit(uint32_t bar) {   // arrives when every MMA issued so far has completed
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (+)= A * B, M = 128, K = 16; A in tensor memory
template <bool ACC>
BK_DEVINL void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred pz;\n\tsetp.ne.b32 pz, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pz;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
               "n"(ACC ? 1 : 0)
               : "memory");
}
// Operand B in shared memory, rows of 128 bytes swizzled in groups of 8 (1,024 bytes).  K-major (keys): group_stride between groups of 8 keys.
// MN-major (values): 64 dims are a row of a key; block_stride between blocks of 64 dims, group_stride between groups of 8 keys.
BK_DEVINL uint64_t smem_desc(uint32_t addr, uint32_t block_stride, uint32_t group_stride) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((block_stride >> 4) & 0x3fffu) << 16) | ((uint64_t)((group_stride >> 4) & 0x3fffu) << 32) | (1ull << 46) | (2ull << 61);
}
// bf16 x bf16 -> f32, M = 128
__host__ __device__ constexpr uint32_t mma_shape(int n, bool b_mn_major) { return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24); }

BK_DEVINL void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
BK_DEVINL bool elect_lane() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}
// A wait of a warp that stays together: whether the phase has completed.  Bounded by time (a poll may sleep): the first wait of a CTA that gives up, after
// 2^31 cycles, sets the status word and `dead`, after which the others return at once and the kernel runs to its end.  Who was to arm a barrier, issue a copy
// or MMAs after a wait that gave up does not, so that what is on its way can be waited for at the end.
BK_DEVINL bool bar_wait_warp(uint32_t bar, uint32_t parity, int* status, volatile int* dead) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long from = clock64();
#pragma unroll 1
  do {
    const bool here = mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, here || *dead)) return __all_sync(0xffffffffu, here);
  } while (__any_sync(0xffffffffu, clock64() - from < (1ll << 31)));
  *dead = 1;
  atomicExch(status, 10003 /* BK_ERR_TIMEOUT */);
  return false;
}
// The end of a CTA where a wait gave up: no longer than 2^16 polls.
BK_DEVINL void bar_settle(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int it = 0; it < (1 << 16) && !mbar_try_wait(bar, parity); it++) {
  }
}
BK_DEVINL void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
BK_DEVINL float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
BK_DEVINL float exp2_approx(float x) {   // 2^x to 2 ulp or so; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two bf16 values, zeros in the place of those that are not finite
BK_DEVINL uint32_t finite_pair(uint32_t v) {
  return ((v & 0x7f80u) == 0x7f80u ? 0u : v & 0xffffu) | ((v & 0x7f800000u) == 0x7f800000u ? 0u : v & 0xffff0000u);
}
// an f32 sum, plus a bf16 value if that is not finite
BK_DEVINL uint32_t odd_value(uint32_t sum, uint16_t v) {
  return (v & 0x7f80u) == 0x7f80u ? __float_as_uint(__fadd_rn(__uint_as_float(sum), bk_bf16_to_f32(v))) : sum;
}

// Adds to a row's sums of 32 dims, d and on, the values of keys k0 to k1 - 1 below the row's limit that are not finite.  Whole warps, of one job.
// (A call: in line it is in the way of every piece, 0.2 us of a short call.)
// (bits, tree: of a row of a tree, whose limit is its first node)
template <bool TREE>
__device__ __noinline__ void add_odd_values(const PagedParams& p, const Job& q, int HD, int d, int k0, int k1, int limit, const uint32_t* bits, Tree tree, uint32_t* o) {
  const int lane = threadIdx.x & 31;
  auto values = [&](int key) {   // (nullptr: rows of zeros)
    const int page = __ldg(p.table + (size_t)max(q.seq, 0) * p.max_pages + key / p.page_rows);
    return page >= 0 && page < p.n_pages ? p.v_pages + (((size_t)page * p.Hkv + q.kvh) * p.page_rows + key % p.page_rows) * HD + d : nullptr;
  };
#pragma unroll 1
  for (int k = k0; k < k1; k += 8) {   // eight keys at once, a lane eight dims of one
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k + (lane >> 2) < k1) {
      const uint16_t* at = values(k + (lane >> 2));
      if (at) v = *reinterpret_cast<const uint4*>(at + (lane & 3) * 8);
    }
    const bool odd = ((v.x ^ finite_pair(v.x)) | (v.y ^ finite_pair(v.y)) | (v.z ^ finite_pair(v.z)) | (v.w ^ finite_pair(v.w))) != 0;
    uint32_t found = __ballot_sync(0xffffffffu, odd);
    while (found) {
      const int i = (__ffs(found) - 1) >> 2;
      found &= ~(15u << (4 * i));
      const uint16_t* at = values(k + i);
      bool sees = k + i < limit;
      if constexpr (TREE) sees = sees || (bits && (seen_keys(bits, tree, k + i) & 1u));
      if (sees) {
#pragma unroll
        for (int y = 0; y < 32; y++) o[y] = odd_value(o[y], at[y]);
      }
    }
  }
}

// positions in the stream of a piece's tiles: K0, K1, V0, K2, V1, ..., V(n-1)
BK_DEVINL int stream_v(int i, int n) { return i < n - 1 ? 2 * i + 2 : 2 * n - 1; }

template <int kStages>
struct TileShared {   // behind the tiles
  uint64_t full[kStages], empty[kStages], q_here, q_empty, q_full, s_full[2], p_full[2], o_full[2], settled;
  float m_s[2][2][kRows];   // [tile & 1][half of the keys]: largest score
  int odd_from[3], odd_to[3];   // [piece mod 3]: keys between which values were not finite and were taken out, see there
  uint32_t tmem_slot;
  int dead;
};
template <int HD>
struct TileCfg {
  static constexpr int kStage = kTile * HD * 2;               // bytes of 64 keys or values
  static constexpr int kStages = HD == 256 ? 5 : 12;
  static constexpr int kQuery = kRows * HD * 2;               // bytes of the queries
  static constexpr int kSmem = kQuery + kStages * kStage + (int)sizeof(TileShared<kStages>);
  static constexpr int kO = 0, kQ = HD, kS = HD + HD / 2;     // tensor memory: output, queries, two buffers of scores (then probabilities)
};
constexpr int kCopyWarp = 8, kMmaWarp = 9, kQueryWarp = 10, kTileThreads = 352;   // warps 0-3 and 4-7: a row each lane, halves of a tile's keys

// S = Q K^T and O += P V on the tensor cores.  Q, S, P and O live in tensor memory, a row per lane (with Q in shared memory its reads, 64 KB a step,
// make a step 500 cycles longer: K, V twice and what TMA writes take three quarters of that bandwidth); a ring of K and V tiles of 64 rows in shared
// memory, by TMA.  Q comes by TMA too, ahead of its turn, and is moved by the lanes that own the rows.  P = 2^(S c - m) with the running maximum m of the row; it overwrites its S as two bf16 matrices, the
// rounded values and what rounding left (16 bits of the value; with 8 the result's error against exact arithmetic is 1.7 times that of its own rounding).
// m is only moved when a score passes it by more than 2^8, since O must be rescaled then.  Row sums are in f32, by the lane that owns the row.
// Bound: the MMAs, 1,650 of the 2,000 cycles that a step of 128 rows and 64 keys takes (HD 256): QK^T once, P V twice for the two matrices.  With P
// rounded once the call of 64 sequences took 85 us for 92 but the error is 0.0029.  Four stages in the ring for five: 92 us for 90.4.
template <int HD, bool TREE>
__global__ void __launch_bounds__(kTileThreads, 1) paged_tile_kernel(const __grid_constant__ TileParams<TREE> P) {
  using C = TileCfg<HD>;
  const Params<TREE>& p = P.g;
  const Layout& L = P.L;
  extern __shared__ __align__(1024) uint8_t q_s[];   // queries [HD / 64][kRows][64], then the ring: stages [HD / 64][kTile][64]
  uint8_t* ring = q_s + C::kQuery;
  TileShared<C::kStages>& sh = *reinterpret_cast<TileShared<C::kStages>*>(ring + C::kStages * C::kStage);
  uint64_t *full = sh.full, *empty = sh.empty, *s_full = sh.s_full, *p_full = sh.p_full, *o_full = sh.o_full;
  uint64_t &q_here = sh.q_here, &q_empty = sh.q_empty, &q_full = sh.q_full;
  auto& m_s = sh.m_s;
  uint32_t& tmem_slot = sh.tmem_slot;
  int& dead_s = sh.dead;
  volatile int* dead = &dead_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    dead_s = 0;
    for (int i = 0; i < 3; i++) {
      sh.odd_from[i] = 0x7fffffff;
      sh.odd_to[i] = -1;
    }
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(smem_u32(full + i), 1);
      mbar_init(smem_u32(empty + i), 1);
    }
    mbar_init(smem_u32(&q_here), 1);
    mbar_init(smem_u32(&q_empty), 8);
    mbar_init(smem_u32(&q_full), 8);
    mbar_init(smem_u32(&sh.settled), 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(s_full + i), 1);
      mbar_init(smem_u32(p_full + i), 8);
      mbar_init(smem_u32(o_full + i), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kCopyWarp && lane < 4)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &P.k_map : lane == 1 ? &P.v_map : P.q_map + (lane - 2)) : "memory");
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  bk_pdl_wait();
  bk_pdl_trigger();   // (the merge reads the plan before its own wait)

  const int4* jobs = jobs_of(L, P.scratch);
  const int cta = blockIdx.x, n_jobs = L.n_p + L.n_s;
  const int4 line = __ldcg(pieces_of(L, P.scratch) + 2 * cta), first = __ldcg(pieces_of(L, P.scratch) + 2 * cta + 1);
  const int u0 = line.x, u1 = line.y;
  int j = line.z - 1;
  // the next piece: a range of common keys, then the line's jobs from j + 1 on
  struct Piece {
    Job q;
    int key1, t0, t1;
    size_t slot;   // of its partial result, among its kind's
  };
  bool began = false;
  auto next_piece = [&](Piece* x) {
    if constexpr (TREE) {
      while (++j < line.w) {
        const int4 team = __ldcg(p.team + j);
        if (team.x >= u1) return false;
        x->q = job_of(p, L, team.y + first.y);
        piece_of(team.x, (team.z - x->q.key0 + kTile - 1) / kTile, u0, u1, &x->t0, &x->t1, tree_overhead(HD));
        if (x->t0 >= x->t1) continue;
        x->key1 = team.z;
        x->slot = team.w + first.x;
        return true;
      }
      return false;
    }
    if (!began) {
      began = true;
      if (line.w >= 0) {
        x->q = job_of(p, L, line.w);
        x->key1 = L.P;
        x->t0 = first.z;
        x->t1 = first.w;
        x->slot = cta;
        return true;
      }
    }
    while (++j < n_jobs) {
      int2 job = make_int2(first.x, first.y);   // start, end of the keys
      if (j != line.z) job = __ldcg(reinterpret_cast<const int2*>(jobs + j));
      if (job.x >= u1) return false;
      piece_of(job.x, tiles_of(L, j, job.y), u0, u1, &x->t0, &x->t1);
      if (x->t0 >= x->t1) continue;
      x->q = job_of(p, L, j);
      x->key1 = job.y;
      x->slot = (j < L.n_p ? j : j - L.n_p) + cta;
      return true;
    }
    return false;
  };
  Piece x;
  int armed = 0;   // copies' barriers so far: of the ring, of the queries

  {
    if (warp == kCopyWarp) {
      // ================= copies: lane (chunk, block) takes box_rows rows x 64 dims =================
      asm volatile("fence.proxy.async;" ::: "memory");   // rows that an earlier kernel stored
      constexpr int kBlocks = HD / 64;
      const int chunks = kTile / P.box_rows, n_box = chunks * kBlocks;
      const int chunk = lane / kBlocks, block = lane % kBlocks;
      const int no_row = p.n_pages * p.Hkv * p.page_rows;   // behind the last row: such a box is filled with zeros
      const uint32_t box_at = block * (kTile * 128) + chunk * P.box_rows * 128;
      int stage = 0;
      uint32_t parity = 1;
      bool going = true;
      while (going && next_piece(&x)) {
        const Job q = x.q;
        const int t0 = x.t0, t1 = x.t1, key1 = x.key1;
        const int* table = p.table + (size_t)max(q.seq, 0) * p.max_pages;
        auto row_of_tile = [&](int i) {   // row of the map that this lane's box of tile i starts at
          const int key = q.key0 + i * kTile + chunk * P.box_rows;
          if (lane >= n_box || i >= t1 || key >= key1 || key / p.page_rows >= p.max_pages) return no_row;
          const int page = __ldg(table + key / p.page_rows);
          return page >= 0 && page < p.n_pages ? (page * p.Hkv + q.kvh) * p.page_rows + key % p.page_rows : no_row;
        };
        auto load = [&](const CUtensorMap* map, int row) {
          if (!bar_wait_warp(smem_u32(empty + stage), parity, P.status, dead)) return false;
          armed++;
          const uint32_t bar = smem_u32(full + stage);
          if (lane == 0) mbar_expect_tx(bar, C::kStage);
          __syncwarp();
          if (lane < n_box) tma_load(smem_u32(ring + (size_t)stage * C::kStage) + box_at, map, block * 64, row, bar);
          if (++stage == C::kStages) {
            stage = 0;
            parity ^= 1u;
          }
          return true;
        };
        int next = row_of_tile(t0), before = 0;
        for (int i = t0; going && i <= t1; i++) {
          const int row = next;
          next = row_of_tile(i + 1);
          if (i < t1) going = load(&P.k_map, row);
          if (going && i > t0) going = load(&P.v_map, before);
          before = row;
        }
      }
    } else if (warp == kMmaWarp) {
      // ================= MMAs =================
      // Scores of tile i, then the output of tile i - 1.  What the second half of a batch does not need is waited for ahead of it, while the
      // first half runs.  Bound: the MMAs (1,650 cycles a step: 16 of 128 x 64 and 8 of 128 x 256) and, while little is queued, what this warp does
      // between them, so addresses are counted up, not made from positions.
      constexpr uint32_t kShapeS = mma_shape(kTile, false), kShapeO = mma_shape(HD, true);
      const uint64_t k_desc0 = smem_desc(smem_u32(ring), 16, 1024), v_desc0 = smem_desc(smem_u32(ring), kTile * 128, 1024);
      const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), s_full0 = smem_u32(s_full), p_full0 = smem_u32(p_full), o_full0 = smem_u32(o_full);
      int stage = 0, tile = 0, pieces = 0;   // tile: counted over all pieces
      uint32_t parity = 0;
      auto next_stage = [&]() {
        if (++stage == C::kStages) {
          stage = 0;
          parity ^= 1u;
        }
      };
      bool going = true;
      auto wait = [&](uint32_t bar, uint32_t par) { going = bar_wait_warp(bar, par, P.status, dead) && going; };
      auto scores = [&](int half, uint64_t desc, int t) {   // (the probabilities that this buffer held have been multiplied: MMAs run in order)
        const uint32_t d = tmem + C::kS + (t & 1) * kTile;
#pragma unroll
        for (int y = 0; y < HD / 32; y++) {
          const int ks = half * (HD / 32) + y;
          const uint64_t at = desc + ((ks >> 2) * (kTile * 128) + (ks & 3) * 32) / 16;
          if (ks == 0) tc_mma<false>(d, tmem + C::kQ + ks * 8, at, kShapeS);
          else tc_mma<true>(d, tmem + C::kQ + ks * 8, at, kShapeS);
        }
      };
      auto output = [&](int half, uint64_t desc, int t, bool first) {   // the rounded probabilities, then what rounding left
        const uint32_t p_at = tmem + C::kS + (t & 1) * kTile + half * 32;
#pragma unroll
        for (int ks = 0; ks < kTile / 16; ks++) {
          if (ks == 0 && half == 0 && first) tc_mma<false>(tmem + C::kO, p_at, desc, kShapeO);
          else tc_mma<true>(tmem + C::kO, p_at + ks * 8, desc + ks * (2048 / 16), kShapeO);
        }
      };
      while (going && next_piece(&x)) {
        const int n = x.t1 - x.t0;
        wait(full0 + stage * 8, parity);
        wait(smem_u32(&q_full), pieces & 1);
        if (!going) break;
        tc_after();
        // the first tile's scores
        if (elect_lane()) {
          scores(0, k_desc0 + stage * (C::kStage / 16), tile);
          scores(1, k_desc0 + stage * (C::kStage / 16), tile);
          tc_commit(empty0 + stage * 8);
          tc_commit(s_full0 + (tile & 1) * 8);
        }
        next_stage();
        if (n > 1) wait(full0 + stage * 8, parity);
        for (int i = 1; i <= n; i++) {
          const int t = tile + i - 1;   // whose output is added
          const uint32_t k_bar = empty0 + stage * 8;
          const uint64_t k_desc = k_desc0 + stage * (C::kStage / 16);
          if (i < n) {
            if (elect_lane()) scores(0, k_desc, t + 1);
            next_stage();
          }
          const uint64_t v_desc = v_desc0 + stage * (C::kStage / 16);
          const uint32_t v_bar = empty0 + stage * 8;
          wait(p_full0 + (t & 1) * 8, (t >> 1) & 1);
          wait(full0 + stage * 8, parity);
          if (!going) break;
          tc_after();
          next_stage();
          if (elect_lane()) {
            if (i < n) {
              scores(1, k_desc, t + 1);
              tc_commit(k_bar);
              tc_commit(s_full0 + ((t + 1) & 1) * 8);
            }
            output(0, v_desc, t, i == 1);
          }
          if (i + 1 < n) wait(full0 + stage * 8, parity);
          if (elect_lane()) {
            output(1, v_desc, t, false);
            tc_commit(v_bar);
            tc_commit(o_full0 + (t & 1) * 8);
          }
        }
        __syncwarp();
        tile += n;
        pieces++;
      }
    } else if (warp == kQueryWarp) {
      // ================= queries of a piece, as soon as those before have moved on =================
      asm volatile("fence.proxy.async;" ::: "memory");   // rows that the kernel before stored
      uint32_t parity = 1;
      while (next_piece(&x)) {
        const bool common = x.q.seq < 0;
        const CUtensorMap* map = P.q_map + common;
        const int rows = P.q_rows[common];
        int row = common ? x.q.kvh * p.B * p.T * (p.Hq / p.Hkv) : (x.q.kvh * p.B + x.q.seq) * p.T * (p.Hq / p.Hkv);
        if constexpr (TREE) {
          if (!common && p.B <= kCompact) row = (x.q.kvh * p.B * p.T + __ldcg(p.first + x.q.seq)) * (p.Hq / p.Hkv);
        }
        if (!bar_wait_warp(smem_u32(&q_empty), parity, P.status, dead)) break;
        armed++;
        if (lane == 0) mbar_expect_tx(smem_u32(&q_here), rows * HD * 2);
        __syncwarp();
        if (lane < HD / 64) tma_load(smem_u32(q_s) + lane * (kRows * 128), map, lane * 64, row + x.q.mt * kRows, smem_u32(&q_here));
        parity ^= 1u;
      }
    } else {
      // ================= rows: thread <-> row of the tile; two groups of four warps have 32 keys of it each =================
      // (A group a tile, taking turns, made the way from a tile's scores to its probabilities twice as long, and with two buffers of scores the
      // MMAs waited for it.)
      const int group = warp >> 2, quarter = warp & 3, i_row = threadIdx.x & 127;
      const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
      const float c = __fmul_rn(p.scale, 1.44269504088896341f);   // scores in powers of two
      int tile = 0, stream = 0, pieces = 0;   // counted over all pieces
      // A wait tells a phase from the next one only, so nobody may be two phases off.  Scores of a tile that are there mean that the output of
      // the tile two before is, so with a barrier for even and one for odd tiles the waits below are within one.
      auto wait_output = [&](int t) {
        bar_wait_warp(smem_u32(o_full + (t & 1)), (t >> 1) & 1, P.status, dead);
        tc_after();
      };
      // (Trees: the next piece is looked up while this one's last output is made; its loads in a row are 1,500 cycles.)
      bool more = TREE && next_piece(&x);
      for (; TREE ? more : next_piece(&x); pieces++) {
        const Job q = x.q;
        const int t0 = x.t0, n = x.t1 - t0, key1 = x.key1;
        int b, t, g, limit = 0x7fffffff;   // (lanes without a row: never masked, never read)
        bool mine = row_at(p, q, i_row, &b, &t, &g);
        if constexpr (TREE) {
          if (q.seq < 0 && p.B <= kCompact) {
            const int at = b * p.T + t;   // (row_at took the rows for T of each sequence)
            mine = mine && at < __ldcg(p.first + p.B);
            const int e = mine ? __ldcg(p.token + at) : 0;
            t = e / p.B;
            b = e - t * p.B;
          }
        }
        Tree tree = {0, 0};
        const uint32_t* bits = nullptr;   // of a row of a tree
        if constexpr (TREE) {
          if (mine) {
            tree = tree_of(p, b);
            mine = t < tree.n;
          }
          if (mine) {
            bits = p.mask + ((size_t)t * p.B + b) * p.words;
            limit = min(tree.base, key1);
          }
        } else if (mine) {
          limit = min(row_of(p, b, t) + 1, key1);
        }
        __syncwarp();
        const bool warp_on = __any_sync(0xffffffffu, mine);
        // Tiles from this key on have a row that does not see all of them.  There a value that is not finite must not meet a zero probability (0 * inf):
        // it is taken out of the tile, and given back at the end to the rows that see it.
        int seen_by_all = key1;
        if (q.seq >= 0) {
          if constexpr (TREE) {
            seen_by_all = tree_of(p, q.seq).base;
          } else {
            const int first = q.mt * kRows / (p.Hq / p.Hkv), count = p.n_new ? min(p.n_new[q.seq], p.T) : p.T;
            seen_by_all = max(0, p.lens[q.seq] - count + first) + 1;
          }
        } else {
          int uneven;
          asm volatile("{ .reg .pred a, b; setp.ne.s32 a, %1, 0; barrier.cta.red.or.pred b, 5, 256, a; selp.s32 %0, 1, 0, b; }"
                       : "=r"(uneven)
                       : "r"((int)(mine && (TREE || limit > 0) && limit < key1))
                       : "memory");
          if (uneven) seen_by_all = 0;
        }
        const int odd = pieces % 3;
        if (threadIdx.x == 0) {   // the next piece's; who read these two pieces ago has moved its queries since
          sh.odd_from[(pieces + 1) % 3] = 0x7fffffff;
          sh.odd_to[(pieces + 1) % 3] = -1;
        }
        uint2 ahead = make_uint2(0, 0);
        if constexpr (TREE) {
          const int key = q.key0 + t0 * kTile + group * 32;
          if (mine && key + 32 > limit) ahead = ask_seen(bits, tree, key);
        }
        // queries into tensor memory, half of the dims a group (the MMAs that read the ones before have completed: their output was there)
        bar_wait_warp(smem_u32(&q_here), pieces & 1, P.status, dead);
        tc_after();
        // Lanes without a row get zeros: their scores are then zeros, which read as probabilities are zeros too, and zeros cost the tensor
        // cores less power than what was there.
#pragma unroll
        for (int d = group * (HD / 128); d < (group + 1) * (HD / 128); d++) {
          uint32_t v[32];
#pragma unroll
          for (int y = 0; y < 8; y++) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (mine) w = *reinterpret_cast<const uint4*>(q_s + d * (kRows * 128) + i_row * 128 + ((y ^ (i_row & 7)) << 4));   // (as TMA swizzles them)
            v[4 * y] = w.x; v[4 * y + 1] = w.y; v[4 * y + 2] = w.z; v[4 * y + 3] = w.w;
          }
          __syncwarp();
          tmem_st32(lanes + C::kQ + d * 32, v);
        }
        tmem_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) {
          bar_arrive(smem_u32(&q_full));
          bar_arrive(smem_u32(&q_empty));   // (in this order: the next queries' turn comes after all of these)
        }
        float m = -INFINITY, l = 0.0f;   // the maximum, and this group's part of the row sum
        for (int i = 0; i < n; i++, tile++) {
          const int tile_key = q.key0 + (t0 + i) * kTile, there = min(kTile, key1 - tile_key), key = tile_key + group * 32;
          const uint32_t s_at = lanes + C::kS + (tile & 1) * kTile;
          const uint2 nodes = ahead;   // of a tree's row, the words of these keys
          if constexpr (TREE) {
            if (mine && i + 1 < n && key + kTile + 32 > limit) ahead = ask_seen(bits, tree, key + kTile);
          }
          bar_wait_warp(smem_u32(s_full + (tile & 1)), (tile >> 1) & 1, P.status, dead);
          tc_after();
          const bool mixed = tile_key + there > seen_by_all;
          // values past the end count as zeros, whatever the page holds there; those that are not finite are taken out where some row does not see them
          auto settle_values = [&]() {
            const int v_pos = stream + stream_v(i, n), v_stage = v_pos % C::kStages;
            bar_wait_warp(smem_u32(full + v_stage), (v_pos / C::kStages) & 1, P.status, dead);
            uint8_t* v_at = ring + (size_t)v_stage * C::kStage;
            for (int y = threadIdx.x; y < (kTile - there) * (HD / 8); y += 256) {
              const int row = there + y / (HD / 8), piece = y % (HD / 8);
              *reinterpret_cast<uint4*>(v_at + (piece >> 3) * (kTile * 128) + row * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            auto take_out = [&](int from) {
              for (int y = threadIdx.x; y < there * (HD / 8); y += 256) {   // (the same rows a thread as it looked at)
                const int row = y / (HD / 8), piece = y % (HD / 8);
                if (row < from) continue;
                uint4* at = reinterpret_cast<uint4*>(v_at + (piece >> 3) * (kTile * 128) + row * 128 + (piece & 7) * 16);
                const uint4 v = *at, w = make_uint4(finite_pair(v.x), finite_pair(v.y), finite_pair(v.z), finite_pair(v.w));
                if (((v.x ^ w.x) | (v.y ^ w.y) | (v.z ^ w.z) | (v.w ^ w.w)) != 0) {
                  *at = w;
                  atomicMin(&sh.odd_from[odd], tile_key + row);
                  atomicMax(&sh.odd_to[odd], tile_key + row);
                }
              }
            };
            if constexpr (TREE) {
              // Most jobs of trees end with such tiles: one look at the rows of the tree (all see those before) with all loads on the way, and no fence where nothing was written.
              bool wrote = there < kTile;
              if (mixed) {
                const int from = max(0, seen_by_all - tile_key);
                uint32_t some = 0;   // bits 15 and 31 of a sum are set by an exponent of ones
#pragma unroll
                for (int z = 0; z < kTile * HD / 8; z += 256) {
                  const int y = z + threadIdx.x, row = y / (HD / 8), piece = y % (HD / 8);
                  if (row >= from && row < there) {
                    const uint4 v = *reinterpret_cast<const uint4*>(v_at + (piece >> 3) * (kTile * 128) + row * 128 + (piece & 7) * 16);
                    some |= ((v.x & 0x7f807f80u) + 0x00800080u) | ((v.y & 0x7f807f80u) + 0x00800080u) | ((v.z & 0x7f807f80u) + 0x00800080u) | ((v.w & 0x7f807f80u) + 0x00800080u);
                  }
                }
                if (some & 0x80008000u) {
                  take_out(from);
                  wrote = true;
                }
              }
              if (wrote) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            } else {
              if (mixed) take_out(0);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
          };
          // Trees: beside the probabilities, which need no values: 1,250 cycles a tile instead of 2,900 ahead of them, with the look above (16 sequences of 16 nodes: 49 to 46 us).
          const bool settle = there < kTile || mixed;
          if (!TREE && settle) settle_values();
          if (warp_on) {
            uint32_t s[32];
            tmem_ld32(s_at + group * 32, s);
            if (!__all_sync(0xffffffffu, key + 32 <= limit)) {
              uint32_t seen = 0xffffffffu;
              if (TREE && mine) {
                seen = tell_seen(nodes, tree, key);
                if (key + 32 > key1) seen &= key >= key1 ? 0u : (1u << (key1 - key)) - 1u;
              }
#pragma unroll
              for (int y = 0; y < 32; y++) s[y] = (TREE ? (seen >> y & 1u) != 0u : key + y < limit) ? s[y] : 0xff800000u;
            }
            float top[4];   // four chains: one alone is 32 results of the instruction before
#pragma unroll
            for (int y = 0; y < 4; y++) top[y] = max3(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1]), __uint_as_float(s[2 * y + 8]));
#pragma unroll
            for (int y = 0; y < 4; y++) top[y] = max3(top[y], __uint_as_float(s[2 * y + 9]), __uint_as_float(s[2 * y + 16]));
#pragma unroll
            for (int y = 0; y < 4; y++) top[y] = max3(top[y], __uint_as_float(s[2 * y + 17]), __uint_as_float(s[2 * y + 24]));
#pragma unroll
            for (int y = 0; y < 4; y++) top[y] = fmaxf(top[y], __uint_as_float(s[2 * y + 25]));
            float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]);
            m_s[tile & 1][group][i_row] = mx;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");   // (both halves have been read, too: probabilities may go over them)
            mx = __fmul_rn(fmaxf(mx, m_s[tile & 1][group ^ 1][i_row]), c);
            const bool move = mine && mx > __fadd_rn(m, 8.0f);
            if (__any_sync(0xffffffffu, move)) {
              const bool rescale = move && m != -INFINITY;
              const float f = rescale ? exp2_approx(__fsub_rn(m, mx)) : 1.0f;
              l = __fmul_rn(l, f);
              if (move) m = mx;
              if (__any_sync(0xffffffffu, rescale)) {   // the output so far, half of the dims a group
                wait_output(tile - 1);
#pragma unroll 1
                for (int d = group * (HD / 64); d < (group + 1) * (HD / 64); d++) {
                  uint32_t o[32];
                  tmem_ld32(lanes + C::kO + d * 32, o);
#pragma unroll
                  for (int y = 0; y < 32; y++) o[y] = __float_as_uint(__fmul_rn(__uint_as_float(o[y]), f));
                  tmem_st32(lanes + C::kO + d * 32, o);
                }
              }
            }
            const float base = m == -INFINITY ? 0.0f : m;
            float2 sum[2];
            uint32_t lo[16];
#pragma unroll
            for (int y = 0; y < 16; y++) {
              const float2 z = bk_fma2(make_float2(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1])), make_float2(c, c), make_float2(-base, -base));
              const float2 e = make_float2(exp2_approx(z.x), exp2_approx(z.y));
              sum[y & 1] = y < 2 ? e : bk_add2(sum[y & 1], e);
              s[y] = bk_f32x2_to_bf16x2(e.x, e.y);
              const float2 left = bk_fma2(make_float2(__uint_as_float(s[y] << 16), __uint_as_float(s[y] & 0xffff0000u)), make_float2(-1.0f, -1.0f), e);
              lo[y] = bk_f32x2_to_bf16x2(left.x, left.y);
            }
            const float2 all = bk_add2(sum[0], sum[1]);
            l = __fadd_rn(l, __fadd_rn(all.x, all.y));
            tmem_st16(s_at + group * 16, s);
            tmem_st16(s_at + 32 + group * 16, lo);
            tmem_wait_st();
          }
          if (TREE && settle) settle_values();   // (a tree's rows are the last tiles of most jobs: their values come while probabilities are made)
          tc_before();
          __syncwarp();
          if (lane == 0) bar_arrive(smem_u32(p_full + (tile & 1)));
        }
        stream += 2 * n;
        const size_t x_slot = x.slot;
        if (TREE) more = next_piece(&x);
        // the piece's part of the result, half of the dims a group
        wait_output(tile - 1);
        if (warp_on) {
          const bool common = q.seq < 0;
          const int rows = common ? kRows : L.rows_s;
          const size_t slot = x_slot * rows;
          float* ml = reinterpret_cast<float*>(P.scratch + (common ? L.ml_p : L.ml_s)) + (slot + i_row) * 4;
          uint4* o_to = reinterpret_cast<uint4*>(P.scratch + (common ? L.o_p : L.o_s)) + slot * (HD / 4) + i_row;   // [HD / 4][rows] x 4 dims: lanes side by side
          if (mine) {
            if (group == 0) ml[0] = m;
            ml[1 + group] = l;
          }
          __syncwarp();
#pragma unroll 1
          for (int d = group * (HD / 64); d < (group + 1) * (HD / 64); d++) {
            uint32_t o[32];
            tmem_ld32(lanes + C::kO + d * 32, o);
            int k0 = *reinterpret_cast<volatile int*>(&sh.odd_from[odd]), k1 = *reinterpret_cast<volatile int*>(&sh.odd_to[odd]) + 1;
            // Where all rows see a value that is not finite it went through the MMAs, and what the two parts of a probability, one of them zero or
            // negative, make of an infinity is NaN.  Sums that are NaN are made anew, of all the piece's values that are not finite; if there are none
            // that this row sees, it is the scores that are NaN.
            const float2 zero = make_float2(0.0f, 0.0f);
            float2 probe[4] = {zero, zero, zero, zero};   // stay zeros while sums are finite (one chain is 0.1 us more)
#pragma unroll
            for (int y = 0; y < 16; y++) probe[y & 3] = bk_fma2(make_float2(__uint_as_float(o[2 * y]), __uint_as_float(o[2 * y + 1])), zero, probe[y & 3]);
            const float2 all = bk_add2(bk_add2(probe[0], probe[1]), bk_add2(probe[2], probe[3]));
            const bool anew = __any_sync(0xffffffffu, mine && (TREE || limit > 0) && __fadd_rn(all.x, all.y) != 0.0f);
            if (anew) {
              k0 = q.key0 + t0 * kTile;
              k1 = min(key1, k0 + n * kTile);
            }
            if (k0 < k1) {   // (nearly never)
              uint32_t z[32];
#pragma unroll
              for (int y = 0; y < 32; y++) z[y] = anew && isnan(__uint_as_float(o[y])) ? 0u : o[y];
              add_odd_values<TREE>(p, q, HD, d * 32, k0, k1, limit, bits, tree, z);
#pragma unroll
              for (int y = 0; y < 32; y++)
                if (!(isnan(__uint_as_float(o[y])) && isfinite(__uint_as_float(z[y])))) o[y] = z[y];
            }
            if (mine) {
#pragma unroll
              for (int y = 0; y < 32; y += 4) o_to[(size_t)(d * 8 + y / 4) * rows] = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
            __syncwarp();
          }
        }
        tc_before();
      }
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  // The MMAs have waited for every copy, and the rows for every MMA, unless a wait gave up: then what is on its way is waited for here.
  if (*dead) {
    if (warp == kCopyWarp) {
      for (int i = 0; i < C::kStages; i++) {
        const int last = bk_ring_last_parity(armed, i, C::kStages);
        if (last >= 0) bar_settle(smem_u32(full + i), last);
      }
    } else if (warp == kQueryWarp) {
      if (armed) bar_settle(smem_u32(&q_here), bk_ring_last_parity(armed, 0, 1));
    } else if (warp == kMmaWarp) {
      if (elect_lane()) tc_commit(smem_u32(&sh.settled));
      bar_settle(smem_u32(&sh.settled), 0);
    }
    __syncwarp();
  }
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// 2^x, x <= 0, as the weight of a piece: never zero, so that what is infinite stays so (NaN stays NaN)
BK_DEVINL float weight_of(float x) {
  const float w = exp2_approx(x);
  return w < 1.17549435e-38f ? 1.17549435e-38f : w;
}

// The pieces' results of a token row and KV head together: a CTA takes 64 dims of the group's heads, whose rows lie side by side in the
// partial results; a thread 4 dims of one head, from every kSlices-th piece.  The common keys' pieces first, each kind in the order of the line.
// Bound: latency, of a chain of loads: the lists of pieces, their sums and results; 2.6 us of a call for one sequence, 5.5 for 32, 6.4 for 64.
// Few CTAs have many pieces to a row, which four slices take together; many CTAs hide one another's latency better when they are small (two
// slices for 64 sequences of 24 heads: 1.5 us more).
template <int HD, int kSlices>
__global__ void __launch_bounds__(256 * kSlices) paged_merge_kernel(const Params<false> p, const Layout L, uint8_t* scratch) {
  __shared__ __align__(16) float4 o_s[kSlices > 1 ? kSlices - 1 : 1][16 * 16];
  __shared__ float2 ml_s[kSlices][16];
  bk_pdl_trigger();
  const int G = p.Hq / p.Hkv, e = blockIdx.x, kvh = blockIdx.y / (HD / 64), d0 = blockIdx.y % (HD / 64) * 16, t = e / p.B, b = e - t * p.B;
  const int g = threadIdx.x % G, d = threadIdx.x / G % 16, slice = threadIdx.x / (G * 16);
  const int rp = (b * p.T + t) * G + g, rs = t * G + g;
  const int jp = kvh * L.mt_p + rp / kRows, js = (b * p.Hkv + kvh) * L.mt_s + rs / kRows;   // within their kind
  const uint16_t* gate = p.fused ? p.qg + ((size_t)e * p.Hq + kvh * G + g) * 2 * HD + HD : p.gate ? p.gate + ((size_t)e * p.Hq + kvh * G + g) * HD : nullptr;
  const int4* jobs = jobs_of(L, scratch);
  const int2 qs = __ldcg(reinterpret_cast<const int2*>(&jobs[L.n_p + js].z));   // first slot; number and distance
  const int2 qp = L.n_p ? __ldcg(reinterpret_cast<const int2*>(&jobs[jp].z)) : make_int2(0, 0);
  const bool here = row_of(p, b, t) >= 0;
  uint2 gv = make_uint2(0, 0);
  if (gate && slice == 0) gv = __ldcg(reinterpret_cast<const uint2*>(gate + (d0 + d) * 4));
  const int np = here ? qp.y & 0xffff : 0, n = here ? np + (qs.y & 0xffff) : 0;
  bk_pdl_wait();   // (what is above was there when the launch before this one began its work)
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int U = kSlices == 1 ? 6 : 4;   // pieces requested together
  for (int i0 = slice; i0 < n; i0 += kSlices * U) {
    float4 v[U], x[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
      const int i = i0 + k * kSlices;
      x[k] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
      if (i < n) {
        const bool common = i < np;
        const size_t slot = common ? qp.x + i * (qp.y >> 16) : qs.x + i - np;
        const int rows = common ? kRows : L.rows_s, row = (common ? rp : rs) % kRows;
        x[k] = __ldcg(reinterpret_cast<const float4*>(scratch + (common ? L.ml_p : L.ml_s)) + slot * rows + row);
        v[k] = __ldcg(reinterpret_cast<const float4*>(scratch + (common ? L.o_p : L.o_s)) + (slot * (HD / 4) + d0 + d) * rows + row);
      }
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < U; k++) {
      // Maxima pass over NaN, sums do not: a piece with a sum and no maximum has NaN scores only, and any maximum will do to bring that in.
      if (x[k].x == -INFINITY && __fadd_rn(x[k].y, x[k].z) != 0.0f) x[k].x = 0.0f;
      mn = fmaxf(mn, x[k].x);
    }
    if (mn == -INFINITY) continue;
    const float f = weight_of(__fsub_rn(m, mn));   // (m = -inf: of zeros)
    l = __fmul_rn(l, f);
    o.x = __fmul_rn(o.x, f); o.y = __fmul_rn(o.y, f); o.z = __fmul_rn(o.z, f); o.w = __fmul_rn(o.w, f);
    m = mn;
#pragma unroll
    for (int k = 0; k < U; k++)
      if (x[k].x != -INFINITY) {
        const float w = weight_of(__fsub_rn(x[k].x, m));
        l = fmaf(w, __fadd_rn(x[k].y, x[k].z), l);
        o.x = fmaf(w, v[k].x, o.x); o.y = fmaf(w, v[k].y, o.y); o.z = fmaf(w, v[k].z, o.z); o.w = fmaf(w, v[k].w, o.w);
      }
  }
  if (slice) o_s[slice - 1][d * 16 + g] = o;
  if (d == 0) ml_s[slice][g] = make_float2(m, l);
  __syncthreads();
  if (slice) return;
  float M = -INFINITY;
#pragma unroll
  for (int k = 0; k < kSlices; k++) M = fmaxf(M, ml_s[k][g].x);
  float sum = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (here) {   // (a token sees its own row at least: without a maximum, -inf, its scores are all -inf, and 0 / 0 it is)
#pragma unroll
    for (int k = 0; k < kSlices; k++) {
      const float2 x = ml_s[k][g];
      const float w = weight_of(__fsub_rn(x.x, M));
      const float4 v = k ? o_s[k - 1][d * 16 + g] : o;
      sum = fmaf(w, x.y, sum);
      y[0] = fmaf(w, v.x, y[0]); y[1] = fmaf(w, v.y, y[1]); y[2] = fmaf(w, v.z, y[2]); y[3] = fmaf(w, v.w, y[3]);
    }
    const uint32_t gw[2] = {gv.x, gv.y};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      y[i] = __fdiv_rn(y[i], sum);
      if (gate) y[i] = __fmul_rn(y[i], bk_sigmoidf(__uint_as_float(i & 1 ? gw[i >> 1] & 0xffff0000u : gw[i >> 1] << 16)));
    }
  }
  *reinterpret_cast<uint2*>(p.out + ((size_t)e * p.Hq + kvh * G + g) * HD + (d0 + d) * 4) = make_uint2(bk_f32x2_to_bf16x2(y[0], y[1]), bk_f32x2_to_bf16x2(y[2], y[3]));
}


// The same for trees.  A thread has kQuads times 4 dims of one head, 64 apart; a CTA 64 kQuads dims of the group's heads, from kSlices slices of pieces.  Many rows have few
// pieces each: one slice and half of the dims, so that the chain of loads (place, lists of pieces, sums and results) is there twice a row and KV head (all dims a CTA, 2,048 tokens of 32
// sequences, 24 heads on 4: with HD 256 84 us a call for 82, with HD 128 66 to 70 for 71 to 73).  Few rows may have a piece of
// every CTA: more slices (2,048 tokens, half of them there, 24 heads on 4: 76 us with 64 dims a CTA and every list read anew, so 35; one token, 16 heads on 2, 8,192 rows: 17.5 us
// with four slices, so 12; caches cold).
template <int HD, int kSlices, int kQuads>
__global__ void __launch_bounds__(256 * (kSlices > 4 ? 4 : kSlices)) tree_merge_kernel(const Params<true> p, const Layout L, uint8_t* scratch) {
  constexpr int U = kQuads == 1 ? 4 : 2, kParts = HD / (64 * kQuads);   // U: pieces requested together
  extern __shared__ __align__(16) uint8_t merge_smem[];
  bk_pdl_trigger();
  const int G = p.Hq / p.Hkv, e = blockIdx.x, kvh = blockIdx.y / kParts, d0 = blockIdx.y % kParts * 16 * kQuads, t = e / p.B, b = e - t * p.B;
  const int g = threadIdx.x % G, d = threadIdx.x / G % 16, slice = threadIdx.x / (G * 16);
  float4* const o_s = reinterpret_cast<float4*>(merge_smem);                                  // [kSlices - 1][kQuads][16][G]
  float2* const ml_s = reinterpret_cast<float2*>(o_s + (kSlices - 1) * kQuads * 16 * G);      // [kSlices][G]
  uint16_t* const out = p.out + ((size_t)e * p.Hq + kvh * G + g) * HD;
  const uint16_t* gate = p.fused ? p.qg + ((size_t)e * p.Hq + kvh * G + g) * 2 * HD + HD : p.gate ? p.gate + ((size_t)e * p.Hq + kvh * G + g) * HD : nullptr;
  uint2 gv[kQuads];
#pragma unroll
  for (int k = 0; k < kQuads; k++)
    if (gate && slice == 0) gv[k] = __ldcg(reinterpret_cast<const uint2*>(gate + (d0 + 16 * k + d) * 4));
  const int place = __ldcg(p.place + e);
  if (place < 0) {
    bk_pdl_wait();   // (nothing of an earlier call may still read or write what is overwritten)
    if (slice == 0)
#pragma unroll
      for (int k = 0; k < kQuads; k++) *reinterpret_cast<uint2*>(out + (d0 + 16 * k + d) * 4) = make_uint2(0, 0);
    return;
  }
  const int rp = place * G + g, rs = t * G + g;
  const int4* jobs = jobs_of(L, scratch);
  const int2 qs = __ldcg(reinterpret_cast<const int2*>(&jobs[L.n_p + (b * p.Hkv + kvh) * L.mt_s + rs / kRows].z));   // first slot; number and distance
  const int2 qp = L.n_p ? __ldcg(reinterpret_cast<const int2*>(&jobs[kvh * L.mt_p + rp / kRows].z)) : make_int2(0, 0);
  const int np = qp.y & 0xffff, n = np + (qs.y & 0xffff);
  bk_pdl_wait();   // (what is above was there when the launch before this one began its work)
  float m = -INFINITY, l = 0.0f;
  float4 o[kQuads];
#pragma unroll
  for (int k = 0; k < kQuads; k++) o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = slice; i0 < n; i0 += kSlices * U) {
    float4 v[U][kQuads], x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * kSlices;
      x[u] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
      if (i < n) {
        const bool common = i < np;
        const size_t slot = common ? qp.x + i * (qp.y >> 16) : qs.x + (i - np) * (qs.y >> 16);
        const int rows = common ? kRows : L.rows_s, row = (common ? rp : rs) % kRows;
        x[u] = __ldcg(reinterpret_cast<const float4*>(scratch + (common ? L.ml_p : L.ml_s)) + slot * rows + row);
#pragma unroll
        for (int k = 0; k < kQuads; k++)
          v[u][k] = __ldcg(reinterpret_cast<const float4*>(scratch + (common ? L.o_p : L.o_s)) + (slot * (HD / 4) + d0 + 16 * k + d) * rows + row);
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; u++) {
      // (a piece with a sum and no maximum has NaN scores only, see paged_merge_kernel)
      if (x[u].x == -INFINITY && __fadd_rn(x[u].y, x[u].z) != 0.0f) x[u].x = 0.0f;
      mn = fmaxf(mn, x[u].x);
    }
    if (mn == -INFINITY) continue;
    const float f = weight_of(__fsub_rn(m, mn));   // (m = -inf: of zeros)
    l = __fmul_rn(l, f);
#pragma unroll
    for (int k = 0; k < kQuads; k++) o[k] = make_float4(__fmul_rn(o[k].x, f), __fmul_rn(o[k].y, f), __fmul_rn(o[k].z, f), __fmul_rn(o[k].w, f));
    m = mn;
#pragma unroll
    for (int u = 0; u < U; u++)
      if (x[u].x != -INFINITY) {
        const float w = weight_of(__fsub_rn(x[u].x, m));
        l = fmaf(w, __fadd_rn(x[u].y, x[u].z), l);
#pragma unroll
        for (int k = 0; k < kQuads; k++) {
          o[k].x = fmaf(w, v[u][k].x, o[k].x); o[k].y = fmaf(w, v[u][k].y, o[k].y); o[k].z = fmaf(w, v[u][k].z, o[k].z); o[k].w = fmaf(w, v[u][k].w, o[k].w);
        }
      }
  }
  if (kSlices > 1) {
    if (slice)
#pragma unroll
      for (int k = 0; k < kQuads; k++) o_s[(((slice - 1) * kQuads + k) * 16 + d) * G + g] = o[k];
    if (d == 0) ml_s[slice * G + g] = make_float2(m, l);
    __syncthreads();
    if (slice) return;
    float M = -INFINITY;
#pragma unroll
    for (int s = 0; s < kSlices; s++) M = fmaxf(M, ml_s[s * G + g].x);
    const float w0 = weight_of(__fsub_rn(m, M));
    l = __fmul_rn(w0, l);
#pragma unroll
    for (int k = 0; k < kQuads; k++) o[k] = make_float4(__fmul_rn(w0, o[k].x), __fmul_rn(w0, o[k].y), __fmul_rn(w0, o[k].z), __fmul_rn(w0, o[k].w));
#pragma unroll
    for (int s = 1; s < kSlices; s++) {
      const float2 x = ml_s[s * G + g];
      const float w = weight_of(__fsub_rn(x.x, M));
      l = fmaf(w, x.y, l);
#pragma unroll
      for (int k = 0; k < kQuads; k++) {
        const float4 v = o_s[(((s - 1) * kQuads + k) * 16 + d) * G + g];
        o[k].x = fmaf(w, v.x, o[k].x); o[k].y = fmaf(w, v.y, o[k].y); o[k].z = fmaf(w, v.z, o[k].z); o[k].w = fmaf(w, v.w, o[k].w);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kQuads; k++) {
    const int at = (d0 + 16 * k + d) * 4;
    float y[4] = {__fdiv_rn(o[k].x, l), __fdiv_rn(o[k].y, l), __fdiv_rn(o[k].z, l), __fdiv_rn(o[k].w, l)};
    if (gate) {
      const uint32_t gw[2] = {gv[k].x, gv[k].y};
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = __fmul_rn(y[i], bk_sigmoidf(__uint_as_float(i & 1 ? gw[i >> 1] & 0xffff0000u : gw[i >> 1] << 16)));
    }
    *reinterpret_cast<uint2*>(out + at) = make_uint2(bk_f32x2_to_bf16x2(y[0], y[1]), bk_f32x2_to_bf16x2(y[2], y[3]));
  }
}

template <int HD, int kSlices, int kQuads>
cudaError_t launch_tree_merge(const Params<true>& p, const Layout& L, uint8_t* scratch) {
  const int G = p.Hq / p.Hkv;
  const size_t smem = kSlices > 1 ? (size_t)(kSlices - 1) * kQuads * 16 * G * 16 + (size_t)kSlices * G * 8 : 0;   // at most 25 KB
  return bk_launch_pdl(tree_merge_kernel<HD, kSlices, kQuads>, dim3(p.T * p.B, p.Hkv * (HD / (64 * kQuads))), dim3(G * 16 * kSlices), smem, p, L, scratch);
}

template <int HD, bool TREE>
int32_t launch_paged(const Params<TREE>& p, const Layout& L, uint64_t scratch) {
  TileParams<TREE> P;
  P.g = p;
  P.L = L;
  P.scratch = bk_ptr<uint8_t>(scratch);
  P.status = bk_ctx().d_status;
  P.box_rows = std::min(p.page_rows, kTile);
  const uint64_t rows = (uint64_t)p.n_pages * p.Hkv * p.page_rows;
  if (!bk_encode_map_2d(&P.k_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)(uintptr_t)p.k_pages, HD, rows, HD * 2, 64, P.box_rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !bk_encode_map_2d(&P.v_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)(uintptr_t)p.v_pages, HD, rows, HD * 2, 64, P.box_rows, CU_TENSOR_MAP_SWIZZLE_128B))
    return bk_fail(BK_ERR_UNSUPPORTED, "bkPagedAttn: the driver refuses a tensor map of %llu rows of %d values", (unsigned long long)rows, HD);
  const uint64_t q_rows = (uint64_t)p.B * p.T * p.Hq;
  for (int common = 0; common < 2; common++) {   // whole groups of 8 rows; rows of another job are read and not used
    P.q_rows[common] = std::min(kRows, ((common ? p.B : 1) * p.T * (p.Hq / p.Hkv) + 7) / 8 * 8);
    if (!bk_encode_map_2d(&P.q_map[common], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, scratch + L.q, HD, q_rows, HD * 2, 64, P.q_rows[common], CU_TENSOR_MAP_SWIZZLE_128B))
      return bk_fail(BK_ERR_UNSUPPORTED, "bkPagedAttn: the driver refuses a tensor map of %llu rows of %d queries", (unsigned long long)q_rows, HD);
  }
  int heads = p.Hq + (p.k ? p.Hkv : 0);
  if constexpr (TREE) heads = (heads + p.each - 1) / p.each;
  BK_CUDA(bk_launch_pdl(paged_prepare_kernel<HD, TREE>, dim3((p.T * p.B * heads + kPrepThreads / 32 - 1) / (kPrepThreads / 32) + 1), dim3(kPrepThreads), 0, p, L, P.scratch));
  BK_CHECK_LAUNCH();
  static bool configured = false;
  if (!configured) {
    BK_CUDA(cudaFuncSetAttribute(paged_tile_kernel<HD, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<HD>::kSmem));
    configured = true;
  }
  BK_CUDA(bk_launch_pdl(paged_tile_kernel<HD, TREE>, dim3(L.ctas), dim3(kTileThreads), TileCfg<HD>::kSmem, P));
  BK_CHECK_LAUNCH();
  const dim3 merge(p.T * p.B, p.Hkv * (HD / 64));
  if constexpr (TREE) {
    // by rows: eight slices of pieces (16 rows: 22 us a call, with four 34), four (1,024 rows: 25 and 32 us, with eight 30 and 42, with two 28 and 36), two (4,096 rows: 49 us, with
    // four 53, with one 51), one (24,576 rows: 72 us, with two 80)
    const long long rows = (long long)p.T * p.B * p.Hq, sms = bk_ctx().sm_count;
    if (rows <= 2 * sms && p.Hq / p.Hkv <= 8) BK_CUDA((launch_tree_merge<HD, 8, 1>(p, L, P.scratch)));
    else if (rows <= 10 * sms) BK_CUDA((launch_tree_merge<HD, 4, HD / 128>(p, L, P.scratch)));
    else if (rows <= 40 * sms) BK_CUDA((launch_tree_merge<HD, 2, HD / 128>(p, L, P.scratch)));
    else BK_CUDA((launch_tree_merge<HD, 1, HD / 128>(p, L, P.scratch)));
  } else if ((long long)merge.x * merge.y <= 2 * bk_ctx().sm_count) {
    BK_CUDA(bk_launch_pdl(paged_merge_kernel<HD, 4>, merge, dim3(p.Hq / p.Hkv * 64), 0, p, L, P.scratch));
  } else {
    BK_CUDA(bk_launch_pdl(paged_merge_kernel<HD, 1>, merge, dim3(p.Hq / p.Hkv * 16), 0, p, L, P.scratch));
  }
  BK_CHECK_LAUNCH();
  return BK_OK;
}

// what the layout takes with what trees have behind it
size_t tree_bytes(const Layout& L, int B, int T) { return L.bytes + (size_t)(L.n_p + L.n_s) * 16 + ((size_t)B + 1 + 2 * (size_t)B * T) * 4; }

// the checks of a call, its parameters and layout
template <typename P>
int32_t read_args(const char* what, const bkPagedAttnArgs& a, P* out, Layout* layout) {
  BK_ARG(a.HD == 128 || a.HD == 256, "%s: head_dim %d unsupported (128 and 256)", what, a.HD);
  BK_ARG(a.Hq > 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0 && a.Hq / a.Hkv <= 16 && a.Hkv <= 1024, "%s: bad head counts Hq=%d Hkv=%d (group size 1..16, at most 1024 KV heads)", what, a.Hq, a.Hkv);
  BK_ARG(a.B > 0 && a.T > 0 && (long long)a.B * a.T * (a.Hq + a.Hkv) < (1 << 24), "%s: B=%d T=%d of %d heads", what, a.B, a.T, a.Hq + a.Hkv);
  BK_ARG(a.page_rows >= 16 && a.page_rows <= 1024 && (a.page_rows & (a.page_rows - 1)) == 0, "%s: page_rows=%d must be a power of two, 16 to 1024", what, a.page_rows);
  BK_ARG(a.n_pages > 0 && a.max_pages > 0 && (long long)a.n_pages * a.Hkv * a.page_rows < (1ll << 31), "%s: n_pages=%d max_pages=%d (n_pages * Hkv * page_rows below 2^31)", what, a.n_pages, a.max_pages);
  BK_ARG(a.max_len > 0 && a.prefix_rows >= 0 && a.prefix_rows <= a.max_len, "%s: prefix_rows=%d max_len=%d", what, a.prefix_rows, a.max_len);
  BK_ARG(a.scale > 0.0f && a.scale < INFINITY, "%s: scale=%g must be positive", what, (double)a.scale);
  BK_ARG(a.qg && a.k_pages && a.v_pages && a.table && a.lens && a.out && a.scratch, "%s: null pointer", what);
  BK_ARG(((a.qg | a.k | a.v | a.gate | a.k_pages | a.v_pages | a.out | a.scratch) & 15) == 0, "%s: tensors must be 16-byte aligned", what);
  BK_ARG(((a.table | a.lens | a.n_new) & 3) == 0, "%s: table, lens and n_new must be int32 arrays", what);
  BK_ARG((a.k != 0) == (a.v != 0), "%s: k and v go together", what);
  if (a.fused_norm_rope) {
    BK_ARG(a.k && a.q_norm_w && a.k_norm_w && a.cos_t && a.sin_t, "%s: fused mode needs k, v, norm weights and tables", what);
    BK_ARG(((a.q_norm_w | a.k_norm_w) & 15) == 0 && ((a.cos_t | a.sin_t) & 3) == 0, "%s: norm weights must be 16-byte aligned, tables f32 arrays", what);
    BK_ARG(a.rot_half > 0 && 2 * a.rot_half <= a.HD, "%s: rot_half=%d", what, a.rot_half);
    BK_ARG(a.gate == 0, "%s: fused mode takes the gate from qg", what);
  }
  const uint64_t need = bkPagedAttnScratchBytes(a.B, a.T, a.Hq, a.Hkv, a.HD, a.prefix_rows);
  BK_ARG(a.scratch_bytes >= need, "%s: scratch of %llu bytes, %llu needed", what, (unsigned long long)a.scratch_bytes, (unsigned long long)need);
  P& p = *out;
  memset(&p, 0, sizeof(p));
  p.qg = bk_ptr<uint16_t>(a.qg); p.k = bk_ptr<uint16_t>(a.k); p.v = bk_ptr<uint16_t>(a.v); p.gate = bk_ptr<uint16_t>(a.gate);
  p.q_norm_w = bk_ptr<uint16_t>(a.q_norm_w); p.k_norm_w = bk_ptr<uint16_t>(a.k_norm_w); p.cos_t = bk_ptr<float>(a.cos_t); p.sin_t = bk_ptr<float>(a.sin_t);
  p.k_pages = bk_ptr<uint16_t>(a.k_pages); p.v_pages = bk_ptr<uint16_t>(a.v_pages);
  p.table = bk_ptr<int>(a.table); p.lens = bk_ptr<int>(a.lens); p.n_new = bk_ptr<int>(a.n_new); p.out = bk_ptr<uint16_t>(a.out);
  p.q = bk_ptr<uint16_t>(a.scratch);
  p.B = a.B; p.T = a.T; p.Hq = a.Hq; p.Hkv = a.Hkv; p.rot_half = a.rot_half; p.n_pages = a.n_pages; p.page_rows = a.page_rows; p.max_pages = a.max_pages;
  p.max_rows = (int)std::min<long long>(a.max_len, (long long)a.max_pages * a.page_rows); p.fused = a.fused_norm_rope != 0; p.scale = a.scale; p.eps = a.eps;
  Layout& L = *layout;
  L = make_layout(a.B, a.T, a.Hq, a.Hkv, a.HD, a.prefix_rows, a.page_rows, bk_ctx().sm_count);
  const int overhead = std::is_same<P, Params<true>>::value ? tree_overhead(a.HD) : kOverhead;
  BK_ARG((long long)(L.n_p + L.n_s) * ((long long)p.max_rows / kTile + 1 + overhead) < (1ll << 31), "%s: B=%d T=%d Hkv=%d with %d rows a sequence: too much for one call", what, a.B,
         a.T, a.Hkv, p.max_rows);
  return BK_OK;
}

}  // namespace

extern "C" {

uint64_t bkPagedAttnScratchBytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t HD, int32_t prefix_rows) {
  if (B <= 0 || T <= 0 || Hkv <= 0 || Hq < Hkv || HD <= 0 || prefix_rows < 0 || !bk_ctx().ready) return 0;
  return make_layout(B, T, Hq, Hkv, HD, prefix_rows, 1, bk_ctx().sm_count).bytes;   // (a page shape can only make the common part shorter)
}

int32_t bkPagedAttn(const bkPagedAttnArgs* args) {
  BK_REQUIRE_INIT();
  BK_ARG(args != nullptr, "bkPagedAttn: args is null");
  Params<false> p;
  Layout L;
  const int32_t rc = read_args("bkPagedAttn", *args, &p, &L);
  if (rc) return rc;
  return args->HD == 256 ? launch_paged<256, false>(p, L, args->scratch) : launch_paged<128, false>(p, L, args->scratch);
}

uint64_t bkTreeAttnScratchBytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t HD, int32_t prefix_rows) {
  if (bkPagedAttnScratchBytes(B, T, Hq, Hkv, HD, prefix_rows) == 0) return 0;
  return tree_bytes(make_layout(B, T, Hq, Hkv, HD, prefix_rows, 1, bk_ctx().sm_count), B, T);
}

int32_t bkTreeAttn(const bkTreeAttnArgs* args) {
  BK_REQUIRE_INIT();
  BK_ARG(args != nullptr, "bkTreeAttn: args is null");
  const bkTreeAttnArgs& a = *args;
  Params<true> p;
  Layout L;
  const int32_t rc = read_args("bkTreeAttn", a.attn, &p, &L);
  if (rc) return rc;
  BK_ARG(a.mask && (a.mask & 3) == 0 && a.mask_words >= (a.attn.T + 31) / 32, "bkTreeAttn: mask must be a uint32 array of at least %d words a node (mask_words=%d)", (a.attn.T + 31) / 32,
         a.mask_words);
  BK_ARG((a.pos & 3) == 0 && (a.pos || !a.attn.fused_norm_rope), "bkTreeAttn: fused mode needs pos, an int32 array");
  BK_ARG((a.slot & 3) == 0 && (a.slot || !a.attn.k), "bkTreeAttn: k and v need slot, an int32 array");
  const uint64_t need = bkTreeAttnScratchBytes(a.attn.B, a.attn.T, a.attn.Hq, a.attn.Hkv, a.attn.HD, a.attn.prefix_rows);
  BK_ARG(a.attn.scratch_bytes >= need, "bkTreeAttn: scratch of %llu bytes, %llu needed", (unsigned long long)a.attn.scratch_bytes, (unsigned long long)need);
  // heads a warp: one while all warps are on the GPU at once (32 an SM)
  const long long items = (long long)a.attn.B * a.attn.T * (a.attn.Hq + (a.attn.k ? a.attn.Hkv : 0));
  p.each = (int)std::max<long long>(1, std::min<long long>(8, items / (32 * bk_ctx().sm_count)));
  p.team = bk_ptr<int4>(a.attn.scratch + L.bytes);
  p.first = reinterpret_cast<int*>(p.team + L.n_p + L.n_s);
  p.token = p.first + a.attn.B + 1;
  p.place = p.token + (size_t)a.attn.B * a.attn.T;
  p.pos = bk_ptr<int>(a.pos); p.slot = bk_ptr<int>(a.slot); p.mask = bk_ptr<uint32_t>(a.mask); p.words = a.mask_words; p.max_pos = a.attn.max_len;
  return a.attn.HD == 256 ? launch_paged<256, true>(p, L, a.attn.scratch) : launch_paged<128, true>(p, L, a.attn.scratch);
}

}  // extern "C"
