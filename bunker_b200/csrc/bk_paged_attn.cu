// bk_paged_attn.cu -- attention of many sequences over pages of keys and values (bkPagedAttn in bunker_cuda.h has the rules).
//
// No counterpart in the reference (one contiguous cache of 128 rows, src/emitters.ts:188-226).
#include <math.h>
#include <string.h>

#include <algorithm>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

struct PagedParams {
  const uint16_t *qg, *k, *v, *gate, *q_norm_w, *k_norm_w;
  const float *cos_t, *sin_t;
  uint16_t *k_pages, *v_pages;
  const int *table, *lens, *n_new;
  uint16_t* out;
  uint16_t* q;        // ready q [T*B][Hq][HD]: qg, or the scratch buffer
  int B, T, Hq, Hkv, rot_half, n_pages, page_rows, max_pages, max_rows, fused;   // max_rows: what a sequence can have
  float scale, eps;
};

// row of its sequence at which token t of sequence b stands, -1 where it is not there
BK_DEVINL int row_of(const PagedParams& p, int b, int t) {
  const int n = p.n_new ? min(p.n_new[b], p.T) : p.T;
  const long long at = (long long)p.lens[b] - n + t;
  return t < n && at >= 0 && at < p.max_rows ? (int)at : -1;
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
// rows of all sequences, then for each sequence its own keys [P, end).  The work, in tiles of 64 keys and kOverhead more for each job, is
// laid out in one line and cut into equal pieces, one per CTA, so that a long prefix and many short sequences keep every SM busy until the
// end.  The line is made on the device (lengths are there), by one CTA of the first launch.
constexpr int kTile = 64;       // keys of a step
constexpr int kRows = 128;      // rows of a job: the lanes of tensor memory
constexpr int kOverhead = 2;    // what a job's start and end cost, in steps

struct Layout {                 // of the scratch buffer, and the numbers of jobs
  int P;                        // common keys: whole pages
  int mt_p, mt_s;               // row tiles of a KV head: of all sequences together, of one sequence
  int n_p, n_s;                 // jobs over common keys, over a sequence's own
  int rows_s;                   // rows of a partial result of the latter
  int ctas;
  size_t q, starts, ml_p, ml_s, o_p, o_s, bytes;   // byte offsets
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
  L.starts = at;
  at += round16((size_t)(L.n_p + L.n_s + 1) * 8);
  // partial results: a job and a CTA that has a piece of it meet in slot job + CTA, which no other pair has
  const size_t slots_p = L.n_p ? L.n_p + ctas : 0, slots_s = L.n_s + ctas;
  L.ml_p = at;
  at += round16(slots_p * kRows * 8);
  L.ml_s = at;
  at += round16(slots_s * L.rows_s * 8);
  L.o_p = at;
  at += slots_p * kRows * HD * 4;
  L.o_s = at;
  at += slots_s * L.rows_s * HD * 4;
  L.bytes = at;
  return L;
}

struct TileParams {
  PagedParams g;
  Layout L;
  uint8_t* scratch;
  int* status;
  int box_rows;   // rows of a page that one copy takes: min(page_rows, kTile)
  CUtensorMap k_map, v_map;
};

// job j: its KV head, row tile, sequence (-1: all) and the end of its keys
struct Job {
  int seq, kvh, mt, key0, key1;
};
BK_DEVINL Job job_of(const PagedParams& p, const Layout& L, int j) {
  Job q;
  if (j < L.n_p) {
    q.seq = -1;
    q.kvh = j / L.mt_p;
    q.mt = j - q.kvh * L.mt_p;
    q.key0 = 0;
    q.key1 = L.P;
    return q;
  }
  const int i = j - L.n_p, bk = i / L.mt_s;
  q.mt = i - bk * L.mt_s;
  q.seq = bk / p.Hkv;
  q.kvh = bk - q.seq * p.Hkv;
  q.key0 = L.P;
  // the last of the tile's tokens that is there
  const int G = p.Hq / p.Hkv, n = p.n_new ? min(p.n_new[q.seq], p.T) : p.T, last = min(n, (min(p.T * G, (q.mt + 1) * kRows) - 1) / G + 1) - 1;
  q.key1 = L.P;
  for (int t = last; t >= 0 && t >= q.mt * kRows / G; t--) {   // (one turn but for tokens past max_len)
    const int at = row_of(p, q.seq, t);
    if (at >= 0) {
      q.key1 = max(L.P, at + 1);
      break;
    }
  }
  return q;
}
BK_DEVINL int tiles_of(const Job& q) { return (q.key1 - q.key0 + kTile - 1) / kTile; }

// starts[j]: where job j begins on the line; one CTA of 128 threads
BK_DEVINL void plan_jobs(const PagedParams& p, const Layout& L, long long* starts) {
  __shared__ long long warp_s[4];
  const int n = L.n_p + L.n_s, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long base = 0;
  for (int j0 = 0; j0 < n; j0 += 128) {
    const int j = j0 + (int)threadIdx.x;
    long long units = 0;
    if (j < n) {
      const int tiles = tiles_of(job_of(p, L, j));
      units = tiles ? tiles + kOverhead : 0;
    }
    long long v = units;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v += o;
    }
    if (lane == 31) warp_s[warp] = v;
    __syncthreads();
    long long before = base;
    for (int w = 0; w < 4; w++) {
      if (w < warp) before += warp_s[w];
      base += warp_s[w];
    }
    if (j < n) starts[j] = before + v - units;
    __syncthreads();
  }
  if (threadIdx.x == 0) starts[n] = base;
}

// CTA c of the line's C pieces: units [bound(c), bound(c + 1))
BK_DEVINL long long bound_of(long long units, int c, int C) { return units * c / C; }
BK_DEVINL int cta_at(long long units, long long x, int C) { return (int)(((x + 1) * C - 1) / units); }
// the tiles of a job that starts at s and has n tiles which lie in units [u0, u1)
BK_DEVINL void piece_of(long long s, int n, long long u0, long long u1, int* t0, int* t1) {
  *t0 = (int)max(0ll, min((long long)n, u0 - s - kOverhead));
  *t1 = (int)max(0ll, min((long long)n, u1 - s - kOverhead));
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

// One warp per (token row, head): q heads to the scratch buffer, k and v heads into their page.  The last CTA lays out the work of the next launch.
template <int HD>
__global__ void __launch_bounds__(128) paged_prepare_kernel(const PagedParams p, const Layout L, uint8_t* scratch) {
  constexpr int PER = HD / 32;
  __shared__ float y_s[4][HD];
  bk_pdl_trigger();
  bk_pdl_wait();
  if (blockIdx.x == gridDim.x - 1) {
    plan_jobs(p, L, reinterpret_cast<long long*>(scratch + L.starts));
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = (p.fused ? p.Hq : 0) + (p.k ? p.Hkv : 0);
  const int item = blockIdx.x * 4 + warp;
  if (item >= p.T * p.B * heads) return;
  const int e = item / heads, h = item - e * heads, t = e / p.B, b = e - t * p.B;
  const int at = row_of(p, b, t);
  if (at < 0) return;
  const bool is_q = p.fused && h < p.Hq;
  const int kvh = h - (p.fused ? p.Hq : 0);
  const uint16_t* src = is_q ? p.qg + ((size_t)e * p.Hq + h) * 2 * HD : p.k + ((size_t)e * p.Hkv + kvh) * HD;
  uint16_t* dst = p.q + ((size_t)e * p.Hq + h) * HD;
  if (!is_q) {
    const int page = p.table[(size_t)b * p.max_pages + at / p.page_rows];
    if (page < 0 || page >= p.n_pages) return;
    const size_t row = (((size_t)page * p.Hkv + kvh) * p.page_rows + at % p.page_rows) * HD;
    dst = p.k_pages + row;
    const uint16_t* vs = p.v + ((size_t)e * p.Hkv + kvh) * HD;
#pragma unroll
    for (int i = 0; i < PER; i += 4) *reinterpret_cast<uint2*>(p.v_pages + row + lane * PER + i) = *reinterpret_cast<const uint2*>(vs + lane * PER + i);
  }
  float x[PER];
  load_bf16(src + lane * PER, x);
  if (p.fused) {
    float w[PER], sum = 0.0f;
    load_bf16((is_q ? p.q_norm_w : p.k_norm_w) + lane * PER, w);
#pragma unroll
    for (int i = 0; i < PER; i++) sum = fmaf(x[i], x[i], sum);
    const float rstd = bk_rcp_sqrt(__fadd_rn(__fdiv_rn(bk_warp_sum(sum), (float)HD), p.eps));
#pragma unroll
    for (int i = 0; i < PER; i++) y_s[warp][lane * PER + i] = __fmul_rn(__fmul_rn(x[i], rstd), __fadd_rn(1.0f, w[i]));
    __syncwarp();
    const float *cr = p.cos_t + (size_t)at * p.rot_half, *sr = p.sin_t + (size_t)at * p.rot_half;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int d = lane * PER + i;
      const float y = y_s[warp][d];
      if (d < p.rot_half) x[i] = __fsub_rn(__fmul_rn(y, cr[d]), __fmul_rn(y_s[warp][d + p.rot_half], sr[d]));
      else if (d < 2 * p.rot_half) x[i] = __fadd_rn(__fmul_rn(y, cr[d - p.rot_half]), __fmul_rn(y_s[warp][d - p.rot_half], sr[d - p.rot_half]));
      else x[i] = y;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; i += 4) *reinterpret_cast<uint2*>(dst + lane * PER + i) = make_uint2(bk_f32x2_to_bf16x2(x[i], x[i + 1]), bk_f32x2_to_bf16x2(x[i + 2], x[i + 3]));
}

// ---- tensor memory and its instructions ------------------------------------------------
#define BK_R32(F, v, o) F(v[o]), F(v[o + 1]), F(v[o + 2]), F(v[o + 3]), F(v[o + 4]), F(v[o + 5]), F(v[o + 6]), F(v[o + 7]), F(v[o + 8]), F(v[o + 9]), F(v[o + 10]), \
    F(v[o + 11]), F(v[o + 12]), F(v[o + 13]), F(v[o + 14]), F(v[o + 15]), F(v[o + 16]), F(v[o + 17]), F(v[o + 18]), F(v[o + 19]), F(v[o + 20]), F(v[o + 21]), F(v[o + 22]), \
    F(v[o + 23]), F(v[o + 24]), F(v[o + 25]), F(v[o + 26]), F(v[o + 27]), F(v[o + 28]), F(v[o + 29]), F(v[o + 30]), F(v[o + 31])
#define BK_OUT(x) "=r"(x)
#define BK_IN(x) "r"(x)
// 32 or 64 columns of the calling lane's row.  The wait is part of it, so that no use of a register can come before.
BK_DEVINL void tmem_ld32(uint32_t at, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : BK_R32(BK_OUT, v, 0)
      : "r"(at)
      : "memory");
}
BK_DEVINL void tmem_ld64(uint32_t at, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, "
      "%53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : BK_R32(BK_OUT, v, 0), BK_R32(BK_OUT, v, 32)
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
BK_DEVINL void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
BK_DEVINL void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
BK_DEVINL void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
BK_DEVINL void tc_commit(uint32_t bar) {   // arrives when every MMA issued so far has completed
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (+)= A * B, M = 128, K = 16; A in tensor memory
BK_DEVINL void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile("{\n\t.reg .pred pz;\n\tsetp.ne.b32 pz, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pz;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
               "r"(acc ? 1u : 0u)
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
// A wait of a warp that stays together.  Bounded by time (a poll may sleep): the first wait of a CTA that gives up, after 2^31 cycles, sets the
// status word and `dead`, after which the others return at once and the kernel runs to its end.
BK_DEVINL void bar_wait_warp(uint32_t bar, uint32_t parity, int* status, volatile int* dead) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
  const long long from = clock64();
#pragma unroll 1
  do {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity) || *dead)) return;
  } while (__any_sync(0xffffffffu, clock64() - from < (1ll << 31)));
  *dead = 1;
  atomicExch(status, 10003 /* BK_ERR_TIMEOUT */);
}
BK_DEVINL void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
BK_DEVINL float exp2_approx(float x) {   // 2^x to 2 ulp or so; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// positions in the stream of a piece's tiles: K0, K1, V0, K2, V1, ..., V(n-1)
BK_DEVINL int stream_v(int i, int n) { return i < n - 1 ? 2 * i + 2 : 2 * n - 1; }

template <int HD>
struct TileCfg {
  static constexpr int kStage = kTile * HD * 2;               // bytes of 64 keys or values
  static constexpr int kStages = HD == 256 ? 6 : 12;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kO = 0, kQ = HD, kS = HD + HD / 2;     // tensor memory: output, queries, two buffers of scores (then probabilities)
};
constexpr int kTileThreads = 192;   // warps 0-3: a row each lane; 4: copies; 5: MMAs

// S = Q K^T and O += P V on the tensor cores.  Q (operand A), S, P and O live in tensor memory, a row per lane; K and V tiles of 64 rows come
// through a ring in shared memory.  P = 2^(S c - m) with the running maximum m of the row; it overwrites its S as two bf16 matrices, the
// rounded values and what rounding left (16 bits of the value; with 8 the result's error against exact arithmetic is 1.7 times that of its own rounding).
// m is only moved when a score passes it by more than 2^8, since O must be rescaled then.  Row sums are in f32, by the lane that owns the row.
template <int HD>
__global__ void __launch_bounds__(kTileThreads, 1) paged_tile_kernel(const __grid_constant__ TileParams P) {
  using C = TileCfg<HD>;
  const PagedParams& p = P.g;
  const Layout& L = P.L;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], q_full, s_full[2], p_full[2], o_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_s;
  volatile int* dead = &dead_s;
  bk_pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    dead_s = 0;
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(smem_u32(full + i), 1);
      mbar_init(smem_u32(empty + i), 1);
    }
    mbar_init(smem_u32(&q_full), 128);
    for (int i = 0; i < 2; i++) {
      mbar_init(smem_u32(s_full + i), 1);
      mbar_init(smem_u32(p_full + i), 128);
    }
    mbar_init(smem_u32(&o_full), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  bk_pdl_wait();

  const long long* starts = reinterpret_cast<const long long*>(P.scratch + L.starts);
  const int n_jobs = L.n_p + L.n_s, cta = blockIdx.x;
  const long long units = __ldcg(starts + n_jobs), u0 = bound_of(units, cta, L.ctas), u1 = bound_of(units, cta + 1, L.ctas);
  // the first job that ends behind u0
  int j = 0;
  {
    int lo = 0, hi = n_jobs;   // starts[lo] <= u0 < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldcg(starts + mid) <= u0) lo = mid;
      else hi = mid;
    }
    j = lo;
  }

  if (u1 > u0) {
    if (warp == 4) {
      // ================= copies: lane (chunk, block) takes box_rows rows x 64 dims =================
      asm volatile("fence.proxy.async;" ::: "memory");   // rows that an earlier kernel stored
      constexpr int kBlocks = HD / 64;
      const int chunks = kTile / P.box_rows, n_box = chunks * kBlocks;
      const int chunk = lane / kBlocks, block = lane % kBlocks;
      const int no_row = p.n_pages * p.Hkv * p.page_rows;   // behind the last row: such a box is filled with zeros
      const uint32_t box_at = block * (kTile * 128) + chunk * P.box_rows * 128;
      int stage = 0;
      uint32_t parity = 1;
      for (; j < n_jobs; j++) {
        const long long s = __ldcg(starts + j);
        if (s >= u1) break;
        const Job q = job_of(p, L, j);
        int t0, t1;
        piece_of(s, tiles_of(q), u0, u1, &t0, &t1);
        if (t0 >= t1) continue;
        const int* table = p.table + (size_t)max(q.seq, 0) * p.max_pages;
        auto row_of_tile = [&](int i) {   // row of the map that this lane's box of tile i starts at
          const int key = q.key0 + i * kTile + chunk * P.box_rows;
          if (lane >= n_box || i >= t1 || key >= q.key1 || key / p.page_rows >= p.max_pages) return no_row;
          const int page = __ldg(table + key / p.page_rows);
          return page >= 0 && page < p.n_pages ? (page * p.Hkv + q.kvh) * p.page_rows + key % p.page_rows : no_row;
        };
        auto load = [&](const CUtensorMap* map, int row) {
          bar_wait_warp(smem_u32(empty + stage), parity, P.status, dead);
          const uint32_t bar = smem_u32(full + stage);
          if (lane == 0) mbar_expect_tx(bar, C::kStage);
          __syncwarp();
          if (lane < n_box) tma_load(smem_u32(ring + (size_t)stage * C::kStage) + box_at, map, block * 64, row, bar);
          if (++stage == C::kStages) {
            stage = 0;
            parity ^= 1u;
          }
        };
        int next = row_of_tile(t0), before = 0;
        for (int i = t0; i <= t1; i++) {
          const int row = next;
          next = row_of_tile(i + 1);
          if (i < t1) load(&P.k_map, row);
          if (i > t0) load(&P.v_map, before);
          before = row;
        }
      }
      // the last copies have landed before the CTA ends: the MMAs waited for them (or the waits below do, where a wait gave up)
      if (*dead) {
        for (int i = 0; i < C::kStages; i++) {
          for (int it = 0; it < (1 << 16) && !mbar_try_wait(smem_u32(full + stage), parity ^ 1u); it++) {
          }
          if (++stage == C::kStages) {
            stage = 0;
            parity ^= 1u;
          }
        }
      }
    } else if (warp == 5) {
      // ================= MMAs =================
      constexpr uint32_t kShapeS = mma_shape(kTile, false), kShapeO = mma_shape(HD, true);
      int stage = 0, tile = 0, pieces = 0;   // tile: counted over all pieces
      uint32_t parity = 0;
      auto next_stage = [&]() {
        if (++stage == C::kStages) {
          stage = 0;
          parity ^= 1u;
        }
      };
      for (; j < n_jobs; j++) {
        const long long s = __ldcg(starts + j);
        if (s >= u1) break;
        int t0, t1;
        piece_of(s, tiles_of(job_of(p, L, j)), u0, u1, &t0, &t1);
        if (t0 >= t1) continue;
        bar_wait_warp(smem_u32(&q_full), pieces & 1, P.status, dead);
        tc_after();
        for (int i = t0; i <= t1; i++) {
          if (i < t1) {   // scores of tile i; the probabilities that this buffer held have been multiplied: MMAs run in order
            bar_wait_warp(smem_u32(full + stage), parity, P.status, dead);
            const uint32_t k_at = smem_u32(ring + (size_t)stage * C::kStage);
            if (elect_lane()) {
#pragma unroll
              for (int ks = 0; ks < HD / 16; ks++)
                tc_mma(tmem + C::kS + (tile & 1) * kTile, tmem + C::kQ + ks * 8, smem_desc(k_at + (ks >> 2) * (kTile * 128) + (ks & 3) * 32, 16, 1024), kShapeS, ks > 0);
              tc_commit(smem_u32(empty + stage));
              tc_commit(smem_u32(s_full + (tile & 1)));
            }
            __syncwarp();
            next_stage();
            tile++;
          }
          if (i > t0) {   // output of tile i - 1
            const int prev = i < t1 ? tile - 2 : tile - 1;
            bar_wait_warp(smem_u32(p_full + (prev & 1)), (prev >> 1) & 1, P.status, dead);
            bar_wait_warp(smem_u32(full + stage), parity, P.status, dead);
            tc_after();
            const uint32_t v_at = smem_u32(ring + (size_t)stage * C::kStage);
            if (elect_lane()) {
#pragma unroll
              for (int half = 0; half < 2; half++)
#pragma unroll
                for (int ks = 0; ks < kTile / 16; ks++)
                  tc_mma(tmem + C::kO, tmem + C::kS + (prev & 1) * kTile + half * 32 + ks * 8, smem_desc(v_at + ks * 2048, kTile * 128, 1024), kShapeO,
                         i - 1 > t0 || half > 0 || ks > 0);
              tc_commit(smem_u32(empty + stage));
              tc_commit(smem_u32(&o_full));
            }
            __syncwarp();
            next_stage();
          }
        }
        pieces++;
      }
    } else {
      // ================= rows: thread <-> row of the tile =================
      const int i_row = threadIdx.x;
      const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
      const float c = __fmul_rn(p.scale, 1.44269504088896341f);   // scores in powers of two
      int tile = 0, stream = 0;   // counted over all pieces
      for (; j < n_jobs; j++) {
        const long long s0 = __ldcg(starts + j);
        if (s0 >= u1) break;
        const Job q = job_of(p, L, j);
        int t0, t1;
        piece_of(s0, tiles_of(q), u0, u1, &t0, &t1);
        if (t0 >= t1) continue;
        const int n = t1 - t0;
        int b, t, g, limit = 0;
        const bool mine = row_at(p, q, i_row, &b, &t, &g);
        if (mine) limit = min(row_of(p, b, t) + 1, q.key1);
        __syncwarp();
        const bool warp_on = __any_sync(0xffffffffu, mine);
        {   // queries into tensor memory (the MMAs that read the ones before have completed: their scores were there)
          const uint16_t* src = p.q + ((size_t)(t * p.B + b) * p.Hq + q.kvh * (p.Hq / p.Hkv) + g) * HD;
          tc_after();
          if (warp_on) {
#pragma unroll
            for (int d = 0; d < HD / 64; d++) {
              uint32_t v[32];
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const uint4 w = limit > 0 ? __ldcg(reinterpret_cast<const uint4*>(src + d * 64 + e * 8)) : make_uint4(0, 0, 0, 0);
                v[4 * e] = w.x; v[4 * e + 1] = w.y; v[4 * e + 2] = w.z; v[4 * e + 3] = w.w;
              }
              tmem_st32(lanes + C::kQ + d * 32, v);
            }
            tmem_wait_st();
          }
          tc_before();
          bar_arrive(smem_u32(&q_full));
        }
        float m = -INFINITY, l = 0.0f;
        for (int i = 0; i < n; i++, tile++) {
          const int key0 = q.key0 + (t0 + i) * kTile, there = min(kTile, q.key1 - key0);
          const uint32_t s_at = lanes + C::kS + (tile & 1) * kTile;
          bar_wait_warp(smem_u32(s_full + (tile & 1)), (tile >> 1) & 1, P.status, dead);
          tc_after();
          if (there < kTile) {   // values past the end count as zeros, whatever the page holds there
            const int v_pos = stream + stream_v(i, n), v_stage = v_pos % C::kStages;
            bar_wait_warp(smem_u32(full + v_stage), (v_pos / C::kStages) & 1, P.status, dead);
            uint8_t* v_at = ring + (size_t)v_stage * C::kStage;
            for (int x = threadIdx.x; x < (kTile - there) * (HD / 8); x += 128) {
              const int row = there + x / (HD / 8), piece = x % (HD / 8);
              *reinterpret_cast<uint4*>(v_at + (piece >> 3) * (kTile * 128) + row * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (warp_on) {
            float s[64];
            {
              uint32_t v[64];
              tmem_ld64(s_at, v);
#pragma unroll
              for (int x = 0; x < 64; x++) s[x] = __uint_as_float(v[x]);
            }
            if (!__all_sync(0xffffffffu, key0 + kTile <= limit)) {
#pragma unroll
              for (int x = 0; x < 64; x++) s[x] = key0 + x < limit ? s[x] : -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int x = 1; x < 64; x++) mx = fmaxf(mx, s[x]);
            mx = __fmul_rn(mx, c);
            const bool move = mx > __fadd_rn(m, 8.0f);
            if (__any_sync(0xffffffffu, move)) {
              const float to = move ? mx : m;
              const float f = m == to || m == -INFINITY ? 1.0f : exp2_approx(__fsub_rn(m, to));
              const bool rescale = move && m != -INFINITY;
              m = to;
              l = __fmul_rn(l, f);
              if (__any_sync(0xffffffffu, rescale)) {
                bar_wait_warp(smem_u32(&o_full), (tile - 1) & 1, P.status, dead);   // tile i - 1 has been added to the output
                tc_after();
#pragma unroll 1
                for (int d = 0; d < HD / 32; d++) {
                  uint32_t o[32];
                  tmem_ld32(lanes + C::kO + d * 32, o);
#pragma unroll
                  for (int x = 0; x < 32; x++) o[x] = __float_as_uint(__fmul_rn(__uint_as_float(o[x]), f));
                  tmem_st32(lanes + C::kO + d * 32, o);
                }
              }
            }
            const float base = m == -INFINITY ? 0.0f : m;
            uint32_t hi[32], lo[32];
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < 32; x++) {
              const float2 y = bk_fma2(make_float2(s[2 * x], s[2 * x + 1]), make_float2(c, c), make_float2(-base, -base));
              const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
              sum = bk_add2(sum, e);
              hi[x] = bk_f32x2_to_bf16x2(e.x, e.y);
              lo[x] = bk_f32x2_to_bf16x2(__fsub_rn(e.x, __uint_as_float(hi[x] << 16)), __fsub_rn(e.y, __uint_as_float(hi[x] & 0xffff0000u)));
            }
            l = __fadd_rn(l, __fadd_rn(sum.x, sum.y));
            tmem_st32(s_at, hi);
            tmem_st32(s_at + 32, lo);
            tmem_wait_st();
          }
          tc_before();
          bar_arrive(smem_u32(p_full + (tile & 1)));
        }
        stream += 2 * n;
        // the piece's part of the result
        if (n > 1) bar_wait_warp(smem_u32(&o_full), (tile - 2) & 1, P.status, dead);   // (a wait must not be two phases ahead)
        bar_wait_warp(smem_u32(&o_full), (tile - 1) & 1, P.status, dead);
        tc_after();
        if (warp_on) {
          const bool common = q.seq < 0;
          const size_t slot = common ? (size_t)(j + cta) * kRows : (size_t)(j - L.n_p + cta) * L.rows_s;
          float2* ml = reinterpret_cast<float2*>(P.scratch + (common ? L.ml_p : L.ml_s)) + slot + i_row;
          float* o_to = reinterpret_cast<float*>(P.scratch + (common ? L.o_p : L.o_s)) + (slot + i_row) * HD;
          if (mine) *ml = make_float2(m, l);
          __syncwarp();
#pragma unroll 1
          for (int d = 0; d < HD / 32; d++) {
            uint32_t o[32];
            tmem_ld32(lanes + C::kO + d * 32, o);
            if (mine) {
#pragma unroll
              for (int x = 0; x < 32; x += 4) *reinterpret_cast<uint4*>(o_to + d * 32 + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
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
  if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// One CTA per (token row, query head): out = sum of the pieces' results, the common keys' first, each in the order of the line.
template <int HD>
__global__ void __launch_bounds__(HD / 4) paged_merge_kernel(const PagedParams p, const Layout L, const uint8_t* scratch) {
  bk_pdl_trigger();
  bk_pdl_wait();
  const int h = blockIdx.y, e = blockIdx.x, t = e / p.B, b = e - t * p.B, G = p.Hq / p.Hkv, kvh = h / G, g = h - kvh * G;
  const long long* starts = reinterpret_cast<const long long*>(scratch + L.starts);
  const long long units = __ldcg(starts + L.n_p + L.n_s);
  const bool here = row_of(p, b, t) >= 0;
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int part = 0; part < 2 && here; part++) {
    const bool common = part == 0;
    if (common && L.n_p == 0) continue;
    const int r = common ? (b * p.T + t) * G + g : t * G + g, mt = r / kRows, row = r - mt * kRows;
    const int j = common ? kvh * L.mt_p + mt : (b * p.Hkv + kvh) * L.mt_s + mt;   // within its kind
    const int job = common ? j : L.n_p + j;
    const long long s = __ldcg(starts + job), s_end = __ldcg(starts + job + 1);
    if (s == s_end) continue;
    const int tiles = (int)(s_end - s) - kOverhead, c1 = cta_at(units, s_end - 1, L.ctas);
    const int rows = common ? kRows : L.rows_s;
    const float2* ml = reinterpret_cast<const float2*>(scratch + (common ? L.ml_p : L.ml_s));
    const float* os = reinterpret_cast<const float*>(scratch + (common ? L.o_p : L.o_s));
    for (int c = cta_at(units, s, L.ctas); c <= c1; c++) {
      int t0, t1;
      piece_of(s, tiles, bound_of(units, c, L.ctas), bound_of(units, c + 1, L.ctas), &t0, &t1);
      if (t0 >= t1) continue;
      const size_t at = (size_t)(j + c) * rows + row;
      const float2 x = __ldcg(ml + at);
      if (x.x == -INFINITY) continue;
      const float4 v = __ldcg(reinterpret_cast<const float4*>(os + at * HD) + threadIdx.x);
      const float mn = fmaxf(m, x.x), f = exp2_approx(__fsub_rn(m, mn)), w = exp2_approx(__fsub_rn(x.x, mn));   // (m = -inf: f = 0)
      l = fmaf(l, f, __fmul_rn(w, x.y));
      o.x = fmaf(o.x, f, __fmul_rn(w, v.x)); o.y = fmaf(o.y, f, __fmul_rn(w, v.y));
      o.z = fmaf(o.z, f, __fmul_rn(w, v.z)); o.w = fmaf(o.w, f, __fmul_rn(w, v.w));
      m = mn;
    }
  }
  float y[4] = {o.x, o.y, o.z, o.w};
  const bool any = m != -INFINITY;
  const uint16_t* gate = p.fused ? p.qg + ((size_t)e * p.Hq + h) * 2 * HD + HD : p.gate ? p.gate + ((size_t)e * p.Hq + h) * HD : nullptr;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    y[i] = any ? __fdiv_rn(y[i], l) : 0.0f;
    if (gate && any) y[i] = __fmul_rn(y[i], bk_sigmoidf(bk_bf16_to_f32(gate[threadIdx.x * 4 + i])));
  }
  *reinterpret_cast<uint2*>(p.out + ((size_t)e * p.Hq + h) * HD + threadIdx.x * 4) = make_uint2(bk_f32x2_to_bf16x2(y[0], y[1]), bk_f32x2_to_bf16x2(y[2], y[3]));
}

template <int HD>
int32_t launch_paged(const PagedParams& p, const Layout& L, uint64_t scratch) {
  TileParams P;
  P.g = p;
  P.L = L;
  P.scratch = bk_ptr<uint8_t>(scratch);
  P.status = bk_ctx().d_status;
  P.box_rows = std::min(p.page_rows, kTile);
  const uint64_t rows = (uint64_t)p.n_pages * p.Hkv * p.page_rows;
  if (!bk_encode_map_2d(&P.k_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)(uintptr_t)p.k_pages, HD, rows, HD * 2, 64, P.box_rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !bk_encode_map_2d(&P.v_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)(uintptr_t)p.v_pages, HD, rows, HD * 2, 64, P.box_rows, CU_TENSOR_MAP_SWIZZLE_128B))
    return bk_fail(BK_ERR_UNSUPPORTED, "bkPagedAttn: the driver refuses a tensor map of %llu rows of %d values", (unsigned long long)rows, HD);
  const int heads = (p.fused ? p.Hq : 0) + (p.k ? p.Hkv : 0);
  BK_CUDA(bk_launch_pdl(paged_prepare_kernel<HD>, dim3((p.T * p.B * heads + 3) / 4 + 1), dim3(128), 0, p, L, P.scratch));
  BK_CHECK_LAUNCH();
  static bool configured = false;
  if (!configured) {
    BK_CUDA(cudaFuncSetAttribute(paged_tile_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<HD>::kSmem));
    configured = true;
  }
  BK_CUDA(bk_launch_pdl(paged_tile_kernel<HD>, dim3(L.ctas), dim3(kTileThreads), TileCfg<HD>::kSmem, P));
  BK_CHECK_LAUNCH();
  BK_CUDA(bk_launch_pdl(paged_merge_kernel<HD>, dim3(p.T * p.B, p.Hq), dim3(HD / 4), 0, p, L, P.scratch));
  BK_CHECK_LAUNCH();
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
  const bkPagedAttnArgs& a = *args;
  BK_ARG(a.HD == 128 || a.HD == 256, "bkPagedAttn: head_dim %d unsupported (128 and 256)", a.HD);
  BK_ARG(a.Hq > 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0 && a.Hq / a.Hkv <= 16, "bkPagedAttn: bad head counts Hq=%d Hkv=%d (group size 1..16)", a.Hq, a.Hkv);
  BK_ARG(a.B > 0 && a.T > 0 && (long long)a.B * a.T * (a.Hq + a.Hkv) < (1 << 24), "bkPagedAttn: B=%d T=%d of %d heads", a.B, a.T, a.Hq + a.Hkv);
  BK_ARG(a.page_rows >= 16 && a.page_rows <= 1024 && (a.page_rows & (a.page_rows - 1)) == 0, "bkPagedAttn: page_rows=%d must be a power of two, 16 to 1024", a.page_rows);
  BK_ARG(a.n_pages > 0 && a.max_pages > 0 && (long long)a.n_pages * a.Hkv * a.page_rows < (1ll << 31), "bkPagedAttn: n_pages=%d max_pages=%d (n_pages * Hkv * page_rows below 2^31)", a.n_pages, a.max_pages);
  BK_ARG(a.max_len > 0 && a.prefix_rows >= 0 && a.prefix_rows <= a.max_len, "bkPagedAttn: prefix_rows=%d max_len=%d", a.prefix_rows, a.max_len);
  BK_ARG(a.scale > 0.0f && a.scale < INFINITY, "bkPagedAttn: scale=%g must be positive", (double)a.scale);
  BK_ARG(a.qg && a.k_pages && a.v_pages && a.table && a.lens && a.out && a.scratch, "bkPagedAttn: null pointer");
  BK_ARG(((a.qg | a.k | a.v | a.gate | a.k_pages | a.v_pages | a.out | a.scratch) & 15) == 0, "bkPagedAttn: tensors must be 16-byte aligned");
  BK_ARG(((a.table | a.lens | a.n_new) & 3) == 0, "bkPagedAttn: table, lens and n_new must be int32 arrays");
  BK_ARG((a.k != 0) == (a.v != 0), "bkPagedAttn: k and v go together");
  if (a.fused_norm_rope) {
    BK_ARG(a.k && a.q_norm_w && a.k_norm_w && a.cos_t && a.sin_t, "bkPagedAttn: fused mode needs k, v, norm weights and tables");
    BK_ARG(((a.q_norm_w | a.k_norm_w) & 15) == 0 && ((a.cos_t | a.sin_t) & 3) == 0, "bkPagedAttn: norm weights must be 16-byte aligned, tables f32 arrays");
    BK_ARG(a.rot_half > 0 && 2 * a.rot_half <= a.HD, "bkPagedAttn: rot_half=%d", a.rot_half);
    BK_ARG(a.gate == 0, "bkPagedAttn: fused mode takes the gate from qg");
  }
  const uint64_t need = bkPagedAttnScratchBytes(a.B, a.T, a.Hq, a.Hkv, a.HD, a.prefix_rows);
  BK_ARG(a.scratch_bytes >= need, "bkPagedAttn: scratch of %llu bytes, %llu needed", (unsigned long long)a.scratch_bytes, (unsigned long long)need);
  PagedParams p;
  memset(&p, 0, sizeof(p));
  p.qg = bk_ptr<uint16_t>(a.qg); p.k = bk_ptr<uint16_t>(a.k); p.v = bk_ptr<uint16_t>(a.v); p.gate = bk_ptr<uint16_t>(a.gate);
  p.q_norm_w = bk_ptr<uint16_t>(a.q_norm_w); p.k_norm_w = bk_ptr<uint16_t>(a.k_norm_w); p.cos_t = bk_ptr<float>(a.cos_t); p.sin_t = bk_ptr<float>(a.sin_t);
  p.k_pages = bk_ptr<uint16_t>(a.k_pages); p.v_pages = bk_ptr<uint16_t>(a.v_pages);
  p.table = bk_ptr<int>(a.table); p.lens = bk_ptr<int>(a.lens); p.n_new = bk_ptr<int>(a.n_new); p.out = bk_ptr<uint16_t>(a.out);
  p.q = a.fused_norm_rope ? bk_ptr<uint16_t>(a.scratch) : bk_ptr<uint16_t>(a.qg);
  p.B = a.B; p.T = a.T; p.Hq = a.Hq; p.Hkv = a.Hkv; p.rot_half = a.rot_half; p.n_pages = a.n_pages; p.page_rows = a.page_rows; p.max_pages = a.max_pages;
  p.max_rows = (int)std::min<long long>(a.max_len, (long long)a.max_pages * a.page_rows); p.fused = a.fused_norm_rope != 0; p.scale = a.scale; p.eps = a.eps;
  const Layout L = make_layout(a.B, a.T, a.Hq, a.Hkv, a.HD, a.prefix_rows, a.page_rows, bk_ctx().sm_count);
  return a.HD == 256 ? launch_paged<256>(p, L, a.scratch) : launch_paged<128>(p, L, a.scratch);
}

}  // extern "C"
