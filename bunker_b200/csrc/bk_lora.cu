// bk_lora.cu -- low-rank adapters of many requests beside a shared projection: out[b] = base[b] + s_a Bm_a (A_a x_b), a = ids[b].
//
// No counterpart in the reference.  Two launches: u = A x, split over K so that few requests fill the GPU too, then out = base + s Bm u.
// A CTA takes all columns of one adapter, so an adapter's weights are read once whatever the number
// of requests that share it.  Both products are m16n8k16 MMAs on fragments that lanes load from memory as they lie: the order of the
// contraction's index is free as long as both operands have the same, so a lane takes 8 or 16 consecutive bytes of a row.  (With one row of weights
// a thread, or a few lanes, and FMAs, unpacking and reducing were 200 instructions for 32 rows and a column.)  x and the weights are
// bf16, exact; u goes in as three bf16 matrices, eight of its 24 bits in each.  Sums in f32, the parts of K added
// in ascending order: the same call gives the same bits.
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxB = 64, kMaxRank = 128;

struct LoraSeg {
  const uint16_t *A, *Bm;
  const void* base;
  void* out;
  int n_rows, f32, ld_out, col_off, u_seg, tile0;   // u_seg: its number in u; tile0: its first CTA in the expanding launch
};
struct LoraParams {
  const uint16_t* x;
  const int* ids;
  const float* scale;
  float* u;   // [part of K][segment][column][rank]
  int K, B, n_segs, rank, n_adapters, parts, chunk, per, u_segs, by_adapter;   // u_segs: segments that u has
  LoraSeg segs[4];
};

// The adapter of CTAs y and its columns, a bit each.  by_adapter: adapter y, if there are as few; else column y's, for the first of its columns
// (64 columns of 7 adapters by columns: 57 of 64 CTAs come to find nothing to do, 24 us for 13).  0: nothing here; *adapter -1: no adapter.  Whole warps call.
BK_DEVINL unsigned long long columns_of(const LoraParams& p, int y, int* adapter) {
  const int lane = threadIdx.x & 31;
  const int lo = lane < p.B ? __ldg(p.ids + lane) : -1, hi = lane + 32 < p.B ? __ldg(p.ids + lane + 32) : -1;
  const int a = p.by_adapter ? y : __shfl_sync(0xffffffffu, y < 32 ? lo : hi, y & 31);
  const bool there = a >= 0 && a < p.n_adapters;
  *adapter = there ? a : -1;
  const unsigned long long same = (unsigned long long)__ballot_sync(0xffffffffu, hi == a) << 32 | __ballot_sync(0xffffffffu, lo == a);
  return there && (p.by_adapter || __ffsll(same) - 1 == y) ? same : 0;
}

// D += A B; a: rows lane/4 and +8, two pairs of the contraction's index; b: column lane/4, the same pairs; d: rows lane/4 and +8, columns 2(lane mod 4), +1
BK_DEVINL void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kWarps = kThreads / 32;

// The adapter's columns as a list; whole CTA, one barrier
BK_DEVINL void list_columns(unsigned long long cols, int* list) {
  if (threadIdx.x < 64 && (cols >> threadIdx.x & 1)) list[__popcll(cols & ((1ull << threadIdx.x) - 1))] = threadIdx.x;
  __syncthreads();
}

// u[r] = sum over k of A[r][k] x[k].  grid (part of K, adapter or column, segment).  A warp has 16 rows of A, up to 8 columns of x and every S-th 32 of
// the CTA's K, 8 KB of weights on the way.  (All rows a warp, with what a long rank leaves of the registers: 56 adapters of rank 128, K = N = 5,120
// 62 us, so 29; rank 64 32, so 20.)  Bound: memory for long ranks (73 MB in 15 us), else the latency of ids, weights and the warps' sums: 42 adapters of
// rank 32, K = 5,120, two segments about 8 us, 28 MB at 3.4 TB/s.  Parts of K: as many CTAs as stay on the GPU, two an SM (three with half as much on
// the way: rank 128 30.0, rank 64 20.9; four: 34.1 and 24.5).
template <int MT>
__global__ void __launch_bounds__(kThreads, 2) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  constexpr int S = kWarps / MT, U = 8;   // U: of 32 values of K requested together
  __shared__ int list[kMaxB];
  __shared__ float part_s[S][MT * 16][8];
  // The wait comes first: a launch behind this call may read, before its own wait, what a launch before this call wrote (weights, settled caches).
  bk_pdl_wait();
  bk_pdl_trigger();
  int a;
  const unsigned long long cols = columns_of(p, blockIdx.y, &a);
  if (!cols) return;
  list_columns(cols, list);
  const int n = __popcll(cols), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane >> 2, j = lane & 3, r0 = warp / S * 16, slice = warp % S;
  const int k0 = blockIdx.x * p.chunk, k1 = min(p.K, k0 + p.chunk);
  const bool row[2] = {r0 < p.rank, r0 + 8 < p.rank};   // (the rank is a multiple of 8)
  const uint16_t* A = p.segs[blockIdx.z].A + ((size_t)a * p.rank + r0 + q) * p.K + j * 8;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int c0 = 0; c0 < n; c0 += 8) {
    const uint16_t* x = p.x + (size_t)list[min(c0 + q, n - 1)] * p.K + j * 8;
    const bool col = c0 + q < n;
    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int kb = k0 + slice * 32; kb < k1; kb += S * 32 * U) {
      uint4 w[U][2], v[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int k = kb + u * S * 32;
        const bool in = k + j * 8 < k1;   // (K and the parts are multiples of 8)
#pragma unroll
        for (int h = 0; h < 2; h++) w[u][h] = in && row[h] ? __ldg(reinterpret_cast<const uint4*>(A + (size_t)(h * 8) * p.K + k)) : zero;
        v[u] = in && col ? __ldg(reinterpret_cast<const uint4*>(x + k)) : zero;
      }
      // Short chains of MMAs, whose sums are rounded worse than an addition: all of a part in one chain, the result's error is 3.1e-7 for 0.9e-7.
#pragma unroll
      for (int u = 0; u < U; u += 2) {
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = u; t < u + 2; t++) {
          mma_bf16(y, w[t][0].x, w[t][1].x, w[t][0].y, w[t][1].y, v[t].x, v[t].y);
          mma_bf16(y, w[t][0].z, w[t][1].z, w[t][0].w, w[t][1].w, v[t].z, v[t].w);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = __fadd_rn(d[e], y[e]);
      }
    }
    if (c0) __syncthreads();   // the sums before have been taken
#pragma unroll
    for (int e = 0; e < 4; e++) part_s[slice][r0 + (e >> 1) * 8 + q][2 * j + (e & 1)] = d[e];
    __syncthreads();
    for (int i = threadIdx.x; i < p.rank * 8; i += kThreads) {
      const int r = i >> 3, c = c0 + (i & 7);
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < S; w++) y = __fadd_rn(y, part_s[w][r][i & 7]);
      if (c < n) p.u[(((size_t)blockIdx.x * p.n_segs + blockIdx.z) * p.B + list[c]) * p.rank + r] = y;
    }
  }
}

// u as three bf16 values, eight of its 24 bits each, cut off: none has another sign than u, and where a part would be zero beside a u that is not it is the
// least normal value, 2^-126.  So an infinite weight, or an infinite u, makes the sum of the products infinite and not NaN (inf * 0, inf - inf).
BK_DEVINL void split3(float u, uint16_t (&o)[3]) {
  const uint32_t bits = __float_as_uint(u);
  o[0] = isnan(u) ? 0x7fc0 : bits >> 16;
  const float r = isfinite(u) ? __fsub_rn(u, bk_bf16_to_f32(o[0])) : 0.0f;
  o[1] = __float_as_uint(r) >> 16;
  o[2] = __float_as_uint(__fsub_rn(r, bk_bf16_to_f32(o[1]))) >> 16;
  if (u != 0.0f) {
#pragma unroll
    for (int t = 0; t < 3; t++)
      if ((o[t] & 0x7fff) == 0) o[t] = (bits >> 16 & 0x8000) | 0x0080;
  }
}

template <bool F32>
BK_DEVINL float load_as(const uint8_t* at) { return F32 ? *reinterpret_cast<const float*>(at) : bk_bf16_to_f32(*reinterpret_cast<const uint16_t*>(at)); }
template <bool F32>
BK_DEVINL void store_as(uint8_t* at, float v) {
  if (F32) *reinterpret_cast<float*>(at) = v;
  else *reinterpret_cast<uint16_t*>(at) = bk_f32_to_bf16(v);
}
template <int KS>
constexpr int kAhead = KS <= 4 ? 2 : 1;   // tiles requested ahead where one or two columns share the weights (three spill: 35.1 us for 31.1)

// out = base + Bm (s u).  grid (p.per tiles of 256 rows, column).  A warp has 32 rows of a tile, KS steps of 16 of the rank; the next tiles' weights are
// requested before these are used up.  WIDE (rank a multiple of 32): a lane's 16 bytes are two steps of a row.  Bound: memory; 64 requests of 42 adapters,
// rank 32, 2 x 17,408 rows: 20 us, 111 MB at 5.5 TB/s.  Instructions come next: with three MMAs for the parts of u and a store for
// each of a row tile's eighths, adapters of one or two columns were bound by them (460 a warp and 32 rows; the call 37 us, now 28.7).
template <int KS, bool WIDE, bool F32>
__global__ void __launch_bounds__(kThreads, KS <= 2 ? 3 : 2) lora_expand_kernel(const __grid_constant__ LoraParams p) {
  constexpr int R = KS * 16, SZ = F32 ? 4 : 2;
  extern __shared__ __align__(16) uint16_t u_s[];   // [3][columns of the adapter][R]
  __shared__ int list[kMaxB];
  bk_pdl_trigger();
  int seg = 0;
  while (seg + 1 < p.n_segs && (int)blockIdx.x >= p.segs[seg + 1].tile0) seg++;
  const LoraSeg& s = p.segs[seg];
  const int lane = threadIdx.x & 31, q = lane >> 2, j = lane & 3;
  const int row0 = ((int)blockIdx.x - s.tile0) * (p.per * kThreads) + (threadIdx.x >> 5) * 32, row_end = min(s.n_rows, row0 + p.per * kThreads);   // of this warp
  int a;
  const unsigned long long cols = columns_of(p, blockIdx.y, &a);
  const uint8_t* const base0 = reinterpret_cast<const uint8_t*>(s.base);   // (0: zeros)
  uint8_t* const out0 = reinterpret_cast<uint8_t*>(s.out);
  const int n_rows = s.n_rows, rank = WIDE ? R : p.rank, ld = s.ld_out, col_off = s.col_off;
  if (a < 0) {   // no adapter: this column, or those of eight
    bk_pdl_wait();
    if (base0 == out0) return;
    const int b0 = p.by_adapter ? ((int)blockIdx.y - p.n_adapters) * 8 : (int)blockIdx.y, b1 = p.by_adapter ? min(p.B, b0 + 8) : b0 + 1;
    for (int b = b0; b < b1; b++) {
      const int id = __ldg(p.ids + b);
      if (id >= 0 && id < p.n_adapters) continue;
      for (int row = row0 + lane; row < row_end; row += kThreads) {
        const size_t at = ((size_t)b * ld + col_off + row) * SZ;
        store_as<F32>(out0 + at, base0 ? load_as<F32>(base0 + at) : 0.0f);
      }
    }
    return;
  }
  if (!cols) {
    bk_pdl_wait();   // (no launch of this call outlives the one behind it)
    return;
  }
  const int n = __popcll(cols);
  // weights first: what is needed beside them is small and near
  const uint16_t* from = s.Bm + ((size_t)a * n_rows + q) * rank + j * (WIDE ? 8 : 4);
  auto request = [&](int row, uint2 (&w)[4][KS]) {   // rows below row_end
    const uint16_t* at = from + (size_t)row * rank;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const bool in = row + i * 8 + q < row_end;
      if (WIDE) {
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          const uint4 v = in ? __ldg(reinterpret_cast<const uint4*>(at + i * 8 * rank + k * 16)) : make_uint4(0, 0, 0, 0);
          w[i][k] = make_uint2(v.x, v.y);
          w[i][k + 1 < KS ? k + 1 : k] = make_uint2(v.z, v.w);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; k++) w[i][k] = in && k * 16 + j * 4 < rank ? __ldg(reinterpret_cast<const uint2*>(at + i * 8 * rank + k * 16)) : make_uint2(0, 0);
      }
    }
  };
  // u of the adapter's columns into u_s, V values a thread at a time; whole CTA
  auto take_u = [&](auto width) {
    constexpr int V = decltype(width)::value;
    const float scale = p.scale ? __ldg(p.scale + a) : 1.0f;
    bk_pdl_wait();   // (all but u is older than this call, and the launch before this one began after that)
    for (int i = threadIdx.x * V; i < n * R; i += kThreads * V) {   // (zeros behind the rank, a multiple of 8)
      const int c = i / R, r = i % R;
      float y[V] = {};
      if (r < rank) {
        const float* u = p.u + ((size_t)s.u_seg * p.B + list[c]) * rank + r;
#pragma unroll 4
        for (int part = 0; part < p.parts; part++) {
          alignas(16) float x[V];
          if (V == 4) *reinterpret_cast<float4*>(x) = __ldcg(reinterpret_cast<const float4*>(u + (size_t)part * p.u_segs * p.B * rank));
          else x[0] = __ldcg(u + (size_t)part * p.u_segs * p.B * rank);
#pragma unroll
          for (int e = 0; e < V; e++) y[e] = __fadd_rn(y[e], x[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        uint16_t o[3];
        split3(__fmul_rn(scale, y[e]), o);
#pragma unroll
        for (int t = 0; t < 3; t++) u_s[(size_t)t * n * R + i + e] = o[t];
      }
    }
    __syncthreads();
  };
  auto u_at = [&](int t, int c, int k) {   // part t of column c, this lane's values of step k
    return *reinterpret_cast<const uint2*>(u_s + ((size_t)t * n + c) * R + (WIDE ? (k >> 1) * 32 + j * 8 + (k & 1) * 4 : k * 16 + j * 4));
  };

  if (n <= 2) {
    // One or two columns: their three parts side by side as six of the eight columns of one operand B, a third of the MMAs.  The parts then lie in lanes
    // j = 0, 1, 2 of a row's four, which add them up and keep one of the tile's four rows q each.
    constexpr int D = kAhead<KS>;
    uint2 w[D][4][KS];
    float base[D][2];
#pragma unroll
    for (int d = 0; d < D; d++) request(row0 + d * kThreads, w[d]);
    list_columns(cols, list);
    const int mine = (j & 1) * 16 + (j >> 1) * 8 + q;
    size_t col[2];
#pragma unroll
    for (int c = 0; c < 2; c++) col[c] = ((size_t)list[min(c, n - 1)] * ld + col_off + mine) * SZ;
    auto request_base = [&](int row, float (&base)[2]) {
#pragma unroll
      for (int c = 0; c < 2; c++) base[c] = base0 && c < n && row + mine < row_end ? load_as<F32>(base0 + col[c] + (size_t)row * SZ) : 0.0f;
    };
#pragma unroll
    for (int d = 0; d < D; d++) request_base(row0 + d * kThreads, base[d]);
    take_u(std::integral_constant<int, 1>());
    uint2 u[KS];
#pragma unroll
    for (int k = 0; k < KS; k++) u[k] = q < 6 && (q & 1) < n ? u_at(q >> 1, q & 1, k) : make_uint2(0, 0);
#pragma unroll 1
    for (int first = row0; first < row_end; first += D * kThreads) {
#pragma unroll
      for (int d = 0; d < D; d++) {
        const int row = first + d * kThreads;
        float v[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) v[t][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int t = 0; t < 2; t++) mma_bf16(v[t], w[d][2 * t][k].x, w[d][2 * t + 1][k].x, w[d][2 * t][k].y, w[d][2 * t + 1][k].y, u[k].x, u[k].y);
        request(row + D * kThreads, w[d]);
        float half[4], sum[2];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (j == 3) v[0][e] = v[1][e] = 0.0f;   // (a weight that is not finite made it NaN)
          half[e] = __fadd_rn(j & 1 ? v[1][e] : v[0][e], __shfl_xor_sync(0xffffffffu, j & 1 ? v[0][e] : v[1][e], 1));
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
          sum[c] = __fadd_rn(j & 2 ? half[2 + c] : half[c], __shfl_xor_sync(0xffffffffu, j & 2 ? half[c] : half[2 + c], 2));
          if (c < n && row + mine < row_end) store_as<F32>(out0 + col[c] + (size_t)row * SZ, __fadd_rn(base[d][c], sum[c]));
        }
        request_base(row + D * kThreads, base[d]);
      }
    }
    return;
  }

  uint2 w[4][KS];
  request(row0, w);
  list_columns(cols, list);
  // this lane's two of eight columns, at row q; base a tile ahead where these are all
  size_t col[2];
  bool has[2];
  auto columns_at = [&](int c0) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
      has[e] = c0 + 2 * j + e < n;
      col[e] = ((size_t)(has[e] ? list[c0 + 2 * j + e] : 0) * ld + col_off + q) * SZ;
    }
  };
  columns_at(0);
  float base[2][4];
  auto request_base = [&](int row) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
      for (int i = 0; i < 4; i++) base[e][i] = 0.0f;
      if (has[e] && base0) {
        const uint8_t* at = base0 + col[e] + (size_t)row * SZ;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (row + i * 8 + q < n_rows) base[e][i] = load_as<F32>(at + i * 8 * SZ);
      }
    }
  };
  request_base(row0);
  take_u(std::integral_constant<int, 4>());   // (64 columns of one adapter: 25.8 us with one value, 20.5 with four)
  constexpr bool kKeep = KS <= 2;   // operand B of eight columns in registers (longer ranks: from shared memory each time, for two CTAs an SM: 8 columns, rank 128 37.9 us with one CTA, 24.5 with two)
  uint2 u[3][kKeep ? KS : 1];
  auto columns_from = [&](int c0) {
#pragma unroll
    for (int t = 0; t < 3; t++)
#pragma unroll
      for (int k = 0; k < (kKeep ? KS : 0); k++) u[t][k] = c0 + q < n ? u_at(t, c0 + q, k) : make_uint2(0, 0);
  };
  columns_from(0);
#pragma unroll 1
  for (int row = row0; row < row_end; row += kThreads) {
#pragma unroll 1
    for (int c0 = 0; c0 < n; c0 += 8) {
      if (n > 8) {
        columns_from(c0);
        columns_at(c0);
        request_base(row);
      }
      float d[2][4];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) d[t][e] = 0.0f;
#pragma unroll
      for (int part = 2; part >= 0; part--)   // the smallest first
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const uint2 y = kKeep ? u[part][kKeep ? k : 0] : c0 + q < n ? u_at(part, c0 + q, k) : make_uint2(0, 0);
#pragma unroll
          for (int t = 0; t < 2; t++) mma_bf16(d[t], w[2 * t][k].x, w[2 * t + 1][k].x, w[2 * t][k].y, w[2 * t + 1][k].y, y.x, y.y);
        }
      float now[2][4];
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) now[e][i] = __fadd_rn(base[e][i], d[i >> 1][(i & 1) * 2 + e]);
      if (c0 + 8 >= n && row + kThreads < row_end) {   // (the last use of these weights)
        request(row + kThreads, w);
        if (n <= 8) request_base(row + kThreads);
      }
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (has[e]) {
          uint8_t* at = out0 + col[e] + (size_t)row * SZ;
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (row + i * 8 + q < n_rows) store_as<F32>(at + i * 8 * SZ, now[e][i]);
        }
    }
  }
}

// A CTA takes one tile where there are few, else as many as leave four CTAs an SM: its start, a chain of ids, u and the first weights, costs several
// tiles' time (eight an SM: 56 adapters of rank 16 to 17,408 rows 23.1 us for 17.0; three: 42 of rank 32 to 34,816 31.9 for 28.7).  In whole turns of what
// it requests ahead: an odd one costs a turn of MMAs on nothing (five tiles 31.2 us, four or six 30.0).
template <int KS, bool WIDE, bool F32>
int32_t launch_expand_as(LoraParams& p) {
  long long tiles = 0;
  for (int i = 0; i < p.n_segs; i++) tiles += (p.segs[i].n_rows + kThreads - 1) / kThreads;
  p.per = (int)std::min(16ll, (tiles * std::min(p.B, p.n_adapters) + 2 * bk_ctx().sm_count) / (4 * bk_ctx().sm_count));
  p.per = std::max(1, p.per / kAhead<KS> * kAhead<KS>);
  int ctas = 0;
  for (int i = 0; i < p.n_segs; i++) {
    p.segs[i].tile0 = ctas;
    ctas += (p.segs[i].n_rows + p.per * kThreads - 1) / (p.per * kThreads);
  }
  const size_t smem = (size_t)3 * p.B * KS * 16 * 2;
  static bool configured = false;
  if (!configured) {
    BK_CUDA(cudaFuncSetAttribute(lora_expand_kernel<KS, WIDE, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * kMaxB * KS * 16 * 2));
    configured = true;
  }
  int ys = p.B;
  if (p.by_adapter) {
    ys = p.n_adapters;
    for (int i = 0; i < p.n_segs; i++)
      if (p.segs[i].base != p.segs[i].out) ys = p.n_adapters + (p.B + 7) / 8;
  }
  BK_CUDA(bk_launch_pdl(lora_expand_kernel<KS, WIDE, F32>, dim3(ctas, ys), dim3(kThreads), smem, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}
// The segments of one type at a time: a launch for each that there is.
template <int KS, bool WIDE>
int32_t launch_expand(const LoraParams& all) {
  for (int f32 = 0; f32 < 2; f32++) {
    LoraParams p = all;
    int n = 0;
    for (int i = 0; i < all.n_segs; i++)
      if (all.segs[i].f32 == f32) {
        p.segs[n] = all.segs[i];
        p.segs[n++].u_seg = i;
      }
    p.n_segs = n;
    if (n == 0) continue;
    const int32_t rc = f32 ? launch_expand_as<KS, WIDE, true>(p) : launch_expand_as<KS, WIDE, false>(p);
    if (rc) return rc;
  }
  return BK_OK;
}
template <int MT>
int32_t launch_shrink(LoraParams& p) {
  BK_CUDA(bk_launch_pdl(lora_shrink_kernel<MT>, dim3(p.parts, p.by_adapter ? p.n_adapters : p.B, p.n_segs), dim3(kThreads), 0, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

}  // namespace

extern "C" {

uint64_t bkLoraScratchBytes(int32_t K, int32_t B, int32_t rank, int32_t n_segs) {
  if (K <= 0 || B <= 0 || rank <= 0 || n_segs <= 0) return 0;
  return (uint64_t)((K + 255) / 256) * n_segs * B * rank * 4;
}

int32_t bkLora(const bkLoraArgs* args) {
  BK_REQUIRE_INIT();
  BK_ARG(args != nullptr, "bkLora: args is null");
  const bkLoraArgs& a = *args;
  BK_ARG(a.K > 0 && a.K % 8 == 0, "bkLora: K=%d must be a positive multiple of 8", a.K);
  BK_ARG(a.B >= 1 && a.B <= kMaxB, "bkLora: B=%d (1 to %d)", a.B, kMaxB);
  BK_ARG(a.n_segs >= 1 && a.n_segs <= 4, "bkLora: n_segs=%d (1 to 4)", a.n_segs);
  BK_ARG(a.rank >= 8 && a.rank <= kMaxRank && a.rank % 8 == 0, "bkLora: rank=%d must be a multiple of 8, 8 to %d", a.rank, kMaxRank);
  BK_ARG(a.n_adapters >= 1, "bkLora: n_adapters=%d", a.n_adapters);
  BK_ARG(a.x && (a.x & 15) == 0 && a.ids && ((a.ids | a.scale) & 3) == 0, "bkLora: x must be 16-byte aligned, ids an int32 and scale an f32 array");
  BK_ARG(a.scratch && (a.scratch & 15) == 0 && a.scratch_bytes >= bkLoraScratchBytes(a.K, a.B, a.rank, a.n_segs), "bkLora: scratch of %llu bytes, %llu needed, 16-byte aligned",
         (unsigned long long)a.scratch_bytes, (unsigned long long)bkLoraScratchBytes(a.K, a.B, a.rank, a.n_segs));
  LoraParams p;
  memset(&p, 0, sizeof(p));
  p.x = bk_ptr<uint16_t>(a.x); p.ids = bk_ptr<int>(a.ids); p.scale = bk_ptr<float>(a.scale); p.u = bk_ptr<float>(a.scratch);
  p.K = a.K; p.B = a.B; p.n_segs = p.u_segs = a.n_segs; p.rank = a.rank; p.n_adapters = a.n_adapters; p.by_adapter = a.n_adapters <= a.B;
  for (int i = 0; i < a.n_segs; i++) {
    const bkLoraSeg& s = a.segs[i];
    BK_ARG(s.n_rows > 0 && s.n_rows < (1 << 30) && s.col_off >= 0 && (long long)s.col_off + s.n_rows <= s.ld_out, "bkLora: segment %d: n_rows=%d col_off=%d ld_out=%d", i, s.n_rows, s.col_off,
           s.ld_out);
    BK_ARG(s.dtype == BK_DTYPE_F32 || s.dtype == BK_DTYPE_BF16, "bkLora: segment %d: dtype %d", i, s.dtype);
    const uint64_t mask = s.dtype == BK_DTYPE_F32 ? 3 : 1;
    BK_ARG(s.A && s.Bm && s.out && ((s.A | s.Bm) & 15) == 0 && ((s.base | s.out) & mask) == 0, "bkLora: segment %d: A and Bm must be 16-byte aligned, out non-null, base and out aligned to their type", i);
    p.segs[i] = LoraSeg{bk_ptr<uint16_t>(s.A), bk_ptr<uint16_t>(s.Bm), bk_ptr<void>(s.base), bk_ptr<void>(s.out), s.n_rows, s.dtype == BK_DTYPE_F32, s.ld_out, s.col_off, i, 0};
  }
  // Parts of K, multiples of 256: about two CTAs an SM, no more than 16 for the expanding launch to add up.
  const int units = (a.K + 255) / 256;
  const int parts = std::max(1, std::min({units, 16, 2 * bk_ctx().sm_count / (a.n_segs * std::min(a.B, a.n_adapters))}));
  p.chunk = (units + parts - 1) / parts * 256;
  p.parts = (a.K + p.chunk - 1) / p.chunk;
  const int32_t rc = a.rank <= 16 ? launch_shrink<1>(p) : a.rank <= 32 ? launch_shrink<2>(p) : a.rank <= 64 ? launch_shrink<4>(p) : launch_shrink<8>(p);
  if (rc) return rc;
  const bool wide = a.rank % 32 == 0;
  return a.rank <= 16   ? launch_expand<1, false>(p)
         : a.rank <= 32 ? (wide ? launch_expand<2, true>(p) : launch_expand<2, false>(p))
         : a.rank <= 64 ? (wide ? launch_expand<4, true>(p) : launch_expand<4, false>(p))
                        : (wide ? a.rank == 96 ? launch_expand<6, true>(p) : launch_expand<8, true>(p) : launch_expand<8, false>(p));
}

}  // extern "C"
