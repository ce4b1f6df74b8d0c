// bk_lora.cu -- low-rank adapters of many requests beside a shared projection: out[b] = base[b] + s_a Bm_a (A_a x_b), a = ids[b].
//
// No counterpart in the reference.  Two launches: u = A x, split over K so that few requests fill the GPU too, then out = base + s Bm u.
// A CTA takes all columns of one adapter (it belongs to the first of them), so an adapter's weights are read once whatever the number
// of requests that share it.  Sums in f32; the parts of K are added in ascending order, so results do not depend on the launch.
#include <string.h>

#include <algorithm>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxB = 64, kMaxRank = 128;

struct LoraSeg {
  const uint16_t *A, *Bm;
  const void* base;
  void* out;
  int n_rows, f32, ld_out, col_off, tile0;   // tile0: first CTA of the segment in the expanding launch
};
struct LoraParams {
  const uint16_t* x;
  const int* ids;
  const float* scale;
  float* u;   // [part of K][segment][column][rank]
  int K, B, n_segs, rank, n_adapters, parts, chunk, per;
  LoraSeg segs[4];
};

// Column b's adapter and the columns that share it, a bit each, if b is the first of them (0: it is not, or has no adapter: *adapter = -1).  Whole
// warps call.
BK_DEVINL unsigned long long columns_of(const LoraParams& p, int b, int* adapter) {
  const int lane = threadIdx.x & 31;
  const int lo = lane < p.B ? __ldg(p.ids + lane) : -1, hi = lane + 32 < p.B ? __ldg(p.ids + lane + 32) : -1;
  const int a = __shfl_sync(0xffffffffu, b < 32 ? lo : hi, b & 31);
  const bool there = a >= 0 && a < p.n_adapters;
  *adapter = there ? a : -1;
  const unsigned long long same = (unsigned long long)__ballot_sync(0xffffffffu, hi == a) << 32 | __ballot_sync(0xffffffffu, lo == a);
  return there && __ffsll(same) - 1 == b ? same : 0;
}

BK_DEVINL void unpack8(uint4 v, float (&y)[8]) {
  y[0] = __uint_as_float(v.x << 16); y[1] = __uint_as_float(v.x & 0xffff0000u);
  y[2] = __uint_as_float(v.y << 16); y[3] = __uint_as_float(v.y & 0xffff0000u);
  y[4] = __uint_as_float(v.z << 16); y[5] = __uint_as_float(v.z & 0xffff0000u);
  y[6] = __uint_as_float(v.w << 16); y[7] = __uint_as_float(v.w & 0xffff0000u);
}

constexpr int kChunk = 2048;   // of K, at most: what a CTA keeps of x, for kCols columns
constexpr int kCols = 4;

// 1,024 values of two rows of A, 4 KB a warp
BK_DEVINL void load_rows(const uint16_t* row0, const uint16_t* row1, int kb, int len, uint4 (&w)[2][4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int k = kb + i * 256 + (threadIdx.x & 31) * 8;
    w[0][i] = k < len ? __ldg(reinterpret_cast<const uint4*>(row0 + k)) : make_uint4(0, 0, 0, 0);
    w[1][i] = k < len ? __ldg(reinterpret_cast<const uint4*>(row1 + k)) : make_uint4(0, 0, 0, 0);
  }
}
// u of C columns (n of them are there): two rows of A a warp at a time, the first of them in w already, x from shared memory
template <int C>
BK_DEVINL void shrink_rows(const LoraParams& p, const uint16_t* A, const uint16_t* x_s, int k0, int len, int seg, int part, const int* cols, int n, uint4 (&w)[2][4]) {
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < p.rank; r += 2 * kThreads / 32) {
    const bool two = r + kThreads / 32 < p.rank;
    const uint16_t* row0 = A + (size_t)r * p.K + k0;
    const uint16_t* row1 = two ? row0 + (size_t)(kThreads / 32) * p.K : row0;
    float acc[2][C];
#pragma unroll
    for (int c = 0; c < C; c++) acc[0][c] = acc[1][c] = 0.0f;
    for (int kb = 0; kb < len; kb += 1024) {
      if (kb || r != (threadIdx.x >> 5)) load_rows(row0, row1, kb, len, w);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int k = kb + i * 256 + lane * 8;
        if (k < len) {
          float w0[8], w1[8];
          unpack8(w[0][i], w0);
          unpack8(w[1][i], w1);
#pragma unroll
          for (int c = 0; c < C; c++) {
            float x[8];
            unpack8(*reinterpret_cast<const uint4*>(x_s + c * kChunk + k), x);
#pragma unroll
            for (int e = 0; e < 8; e++) {
              acc[0][c] = fmaf(w0[e], x[e], acc[0][c]);
              acc[1][c] = fmaf(w1[e], x[e], acc[1][c]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
      const float y0 = bk_warp_sum(acc[0][c]), y1 = bk_warp_sum(acc[1][c]);
      if (lane == 0 && c < n) {
        float* u = p.u + (((size_t)part * p.n_segs + seg) * p.B + cols[c]) * p.rank + r;
        u[0] = y0;
        if (two) u[kThreads / 32] = y1;
      }
    }
  }
}

// grid (part of K, column, segment).  Bound: latency, of ids, then of the first rows of A (requested before x is staged).
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  __shared__ __align__(16) uint16_t x_s[kCols * kChunk];
  bk_pdl_trigger();
  bk_pdl_wait();
  int a;
  unsigned long long left = columns_of(p, blockIdx.y, &a);
  if (!left) return;
  const uint16_t* A = p.segs[blockIdx.z].A + (size_t)a * p.rank * p.K;
  const int k0 = blockIdx.x * p.chunk, len = min(p.K - k0, p.chunk), r0 = threadIdx.x >> 5;
  uint4 w[2][4];
  bool first = true;
  while (left) {
    const uint16_t* row0 = A + (size_t)r0 * p.K + k0;   // (rank is at least the number of warps)
    load_rows(row0, r0 + kThreads / 32 < p.rank ? row0 + (size_t)(kThreads / 32) * p.K : row0, 0, len, w);
    int cols[kCols], m = 0;
#pragma unroll
    for (int c = 0; c < kCols; c++) {   // (a column that is not there is a copy of the last one that is: what it gives is not used)
      if (left) {
        cols[c] = __ffsll(left) - 1;
        left &= left - 1;
        m++;
      } else cols[c] = cols[c ? c - 1 : 0];
    }
    if (!first) __syncthreads();
    first = false;
#pragma unroll
    for (int c = 0; c < kCols; c++)
      if (c < m || m > 1)
        for (int k = threadIdx.x * 8; k < len; k += kThreads * 8) *reinterpret_cast<uint4*>(x_s + c * kChunk + k) = *reinterpret_cast<const uint4*>(p.x + (size_t)cols[c] * p.K + k0 + k);
    __syncthreads();
    if (m == 1) shrink_rows<1>(p, A, x_s, k0, len, blockIdx.z, blockIdx.x, cols, m, w);
    else shrink_rows<kCols>(p, A, x_s, k0, len, blockIdx.z, blockIdx.x, cols, m, w);
  }
}

BK_DEVINL float load_base(const LoraSeg& s, size_t at) {
  return !s.base ? 0.0f : s.f32 ? reinterpret_cast<const float*>(s.base)[at] : bk_bf16_to_f32(reinterpret_cast<const uint16_t*>(s.base)[at]);
}
BK_DEVINL void store_out(const LoraSeg& s, size_t at, float v) {
  if (s.f32) reinterpret_cast<float*>(s.out)[at] = v;
  else reinterpret_cast<uint16_t*>(s.out)[at] = bk_f32_to_bf16(v);
}

// P lanes read a row of Bm (16 bytes each, rank <= 8 P), so that a warp's loads are whole lines; P loads a lane are 32 rows of a warp, a CTA's 256 are
// a tile.  The sums of the P lanes of a row are halved out so that every lane ends up with one row.  A CTA takes p.per times M tiles; the next M are
// requested before these are multiplied.
template <int P>
BK_DEVINL void load_weights(const LoraSeg& s, const uint16_t* from, int rank, int row, uint4* w) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int r = row + i * (32 / P) + lane / P;
    w[i] = r < s.n_rows && lane % P * 8 < rank ? __ldg(reinterpret_cast<const uint4*>(from + (size_t)r * rank)) : make_uint4(0, 0, 0, 0);
  }
}
// grid (M * p.per tiles of rows, column)
template <int P, int M>
__global__ void __launch_bounds__(kThreads, P <= 4 ? 4 : 1) lora_expand_kernel(const __grid_constant__ LoraParams p) {
  extern __shared__ __align__(16) float u_s[];   // [columns of the adapter][8 P]
  bk_pdl_trigger();
  bk_pdl_wait();
  int seg = 0;
  while (seg + 1 < p.n_segs && (int)blockIdx.x >= p.segs[seg + 1].tile0) seg++;
  const LoraSeg& s = p.segs[seg];
  const int lane = threadIdx.x & 31, b = blockIdx.y, piece = lane % P;
  const int row0 = ((int)blockIdx.x - s.tile0) * (p.per * M * kThreads) + (threadIdx.x >> 5) * 32, row_end = min(s.n_rows, row0 + p.per * M * kThreads);   // of this warp: 32 rows of every tile
  int a;
  unsigned long long cols = columns_of(p, b, &a);
  if (a < 0) {   // no adapter
    if (s.base == s.out) return;
    for (int row = row0 + lane; row < row_end; row += kThreads) {
      const size_t at = (size_t)b * s.ld_out + s.col_off + row;
      store_out(s, at, load_base(s, at));
    }
    return;
  }
  if (!cols) return;
  // weights first: what is needed beside them is small and near
  const uint16_t* from = s.Bm + (size_t)a * s.n_rows * p.rank + piece * 8;
  const size_t first_col = (size_t)b * s.ld_out + s.col_off;
  // the row that this lane ends up with of each 32: the halving leaves the first half of the loads to the lanes whose first bit of `piece` is 0
  int turn = 0;
#pragma unroll
  for (int bit = 1; bit < P; bit <<= 1) turn = turn << 1 | ((piece / bit) & 1);
  const int my_row = turn * (32 / P) + lane / P;
  uint4 w[M][P];
  float base[M];
  auto request = [&](int row) {
#pragma unroll
    for (int m = 0; m < M; m++) {
      load_weights<P>(s, from, p.rank, row + m * kThreads, w[m]);
      base[m] = row + m * kThreads + my_row < s.n_rows ? load_base(s, first_col + row + m * kThreads + my_row) : 0.0f;
    }
  };
  request(row0);
  const float scale = p.scale ? __ldg(p.scale + a) : 1.0f;
  const int n = __popcll(cols);
  {
    unsigned long long rest = cols;
    for (int c = 0; c < n; c++, rest &= rest - 1) {
      const int col = __ffsll(rest) - 1;
      for (int r = threadIdx.x; r < 8 * P; r += kThreads) {   // (rows of 8 P, zeros behind the rank)
        float y = 0.0f;
        if (r < p.rank)
#pragma unroll 4
          for (int part = 0; part < p.parts; part++) y = __fadd_rn(y, __ldcg(p.u + (((size_t)part * p.n_segs + seg) * p.B + col) * p.rank + r));
        u_s[c * 8 * P + r] = __fmul_rn(scale, y);
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int row = row0; row < row_end; row += M * kThreads) {
    uint4 now[M][P];
    float base_now[M];
#pragma unroll
    for (int m = 0; m < M; m++) {
      base_now[m] = base[m];
#pragma unroll
      for (int i = 0; i < P; i++) now[m][i] = w[m][i];
    }
    if (row + M * kThreads < row_end) request(row + M * kThreads);
    unsigned long long rest = cols;
#pragma unroll 1
    for (int c = 0; c < n; c++, rest &= rest - 1) {
      float u[8];
      *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(u_s + c * 8 * P + piece * 8);
      *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(u_s + c * 8 * P + piece * 8 + 4);
      const size_t col = (size_t)(__ffsll(rest) - 1) * s.ld_out + s.col_off;
#pragma unroll
      for (int m = 0; m < M; m++) {
        float y[P];
#pragma unroll
        for (int i = 0; i < P; i++) {
          float v[8];
          unpack8(now[m][i], v);
          y[i] = __fmul_rn(v[0], u[0]);
#pragma unroll
          for (int e = 1; e < 8; e++) y[i] = fmaf(v[e], u[e], y[i]);
        }
        // the lanes of a row: a lane keeps the half of its sums that its bit of `piece` says and gets the partner's
#pragma unroll
        for (int half = P / 2, bit = 1; half >= 1; half >>= 1, bit <<= 1) {
          const bool upper = piece & bit;
#pragma unroll
          for (int i = 0; i < half; i++) {
            const float send = upper ? y[i] : y[i + half], keep = upper ? y[i + half] : y[i];
            y[i] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, send, bit));
          }
        }
        const int r = row + m * kThreads + my_row;
        if (r < s.n_rows) store_out(s, col + r, __fadd_rn(c == 0 ? base_now[m] : load_base(s, col + r), y[0]));
      }
    }
  }
}

template <int P, int M>
int32_t launch_expand_as(LoraParams& p, int per) {
  int ctas = 0;
  p.per = per;
  for (int i = 0; i < p.n_segs; i++) {
    p.segs[i].tile0 = ctas;
    ctas += (p.segs[i].n_rows + per * M * kThreads - 1) / (per * M * kThreads);
  }
  BK_CUDA(bk_launch_pdl(lora_expand_kernel<P, M>, dim3(ctas, p.B), dim3(kThreads), (size_t)p.B * 8 * P * 4, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}
// A CTA takes one tile where there are few, else as many as leave eight CTAs an SM.
template <int P>
int32_t launch_expand(LoraParams& p) {
  long long tiles = 0;
  for (int i = 0; i < p.n_segs; i++) tiles += (p.segs[i].n_rows + kThreads - 1) / kThreads;
  const long long each = tiles * std::min(p.B, p.n_adapters) / (8 * bk_ctx().sm_count);
  constexpr int M = P >= 4 ? 1 : 4 / P;
  if (each < M) return launch_expand_as<P, 1>(p, 1);
  return launch_expand_as<P, M>(p, (int)std::min(16ll, each / M));
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
  p.K = a.K; p.B = a.B; p.n_segs = a.n_segs; p.rank = a.rank; p.n_adapters = a.n_adapters;
  for (int i = 0; i < a.n_segs; i++) {
    const bkLoraSeg& s = a.segs[i];
    BK_ARG(s.n_rows > 0 && s.n_rows < (1 << 30) && s.col_off >= 0 && (long long)s.col_off + s.n_rows <= s.ld_out, "bkLora: segment %d: n_rows=%d col_off=%d ld_out=%d", i, s.n_rows, s.col_off,
           s.ld_out);
    BK_ARG(s.dtype == BK_DTYPE_F32 || s.dtype == BK_DTYPE_BF16, "bkLora: segment %d: dtype %d", i, s.dtype);
    const uint64_t mask = s.dtype == BK_DTYPE_F32 ? 3 : 1;
    BK_ARG(s.A && s.Bm && s.out && ((s.A | s.Bm) & 15) == 0 && ((s.base | s.out) & mask) == 0, "bkLora: segment %d: A and Bm must be 16-byte aligned, out non-null, base and out aligned to their type", i);
    p.segs[i] = LoraSeg{bk_ptr<uint16_t>(s.A), bk_ptr<uint16_t>(s.Bm), bk_ptr<void>(s.base), bk_ptr<void>(s.out), s.n_rows, s.dtype == BK_DTYPE_F32, s.ld_out, s.col_off, 0};
  }
  // Parts of K, multiples of 256: about four CTAs an SM, but no more than 512 partial rows of u for an expanding CTA to add up, and x in its place.
  const int units = (a.K + 255) / 256, least = (units + kChunk / 256 - 1) / (kChunk / 256);
  int parts = std::max(1, std::min(units, 4 * bk_ctx().sm_count / (a.n_segs * std::min(a.B, a.n_adapters))));
  parts = std::max(least, std::min(parts, std::max(1, 512 / a.B)));
  p.chunk = (units + parts - 1) / parts * 256;
  p.parts = (a.K + p.chunk - 1) / p.chunk;
  BK_CUDA(bk_launch_pdl(lora_shrink_kernel, dim3(p.parts, a.B, a.n_segs), dim3(kThreads), 0, p));
  BK_CHECK_LAUNCH();
  return a.rank <= 8 ? launch_expand<1>(p) : a.rank <= 16 ? launch_expand<2>(p) : a.rank <= 32 ? launch_expand<4>(p) : a.rank <= 64 ? launch_expand<8>(p) : launch_expand<16>(p);
}

}  // extern "C"
