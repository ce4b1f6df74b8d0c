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
  int n_rows, f32, ld_out, col_off, tile0;   // tile0: first row tile of the segment in the expanding launch
};
struct LoraParams {
  const uint16_t* x;
  const int* ids;
  const float* scale;
  float* u;   // [part of K][segment][column][rank]
  int K, B, n_segs, rank, n_adapters, parts, chunk;
  LoraSeg segs[4];
};

// The columns that share column b's adapter, if b is the first of them: their number (0: b is not, or has no adapter), list in cols[].  All
// threads call.
BK_DEVINL int columns_of(const LoraParams& p, int b, int* cols, int* adapter) {
  __shared__ int n_s;
  const int a = p.ids[b];
  *adapter = a;
  if (a < 0 || a >= p.n_adapters) return 0;
  if (threadIdx.x < 32) {
    int n = 0;
    bool first = true;
    for (int j0 = 0; j0 < p.B; j0 += 32) {
      const int j = j0 + (int)threadIdx.x;
      const unsigned int same = __ballot_sync(0xffffffffu, j < p.B && p.ids[j] == a);
      if (first && same && j0 + __ffs(same) - 1 < b) {
        n = 0;
        break;
      }
      if (same) first = false;
      if ((same >> threadIdx.x) & 1) cols[n + __popc(same & ((1u << threadIdx.x) - 1))] = j;
      n += __popc(same);
    }
    if (threadIdx.x == 0) n_s = n;
  }
  __syncthreads();
  return n_s;
}

BK_DEVINL void unpack8(uint4 v, float (&y)[8]) {
  y[0] = __uint_as_float(v.x << 16); y[1] = __uint_as_float(v.x & 0xffff0000u);
  y[2] = __uint_as_float(v.y << 16); y[3] = __uint_as_float(v.y & 0xffff0000u);
  y[4] = __uint_as_float(v.z << 16); y[5] = __uint_as_float(v.z & 0xffff0000u);
  y[6] = __uint_as_float(v.w << 16); y[7] = __uint_as_float(v.w & 0xffff0000u);
}

// rows of A of one warp times C columns
template <int C>
BK_DEVINL void shrink_rows(const LoraParams& p, const uint16_t* A, int seg, int part, const int* cols, int n) {
  const int lane = threadIdx.x & 31, k0 = part * p.chunk, k1 = min(p.K, k0 + p.chunk);
  for (int r = threadIdx.x >> 5; r < p.rank; r += kThreads / 32) {
    float acc[C];
#pragma unroll
    for (int c = 0; c < C; c++) acc[c] = 0.0f;
    for (int k = k0 + lane * 8; k < k1; k += 256) {
      float w[8];
      unpack8(__ldg(reinterpret_cast<const uint4*>(A + (size_t)r * p.K + k)), w);
#pragma unroll
      for (int c = 0; c < C; c++) {
        float x[8];
        unpack8(*reinterpret_cast<const uint4*>(p.x + (size_t)cols[min(c, n - 1)] * p.K + k), x);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[c] = fmaf(w[e], x[e], acc[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
      const float y = bk_warp_sum(acc[c]);
      if (lane == 0 && c < n) p.u[(((size_t)part * p.n_segs + seg) * p.B + cols[c]) * p.rank + r] = y;
    }
  }
}

// grid (part of K, column, segment)
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  __shared__ int cols[kMaxB];
  bk_pdl_trigger();
  bk_pdl_wait();
  int a;
  const int n = columns_of(p, blockIdx.y, cols, &a);
  const uint16_t* A = p.segs[blockIdx.z].A + (size_t)a * p.rank * p.K;
  for (int c = 0; c < n; c += 4) {
    if (n - c == 1) shrink_rows<1>(p, A, blockIdx.z, blockIdx.x, cols + c, 1);
    else shrink_rows<4>(p, A, blockIdx.z, blockIdx.x, cols + c, n - c);
  }
}

BK_DEVINL float load_base(const LoraSeg& s, size_t at) {
  return !s.base ? 0.0f : s.f32 ? reinterpret_cast<const float*>(s.base)[at] : bk_bf16_to_f32(reinterpret_cast<const uint16_t*>(s.base)[at]);
}
BK_DEVINL void store_out(const LoraSeg& s, size_t at, float v) {
  if (s.f32) reinterpret_cast<float*>(s.out)[at] = v;
  else reinterpret_cast<uint16_t*>(s.out)[at] = bk_f32_to_bf16(v);
}

// grid (tile of 256 rows, column); a thread has one row
__global__ void __launch_bounds__(kThreads) lora_expand_kernel(const __grid_constant__ LoraParams p) {
  __shared__ int cols[kMaxB];
  __shared__ __align__(16) float u_s[kMaxB * kMaxRank];
  bk_pdl_trigger();
  bk_pdl_wait();
  int seg = 0;
  while (seg + 1 < p.n_segs && (int)blockIdx.x >= p.segs[seg + 1].tile0) seg++;
  const LoraSeg& s = p.segs[seg];
  const int row = ((int)blockIdx.x - s.tile0) * kThreads + (int)threadIdx.x, b = blockIdx.y;
  int a;
  const int n = columns_of(p, b, cols, &a);
  if (a < 0 || a >= p.n_adapters) {
    if (s.base != s.out && row < s.n_rows) {
      const size_t at = (size_t)b * s.ld_out + s.col_off + row;
      store_out(s, at, load_base(s, at));
    }
    return;
  }
  if (n == 0) return;
  const float scale = p.scale ? p.scale[a] : 1.0f;
  for (int i = threadIdx.x; i < n * p.rank; i += kThreads) {
    const int c = i / p.rank, r = i - c * p.rank;
    float y = 0.0f;
    for (int part = 0; part < p.parts; part++) y = __fadd_rn(y, __ldcg(p.u + (((size_t)part * p.n_segs + seg) * p.B + cols[c]) * p.rank + r));
    u_s[i] = __fmul_rn(scale, y);
  }
  __syncthreads();
  if (row >= s.n_rows) return;
  const uint16_t* w_row = s.Bm + ((size_t)a * s.n_rows + row) * p.rank;
  for (int c0 = 0; c0 < n; c0 += 4) {
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int r = 0; r < p.rank; r += 8) {
      float w[8];
      unpack8(__ldg(reinterpret_cast<const uint4*>(w_row + r)), w);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const float* u = u_s + min(c0 + c, n - 1) * p.rank + r;
#pragma unroll
        for (int e = 0; e < 8; e++) acc[c] = fmaf(w[e], u[e], acc[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (c0 + c < n) {
        const size_t at = (size_t)cols[c0 + c] * s.ld_out + s.col_off + row;
        store_out(s, at, __fadd_rn(load_base(s, at), acc[c]));
      }
  }
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
  int tiles = 0;
  for (int i = 0; i < a.n_segs; i++) {
    const bkLoraSeg& s = a.segs[i];
    BK_ARG(s.n_rows > 0 && s.n_rows < (1 << 30) && s.col_off >= 0 && (long long)s.col_off + s.n_rows <= s.ld_out, "bkLora: segment %d: n_rows=%d col_off=%d ld_out=%d", i, s.n_rows, s.col_off,
           s.ld_out);
    BK_ARG(s.dtype == BK_DTYPE_F32 || s.dtype == BK_DTYPE_BF16, "bkLora: segment %d: dtype %d", i, s.dtype);
    const uint64_t mask = s.dtype == BK_DTYPE_F32 ? 3 : 1;
    BK_ARG(s.A && s.Bm && s.out && ((s.A | s.Bm) & 15) == 0 && ((s.base | s.out) & mask) == 0, "bkLora: segment %d: A and Bm must be 16-byte aligned, out non-null, base and out aligned to their type", i);
    p.segs[i] = LoraSeg{bk_ptr<uint16_t>(s.A), bk_ptr<uint16_t>(s.Bm), bk_ptr<void>(s.base), bk_ptr<void>(s.out), s.n_rows, s.dtype == BK_DTYPE_F32, s.ld_out, s.col_off, tiles};
    tiles += (s.n_rows + kThreads - 1) / kThreads;
  }
  const int units = (a.K + 255) / 256;   // the least that a warp takes of K at a time
  int parts = std::max(1, std::min(units, 2 * bk_ctx().sm_count / (a.n_segs * std::min(a.B, a.n_adapters))));
  parts = std::min(parts, std::max(1, 512 / a.B));
  p.chunk = (units + parts - 1) / parts * 256;
  p.parts = (a.K + p.chunk - 1) / p.chunk;
  BK_CUDA(bk_launch_pdl(lora_shrink_kernel, dim3(p.parts, a.B, a.n_segs), dim3(kThreads), 0, p));
  BK_CHECK_LAUNCH();
  BK_CUDA(bk_launch_pdl(lora_expand_kernel, dim3(tiles, a.B), dim3(kThreads), 0, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

}  // extern "C"
