// bk_paged_attn.cu -- attention of many sequences over pages of keys and values (bkPagedAttn in bunker_cuda.h has the rules).
//
// No counterpart in the reference (one contiguous cache of 128 rows, src/emitters.ts:188-226).
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
  int B, T, Hq, Hkv, rot_half, n_pages, page_rows, max_pages, max_len, fused;
  float scale, eps;
};

// row of its sequence at which token t of sequence b stands, -1 where it is not there
BK_DEVINL int row_of(const PagedParams& p, int b, int t) {
  const int n = p.n_new ? min(p.n_new[b], p.T) : p.T;
  const long long at = (long long)p.lens[b] - n + t;
  return t < n && at >= 0 && at < p.max_len ? (int)at : -1;
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

// One warp per (token row, head): q heads to the scratch buffer, k and v heads into their page.
template <int HD>
__global__ void __launch_bounds__(128) paged_prepare_kernel(const PagedParams p) {
  constexpr int PER = HD / 32;
  __shared__ float y_s[4][HD];
  bk_pdl_trigger();
  bk_pdl_wait();
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
    const int page = p.table[(size_t)b * p.max_pages + min(at / p.page_rows, p.max_pages - 1)];
    if (page < 0 || page >= p.n_pages || at / p.page_rows >= p.max_pages) return;
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

// One warp per (token row, query head).
template <int HD>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedParams p) {
  constexpr int PER = HD / 32;
  bk_pdl_trigger();
  bk_pdl_wait();
  const int lane = threadIdx.x & 31, item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= p.T * p.B * p.Hq) return;
  const int e = item / p.Hq, h = item - e * p.Hq, t = e / p.B, b = e - t * p.B, kvh = h / (p.Hq / p.Hkv);
  uint16_t* out = p.out + ((size_t)e * p.Hq + h) * HD + lane * PER;
  float q[PER], o[PER], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; i++) o[i] = 0.0f;
  const int at = row_of(p, b, t);
  if (at >= 0) load_bf16(p.q + ((size_t)e * p.Hq + h) * HD + lane * PER, q);
  for (int j = 0; j <= at; j++) {
    if (j / p.page_rows >= p.max_pages) break;
    const int page = p.table[(size_t)b * p.max_pages + j / p.page_rows];
    if (page < 0 || page >= p.n_pages) continue;
    const size_t row = (((size_t)page * p.Hkv + kvh) * p.page_rows + j % p.page_rows) * HD + lane * PER;
    float k[PER], v[PER], s = 0.0f;
    load_bf16(p.k_pages + row, k);
    load_bf16(p.v_pages + row, v);
#pragma unroll
    for (int i = 0; i < PER; i++) s = fmaf(q[i], k[i], s);
    s = __fmul_rn(bk_warp_sum(s), p.scale);
    const float mn = fmaxf(m, s);
    const float c = m == -INFINITY ? 0.0f : bk_expf(__fsub_rn(m, mn)), w = bk_expf(__fsub_rn(s, mn));
    l = fmaf(l, c, w);
#pragma unroll
    for (int i = 0; i < PER; i++) o[i] = fmaf(o[i], c, __fmul_rn(w, v[i]));
    m = mn;
  }
  const uint16_t* gate = p.fused ? p.qg + ((size_t)e * p.Hq + h) * 2 * HD + HD : p.gate ? p.gate + ((size_t)e * p.Hq + h) * HD : nullptr;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    o[i] = l > 0.0f ? __fdiv_rn(o[i], l) : 0.0f;
    if (gate && l > 0.0f) o[i] = __fmul_rn(o[i], bk_sigmoidf(bk_bf16_to_f32(gate[lane * PER + i])));
  }
#pragma unroll
  for (int i = 0; i < PER; i += 4) *reinterpret_cast<uint2*>(out + i) = make_uint2(bk_f32x2_to_bf16x2(o[i], o[i + 1]), bk_f32x2_to_bf16x2(o[i + 2], o[i + 3]));
}

template <int HD>
int32_t launch_paged(const PagedParams& p) {
  const int heads = (p.fused ? p.Hq : 0) + (p.k ? p.Hkv : 0);
  if (heads) {
    BK_CUDA(bk_launch_pdl(paged_prepare_kernel<HD>, dim3((p.T * p.B * heads + 3) / 4), dim3(128), 0, p));
    BK_CHECK_LAUNCH();
  }
  BK_CUDA(bk_launch_pdl(paged_attn_kernel<HD>, dim3((p.T * p.B * p.Hq + 3) / 4), dim3(128), 0, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}

}  // namespace

extern "C" {

uint64_t bkPagedAttnScratchBytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t HD, int32_t prefix_rows) {
  (void)Hkv;
  (void)prefix_rows;
  if (B <= 0 || T <= 0 || Hq <= 0 || HD <= 0) return 0;
  return (uint64_t)B * T * Hq * HD * 2;
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
  p.max_len = a.max_len; p.fused = a.fused_norm_rope != 0; p.scale = a.scale; p.eps = a.eps;
  return a.HD == 256 ? launch_paged<256>(p) : launch_paged<128>(p);
}

}  // extern "C"
