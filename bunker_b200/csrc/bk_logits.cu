// bk_logits.cu -- penalties for repeated tokens, biases and grammar masks on logits, in place (bkAdjustLogits in bunker_cuda.h has the rules).
//
// What a row needs is sparse (the tokens of a history, of a path in a drafted tree, of a list of biases) but for the mask, so a row is not read as a
// whole: a CTA has a slice of the vocabulary of one request, counts the request's tokens of that slice in shared memory, and reads and writes only the
// quads of logits that something names; quads that a mask hides whole are written without being read.  Rows of one request (the nodes of its tree) share the
// counts: a row adds its path's tokens and takes them back.  Counts are integers, so results do not depend on the order of threads.
//
// No counterpart in the reference, which takes the argmax of the logits as they are (prototypes/decode.ts:749-791).
#include <math.h>

#include <algorithm>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

constexpr int kThreads = 512;
constexpr int kQuads = 4;   // quads of logits that a thread has on the way

// A token's word: how often it was said (20 bits), 1 + the place of its bias (11 bits), whether it is in the prompt.
constexpr uint32_t kSaid = (1u << 20) - 1, kInPrompt = 1u << 31;
constexpr int kBiasShift = 20;
constexpr int kMaxHistory = (1 << 20) - 1 - 1024;   // with a path of up to 1,024 nodes behind it
constexpr int kMaxNodes = 1024;

struct LogitsParams {
  float* logits;
  const int *seqs, *history, *hist_len, *prompt_len;
  const float *repetition, *presence, *frequency;
  const int* draft;
  const uint32_t* path;
  const int* bias_token;
  const float* bias_value;
  const int* bias_n;
  const uint32_t* allowed;
  const int* mask_id;
  int B, T, V, n_seqs, history_ld, bias_ld, path_words, n_masks, allowed_words;
  int slice, rows;   // tokens, and rows of a request, that a CTA has
  long long ld;
};

struct Penalty {
  float repetition, presence, frequency;
};
BK_DEVINL float adjusted(float x, uint32_t w, const Penalty& a, const float* bias) {
  const uint32_t n = w & kSaid, at = w >> kBiasShift & 2047u;
  if (n || w & kInPrompt) {
    x = x > 0.0f ? __fdiv_rn(x, a.repetition) : __fmul_rn(x, a.repetition);
    x = __fsub_rn(x, __fadd_rn(__fmul_rn(a.frequency, (float)n), n ? a.presence : 0.0f));
  }
  return at ? __fadd_rn(x, bias[at - 1]) : x;
}

// VEC: rows start on 16 bytes
template <bool VEC>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(const __grid_constant__ LogitsParams p) {
  extern __shared__ __align__(16) uint32_t word_s[];   // [slice]
  __shared__ int bias_at_s[BK_LOGITS_MAX_BIAS], warp_s[kThreads / 32];
  __shared__ float bias_s[BK_LOGITS_MAX_BIAS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y, lo = blockIdx.x * p.slice, n = min(p.slice, p.V - lo);
  for (int i = tid; i < p.slice / 4; i += kThreads) reinterpret_cast<uint4*>(word_s)[i] = make_uint4(0, 0, 0, 0);
  bk_pdl_wait();
  bk_pdl_trigger();
  const int s = p.seqs ? p.seqs[b] : b;
  const bool known = s >= 0 && s < p.n_seqs;
  Penalty a = {1.0f, 0.0f, 0.0f};
  if (known) {
    if (p.repetition) a.repetition = p.repetition[s];
    if (p.presence) a.presence = p.presence[s];
    if (p.frequency) a.frequency = p.frequency[s];
  }
  __syncthreads();
  if (known && p.history) {
    const int said = max(0, min(p.hist_len[s], p.history_ld)), prompt = p.prompt_len ? p.prompt_len[s] : 0;
    const int* h = p.history + (size_t)s * p.history_ld;
    auto count = [&](int token, int i) {
      const uint32_t o = (uint32_t)token - (uint32_t)lo;
      if (o < (uint32_t)n) {
        if (i < prompt) atomicOr(word_s + o, kInPrompt);
        else atomicAdd(word_s + o, 1u);
      }
    };
    const int head = min(said, (int)((16 - ((uintptr_t)h & 15)) & 15) / 4), quads = (said - head) / 4;
    if (tid < head) count(h[tid], tid);
#pragma unroll 4
    for (int q = tid; q < quads; q += kThreads) {
      const int4 v = __ldcg(reinterpret_cast<const int4*>(h + head) + q);
      const int i = head + 4 * q;
      count(v.x, i); count(v.y, i + 1); count(v.z, i + 2); count(v.w, i + 3);
    }
    const int i = head + 4 * quads + tid;
    if (i < said) count(h[i], i);
  }
  if (known && p.bias_token) {
    // the slice's entries, in the list's order
    const int listed = max(0, min(p.bias_n[s], p.bias_ld));
    int m = 0;
    for (int i0 = 0; i0 < listed; i0 += kThreads) {
      const int i = i0 + tid;
      const uint32_t o = i < listed ? (uint32_t)p.bias_token[(size_t)s * p.bias_ld + i] - (uint32_t)lo : 0xffffffffu;
      const bool mine = o < (uint32_t)n;
      const uint32_t votes = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) warp_s[warp] = __popc(votes);
      __syncthreads();
      int at = m + __popc(votes & ((1u << lane) - 1u));
      for (int w = 0; w < kThreads / 32; w++) {
        if (w < warp) at += warp_s[w];
        m += warp_s[w];
      }
      if (mine) {
        bias_at_s[at] = (int)o;
        bias_s[at] = p.bias_value[(size_t)s * p.bias_ld + i];
      }
      __syncthreads();
    }
    // a token's first entry gets the sum of all of its (a thread may only write its own, so sums are stored behind a barrier)
    float sum[BK_LOGITS_MAX_BIAS / kThreads];
    int first = 0;   // bit k: entry tid + k * kThreads is its token's first
#pragma unroll
    for (int k = 0; k < BK_LOGITS_MAX_BIAS / kThreads; k++) {
      const int i = tid + k * kThreads;
      if (i >= m) continue;
      const int o = bias_at_s[i];
      bool earlier = false;
      float y = 0.0f;
      for (int j = 0; j < m; j++)
        if (bias_at_s[j] == o) {
          if (j < i) earlier = true;
          else y = j == i ? bias_s[j] : __fadd_rn(y, bias_s[j]);
        }
      sum[k] = y;
      if (!earlier) first |= 1 << k;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BK_LOGITS_MAX_BIAS / kThreads; k++)
      if (first >> k & 1) {
        const int i = tid + k * kThreads;
        bias_s[i] = sum[k];
        atomicOr(word_s + bias_at_s[i], (uint32_t)(i + 1) << kBiasShift);
      }
  }
  __syncthreads();

  const int t1 = min(p.T, (int)(blockIdx.z + 1) * p.rows);
  for (int t = blockIdx.z * p.rows; t < t1; t++) {
    const size_t row = (size_t)t * p.B + b;
    // the path's tokens, for this row only
    auto path = [&](uint32_t by) {
      for (int u = tid; u < p.T; u += kThreads)
        if (p.path[row * p.path_words + (u >> 5)] >> (u & 31) & 1u) {
          const uint32_t o = (uint32_t)p.draft[(size_t)u * p.B + b] - (uint32_t)lo;
          if (o < (uint32_t)n) atomicAdd(word_s + o, by);
        }
    };
    if (p.path) {
      path(1u);
      __syncthreads();
    }
    const int id = p.mask_id ? p.mask_id[row] : -1;
    const uint32_t* allowed = id >= 0 && id < p.n_masks ? p.allowed + (size_t)id * p.allowed_words + lo / 32 : nullptr;
    float* x = p.logits + row * p.ld + lo;
    const int quads = (n + 3) / 4;
    for (int q0 = tid; q0 < quads; q0 += kThreads * kQuads) {
      uint4 w[kQuads];
      uint32_t open[kQuads];   // bit e: token e of the quad is allowed
      float v[kQuads][4];
      int todo = 0;
#pragma unroll
      for (int k = 0; k < kQuads; k++) {
        const int q = q0 + k * kThreads;
        w[k] = make_uint4(0, 0, 0, 0);
        open[k] = 15;
        if (q >= quads) continue;
        w[k] = reinterpret_cast<const uint4*>(word_s)[q];
        if (allowed) open[k] = __ldg(allowed + (q >> 3)) >> (q & 7) * 4 & 15u;
        if ((w[k].x | w[k].y | w[k].z | w[k].w) == 0 && open[k] == 15) continue;
        todo |= 1 << k;
        if (open[k] == 0) continue;   // (written without being read)
        if (VEC && 4 * q + 4 <= n) {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(x) + q);
          v[k][0] = y.x; v[k][1] = y.y; v[k][2] = y.z; v[k][3] = y.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (4 * q + e < n) v[k][e] = __ldcg(x + 4 * q + e);
        }
      }
#pragma unroll
      for (int k = 0; k < kQuads; k++) {
        if (!(todo >> k & 1)) continue;
        const int q = q0 + k * kThreads;
        const uint32_t words[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
        for (int e = 0; e < 4; e++) v[k][e] = open[k] >> e & 1 ? words[e] ? adjusted(v[k][e], words[e], a, bias_s) : v[k][e] : -INFINITY;
        if (VEC && 4 * q + 4 <= n) {
          reinterpret_cast<float4*>(x)[q] = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (4 * q + e < n) x[4 * q + e] = v[k][e];
        }
      }
    }
    if (p.path && t + 1 < t1) {
      __syncthreads();
      path(0xffffffffu);
      __syncthreads();
    }
  }
}

}  // namespace

extern "C" int32_t bkAdjustLogits(const bkLogitsArgs* args) {
  BK_REQUIRE_INIT();
  BK_ARG(args != nullptr, "bkAdjustLogits: args is null");
  const bkLogitsArgs& a = *args;
  BK_ARG(a.logits && (a.logits & 3) == 0, "bkAdjustLogits: logits must be a non-null f32 array");
  BK_ARG(a.B > 0 && a.B <= 65535 && a.T > 0 && a.T <= kMaxNodes && a.V > 0 && a.V <= (1 << 30), "bkAdjustLogits: B=%d (1 to 65535) T=%d (1 to %d) V=%d", a.B, a.T, kMaxNodes, a.V);
  BK_ARG(a.ld == 0 || a.ld >= a.V, "bkAdjustLogits: ld=%d for %d logits", a.ld, a.V);
  BK_ARG(a.n_seqs >= 0, "bkAdjustLogits: n_seqs=%d", a.n_seqs);
  BK_ARG(((a.seqs | a.history | a.hist_len | a.prompt_len | a.repetition | a.presence | a.frequency | a.draft | a.path | a.bias_token | a.bias_value | a.bias_n | a.allowed | a.mask_id) & 3) == 0,
         "bkAdjustLogits: all arrays are of 32-bit words");
  BK_ARG(!a.history || (a.hist_len && a.history_ld > 0 && a.history_ld <= kMaxHistory), "bkAdjustLogits: history needs hist_len and history_ld (%d; 1 to %d)", a.history_ld, kMaxHistory);
  BK_ARG((a.path != 0) == (a.draft != 0) && (!a.path || a.path_words >= (a.T + 31) / 32), "bkAdjustLogits: draft and path go together, path_words=%d for %d nodes", a.path_words, a.T);
  BK_ARG((a.bias_token != 0) == (a.bias_value != 0) && (a.bias_token != 0) == (a.bias_n != 0) && (!a.bias_token || (a.bias_ld > 0 && a.bias_ld <= BK_LOGITS_MAX_BIAS)),
         "bkAdjustLogits: bias_token, bias_value and bias_n go together, bias_ld=%d (1 to %d)", a.bias_ld, BK_LOGITS_MAX_BIAS);
  BK_ARG((a.allowed != 0) == (a.mask_id != 0) && (!a.allowed || (a.n_masks > 0 && a.allowed_words >= (a.V + 31) / 32)),
         "bkAdjustLogits: allowed and mask_id go together, n_masks=%d allowed_words=%d for %d tokens", a.n_masks, a.allowed_words, a.V);
  LogitsParams p = {bk_ptr<float>(a.logits), bk_ptr<int>(a.seqs), bk_ptr<int>(a.history), bk_ptr<int>(a.hist_len), bk_ptr<int>(a.prompt_len), bk_ptr<float>(a.repetition),
                    bk_ptr<float>(a.presence), bk_ptr<float>(a.frequency), bk_ptr<int>(a.draft), bk_ptr<uint32_t>(a.path), bk_ptr<int>(a.bias_token), bk_ptr<float>(a.bias_value),
                    bk_ptr<int>(a.bias_n), bk_ptr<uint32_t>(a.allowed), bk_ptr<int>(a.mask_id), a.B, a.T, a.V, a.n_seqs ? a.n_seqs : a.B, a.history_ld, a.bias_ld, a.path_words,
                    a.n_masks, a.allowed_words, 0, 0, a.ld ? a.ld : a.V};
  // Slices of 8,192 tokens (32 KB of words, four CTAs an SM), shorter while that leaves SMs without one; then rows apart, until each SM has four.
  const long long sms = bk_ctx().sm_count;
  p.slice = 8192;
  while (p.slice > 1024 && (long long)((a.V + p.slice - 1) / p.slice) * a.B * a.T < sms) p.slice /= 2;
  const long long ctas = (long long)((a.V + p.slice - 1) / p.slice) * a.B;
  const int parts = (int)std::min<long long>(a.T, (4 * sms + ctas - 1) / ctas);
  p.rows = (a.T + parts - 1) / parts;
  const dim3 grid((a.V + p.slice - 1) / p.slice, a.B, (a.T + p.rows - 1) / p.rows);
  const bool vec = (a.logits & 15) == 0 && p.ld % 4 == 0;
  if (vec) BK_CUDA(bk_launch_pdl(adjust_logits_kernel<true>, grid, dim3(kThreads), (size_t)p.slice * 4, p));
  else BK_CUDA(bk_launch_pdl(adjust_logits_kernel<false>, grid, dim3(kThreads), (size_t)p.slice * 4, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}
