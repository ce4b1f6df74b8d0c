// bk_logits.cu -- penalties for repeated tokens, biases and grammar masks on logits, in place (bkAdjustLogits in bunker_cuda.h has the rules).
//
// Two kinds of CTAs, of one launch, which never touch the same logit.  Some hide what the masks forbid: a warp has 1,024 tokens of a row, a lane's mask word
// at a time for all lanes, and only writes.  The others do what is named (tokens of a history, of a path in a drafted tree, of a list of biases), which is sparse: a CTA has a
// slice of the vocabulary of one request (every 2^k-th block of 512 tokens, since frequent tokens have numbers near one another), counts the tokens of the history that
// lie there in shared memory (a word for each token of the slice, or, for short histories, a table of those that occur), lists them, and goes over (listed token, row) pairs; the rows of a request, the nodes of its tree, share counts and list.  Tokens that are
// drafted somewhere in the tree, or have a bias, are marked and left to a loop of their own.  Counts are integers, so results do not depend on the order of threads.
//
// No counterpart in the reference, which takes the argmax of the logits as they are (prototypes/decode.ts:749-791).
#include <math.h>

#include <algorithm>

#include "bk_common.cuh"
#include "bk_internal.h"

namespace {

constexpr int kThreads = 512;
constexpr int kUnits = 6;        // logits that a thread has on the way
constexpr int kMaxNodes = 1024;  // of a tree
constexpr int kMaxSlice = 8192;  // words
constexpr int kMaxTable = 8192;  // entries of a table (of 8 bytes), a quarter of them free
constexpr int kBlock = 512;      // tokens that lie together in a slice (64: 3 % slower, where memory is the bound)
constexpr int kAhead = 1;        // groups of four tokens of the history that a thread asks for before it knows the history's length

// A token's word: how often it was said, whether the request names a bias of it again, whether the last loop has it, whether it is in the prompt.
constexpr uint32_t kSaid = (1u << 29) - 1, kAgain = 1u << 29, kMarked = 1u << 30, kInPrompt = 1u << 31;
constexpr int kMaxHistory = 1 << 28;

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
  int shift, slice, rows, parts;   // log2 of the number of slices; words, and rows of a request, that a CTA has; CTAs that share a request's rows
  int naming, hiding;              // CTAs of each kind
  long long ld;
};

struct Penalty {
  float down, up, presence, frequency;   // of positive and other logits: 1 / repetition, rounded (a second rounding beside the product's), and repetition
};
BK_DEVINL float taken(uint32_t n, const Penalty& a) { return fmaf(a.frequency, (float)n, n ? a.presence : 0.0f); }
BK_DEVINL float adjusted(float x, float sub, const Penalty& a) { return fmaf(x, x > 0.0f ? a.down : a.up, -sub); }

// Hides what the masks forbid.  Bound: the writes, 4 bytes a token at least (a sector that is written in part is read by the memory beside it).
BK_DEVINL void hide(const LogitsParams& p, int cta) {
  const int lane = threadIdx.x & 31, chunks = (p.V + 1023) / 1024;
  const long long items = (long long)p.T * p.B * chunks, warps = (long long)p.hiding * (kThreads / 32), w = (long long)cta * (kThreads / 32) + (threadIdx.x >> 5);
  const long long i1 = items * (w + 1) / warps;
  long long i = items * w / warps;
  long long row = i / chunks;
  int chunk = (int)(i - row * chunks);
  auto id_of = [&]() {
    const int id = i < i1 ? __ldg(p.mask_id + row) : -1;
    return id >= 0 && id < p.n_masks ? id : -1;
  };
  auto word_of = [&](int id) {   // this lane's 32 tokens; one behind the vocabulary is not hidden
    const int at = chunk * 32 + lane, left = p.V - at * 32;
    if (id < 0 || left <= 0) return 0xffffffffu;
    return __ldg(p.allowed + (size_t)id * p.allowed_words + at) | (left < 32 ? 0xffffffffu << left : 0u);
  };
  int id = id_of();
  uint32_t word = word_of(id);
  while (i < i1) {
    float* x = p.logits + row * p.ld + chunk * 1024 + lane;
    const uint32_t now = word;
    i++;
    if (++chunk == chunks) {
      chunk = 0;
      row++;
      id = id_of();
    }
    word = i < i1 ? word_of(id) : 0xffffffffu;
    if (!__any_sync(0xffffffffu, now != 0xffffffffu)) continue;
#pragma unroll
    for (int j = 0; j < 32; j++)
      if (!(__shfl_sync(0xffffffffu, now, j) >> lane & 1u)) x[j * 32] = -INFINITY;
  }
}

// TABLE: words belong to the tokens of a table (open addressing), not to all of the slice's
template <bool TABLE>
__global__ void __launch_bounds__(kThreads, 2) adjust_logits_kernel(const __grid_constant__ LogitsParams p) {
  extern __shared__ __align__(16) uint32_t word_s[];        // [slice], then lists, see there
  __shared__ int node_s[kMaxNodes], warp_s[kThreads / 32];  // nodes whose token lies in the slice: node << 16 | place
  __shared__ int n_node_s, n_marked_s, n_listed_s, mask_s[kMaxNodes];   // mask_s: of each row, -1 where it has none
  bk_pdl_wait();
  bk_pdl_trigger();
  // Every third CTA hides, while there are two that name to one that hides: the ones are bound by memory, the others by latency (512 rows: 122 us with all that hide
  // behind, 111 so).
  const int triples = min(p.hiding, p.naming / 2), i_cta = blockIdx.x, behind = i_cta - 3 * triples;
  const int i_name = behind < 0 ? (i_cta % 3 < 2 ? i_cta - i_cta / 3 : -1) : behind < p.naming - 2 * triples ? behind + 2 * triples : -1;
  if (i_name < 0) {
    hide(p, behind < 0 ? i_cta / 3 : behind - (p.naming - 2 * triples) + triples);
    return;
  }
  const int marks = p.bias_ld + (p.path ? p.T : 0);
  float* const bias_s = reinterpret_cast<float*>(word_s + p.slice);           // [bias_ld]: the slice's biases
  float* const sum_s = bias_s + p.bias_ld;                                    // [marks]: of a marked token
  uint16_t* const marked_s = reinterpret_cast<uint16_t*>(sum_s + marks);      // [marks]
  uint16_t* const bias_at_s = marked_s + marks;                               // [bias_ld]
  uint16_t* const listed_s = bias_at_s + p.bias_ld;                           // [slice]: places of tokens that something but a mark names
  int* const key_s = reinterpret_cast<int*>(listed_s + p.slice + ((marks + p.bias_ld) & 1));   // TABLE: [slice] tokens, -1: free
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = i_name & ((1 << p.shift) - 1), group = i_name >> p.shift, b = group / p.parts,
            t0 = (group - b * p.parts) * p.rows, rows = min(p.rows, p.T - t0);
  if (rows <= 0) return;
  // token -> its place in the slice, -1: not in it; place -> token
  auto place = [&](int token) {
    const uint32_t block = (uint32_t)token / kBlock;
    if ((uint32_t)token >= (uint32_t)p.V || (block & ((1u << p.shift) - 1u)) != (uint32_t)part) return -1;
    if (!TABLE) return (int)(block >> p.shift) * kBlock + token % kBlock;
    int at = (int)((uint32_t)token * 2654435761u >> 16 & (uint32_t)(p.slice - 1));
    while (true) {   // (ends: the table has more entries than the request names tokens)
      int there = *reinterpret_cast<volatile int*>(key_s + at);   // (most are there already: equal addresses are one read, but one atomic after the other)
      if (there == -1) there = atomicCAS(key_s + at, -1, token);
      if (there == -1 || there == token) return at;
      at = (at + 1) & (p.slice - 1);
    }
  };
  auto token_of = [&](int at) { return TABLE ? key_s[at] : ((at / kBlock << p.shift) + part) * kBlock + at % kBlock; };
  const int s = p.seqs ? p.seqs[b] : b;
  const bool known = s >= 0 && s < p.n_seqs;
  // everything that the request has is asked for at once, beyond what counts where its arrays are longer
  Penalty a = {1.0f, 1.0f, 0.0f, 0.0f};
  int said = 0, prompt = 0, listed = 0, head = 0;
  const int* h = p.history + (known ? (size_t)s * p.history_ld : 0);
  int4 ahead[kAhead];
  int bias_token[BK_LOGITS_MAX_BIAS / kThreads], draft[kMaxNodes / kThreads];
  float bias_value[BK_LOGITS_MAX_BIAS / kThreads];
  if (known) {
    if (p.history) {
      said = p.hist_len[s];
      head = min(p.history_ld, (int)((16 - ((uintptr_t)h & 15)) & 15) / 4);
#pragma unroll
      for (int k = 0; k < kAhead; k++)
        if (head + 4 * (tid + k * kThreads) + 4 <= p.history_ld) ahead[k] = __ldcg(reinterpret_cast<const int4*>(h + head) + tid + k * kThreads);
    }
    if (p.prompt_len) prompt = p.prompt_len[s];
    if (p.repetition) a.up = p.repetition[s];
    if (p.presence) a.presence = p.presence[s];
    if (p.frequency) a.frequency = p.frequency[s];
    if (p.bias_ld) {
      listed = p.bias_n[s];
#pragma unroll
      for (int k = 0; k < BK_LOGITS_MAX_BIAS / kThreads; k++) {
        const int i = tid + k * kThreads;
        if (i < p.bias_ld) {
          bias_token[k] = p.bias_token[(size_t)s * p.bias_ld + i];
          bias_value[k] = p.bias_value[(size_t)s * p.bias_ld + i];
        }
      }
    }
  }
  if (p.path) {
#pragma unroll
    for (int k = 0; k < kMaxNodes / kThreads; k++)
      if (tid + k * kThreads < p.T) draft[k] = p.draft[(size_t)(tid + k * kThreads) * p.B + b];
  }
  for (int t = tid; t < rows; t += kThreads) {
    const int id = p.mask_id ? p.mask_id[(size_t)(t0 + t) * p.B + b] : -1;
    mask_s[t] = id >= 0 && id < p.n_masks ? id : -1;
  }
  for (int i = tid; i < p.slice / 4; i += kThreads) reinterpret_cast<uint4*>(word_s)[i] = make_uint4(0, 0, 0, 0);
  if (TABLE)
    for (int i = tid; i < p.slice; i += kThreads) key_s[i] = -1;
  if (tid == 0) n_node_s = n_marked_s = n_listed_s = 0;
  said = max(0, min(said, p.history_ld));
  listed = max(0, min(listed, p.bias_ld));
  a.down = __fdiv_rn(1.0f, a.up);
  __syncthreads();
  if (said) {
    head = min(head, said);
    auto count = [&](int token, int i) {
      const int o = place(token);
      if (o >= 0) {
        if (i < prompt) atomicOr(word_s + o, kInPrompt);
        else atomicAdd(word_s + o, 1u);
      }
    };
    const int quads = (said - head) / 4;
    auto count4 = [&](int4 v, int q) {
      const int i = head + 4 * q;
      count(v.x, i); count(v.y, i + 1); count(v.z, i + 2); count(v.w, i + 3);
    };
    if (tid < head) count(h[tid], tid);
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (tid + k * kThreads < quads) count4(ahead[k], tid + k * kThreads);
#pragma unroll 4
    for (int q = tid + kAhead * kThreads; q < quads; q += kThreads) count4(__ldcg(reinterpret_cast<const int4*>(h + head) + q), q);
    const int i = head + 4 * quads + tid;
    if (i < said) count(h[i], i);
  }
  // marked tokens: who sets a token's mark writes it down
  auto mark = [&](int o, bool bias, float value) {
    if (!(atomicOr(word_s + o, kMarked) & kMarked)) {
      const int i = atomicAdd(&n_marked_s, 1);
      marked_s[i] = (uint16_t)o;
      sum_s[i] = value;
    } else if (bias) {
      atomicOr(word_s + o, kAgain);
    }
  };
  int m = 0;   // biases of the slice, in the list's order
#pragma unroll
  for (int k = 0; k < BK_LOGITS_MAX_BIAS / kThreads; k++) {
    if (k * kThreads >= listed) break;
    const int o = tid + k * kThreads < listed ? place(bias_token[k]) : -1;
    const uint32_t votes = __ballot_sync(0xffffffffu, o >= 0);
    if (k) __syncthreads();
    if (lane == 0) warp_s[warp] = __popc(votes);
    __syncthreads();
    int at = m + __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < kThreads / 32; w++) {
      if (w < warp) at += warp_s[w];
      m += warp_s[w];
    }
    if (o >= 0) {
      bias_at_s[at] = (uint16_t)o;
      bias_s[at] = bias_value[k];
      mark(o, true, bias_value[k]);
    }
  }
  if (p.bias_ld && p.path) __syncthreads();   // (a token that has a bias too is marked with that)
  if (p.path) {
#pragma unroll
    for (int k = 0; k < kMaxNodes / kThreads; k++) {
      const int u = tid + k * kThreads, o = u < p.T ? place(draft[k]) : -1;
      if (o >= 0) {
        node_s[atomicAdd(&n_node_s, 1)] = u << 16 | o;
        mark(o, false, -0.0f);   // (adds nothing, not even to a zero's sign)
      }
    }
  }
  __syncthreads();
  const int marked = n_marked_s, nodes = n_node_s;
  for (int i = tid; i < marked; i += kThreads) {   // several biases of a token: their sum, in the list's order
    const int o = marked_s[i];
    if (!(word_s[o] & kAgain)) continue;
    float y = 0.0f;
    bool any = false;
    for (int j = 0; j < m; j++)
      if (bias_at_s[j] == o) {
        y = any ? __fadd_rn(y, bias_s[j]) : bias_s[j];
        any = true;
      }
    sum_s[i] = y;
  }
  if (said) {   // the others that are named: a warp's in one piece
    for (int q0 = warp * 32; q0 < p.slice / 4; q0 += kThreads) {
      const int q = q0 + lane;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (q < p.slice / 4) w = reinterpret_cast<const uint4*>(word_s)[q];
      auto here = [](uint32_t u) { return u != 0 && !(u & kMarked); };
      const int n = here(w.x) + here(w.y) + here(w.z) + here(w.w);
      if (!__any_sync(0xffffffffu, n)) continue;
      int upto = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += y;
      }
      int at = 0;
      if (lane == 31) at = atomicAdd(&n_listed_s, upto);
      at = __shfl_sync(0xffffffffu, at, 31) + upto - n;
      if (here(w.x)) listed_s[at++] = (uint16_t)(4 * q);
      if (here(w.y)) listed_s[at++] = (uint16_t)(4 * q + 1);
      if (here(w.z)) listed_s[at++] = (uint16_t)(4 * q + 2);
      if (here(w.w)) listed_s[at++] = (uint16_t)(4 * q + 3);
    }
  }
  __syncthreads();

  // (named token, row) pairs, tokens first: kUnits of a thread on the way at once
  const int n_listed = n_listed_s, pairs = n_listed * rows;
  const size_t next = (size_t)p.B * p.ld;   // floats from a row to the request's next
  float* const x0 = p.logits + ((size_t)t0 * p.B + b) * p.ld;
  auto hidden = [&](int t, int token) {
    const int id = mask_s[t];
    return id >= 0 && !(__ldg(p.allowed + (size_t)id * p.allowed_words + (token >> 5)) >> (token & 31) & 1u);
  };
  for (int it0 = tid; it0 < pairs; it0 += kThreads * kUnits) {
    float* at[kUnits];
    float x[kUnits], sub[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
      const int it = it0 + k * kThreads;
      at[k] = nullptr;
      if (it >= pairs) continue;
      const int t = it / n_listed, o = listed_s[it - t * n_listed], token = token_of(o);
      if (hidden(t, token)) continue;
      at[k] = x0 + t * next + token;
      x[k] = __ldcg(at[k]);
      sub[k] = taken(word_s[o] & kSaid, a);
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++)
      if (at[k]) *at[k] = adjusted(x[k], sub[k], a);
  }
  for (int it = tid; it < marked * rows; it += kThreads) {
    const int t = it / marked, i = it - t * marked, o = marked_s[i], token = token_of(o);
    if (hidden(t, token)) continue;
    const size_t row = (size_t)(t0 + t) * p.B + b;
    const uint32_t w = word_s[o];
    uint32_t said_here = w & kSaid;
    for (int j = 0; j < nodes; j++) {
      const int u = node_s[j] >> 16;
      if ((node_s[j] & 0xffff) == o) said_here += __ldg(p.path + row * p.path_words + (u >> 5)) >> (u & 31) & 1u;
    }
    const bool penalised = said_here || w & kInPrompt;
    if (!penalised && __float_as_uint(sum_s[i]) == 0x80000000u) continue;   // (drafted elsewhere in the tree)
    float* x = x0 + t * next + token;
    float y = __ldcg(x);
    if (penalised) y = adjusted(y, taken(said_here, a), a);
    *x = __fadd_rn(y, sum_s[i]);
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
  BK_ARG(!a.history || (a.hist_len && a.history_ld > 0 && a.history_ld <= kMaxHistory), "bkAdjustLogits: history needs hist_len and history_ld (%d; 1 to 2^28)", a.history_ld);
  BK_ARG((a.path != 0) == (a.draft != 0) && (!a.path || a.path_words >= (a.T + 31) / 32), "bkAdjustLogits: draft and path go together, path_words=%d for %d nodes", a.path_words, a.T);
  BK_ARG((a.bias_token != 0) == (a.bias_value != 0) && (a.bias_token != 0) == (a.bias_n != 0) && (!a.bias_token || (a.bias_ld > 0 && a.bias_ld <= BK_LOGITS_MAX_BIAS)),
         "bkAdjustLogits: bias_token, bias_value and bias_n go together, bias_ld=%d (1 to %d)", a.bias_ld, BK_LOGITS_MAX_BIAS);
  BK_ARG((a.allowed != 0) == (a.mask_id != 0) && (!a.allowed || (a.n_masks > 0 && a.allowed_words >= (a.V + 31) / 32)),
         "bkAdjustLogits: allowed and mask_id go together, n_masks=%d allowed_words=%d for %d tokens", a.n_masks, a.allowed_words, a.V);
  LogitsParams p = {bk_ptr<float>(a.logits), bk_ptr<int>(a.seqs), bk_ptr<int>(a.history), bk_ptr<int>(a.hist_len), bk_ptr<int>(a.prompt_len), bk_ptr<float>(a.repetition),
                    bk_ptr<float>(a.presence), bk_ptr<float>(a.frequency), bk_ptr<int>(a.draft), bk_ptr<uint32_t>(a.path), bk_ptr<int>(a.bias_token), bk_ptr<float>(a.bias_value),
                    bk_ptr<int>(a.bias_n), bk_ptr<uint32_t>(a.allowed), bk_ptr<int>(a.mask_id), a.B, a.T, a.V, a.n_seqs ? a.n_seqs : a.B, a.history_ld, a.bias_ld, a.path_words,
                    a.n_masks, a.allowed_words, 0, 0, 0, 0, 0, 0, a.ld ? a.ld : a.V};
  if (!a.bias_token) p.bias_ld = 0;
  // (Figures: 151,936 logits, 148 SMs.)  Who names: slices of at most 8,192 words (48 KB with the list; 512 rows behind 16,000 tokens 111 us, with half as many words 116, with twice as many
  // 112; 4 requests, 10 rows, 9,000 tokens 11.7, 11.3 and 14.2), shorter while that leaves SMs without a CTA, to 1,024; then rows apart, until each SM has two (one request of 100 rows behind
  // 30,000 tokens 35 us, none apart 74; 512 rows, which are not taken apart so, 111, until each SM has four 116), but no fewer rows than half the slices, each of which counts the whole history (4 requests,
  // 10 rows, 9,000 tokens, 32 slices: 11.7 us with ten rows a CTA, 14.6 with four; 100 rows behind 30,000 34.7 and 41.5; against it one request of 32 rows behind 16,000, 15.9 and 12.6).
  // Where such a slice has more than 4,096 words and the request's tokens fit a table, fewer CTAs with a table each (64 requests, 5,000 tokens: 15.4 us with four tables, 46 with slices of
  // words; against it 4 requests, 10 rows, 6,000 tokens, 12.4 and 9.0; below 4,096 words 4 requests, 2,000 tokens: 4.8 us with slices of 2,560 words, 5.7 with tables).  A request's tokens are
  // what its arrays hold (history_ld, bias_ld, T): its lengths are on the device.
  // Who hides: four CTAs an SM, no more than have 4,096 tokens each.
  const long long sms = bk_ctx().sm_count;
  const int blocks = (a.V + kBlock - 1) / kBlock;
  const long long names = (a.history ? a.history_ld : 0) + p.bias_ld + (a.path ? a.T : 0);
  int table = 512;
  while (table <= kMaxTable && 3ll * table < 4 * names) table *= 2;
  auto slice_of = [&](int shift) { return ((blocks + (1 << shift) - 1) >> shift) * kBlock; };
  while (slice_of(p.shift) > kMaxSlice || (slice_of(p.shift) > 1024 && ((long long)a.B * a.T << p.shift) < sms)) p.shift++;
  p.slice = slice_of(p.shift);
  const bool use_table = table <= kMaxTable && p.slice > 4096;
  if (use_table) {
    p.slice = table;
    while (p.shift > 0 && ((long long)a.B * a.T << (p.shift - 1)) >= sms) p.shift--;
  }
  const long long ctas = (long long)a.B << p.shift;
  p.parts = (int)std::max<long long>(1, std::min<long long>(std::min<long long>(a.T, (2 * sms + ctas - 1) / ctas), 2ll * a.T >> p.shift));
  p.rows = (a.T + p.parts - 1) / p.parts;
  if (a.allowed) p.hiding = (int)std::max<long long>(1, std::min<long long>(4 * sms, (long long)a.T * a.B * a.V / 4096));
  BK_ARG(ctas * p.parts + p.hiding < (1ll << 31), "bkAdjustLogits: B=%d rows of %d logits: too much for one call", a.B, a.V);
  if (a.history || a.bias_token || a.path) p.naming = (int)ctas * p.parts;
  if (p.naming + p.hiding == 0) return BK_OK;
  const size_t marks = (size_t)p.bias_ld + (a.path ? a.T : 0), smem = (size_t)p.slice * (use_table ? 10 : 6) + (size_t)p.bias_ld * 6 + marks * 6 + 4;   // at most 80 + 6 + 12 KB
  auto* kernel = use_table ? adjust_logits_kernel<true> : adjust_logits_kernel<false>;
  static bool configured[2] = {false, false};
  if (!configured[use_table]) {
    BK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 116 << 10));
    configured[use_table] = true;
  }
  BK_CUDA(bk_launch_pdl(kernel, dim3(p.naming + p.hiding), dim3(kThreads), smem, p));
  BK_CHECK_LAUNCH();
  return BK_OK;
}
