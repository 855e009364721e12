// What sampling asks of the logits before it draws, in one pass: penalties for tokens that occur already, biases of single
// tokens and masks of what a grammar allows.  The tokens that occur are counted here, from the requests' token histories and, where
// a row is a node of a drafted tree, from the tokens on the path to it.
// Counterpart in the reference: the penalties of core/src/model_executor/layers/sampler.rs:48-137 (order and formulas:
// repetition, frequency, presence); biases and masks have none.
#include "common.cuh"

LMSF_DEFINE_LAST_ERROR(lmsf_adjust_logits)

namespace lmsf {

constexpr int kErrOptions = 5;             // value of the error word
constexpr int kChunk = 4096;               // values of a row that a block takes
constexpr int kThreads = 256;
constexpr unsigned kInPrompt = 0x80000000u;

struct AdjustArgs {
  float* out; long long out_stride;
  const float* logits; long long stride;
  int n_rows, vocab;
  const int* row_req; int n_reqs;                                // null: row r is request r
  const int* history; long long history_stride; int history_width;   // [n_reqs, width]
  const int* history_len; const int* prompt_len;
  const float* presence; const float* frequency; const float* repetition;
  const int* tree_tokens; const unsigned* tree_mask; const int* cu_q; int words;
  const int* bias_start; const int* bias_token; const float* bias_value; int n_bias;
  const unsigned* allowed; const int* allowed_row; int n_allowed, allowed_words;
  int* error_flag;
};

__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(AdjustArgs a) {
  __shared__ unsigned seen[kChunk];        // how often a token occurs in the output; the top bit: it occurs in the prompt
  __shared__ float bias[kChunk];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int v0 = blockIdx.x * kChunk, width = min(kChunk, a.vocab - v0);
  int req = a.row_req ? a.row_req[r] : r;
  const bool known = req >= 0 && req < a.n_reqs;
  if (!known && a.n_reqs > 0 && tid == 0 && blockIdx.x == 0 && a.error_flag) atomicExch(a.error_flag, kErrOptions);
  const bool penalties = known && a.repetition, biases = known && a.bias_start;
  if (penalties) for (int i = tid; i < kChunk; i += kThreads) seen[i] = 0u;
  if (biases) for (int i = tid; i < kChunk; i += kThreads) bias[i] = 0.f;
  __syncthreads();
  auto note = [&](int token, bool prompt) {
    const unsigned i = (unsigned)(token - v0);
    if (i < (unsigned)width) {
      if (prompt) atomicOr(&seen[i], kInPrompt);
      else atomicAdd(&seen[i], 1u);
    }
  };
  if (penalties) {
    if (a.history) {
      const int* h = a.history + req * a.history_stride;
      const int n = min(max(a.history_len[req], 0), a.history_width), p = a.prompt_len[req];
      for (int i = tid; i < n; i += kThreads) note(h[i], i < p);
    }
    if (a.tree_tokens) {
      const int first = min(max(a.cu_q[req], 0), a.n_rows), nodes = min(a.cu_q[req + 1], a.n_rows) - first;
      for (int i = tid; i < min(nodes, 32 * a.words); i += kThreads)
        if ((a.tree_mask[(size_t)r * a.words + (i >> 5)] >> (i & 31)) & 1u) note(a.tree_tokens[first + i], false);
    }
  }
  if (biases && tid < 32) {
    // In the order of the list, so that a token that is listed twice gets the same sum in every run: one warp, 32 entries
    // at a time, the first lane of those that name one token adds theirs up.
    const int b0 = min(max(a.bias_start[req], 0), a.n_bias), b1 = min(a.bias_start[req + 1], a.n_bias);
    for (int base = b0; base < b1; base += 32) {
      const int e = base + lane;
      const unsigned i = e < b1 ? (unsigned)(a.bias_token[e] - v0) : 0xffffffffu;
      const float value = e < b1 ? a.bias_value[e] : 0.f;
      const bool mine = i < (unsigned)width;
      const unsigned same = __match_any_sync(0xffffffffu, mine ? i : 0xffffffffu);
      if (mine && (same & ((1u << lane) - 1u)) == 0u) bias[i] += value;
      unsigned later = mine && (same & ((1u << lane) - 1u)) == 0u ? same & ~(1u << lane) : 0u;
      if (__any_sync(0xffffffffu, later != 0u)) {
        for (int k = 1; k < 32; ++k) {
          const float other = __shfl_sync(0xffffffffu, value, k);
          if ((later >> k) & 1u) bias[i] += other;
        }
      }
      __syncwarp();
    }
  }
  __syncthreads();
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (penalties) {
    rep = a.repetition[req];
    freq = a.frequency[req];
    pres = a.presence[req];
  }
  const unsigned* allow = nullptr;
  if (a.allowed) {
    const int m = a.allowed_row ? a.allowed_row[r] : r;
    if (m >= a.n_allowed) {
      if (tid == 0 && blockIdx.x == 0 && a.error_flag) atomicExch(a.error_flag, kErrOptions);
    } else if (m >= 0) {
      allow = a.allowed + (size_t)m * a.allowed_words;
    }
  }
  const float* x_row = a.logits + r * a.stride + v0;
  float* out_row = a.out + r * a.out_stride + v0;
  auto one = [&](int i, float x, bool ok) {
    if (penalties) {
      const unsigned c = seen[i];
      if (c) {
        x = x > 0.f ? x / rep : x * rep;
        const unsigned said = c & ~kInPrompt;
        x -= freq * (float)said;
        if (said) x -= pres;
      }
    }
    if (biases) x += bias[i];
    return ok ? x : -INFINITY;
  };
  for (int i = tid; i < width; i += kThreads) {
    const bool ok = !allow || ((allow[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u);
    out_row[i] = one(i, x_row[i], ok);
  }
}

}  // namespace lmsf

// logits, out: float32 [n_rows, vocab] (the same memory, or apart).  Every option may be null.
LMSF_API int lmsf_adjust_logits(float* out, long long out_stride, const float* logits, long long stride, int n_rows, int vocab,
                                const int* row_req, int n_reqs, const int* history, long long history_stride, int history_width,
                                const int* history_len, const int* prompt_len, const float* presence, const float* frequency,
                                const float* repetition, const int* tree_tokens, const unsigned* tree_mask, const int* cu_q, int words,
                                const int* bias_start, const int* bias_token, const float* bias_value, int n_bias,
                                const unsigned* allowed, const int* allowed_row, int n_allowed, int allowed_words, int* error_flag,
                                void* stream) {
  using namespace lmsf;
  if (n_rows <= 0) return 0;
  if (vocab <= 0 || stride < vocab || out_stride < vocab) LMSF_REFUSE("adjust_logits: vocab=%d, strides %lld and %lld", vocab, stride, out_stride);
  if (n_rows > 65535) LMSF_REFUSE("adjust_logits: %d rows are more than one launch takes (65535)", n_rows);
  AdjustArgs a{out, out_stride, logits, stride, n_rows, vocab, row_req, n_reqs, history, history_stride, history_width, history_len,
               prompt_len, presence, frequency, repetition, tree_tokens, tree_mask, cu_q, words, bias_start, bias_token, bias_value, n_bias,
               allowed, allowed_row, n_allowed, allowed_words, error_flag};
  return launch_pdl(adjust_logits_kernel, dim3(ceil_div(vocab, kChunk), n_rows), dim3(kThreads), 0, (cudaStream_t)stream, a);
}
