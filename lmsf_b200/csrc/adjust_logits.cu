// What sampling asks of the logits before it draws, in one pass: penalties for tokens that occur already, biases of single
// tokens and masks of what a grammar allows.  The tokens that occur are counted here, from the requests' token histories and, where
// a row is a node of a drafted tree, from the tokens on the path to it.
// Counterpart in the reference: the penalties of core/src/model_executor/layers/sampler.rs:48-137 (order and formulas:
// repetition, frequency, presence); biases and masks have none.
#include <type_traits>

#include "common.cuh"

LMSF_DEFINE_LAST_ERROR(lmsf_adjust_logits)

namespace lmsf {

constexpr int kErrOptions = 5;             // value of the error word
constexpr int kChunk = 2048;               // values of a row that a block takes
constexpr int kThreads = 256, kPer = kChunk / kThreads;
constexpr int kMaxNodes = 256;             // nodes of a drafted tree
constexpr int kEntries = 2 * kThreads;     // biases that are looked at at once, two a thread
// A value's word: how often its token occurs in the output, and whether it occurs in the prompt, is on a node of the tree, has a bias.
constexpr unsigned kInPrompt = 0x80000000u, kOnTree = 0x40000000u, kHasBias = 0x20000000u, kCount = kHasBias - 1;

struct AdjustArgs {
  float* out; long long out_stride;
  const float* logits; long long stride;
  int n_rows, vocab;
  const int* row_req; int n_reqs;                                // null: row r is request r; -1: no option is a request's
  const int* history; long long history_stride; int history_width;   // [n_reqs, width]
  const int* history_len; const int* prompt_len;
  const float* presence; const float* frequency; const float* repetition;
  const int* tree_tokens; const unsigned* tree_mask; const int* cu_q; int words;
  const int* bias_start; const int* bias_token; const float* bias_value; int n_bias;
  const unsigned* allowed; const int* allowed_row; int n_allowed, allowed_words;
  int* error_flag;
};

// A block takes kChunk values of up to `rows_block` rows in turn.  Few of a row's values have anything to do with its request: those that occur in the
// history, in the tree or in the list of biases; they are marked when a row's request is another than the row's before, so the nodes of a tree share
// one pass over their request's history.  A row's values come into shared memory by copies of their own (cp.async, the next row's while this one
// is worked on; not at all where a grammar hides four neighbours); every thread changes the marked ones among those that it brought, without a barrier, and
// all leave, with -inf for those that are not allowed.  Bound by memory: 8 bytes a value, 4 of them less where they are hidden.
// (With the counts of every value looked at in every row, more than half of the issue slots went to some 34 instructions a value, most of them for divisions
// that one lane of a warp had asked for: 89 us; with the marked ones on a list of the block's, between two barriers, 85.)  Measured: 16 requests with 17 to 32 nodes, 128,256 values, a mask each
// row: 81 us, 397 MB at 4.9 TB/s; 8 single rows 7.1 us, of which the launch and the chain of lengths, history, values and stores are nearly all.  Chunks of 1,024
// values took 116 us, of 4,096 (three blocks an SM) 84.
template <bool kWide>
__global__ void __launch_bounds__(kThreads, 5) adjust_logits_kernel(AdjustArgs a, int rows_block) {
  __shared__ __align__(16) float xs[2][kChunk];
  __shared__ __align__(16) unsigned seen[kChunk];
  __shared__ float bias[kChunk];           // where kHasBias says so
  __shared__ unsigned path[kMaxNodes];     // the tree's nodes whose token is one of the chunk's: node << 16 | value
  __shared__ unsigned on_row[kThreads / 32][kMaxNodes / 32];      // a row's mask of the tree, a copy for every warp
  __shared__ int n_path;
  __shared__ unsigned entry_at[kEntries];  // of so many entries of the list of biases those of the chunk's tokens, in the list's order
  __shared__ float entry_value[kEntries];
  __shared__ int entries_of[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v0 = blockIdx.x * kChunk, width = min(kChunk, a.vocab - v0);
  const int row0 = blockIdx.y * rows_block, row1 = min(row0 + rows_block, a.n_rows);
  // this thread's k-th value; wide: four neighbours at a time
  auto place = [&](int k) { return kWide ? 4 * (tid + kThreads * (k >> 2)) + (k & 3) : tid + kThreads * k; };
  const bool whole = width == kChunk;      // no place of the chunk is behind the vocabulary's end: nothing to look at in the loops over a row
  // Which of this thread's values mask `which` allows.
  auto allowed = [&](int which) {
    if (which < 0 || which >= a.n_allowed) return 0xffffu;
    const unsigned* words = a.allowed + (size_t)which * a.allowed_words + (v0 + place(0)) / 32;
    const int shift = place(0) & 31;       // (v0 and the distances between a thread's places are multiples of 32)
    unsigned ok = 0u;
#pragma unroll
    for (int k = 0; k < kPer; k += kWide ? 4 : 1)
      if (whole || place(k) < width) ok |= ((words[(place(k) - place(0)) / 32] >> shift) & (kWide ? 15u : 1u)) << k;
    return ok;
  };
  auto copy = [&](float* dst, const float* src, auto bytes) {
    if constexpr (decltype(bytes)::value == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
  };
  using Four = std::integral_constant<int, 4>;
  using Sixteen = std::integral_constant<int, 16>;
  // This thread's values of a row, those that are hidden left out.
  auto request = [&](int r, unsigned ok, float* x) {
    const float* x_row = a.logits + r * a.stride + v0;
#pragma unroll
    for (int k = 0; k < kPer; k += kWide ? 4 : 1) {
      const int i = place(k);
      if (!((ok >> k) & (kWide ? 15u : 1u))) continue;
      if constexpr (kWide) {
        if (whole || i + 4 <= width) {
          copy(x + i, x_row + i, Sixteen{});
        } else {
          for (int e = i; e < width; ++e) copy(x + e, x_row + e, Four{});
        }
      } else if (whole || i < width) {
        copy(x + i, x_row + i, Four{});
      }
    }
  };
  auto sent = [&]() { asm volatile("cp.async.commit_group;" ::: "memory"); };
  auto request_of = [&](int r) { return a.row_req ? a.row_req[r] : r; };
  auto mask_of = [&](int r) { return a.allowed_row ? a.allowed_row[r] : -1; };
  int current = -1;                        // the request that seen, bias and path are of
  unsigned touched = 0u;                   // which of this thread's values it has anything to do with
  float rep = 1.f, freq = 0.f, pres = 0.f;
  int req = request_of(row0), which = mask_of(row0);
  unsigned ok = allowed(which);
  request(row0, ok, xs[0]);
  sent();
  for (int r = row0; r < row1; ++r) {
    float* x = xs[(r - row0) & 1];
    const bool known = req >= 0 && req < a.n_reqs, fresh = known && req != current;
    if (((!known && a.n_reqs >= 0) || (a.allowed_row && which >= a.n_allowed)) && tid == 0 && blockIdx.x == 0 && a.error_flag) atomicExch(a.error_flag, kErrOptions);
    const bool penalties = known && a.repetition, biases = known && a.bias_start;
    int next_req = -1, next_which = -1;
    if (r + 1 < row1) {
      next_req = request_of(r + 1);
      next_which = mask_of(r + 1);
    }
    if (fresh) {
      if (current >= 0) __syncthreads();                         // the rows before are done with what is there
      int n_history = 0, n_prompt = 0, first = 0, nodes = 0, b0 = 0, b1 = 0;
      if (a.history) {
        n_history = min(max(a.history_len[req], 0), a.history_width);
        n_prompt = a.prompt_len[req];
      }
      if (penalties) {
        rep = a.repetition[req];
        freq = a.frequency[req];
        pres = a.presence[req];
      }
      if (a.tree_tokens) {
        first = min(max(a.cu_q[req], 0), a.n_rows);
        nodes = min(min(a.cu_q[req + 1], a.n_rows) - first, 32 * a.words);
      }
      if (biases) {
        b0 = min(max(a.bias_start[req], 0), a.n_bias);
        b1 = min(a.bias_start[req + 1], a.n_bias);
      }
      current = req;
      for (int i = tid; i < kChunk / 4; i += kThreads) reinterpret_cast<uint4*>(seen)[i] = make_uint4(0u, 0u, 0u, 0u);
      if (tid == 0) n_path = 0;
      __syncthreads();
      unsigned at[2];
      float value[2];
      auto entries = [&](int base) {                             // this thread's two of them
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int e = base + 2 * tid + k;
          at[k] = e < b1 ? (unsigned)(a.bias_token[e] - v0) : 0xffffffffu;
          value[k] = e < b1 ? a.bias_value[e] : 0.f;
        }
      };
      entries(b0);
      if (penalties) {
        const int* h = a.history + req * a.history_stride;
        for (int i0 = tid; i0 < n_history; i0 += 8 * kThreads) {
          int t[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) t[k] = i0 + k * kThreads < n_history ? h[i0 + k * kThreads] : -1;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const unsigned i = (unsigned)(t[k] - v0);
            if (i0 + k * kThreads < n_history && i < (unsigned)width) {
              if (i0 + k * kThreads < n_prompt) atomicOr(&seen[i], kInPrompt);
              else atomicAdd(&seen[i], 1u);
            }
          }
        }
        for (int j = tid; j < nodes; j += kThreads) {
          const unsigned i = (unsigned)(a.tree_tokens[first + j] - v0);
          if (i < (unsigned)width) {
            path[atomicAdd(&n_path, 1)] = ((unsigned)j << 16) | i;
            atomicOr(&seen[i], kOnTree);
          }
        }
      }
      // In the order of the list, so that a token that is listed twice gets the same sum in every run: the first entry of those that name
      // one token adds theirs up.
      for (int base = b0; base < b1; base += kEntries) {
        const bool mine0 = at[0] < (unsigned)width, mine1 = at[1] < (unsigned)width;
        const unsigned has0 = __ballot_sync(0xffffffffu, mine0), has1 = __ballot_sync(0xffffffffu, mine1), below = (1u << lane) - 1u;
        if (lane == 0) entries_of[warp] = __popc(has0) + __popc(has1);
        __syncthreads();
        int n = 0, to = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
          if (w == warp) to = n;
          n += entries_of[w];
        }
        to += __popc(has0 & below) + __popc(has1 & below);
        if (mine0) {
          entry_at[to] = at[0];
          entry_value[to] = value[0];
        }
        if (mine1) {
          entry_at[to + mine0] = at[1];
          entry_value[to + mine0] = value[1];
        }
        if (base + kEntries < b1) entries(base + kEntries);
        __syncthreads();
        for (int e = tid; e < n; e += kThreads) {
          const unsigned i = entry_at[e];
          bool is_first = true;
          for (int o = 0; o < e; ++o) is_first &= entry_at[o] != i;
          if (!is_first) continue;
          const unsigned before = atomicOr(&seen[i], kHasBias);
          float sum = before & kHasBias ? bias[i] : 0.f;
          for (int o = e; o < n; ++o)
            if (entry_at[o] == i) sum += entry_value[o];
          bias[i] = sum;
        }
      }
      __syncthreads();
      touched = 0u;
#pragma unroll
      for (int k = 0; k < kPer; ++k) touched |= (place(k) < width && seen[place(k)] ? 1u : 0u) << k;
    }
    const unsigned next_ok = r + 1 < row1 ? allowed(next_which) : 0u;
    if (r + 1 < row1) request(r + 1, next_ok, xs[(r + 1 - row0) & 1]);
    sent();
    const int on_path = penalties && a.tree_tokens ? n_path : 0;
    if (on_path > 0) {
      if (lane < a.words) on_row[warp][lane] = a.tree_mask[(size_t)r * a.words + lane];
      __syncwarp();
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");         // (a thread works on values that it brought itself)
    if (penalties || biases) {
      for (unsigned left = touched & ok; left; left &= left - 1) {
        const int i = place(__ffs((int)left) - 1);
        const unsigned word = seen[i];
        unsigned said = word & kCount;
        if (word & kOnTree)
          for (int e = 0; e < on_path; ++e) {
            const unsigned node = path[e] >> 16;
            if ((path[e] & 0xffffu) == i) said += (on_row[warp][node >> 5] >> (node & 31)) & 1u;
          }
        float y = x[i];
        if (penalties && (said | (word & kInPrompt))) {
          y = y > 0.f ? y / rep : y * rep;
          y -= freq * (float)said;
          if (said) y -= pres;
        }
        if (word & kHasBias) y += bias[i];
        x[i] = y;
      }
      __syncwarp();
    }
    float* out_row = a.out + r * a.out_stride + v0;
#pragma unroll
    for (int k = 0; k < kPer; k += kWide ? 4 : 1) {
      const int i = place(k);
      if (!whole && i >= width) continue;
      if constexpr (kWide) {               // (x is whole, also behind the vocabulary's end)
        const float4 f = *reinterpret_cast<const float4*>(x + i);
        float y[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((ok >> (k + e)) & 1u)) y[e] = -INFINITY;
        if (whole || i + 4 <= width) {
          *reinterpret_cast<float4*>(out_row + i) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (i + e < width) out_row[i + e] = y[e];
        }
      } else {
        out_row[i] = (ok >> k) & 1u ? x[i] : -INFINITY;
      }
    }
    req = next_req;
    which = next_which;
    ok = next_ok;
  }
}

}  // namespace lmsf

// logits, out: float32 [n_rows, vocab] (the same memory, or apart).  Every option may be null; n_reqs -1: there are neither penalties nor biases.
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
  if (history_width > (1 << 28)) LMSF_REFUSE("adjust_logits: a history of %d tokens is more than its counts hold", history_width);
  if (tree_tokens && (words < 1 || words > kMaxNodes / 32)) LMSF_REFUSE("adjust_logits: a tree's mask has 1 to %d words a row, not %d", kMaxNodes / 32, words);
  AdjustArgs a{out, out_stride, logits, stride, n_rows, vocab, row_req, n_reqs, history, history_stride, history_width, history_len,
               prompt_len, presence, frequency, repetition, tree_tokens, tree_mask, cu_q, words, bias_start, bias_token, bias_value, n_bias,
               allowed, allowed_row, n_allowed, allowed_words, error_flag};
  // Rows of a block: one, where rows are few; more, where that leaves 16 blocks and more for each of 148 SMs, so that the rows of a request
  // share its list.  (16 requests with 17 to 32 nodes over 128,256 values: 102 us with 4 blocks and more, 87 with 8, 81 with 16, 86 with 32.)
  const int chunks = ceil_div(vocab, kChunk);
  const long long blocks = (long long)chunks * n_rows;
  int rows_block = 1;
  while (rows_block < 32 && blocks / (2 * rows_block) >= 148 * 16) rows_block *= 2;
  while (ceil_div(n_rows, rows_block) > 65535) rows_block *= 2;
  const bool wide = ((unsigned long long)out | (unsigned long long)logits) % 16 == 0 && (n_rows == 1 || (out_stride | stride) % 4 == 0);
  const dim3 grid(chunks, ceil_div(n_rows, rows_block));
  if (wide) return launch_pdl(adjust_logits_kernel<true>, grid, dim3(kThreads), 0, (cudaStream_t)stream, a, rows_block);
  return launch_pdl(adjust_logits_kernel<false>, grid, dim3(kThreads), 0, (cudaStream_t)stream, a, rows_block);
}
