// Steps that check trees of drafted tokens: their layout, made on the device from the requests' lengths and the nodes' parents,
// and the acceptance of a path of drafted tokens with its keys and values.  (The reference decodes one token a step; these
// have no counterpart in it.)
//
// A tree's nodes are numbered so that a parent comes before its children.  Node 0 of a request is the token that was sampled
// last (its keys are not cached yet); a node whose parent is -1 follows the request's cached tokens.
//
// Measured: the layout of a tree of 8 nodes 2.3 us and of 64 trees of 1..64 nodes 3.1 us, launches and three dependent loads; acceptance of a tree of 8 with its keys
// and values in 16 layers of 8 heads of 64 2.9 us, of 64 trees of 33..64 in 32 layers of 8 heads of 128 15 us: 67 MB at 4.5 TB/s.
#include "common.cuh"

LMSF_DEFINE_LAST_ERROR(lmsf_tree)

namespace lmsf {

constexpr int kMaxNodes = 256;             // nodes of one tree: one thread each, their ancestors as eight words
constexpr int kMaxWords = kMaxNodes / 32;
constexpr int kErrNoPage = 2, kErrTree = 5;    // values of the error word

__device__ __forceinline__ void report(int* error_flag, int code) {
  if (error_flag) atomicExch(error_flag, code);
}

struct LayoutArgs {
  int* cu_q; int* token_seq; int* positions; long long* slots; unsigned* mask;      // mask may be null
  const int* parents;                      // null: every node follows the one before it (an ordinary portion)
  const int* tree_len; const int* prefix_len;
  const int* block_table; int max_blocks, block_size;
  int n_seqs, n_rows, words, window;
  int* error_flag;
};

// Nodes of request s that the step has room for in its mask.
__device__ __forceinline__ int nodes_of(const LayoutArgs& a, int s) {
  const int limit = a.mask ? a.words * 32 : (a.parents ? kMaxNodes : 0x7fffffff);
  return min(max(a.tree_len[s], 0), limit);
}

// One block per request.  Every block adds up the lengths before its own (a few kilobytes that lie in L2), so that the whole
// layout is one launch: the time is the launch and three dependent loads, at any size that a step has.  A node's ancestors are
// found by doubling: round k joins to every node's set that of its ancestor 2^k levels up, so a chain of 64 nodes takes
// six rounds where a walk to the root would take 63 dependent loads.
__global__ void __launch_bounds__(kMaxNodes) tree_layout_kernel(LayoutArgs a) {
  __shared__ long long sums[8];
  __shared__ unsigned sets[kMaxNodes][kMaxWords + 1];            // + 1: rows start in different banks
  __shared__ short up[kMaxNodes];
  __shared__ short depths[kMaxNodes];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, tid = threadIdx.x;
  if (s >= a.n_seqs) {                                           // a step of no requests: one block, for cu_q[0]
    if (tid == 0) a.cu_q[0] = 0;
    return;
  }
  long long before = 0;
  for (int j = tid; j < s; j += blockDim.x) before += nodes_of(a, j);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((tid & 31) == 0) sums[tid >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += sums[w];
  const int start = (int)min(before, (long long)a.n_rows);
  const int want = nodes_of(a, s), n = min(want, a.n_rows - start);
  const int prefix = min(max(a.prefix_len[s], 0), 0x7fffffff - n);     // (no place or position of the request passes 32 bits)
  if (tid == 0) {
    if (s == 0) a.cu_q[0] = 0;
    a.cu_q[s + 1] = start + n;
    if (n != a.tree_len[s] || prefix != a.prefix_len[s]) report(a.error_flag, kErrTree);
  }
  const int* table = a.block_table + (size_t)s * a.max_blocks;
  auto slot_of = [&](int place) -> long long {
    const int blk = place / a.block_size;
    const int page = blk < a.max_blocks ? table[blk] : -1;
    return page < 0 ? -1ll : (long long)page * a.block_size + place % a.block_size;
  };
  if (!a.parents) {                                              // a chain: no sets to find, any length
    for (int i = tid; i < n; i += blockDim.x) {
      const int row = start + i;
      a.token_seq[row] = s;
      a.positions[row] = prefix + i;
      a.slots[row] = slot_of(prefix + i);
      if (a.mask) {
        const int first = a.window > 0 ? max(0, i - a.window + 1) : 0;       // the nodes first .. i are seen
        for (int w = 0; w < a.words; ++w) {
          const int lo = min(max(first - 32 * w, 0), 32), hi = min(max(i + 1 - 32 * w, 0), 32);
          const unsigned upto = hi >= 32 ? 0xffffffffu : (1u << hi) - 1u, below = lo >= 32 ? 0xffffffffu : (1u << lo) - 1u;
          a.mask[(size_t)row * a.words + w] = upto & ~below;
        }
      }
    }
    return;
  }
  const bool mine = tid < n;
  unsigned set[kMaxWords];
  int anc = -1;
#pragma unroll
  for (int w = 0; w < kMaxWords; ++w) set[w] = mine && (tid >> 5) == w ? 1u << (tid & 31) : 0u;
  if (mine) {
    anc = a.parents[start + tid];
    if (anc < -1 || anc >= tid) {                                // no tree: the node stands alone
      report(a.error_flag, kErrTree);
      anc = -1;
    }
  }
  while (true) {
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w) sets[tid][w] = set[w];
    up[tid] = (short)anc;
    if (!__syncthreads_or(anc >= 0)) break;
    if (anc >= 0) {
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w) set[w] |= sets[anc][w];
      anc = up[anc];
    }
    __syncthreads();
  }
  int depth = -1;
#pragma unroll
  for (int w = 0; w < kMaxWords; ++w) depth += __popc(set[w]);
  if (a.window > 0) {                                            // ancestors `window` levels up and more are out of sight
    depths[tid] = (short)depth;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w) {
      unsigned left = set[w];
      while (left) {
        const int j = __ffs(left) - 1;
        left &= left - 1;
        if (depths[32 * w + j] <= depth - a.window) set[w] &= ~(1u << j);
      }
    }
  }
  if (!mine) return;
  const int row = start + tid;
  a.token_seq[row] = s;
  a.positions[row] = prefix + depth;
  a.slots[row] = slot_of(prefix + tid);
  if (a.mask) {
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w)
      if (w < a.words) a.mask[(size_t)row * a.words + w] = set[w];
  }
}

struct AcceptArgs {
  int* n_kept; int* path; int* next_token; int* new_len;
  const int* target; const int* tokens; const int* parents; const int* cu_q; const int* prefix_len;
  int n_seqs, n_rows, max_path;
  const long long* slots;                                        // null: nothing is written to a cache
  const char* k; const char* v;                                  // [calls][rows][kv heads x head size]
  long long k_call, k_row, v_call, v_row;                        // their strides in bytes
  char* cache;                                                   // [calls][pages][2][kv head][slot][head size]
  int calls, pages, n_kv_heads, block_size, head_bytes;
  int* error_flag;
};

// grid (shares of the copy, requests).  Every block walks its request's tree (a warp with eight nodes a lane; a level
// is a comparison and a minimum over the warp), then the blocks of a request share the copy of the kept rows out among them:
// what would be a second launch, with the path read back from memory, costs each block the walk.
// Vec: the widest word in which all rows can be moved.
template <typename Vec>
__global__ void __launch_bounds__(256) tree_accept_kernel(AcceptArgs a) {
  __shared__ int chosen[kMaxNodes];
  __shared__ short kept[kMaxNodes];
  __shared__ long long dest[kMaxNodes];
  __shared__ int n_kept_mem;
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int start = min(max(a.cu_q[s], 0), a.n_rows);
  const int all = min(max(a.cu_q[s + 1] - start, 0), a.n_rows - start), n = min(all, kMaxNodes);
  if (all > kMaxNodes && tid == 0 && blockIdx.x == 0) report(a.error_flag, kErrTree);
  if (tid < n) chosen[tid] = a.target[start + tid];
  int par[kMaxNodes / 32], tok[kMaxNodes / 32];
  if (tid < 32) {
#pragma unroll
    for (int i = 0; i < kMaxNodes / 32; ++i) {
      const int node = 32 * i + lane;
      par[i] = node < n ? a.parents[start + node] : -2;
      tok[i] = node < n ? a.tokens[start + node] : 0;
    }
  }
  __syncthreads();
  if (tid < 32) {
    int count = 0, node = 0;
    if (n > 0) {
      while (true) {
        if (lane == 0) kept[count] = (short)node;
        if (++count >= a.max_path) break;
        const int want = chosen[node];
        int best = 0x7fffffff;
#pragma unroll
        for (int i = kMaxNodes / 32 - 1; i >= 0; --i) {
          const int c = 32 * i + lane;
          if (par[i] == node && tok[i] == want && c > node) best = c;        // (c > node: a list that is no tree ends too)
        }
        best = __reduce_min_sync(0xffffffffu, best);
        if (best == 0x7fffffff) break;
        node = best;
      }
    }
    if (lane == 0) {
      n_kept_mem = count;
      if (blockIdx.x == 0) {
        a.n_kept[s] = count;
        a.next_token[s] = count > 0 ? chosen[node] : -1;
        a.new_len[s] = a.prefix_len[s] + count;
      }
    }
    __syncwarp();
    if (blockIdx.x == 0)
      for (int j = lane; j < a.max_path; j += 32) a.path[(size_t)s * a.max_path + j] = j < count ? kept[j] : -1;
    if (a.slots) {
      for (int j = lane; j < count; j += 32) {
        const long long slot = a.slots[start + j];
        const bool ok = slot >= 0 && slot < (long long)a.pages * a.block_size;
        if (!ok && blockIdx.x == 0) report(a.error_flag, kErrNoPage);
        // bytes from the start of a call's tensor to the row of kv head 0
        dest[j] = ok ? ((slot / a.block_size) * 2 * a.n_kv_heads * a.block_size + slot % a.block_size) * a.head_bytes : -1ll;
      }
    }
  }
  __syncthreads();
  if (!a.slots) return;
  const int count = n_kept_mem;
  const int head_vecs = a.head_bytes / (int)sizeof(Vec), row_vecs = a.n_kv_heads * head_vecs;
  const long long head_pitch = (long long)a.block_size * a.head_bytes;       // between kv heads inside a page
  const long long plane = a.n_kv_heads * head_pitch, call_bytes = 2ll * a.pages * plane;
  const int total = a.calls * 2 * row_vecs;
  // a thread keeps its place in the row and goes over the kept tokens
  for (int w = blockIdx.x * blockDim.x + tid; w < total; w += gridDim.x * blockDim.x) {
    const int x = w % row_vecs, cp = w / row_vecs, is_v = cp & 1, call = cp >> 1;
    const char* src = (is_v ? a.v + call * a.v_call + start * a.v_row : a.k + call * a.k_call + start * a.k_row) + (long long)x * sizeof(Vec);
    const long long row = is_v ? a.v_row : a.k_row;
    char* dst = a.cache + call * call_bytes + is_v * plane + (x / head_vecs) * head_pitch + (long long)(x % head_vecs) * sizeof(Vec);
    for (int j0 = 0; j0 < count; j0 += 4) {
      Vec r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < count) r[j] = *reinterpret_cast<const Vec*>(src + kept[j0 + j] * row);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + j < count && dest[j0 + j] >= 0) *reinterpret_cast<Vec*>(dst + dest[j0 + j]) = r[j];
    }
  }
}

}  // namespace lmsf

// All index arrays are int32 but slots (int64).  cu_q [n_seqs + 1]; token_seq, positions, slots [n_rows]; mask [n_rows, words] or
// null; parents [n_rows] or null; tree_len, prefix_len [n_seqs]; block_table [n_seqs, max_blocks].  Rows behind the last
// request's are left as they were.
LMSF_API int lmsf_tree_layout(int* cu_q, int* token_seq, int* positions, long long* slots, unsigned* mask, const int* parents,
                              const int* tree_len, const int* prefix_len, const int* block_table, int max_blocks, int block_size,
                              int n_seqs, int n_rows, int words, int window, int* error_flag, void* stream) {
  using namespace lmsf;
  if (n_seqs < 0 || n_rows < 0) LMSF_REFUSE("tree_layout: %d requests, %d rows", n_seqs, n_rows);
  if (block_size <= 0 || (n_seqs > 0 && max_blocks <= 0)) LMSF_REFUSE("tree_layout: block_size=%d, max_blocks=%d", block_size, max_blocks);
  if (mask && (words < 1 || words > kMaxWords)) LMSF_REFUSE("tree_layout: a mask has 1 to %d words a row, not %d", kMaxWords, words);
  LayoutArgs a{cu_q, token_seq, positions, slots, mask, parents, tree_len, prefix_len, block_table, max_blocks, block_size,
               n_seqs, n_rows, words, window, error_flag};
  return launch_pdl(tree_layout_kernel, dim3(n_seqs > 0 ? n_seqs : 1), dim3(kMaxNodes), 0, (cudaStream_t)stream, a);
}

// Strides in bytes.  slots null: only the path is found.
LMSF_API int lmsf_tree_accept(int* n_kept, int* path, int* next_token, int* new_len, const int* target, const int* tokens,
                              const int* parents, const int* cu_q, const int* prefix_len, int n_seqs, int n_rows, int max_path,
                              const long long* slots, const void* k, const void* v, long long k_call, long long k_row,
                              long long v_call, long long v_row, void* cache, int calls, int pages, int n_kv_heads, int block_size,
                              int head_bytes, int* error_flag, void* stream) {
  using namespace lmsf;
  if (n_seqs <= 0) return 0;
  if (max_path < 1 || max_path > kMaxNodes) LMSF_REFUSE("tree_accept: a path has 1 to %d places, not %d", kMaxNodes, max_path);
  if (n_seqs > 65535) LMSF_REFUSE("tree_accept: %d requests are more than one launch takes (65535)", n_seqs);
  AcceptArgs a{n_kept, path, next_token, new_len, target, tokens, parents, cu_q, prefix_len, n_seqs, n_rows, max_path,
               slots, (const char*)k, (const char*)v, k_call, k_row, v_call, v_row, (char*)cache, calls, pages, n_kv_heads, block_size,
               head_bytes, error_flag};
  cudaStream_t st = (cudaStream_t)stream;
  if (!slots) return launch_pdl(tree_accept_kernel<uint4>, dim3(1, n_seqs), dim3(256), 0, st, a);
  if (!k || !v || !cache || calls <= 0 || pages <= 0 || n_kv_heads <= 0 || block_size <= 0 || head_bytes <= 0)
    LMSF_REFUSE("tree_accept: a cache write needs k, v and a cache");
  const unsigned long long bits = (unsigned long long)k | (unsigned long long)v | (unsigned long long)cache | (unsigned long long)k_call |
                                  (unsigned long long)k_row | (unsigned long long)v_call | (unsigned long long)v_row | (unsigned long long)head_bytes;
  const int vec = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
  if (bits % 2) LMSF_REFUSE("tree_accept: rows must be 2-byte aligned");
  const long long items = 2ll * calls * n_kv_heads * (head_bytes / vec);
  if (items > (1ll << 30)) LMSF_REFUSE("tree_accept: %d calls of %d heads of %d bytes are too many for one launch", calls, n_kv_heads, head_bytes);
  int share = (int)((items + 255) / 256);
  const int most = 1184 / n_seqs > 1 ? 1184 / n_seqs : 1;        // eight blocks for each of 148 SMs
  if (share > most) share = most;
  const dim3 grid(share, n_seqs), block(256);
  if (vec == 16) return launch_pdl(tree_accept_kernel<uint4>, grid, block, 0, st, a);
  if (vec == 8) return launch_pdl(tree_accept_kernel<uint2>, grid, block, 0, st, a);
  if (vec == 4) return launch_pdl(tree_accept_kernel<unsigned>, grid, block, 0, st, a);
  return launch_pdl(tree_accept_kernel<unsigned short>, grid, block, 0, st, a);
}
