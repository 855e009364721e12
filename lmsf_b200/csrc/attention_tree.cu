// Attention of drafted trees on the CUDA cores: float32 throughout for float32 (no TF32), and bfloat16 where the tensor-core
// kernel does not take the shape.  Any head size up to 256, any group, any page size, any stride.
#include "attention_tree.cuh"

LMSF_DEFINE_LAST_ERROR(lmsf_attention_tree)

namespace lmsf {
namespace tree {

constexpr int kRows = 32, kKeys = 64, kThreads = 256;

// Four values of a row from column c on, zeros behind the head size.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int c, int hd, bool wide, float (&v)[4]) {
  if (wide && c + 4 <= hd) {
    ld4(p + c, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = c + e < hd ? to_f32(p[c + e]) : 0.f;
}

// One pass over the keys with the running maximum and sum of the softmax.  A tile of 64 keys lies in shared memory as float32
// (keys for the scores, then values in the same place); thread (ty, tx) = (tid / 16, tid % 16) has the scores of rows 2 ty, 2 ty + 1
// with keys tx + 16 j and the output's columns 64 c + 4 tx .. + 3.
template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads) attention_tree_kernel(Args a, bool wide) {
  constexpr int kPitch = HDP + 4;
  extern __shared__ float smem[];
  float* qs = smem;                                              // [kRows][kPitch]
  float* kv = qs + kRows * kPitch;                               // [kKeys][kPitch]
  float* ps = kv + kKeys * kPitch;                               // [kRows][kKeys + 4]
  int* there = (int*)(ps + kRows * (kKeys + 4));                 // [kKeys] whether any row may see the key
  Lengths* lens = (Lengths*)(there + kKeys);                     // [n_seqs]
  int* offs = (int*)(lens + a.n_seqs);                           // [n_seqs + 1]
  __shared__ int scratch[32];
  constexpr int kPP = kKeys + 4;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  add_up_work<kKeys>(a, kRows, lens, offs, scratch);
  int begin, end;
  share_of_block(offs[a.n_seqs], begin, end);
  const int b = blockIdx.x;
  if (tid == 0) a.notes[b] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  const T* q = (const T*)a.q;
  for (int p = begin; p < end;) {
    const Piece u = piece_at<kKeys, 1>(a, lens, offs, p, end);
    const int row0 = u.item * kRows, rows = min(kRows, u.r.n * a.group - row0);
    const int* table = a.block_table + (size_t)u.s * a.max_blocks;
    __syncthreads();
    for (int i = tid; i < kRows * (HDP / 4); i += kThreads) {
      const int row = i / (HDP / 4), c = (i % (HDP / 4)) * 4, r = row0 + row;
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (row < rows) load4(q + (u.r.start + r / a.group) * a.q_stride + (size_t)(u.kvh * a.group + r % a.group) * a.hd, c, a.hd, wide, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) qs[row * kPitch + c + e] = x[e] * (a.scale * 1.4426950408889634f);
    }
    int node[2], after[2];                                       // of this thread's rows: node, and the cached key behind which it sees
    float m[2], l[2], acc[2][HDP / 64][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 2 * ty + i;
      node[i] = row < rows ? (row0 + row) / a.group : -1;
      after[i] = node[i] >= 0 && a.window > 0 ? a.positions[u.r.start + node[i]] - a.window : -1;
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < HDP / 64; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][c][e] = 0.f;
    }
    for (int t = u.t0; t < u.t1; ++t) {
      const bool nodes = t >= u.r.n_pre;                         // a tile of drafted keys
      const int key0 = nodes ? (t - u.r.n_pre) * kKeys : (u.r.first + t) * kKeys;
      // the address of a key's (or value's) row, null where there is none
      auto row_of = [&](int j, bool value) -> const T* {
        const int key = key0 + j;
        if (nodes) {
          if (key >= u.r.nk) return nullptr;
          return value ? (const T*)a.v + (u.r.start + key) * a.v_stride + (size_t)u.kvh * a.hd
                       : (const T*)a.k + (u.r.start + key) * a.k_stride + (size_t)u.kvh * a.hd;
        }
        if (key < u.r.lo || key >= u.r.prefix) return nullptr;
        const int page = table[key / a.block_size];
        if (page < 0 || page >= a.pages) return nullptr;
        return (const T*)a.cache + page * a.page_stride + (value ? a.v_off : 0) + ((size_t)u.kvh * a.block_size + key % a.block_size) * a.hd;
      };
      __syncthreads();
      for (int i = tid; i < kKeys * (HDP / 4); i += kThreads) {
        const int j = i / (HDP / 4), c = (i % (HDP / 4)) * 4;
        const T* src = row_of(j, false);
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (src) load4(src, c, a.hd, wide, x);
        *reinterpret_cast<float4*>(kv + j * kPitch + c) = make_float4(x[0], x[1], x[2], x[3]);
        if (c == 0) there[j] = src != nullptr;
      }
      __syncthreads();
      float s[2][4] = {};
      const float* q0 = qs + 2 * ty * kPitch;
#pragma unroll 4
      for (int c = 0; c < HDP; c += 4) {
        const float4 x0 = *reinterpret_cast<const float4*>(q0 + c), x1 = *reinterpret_cast<const float4*>(q0 + kPitch + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 y = *reinterpret_cast<const float4*>(kv + (tx + 16 * j) * kPitch + c);
          s[0][j] = fmaf(x0.x, y.x, s[0][j]); s[0][j] = fmaf(x0.y, y.y, s[0][j]); s[0][j] = fmaf(x0.z, y.z, s[0][j]); s[0][j] = fmaf(x0.w, y.w, s[0][j]);
          s[1][j] = fmaf(x1.x, y.x, s[1][j]); s[1][j] = fmaf(x1.y, y.y, s[1][j]); s[1][j] = fmaf(x1.z, y.z, s[1][j]); s[1][j] = fmaf(x1.w, y.w, s[1][j]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        bool sees[4];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + tx + 16 * j;
          sees[j] = node[i] >= 0 && there[tx + 16 * j];
          if (nodes) sees[j] = sees[j] && ((a.mask[(size_t)(u.r.start + node[i]) * a.words + (key >> 5)] >> (key & 31)) & 1u);
          else sees[j] = sees[j] && key > after[i];
          if (sees[j]) top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float now = fmaxf(m[i], top), base = now == -INFINITY ? 0.f : now, keep = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // an unseen key's weight is -0: nothing to the sums, and told from the +0 of a seen one whose score is far below
          const float w = sees[j] ? exp2f(s[i][j] - base) : -0.f;
          sum += w;
          ps[(2 * ty + i) * kPP + tx + 16 * j] = w;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * keep + sum;
        m[i] = now;
#pragma unroll
        for (int c = 0; c < HDP / 64; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][c][e] *= keep;
      }
      __syncthreads();
      bool odd = false;                                          // an infinity or NaN among the values
      for (int i = tid; i < kKeys * (HDP / 4); i += kThreads) {
        const int j = i / (HDP / 4), c = (i % (HDP / 4)) * 4;
        const T* src = row_of(j, true);
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (src) load4(src, c, a.hd, wide, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= !(fabsf(x[e]) <= 3.4028235e38f);
        *reinterpret_cast<float4*>(kv + j * kPitch + c) = make_float4(x[0], x[1], x[2], x[3]);
      }
      const float* p0 = ps + 2 * ty * kPP;
      if (!__syncthreads_or(odd)) {
#pragma unroll 4
        for (int j = 0; j < kKeys; ++j) {
          const float w0 = p0[j], w1 = p0[kPP + j];
#pragma unroll
          for (int c = 0; c < HDP / 64; ++c) {
            const float4 y = *reinterpret_cast<const float4*>(kv + j * kPitch + 64 * c + 4 * tx);
            acc[0][c][0] = fmaf(w0, y.x, acc[0][c][0]); acc[0][c][1] = fmaf(w0, y.y, acc[0][c][1]);
            acc[0][c][2] = fmaf(w0, y.z, acc[0][c][2]); acc[0][c][3] = fmaf(w0, y.w, acc[0][c][3]);
            acc[1][c][0] = fmaf(w1, y.x, acc[1][c][0]); acc[1][c][1] = fmaf(w1, y.y, acc[1][c][1]);
            acc[1][c][2] = fmaf(w1, y.z, acc[1][c][2]); acc[1][c][3] = fmaf(w1, y.w, acc[1][c][3]);
          }
        }
      } else {
        // a value that is no number must not reach the rows that do not see it (0 times infinity)
        for (int j = 0; j < kKeys; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float w = p0[i * kPP + j];
            if (__float_as_uint(w) == 0x80000000u) continue;
#pragma unroll
            for (int c = 0; c < HDP / 64; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][c][e] = fmaf(w, kv[j * kPitch + 64 * c + 4 * tx + e], acc[i][c][e]);
          }
      }
    }
    const bool begins = u.t0 == 0, ends = u.t1 == u.r.tiles;
    if (begins && ends) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (node[i] < 0) continue;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        T* out = (T*)a.out + (u.r.start + node[i]) * a.out_stride + (size_t)(u.kvh * a.group + (row0 + 2 * ty + i) % a.group) * a.hd;
#pragma unroll
        for (int c = 0; c < HDP / 64; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = 64 * c + 4 * tx + e;
            if (col < a.hd) out[col] = from_f32<T>(acc[i][c][e] * inv);
          }
      }
    } else {
      const int slot = 2 * b + (begins ? 1 : 0);
      float* o = a.partials + slot * partial_floats(kRows, a.hd);
      const int quads = (a.hd + 3) / 4;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 2 * ty + i;
        if (row >= rows) continue;
#pragma unroll
        for (int c = 0; c < HDP / 64; ++c) {
          const int quad = 16 * c + tx;
          if (quad < quads) st4(o + ((size_t)quad * kRows + row) * 4, acc[i][c]);
        }
        if (tx == 0) {
          o[(size_t)quads * 4 * kRows + row] = m[i];
          o[(size_t)quads * 4 * kRows + kRows + row] = l[i];
        }
      }
      if (begins && tid == 0) a.notes[b] = make_int4(u.s, u.kvh, row0, rows | (block_of(offs[a.n_seqs], u.last) << 8));
    }
    p = u.next;
  }
}

template <typename T, int HDP>
static int launch(const Args& a, int blocks, bool wide, cudaStream_t st) {
  const size_t smem = sizeof(float) * ((size_t)(kRows + kKeys) * (HDP + 4) + kRows * (kKeys + 4) + kKeys) + work_bytes(a.n_seqs);
  static bool raised[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 64 && !raised[dev]) {
    e = cudaFuncSetAttribute(attention_tree_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != cudaSuccess) return (int)e;
    raised[dev] = true;
  }
  int rc = launch_pdl(attention_tree_kernel<T, HDP>, dim3(blocks), dim3(kThreads), smem, st, a, wide);
  if (rc) return rc;
  const bool wide_out = ((unsigned long long)a.out | (unsigned long long)(a.out_stride * sizeof(T)) | (unsigned long long)(a.hd * sizeof(T))) % 16 == 0;
  return launch_pdl(join_kernel<T, kRows, 1, HDP>, dim3(blocks, 1), dim3(256), 0, st, a, wide_out);
}

}  // namespace tree
}  // namespace lmsf

// Blocks of a launch, and the bytes of workspace that go with them.
LMSF_API int lmsf_attention_tree_blocks(int sms) { return 2 * sms; }
LMSF_API long long lmsf_attention_tree_workspace(int sms, int hd) {
  const long long blocks = lmsf_attention_tree_blocks(sms);
  return blocks * (2 * (long long)lmsf::tree::partial_floats(lmsf::tree::kRows, hd) * 4 + 16);
}

// q, out [n_rows, heads x hd]; k, v [n_rows, kv heads x hd]; strides in elements.  workspace: lmsf_attention_tree_workspace
// bytes, 16-byte aligned, in any state.
LMSF_API int lmsf_attention_tree(const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                 void* out, long long out_stride, const void* cache, long long page_stride, long long v_off, int pages,
                                 const int* block_table, int max_blocks, int block_size, const int* cu_q, const int* prefix_len,
                                 const unsigned* mask, int words, const int* positions, int window, float scale, int n_seqs, int n_rows,
                                 int n_q_heads, int n_kv_heads, int hd, int dtype, void* workspace, int sms, void* stream) {
  using namespace lmsf;
  using namespace lmsf::tree;
  if (n_seqs <= 0 || n_rows <= 0) return 0;
  if (hd < 1 || hd > 256) LMSF_REFUSE("attention_tree: head size %d is not between 1 and 256", hd);
  if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads) LMSF_REFUSE("attention_tree: %d query heads of %d kv heads", n_q_heads, n_kv_heads);
  if (n_seqs > kMaxSeqs) LMSF_REFUSE("attention_tree: %d requests are more than one launch takes (%d)", n_seqs, kMaxSeqs);
  if (words < 1 || block_size < 1 || max_blocks < 1) LMSF_REFUSE("attention_tree: words=%d, block_size=%d, max_blocks=%d", words, block_size, max_blocks);
  if (window > 0 && !positions) LMSF_REFUSE("attention_tree: a window needs the nodes' positions");
  if (dtype != LMSF_F32 && dtype != LMSF_BF16) LMSF_REFUSE("attention_tree: unknown dtype code %d", dtype);
  const long long group = n_q_heads / n_kv_heads;
  const long long tiles = ((long long)max_blocks * block_size + kKeys - 1) / kKeys + (32ll * words + kKeys - 1) / kKeys + 1;
  if (((n_rows * group + kRows - 1) / kRows + n_seqs) * n_kv_heads * tiles > 0x7fffffffll)
    LMSF_REFUSE("attention_tree: %d rows of %d heads over %d pages are too much work for one launch", n_rows, n_q_heads, max_blocks);
  Args a{q, q_stride, k, k_stride, v, v_stride, out, out_stride, cache, page_stride, v_off, pages, block_table, max_blocks, block_size,
         cu_q, prefix_len, mask, words, positions, window, scale, n_seqs, n_rows, n_q_heads, n_kv_heads, (int)group, hd, nullptr, nullptr};
  const int blocks = lmsf_attention_tree_blocks(sms);
  a.notes = (int4*)workspace;
  a.partials = (float*)(a.notes + blocks);
  const int size = dtype == LMSF_F32 ? 4 : 2;
  const unsigned long long bits = (unsigned long long)q | (unsigned long long)k | (unsigned long long)v | (unsigned long long)cache |
                                  (unsigned long long)(size * (q_stride | k_stride | v_stride | page_stride | v_off | hd));
  const bool wide = bits % (4 * size) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LMSF_F32) {
    if (hd <= 64) return launch<float, 64>(a, blocks, wide, st);
    if (hd <= 128) return launch<float, 128>(a, blocks, wide, st);
    return launch<float, 256>(a, blocks, wide, st);
  }
  if (hd <= 64) return launch<bf16, 64>(a, blocks, wide, st);
  if (hd <= 128) return launch<bf16, 128>(a, blocks, wide, st);
  return launch<bf16, 256>(a, blocks, wide, st);
}
