// Attention of drafted trees on the CUDA cores: float32 throughout for float32 (no TF32), and bfloat16 where the tensor-core
// kernel does not take the shape.  Any head size up to 256, any group, any page size, any stride.
// Measured: 3 requests of 13..48 nodes behind 515..1,500 keys, a window of 1,024, 32 heads of 64 over 8, float32: 50 to 54 us, 15 TFLOP/s of some 70.  Bound by
// instructions and their latency: issue slots are 40 % used, a third of that by FMAs, with two warps a scheduler (a block has 89 KB of shared memory).  Tiles of 32 keys with three or
// four blocks an SM took 62 to 72 us, 64 rows and 256 threads a block 55.
#include "attention_tree.cuh"

LMSF_DEFINE_LAST_ERROR(lmsf_attention_tree)

namespace lmsf {
namespace tree {

constexpr int kRows = 32, kThreads = 128;
constexpr int kExtra = 0;                      // places of a unit beside its tiles (1: 56 us where 0 takes 50, as the shares no longer end with units)
// Keys of a tile: two tiles of keys and two of values lie in shared memory, for head sizes up to 128 twice per SM.
template <int HDP> constexpr int kTile = HDP <= 64 ? 64 : 32;
template <typename T, int HDP> constexpr int kPitch = HDP + 16 / (int)sizeof(T);         // of a row in shared memory: 16 bytes more, for the banks
template <typename T, int HDP> constexpr size_t smem_bytes(int n_seqs) {
  return sizeof(float) * kRows * (HDP + 4) + sizeof(T) * 4 * kTile<HDP> * kPitch<T, HDP> + sizeof(float) * kRows * (kTile<HDP> + 4) + sizeof(ulonglong2) * 2 * kTile<HDP>
         + work_bytes(n_seqs);
}

__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void upk2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Four neighbouring values of shared memory as two pairs.
__device__ __forceinline__ void pairs(const float* p, uint64_t& a, uint64_t& b) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  a = v.x;
  b = v.y;
}
__device__ __forceinline__ void pairs(const bf16* p, uint64_t& a, uint64_t& b) {
  float v[4];
  ld4(p, v);
  a = pk2(v[0], v[1]);
  b = pk2(v[2], v[3]);
}
__device__ __forceinline__ void copy16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ bool is_odd(float v) { return !(fabsf(v) <= 3.4028235e38f); }

// One pass over the keys with the running maximum and sum of the softmax.  Thread (ty, tx) = (tid / 16, tid % 16) has the scores of rows
// 4 ty .. 4 ty + 3 with keys tx + 16 j and of the same rows' output the columns 64 c + 4 tx .. + 3, in packed pairs of float32: the products of
// 32 rows with 64 keys are bound by the FMA pipe then (48 shared-memory wavefronts beside 64 cycles of packed FMAs), where 8 scores a
// thread were bound by shared memory.  The next tile's keys are on their way while this one's scores are computed, its values while
// its weights are (cp.async, two tiles each).
template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads) attention_tree_kernel(Args a, bool wide) {
  constexpr int kKeys = kTile<HDP>, kJ = kKeys / 16, kC = HDP / 64, kP = kPitch<T, HDP>, kQP = HDP + 4, kPP = kKeys + 4;
  extern __shared__ __align__(16) unsigned char smem[];
  float* qs = (float*)smem;                                      // [kRows][kQP]
  T* ks = (T*)(qs + kRows * kQP);                                // [2][kKeys][kP]
  T* vs = ks + 2 * kKeys * kP;                                   // [2][kKeys][kP]
  float* ps = (float*)(vs + 2 * kKeys * kP);                     // [kRows][kPP]
  ulonglong2* rows_at = (ulonglong2*)(ps + kRows * kPP);         // [2][kKeys] addresses of a key's and its value's row, 0 where there is none
  Lengths* lens = (Lengths*)(rows_at + 2 * kKeys);               // [n_seqs]
  int* offs = (int*)(lens + a.n_seqs);                           // [n_seqs + 1]
  __shared__ int scratch[32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  add_up_work<kKeys, 1, kExtra>(a, kRows, lens, offs, scratch);
  int begin, end;
  share_of_block<kExtra>(offs[a.n_seqs], begin, end);
  const int b = blockIdx.x;
  if (tid == 0) a.notes[b] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  const T* q = (const T*)a.q;
  for (int p = begin; p < end;) {
    const Piece u = piece_at<kKeys, 1, kExtra>(a, lens, offs, p, end);
    const int row0 = u.item * kRows, rows = min(kRows, u.r.n * a.group - row0);
    const int* table = a.block_table + (size_t)u.s * a.max_blocks;
    // thread j < kKeys: where row j of tile t lies (asked for an iteration before its copies are, which every thread makes some of)
    auto find_row = [&](int t) {
      ulonglong2 at = make_ulonglong2(0ull, 0ull);
      if (tid >= kKeys || t >= u.t1) return at;
      if (t >= u.r.n_pre) {
        const int key = (t - u.r.n_pre) * kKeys + tid;
        if (key < u.r.nk) {
          at.x = (unsigned long long)((const T*)a.k + (u.r.start + key) * a.k_stride + (size_t)u.kvh * a.hd);
          at.y = (unsigned long long)((const T*)a.v + (u.r.start + key) * a.v_stride + (size_t)u.kvh * a.hd);
        }
        return at;
      }
      const int key = (u.r.first + t) * kKeys + tid;
      if (key < u.r.lo || key >= u.r.prefix) return at;
      const int block = key / a.block_size, page = table[block];
      if (page < 0 || page >= a.pages) return at;
      const T* row = (const T*)a.cache + page * a.page_stride + ((size_t)u.kvh * a.block_size + (key - block * a.block_size)) * a.hd;
      at.x = (unsigned long long)row;
      at.y = (unsigned long long)(row + a.v_off);
      return at;
    };
    auto note_row = [&](int t, ulonglong2 at) {
      if (tid < kKeys) rows_at[(t & 1) * kKeys + tid] = at;
    };
    constexpr int kE = 16 / (int)sizeof(T), kChunks = HDP / kE;  // values and copies of 16 bytes
    auto request_tile = [&](int t, bool value) {
      T* dst = (value ? vs : ks) + (t & 1) * kKeys * kP;
#pragma unroll 4
      for (int i = tid; i < kKeys * kChunks; i += kThreads) {
        const int j = i / kChunks, c = (i % kChunks) * kE;
        const ulonglong2 at = rows_at[(t & 1) * kKeys + j];
        const T* src = (const T*)(value ? at.y : at.x);
        if (wide) {                                              // whole rows of 16-byte words
          copy16(dst + j * kP + c, src && c < a.hd ? (const void*)(src + c) : a.k, src && c < a.hd);
        } else {
#pragma unroll
          for (int e = 0; e < kE; ++e) dst[j * kP + c + e] = src && c + e < a.hd ? src[c + e] : from_f32<T>(0.f);
        }
      }
      copies_sent();
    };
    const ulonglong2 at0 = find_row(u.t0), at1 = find_row(u.t0 + 1);
    __syncthreads();
    note_row(u.t0, at0);
    note_row(u.t0 + 1, at1);
    __syncthreads();
    request_tile(u.t0, false);
    request_tile(u.t0, true);
    {
      constexpr int kQuads = HDP / 4, kEach = kRows * kQuads / kThreads;     // groups of four values: of a row, of a thread
      float x[kEach < 8 ? kEach : 8][4];
#pragma unroll
      for (int k0 = 0; k0 < kEach; k0 += 8) {
#pragma unroll
        for (int k = 0; k < 8 && k0 + k < kEach; ++k) {          // all requested before the first is stored
          const int i = tid + (k0 + k) * kThreads, row = i / kQuads, c = (i % kQuads) * 4, r = row0 + row, n = r / a.group;
          const T* src = q + (u.r.start + n) * a.q_stride + (size_t)(u.kvh * a.group + (r - n * a.group)) * a.hd + c;
          if (wide && row < rows && c < a.hd) {
            ld4(src, x[k]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][e] = row < rows && c + e < a.hd ? to_f32(src[e]) : 0.f;
          }
        }
#pragma unroll
        for (int k = 0; k < 8 && k0 + k < kEach; ++k) {
          const int i = tid + (k0 + k) * kThreads;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k][e] *= a.scale * 1.4426950408889634f;
          st4(qs + (i / kQuads) * kQP + (i % kQuads) * 4, x[k]);
        }
      }
    }
    int node[4], after[4];                                       // of this thread's rows: node, and the cached key behind which it sees
    float m[4], l[4];
    uint64_t acc[4][kC][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * ty + i;
      node[i] = row < rows ? (row0 + row) / a.group : -1;
      after[i] = node[i] >= 0 && a.window > 0 ? a.positions[u.r.start + node[i]] - a.window : -1;
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kC; ++c) acc[i][c][0] = acc[i][c][1] = 0ull;
    }
    for (int t = u.t0; t < u.t1; ++t) {
      const bool nodes = t >= u.r.n_pre;                         // a tile of drafted keys
      const int key0 = nodes ? (t - u.r.n_pre) * kKeys : (u.r.first + t) * kKeys;
      // sent so far: k and v up to this tile; k of it is awaited, and the next one's sent behind it
      copies_but<1>();
      __syncthreads();
      if (t + 1 < u.t1) request_tile(t + 1, false);
      else copies_sent();
      const ulonglong2 at_next = find_row(t + 2);
      uint32_t words[4][kKeys / 32];                             // what the rows see of drafted tokens
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < kKeys / 32; ++w)
          words[i][w] = nodes && node[i] >= 0 && key0 / 32 + w < a.words ? a.mask[(size_t)(u.r.start + node[i]) * a.words + key0 / 32 + w] : 0xffffffffu;
      const T* kt = ks + (t & 1) * kKeys * kP;
      uint64_t s2[4][kJ] = {};
      const float* q0 = qs + 4 * ty * kQP;
      // (the next four columns are asked for before these are multiplied: a scheduler has one or two warps of this kernel)
      uint64_t x[2][4][2], y[2][kJ][2];
      auto columns = [&](int g, int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) pairs(q0 + i * kQP + c, x[g][i][0], x[g][i][1]);
#pragma unroll
        for (int j = 0; j < kJ; ++j) pairs(kt + (tx + 16 * j) * kP + c, y[g][j][0], y[g][j][1]);
      };
      columns(0, 0);
#pragma unroll 2
      for (int c = 0; c < HDP; c += 8) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g == 0) columns(1, c + 4);
          else columns(0, c + 8 < HDP ? c + 8 : 0);
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s2[i][j] = fma2(x[g][i][0], y[g][j][0], s2[i][j]);
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s2[i][j] = fma2(x[g][i][1], y[g][j][1], s2[i][j]);
        }
      }
      const ulonglong2* here = rows_at + (t & 1) * kKeys;
      // the four rows side by side: their sixteen threads' maxima and sums pass through the warp in four steps
      float s[4][kJ], top[4], sum[4], keep[4];
      bool sees[4][kJ];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int at = tx + 16 * j;
          float lo, hi;
          upk2(s2[i][j], lo, hi);
          s[i][j] = lo + hi;
          sees[i][j] = node[i] >= 0 && here[at].x != 0ull && ((words[i][j / 2] >> (at & 31)) & 1u) && (nodes || key0 + at > after[i]);
          if (sees[i][j]) top[i] = fmaxf(top[i], s[i][j]);
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float now = fmaxf(m[i], top[i]), base = now == -INFINITY ? 0.f : now;
        keep[i] = exp2f(m[i] - base);
        m[i] = now;
        sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          // an unseen key's weight is -0: nothing to the sums, and told from the +0 of a seen one whose score is far below
          const float w = sees[i][j] ? exp2f(s[i][j] - base) : -0.f;
          sum[i] += w;
          ps[(4 * ty + i) * kPP + tx + 16 * j] = w;
        }
        const uint64_t keep2 = pk2(keep[i], keep[i]);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          acc[i][c][0] = mul2(acc[i][c][0], keep2);
          acc[i][c][1] = mul2(acc[i][c][1], keep2);
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i] = l[i] * keep[i] + sum[i];
      copies_but<1>();                                           // v of this tile
      const T* vt = vs + (t & 1) * kKeys * kP;
      bool odd = false;                                          // an infinity or NaN among the values (each thread looks at those that it brought)
      for (int i = tid; i < kKeys * kChunks; i += kThreads) {
        const T* x = vt + (i / kChunks) * kP + (i % kChunks) * kE;
#pragma unroll
        for (int e = 0; e < kE; e += 4) {
          float y[4];
          ld4(x + e, y);
          odd |= is_odd(y[0]) | is_odd(y[1]) | is_odd(y[2]) | is_odd(y[3]);
        }
      }
      const bool any_odd = __syncthreads_or(odd);
      if (t + 1 < u.t1) request_tile(t + 1, true);
      else copies_sent();
      note_row(t + 2, at_next);                                  // (this tile's rows have been read by all)
      const float* p0 = ps + 4 * ty * kPP;
      if (!any_odd) {
        float w[2][4][2];
        uint64_t y[2][2][kC][2];
        auto two_keys = [&](int g, int j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = *reinterpret_cast<const float2*>(p0 + i * kPP + j);
            w[g][i][0] = f.x;
            w[g][i][1] = f.y;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int c = 0; c < kC; ++c) pairs(vt + (j + e) * kP + 64 * c + 4 * tx, y[g][e][c][0], y[g][e][c][1]);
        };
        two_keys(0, 0);
#pragma unroll 2
        for (int j = 0; j < kKeys; j += 4) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (g == 0) two_keys(1, j + 2);
            else two_keys(0, j + 4 < kKeys ? j + 4 : 0);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint64_t w2 = pk2(w[g][i][e], w[g][i][e]);
                  acc[i][c][0] = fma2(w2, y[g][e][c][0], acc[i][c][0]);
                  acc[i][c][1] = fma2(w2, y[g][e][c][1], acc[i][c][1]);
                }
          }
        }
      } else {
        // a value that is no number must not reach the rows that do not see it (0 times infinity)
        for (int j = 0; j < kKeys; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = p0[i * kPP + j];
            if (__float_as_uint(w) == 0x80000000u) continue;
#pragma unroll
            for (int c = 0; c < kC; ++c) {
              uint64_t y0, y1;
              pairs(vt + j * kP + 64 * c + 4 * tx, y0, y1);
              acc[i][c][0] = fma2(pk2(w, w), y0, acc[i][c][0]);
              acc[i][c][1] = fma2(pk2(w, w), y1, acc[i][c][1]);
            }
          }
      }
    }
    const bool begins = u.t0 == 0, ends = u.t1 == u.r.tiles;
    const int slot = 2 * b + (begins ? 1 : 0), quads = (a.hd + 3) / 4;
    float* o = a.partials + slot * partial_floats(kRows, a.hd);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (node[i] < 0) continue;
      const int row = 4 * ty + i;
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      T* out = (T*)a.out + (u.r.start + node[i]) * a.out_stride + (size_t)(u.kvh * a.group + (row0 + row) % a.group) * a.hd;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        float v[4];
        upk2(acc[i][c][0], v[0], v[1]);
        upk2(acc[i][c][1], v[2], v[3]);
        const int quad = 16 * c + tx;
        if (begins && ends) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * quad + e < a.hd) out[4 * quad + e] = from_f32<T>(v[e] * inv);
        } else if (quad < quads) {
          st4(o + ((size_t)quad * kRows + row) * 4, v);
        }
      }
      if (!(begins && ends) && tx == 0) {
        o[(size_t)quads * 4 * kRows + row] = m[i];
        o[(size_t)quads * 4 * kRows + kRows + row] = l[i];
      }
    }
    if (begins && !ends && tid == 0) a.notes[b] = make_int4(u.s, u.kvh, row0, rows | (block_of<kExtra>(offs[a.n_seqs], u.last) << 8));
    p = u.next;
  }
}

template <typename T, int HDP>
static int launch(const Args& a, int blocks, bool wide, cudaStream_t st) {
  static bool raised[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 64 && !raised[dev]) {
    e = cudaFuncSetAttribute(attention_tree_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<T, HDP>(kMaxSeqs));
    if (e != cudaSuccess) return (int)e;
    raised[dev] = true;
  }
  int rc = launch_pdl(attention_tree_kernel<T, HDP>, dim3(blocks), dim3(kThreads), smem_bytes<T, HDP>(a.n_seqs), st, a, wide);
  if (rc) return rc;
  const bool wide_out = ((unsigned long long)a.out | (unsigned long long)(a.out_stride * sizeof(T)) | (unsigned long long)(a.hd * sizeof(T))) % 16 == 0;
  return launch_pdl(join_kernel<T, kRows, 1, HDP>, dim3(blocks, 1), dim3(256), 0, st, a, wide_out);
}

}  // namespace tree
}  // namespace lmsf

// Blocks of a launch, and the bytes of workspace that go with them.
LMSF_API int lmsf_attention_tree_blocks(int sms, int hd) { return hd <= 128 ? 2 * sms : sms; }
LMSF_API long long lmsf_attention_tree_workspace(int sms, int hd) {
  const long long blocks = lmsf_attention_tree_blocks(sms, hd);
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
  const int keys = hd <= 64 ? kTile<64> : kTile<128>;
  const long long tiles = ((long long)max_blocks * block_size + keys - 1) / keys + (32ll * words + keys - 1) / keys + 1 + kExtra;
  if (((n_rows * group + kRows - 1) / kRows + n_seqs) * n_kv_heads * tiles > 0x7fffffffll)
    LMSF_REFUSE("attention_tree: %d rows of %d heads over %d pages are too much work for one launch", n_rows, n_q_heads, max_blocks);
  Args a{q, q_stride, k, k_stride, v, v_stride, out, out_stride, cache, page_stride, v_off, pages, block_table, max_blocks, block_size,
         cu_q, prefix_len, mask, words, positions, window, scale, n_seqs, n_rows, n_q_heads, n_kv_heads, (int)group, hd, nullptr, nullptr};
  const int blocks = lmsf_attention_tree_blocks(sms, hd);
  a.notes = (int4*)workspace;
  a.partials = (float*)(a.notes + blocks);
  const int size = dtype == LMSF_F32 ? 4 : 2;
  const unsigned long long bits = (unsigned long long)q | (unsigned long long)k | (unsigned long long)v | (unsigned long long)cache |
                                  (unsigned long long)(size * (q_stride | k_stride | v_stride | page_stride | v_off | hd));
  const bool wide = bits % 16 == 0;             // rows of 16-byte words
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
