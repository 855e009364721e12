// Attention of drafted trees: what its kernels share.
//
// A request has `prefix_len` cached keys in pages and n drafted nodes whose keys and values are rows of the step's own k and v.
// A node sees the cached keys (inside its window, if there is one) and the nodes whose bits are set in its mask row.  The rows of
// one kv head of one request are its nodes x the heads of the group, node-major: row = node * group + head of the group.
//
// The work is cut as follows.  A unit is (request, kv head, item of up to kRows rows); it has the request's tiles of kKeys keys: its
// cached keys first, then the nodes.  All units' tiles in a row, requests in order, are shared out evenly over the blocks, whatever the
// lengths are, a tile of a unit of two items counted twice and every unit as kExtra tiles more, for what it costs beside them; no
// plan is made on the host, so a captured launch serves any lengths.  A unit that lies in one block's range is finished there.  Of a unit that is cut every block leaves a partial (unnormalised output, running maximum, sum; float32) in the workspace: at most two for a block (and item), one for the unit
// that it begins with and one for the unit that it ends with.  A second kernel adds them up in the order of the blocks; both
// depend only on lengths and G, so the result is the same in every run.
#pragma once
#include "common.cuh"

namespace lmsf {
namespace tree {

constexpr int kMaxSeqs = 1024;             // requests of a step (what is known of each lies in shared memory)

struct Args {
  const void* q; long long q_stride;
  const void* k; long long k_stride;       // drafted tokens' keys [rows][kv heads x head size], values alike
  const void* v; long long v_stride;
  void* out; long long out_stride;
  const void* cache; long long page_stride, v_off; int pages;   // [page][2][kv head][slot][head size], in elements
  const int* block_table; int max_blocks, block_size;
  const int* cu_q; const int* prefix_len;
  const unsigned* mask; int words;
  const int* positions; int window;        // window > 0: a node at position p sees cached keys > p - window
  float scale;
  int n_seqs, n_rows, n_q_heads, n_kv, group, hd;
  float* partials; int4* notes;            // workspace: for every block and item two partials and a note
};

struct Request { int start, n, nk, prefix, lo, first, n_pre, tiles, items; };
struct __align__(16) Lengths { int start, n, prefix, items; };

// An item has `rows` rows.
__device__ __forceinline__ Lengths lengths(const Args& a, int s, int rows) {
  Lengths l;
  const int from = a.cu_q[s], to = a.cu_q[s + 1], prefix = a.prefix_len[s];
  l.start = min(max(from, 0), a.n_rows);
  l.n = min(max(to - l.start, 0), a.n_rows - l.start);
  l.prefix = (int)min((long long)max(prefix, 0), (long long)a.max_blocks * a.block_size);
  l.items = (l.n * a.group + rows - 1) / rows;
  return l;
}
// kKeys keys a tile.
template <int kKeys>
__device__ __forceinline__ Request request(const Args& a, const Lengths& l) {
  Request r;
  r.start = l.start;
  r.n = l.n;
  r.prefix = l.prefix;
  r.items = l.items;
  r.nk = min(r.n, 32 * a.words);                                 // a node behind the mask's last bit is seen by nobody
  r.lo = a.window > 0 ? min(max(r.prefix - a.window + 1, 0), r.prefix) : 0;    // a node's position is the prefix or behind it
  r.first = r.lo / kKeys;
  r.n_pre = (r.prefix + kKeys - 1) / kKeys - r.first;
  if (r.lo >= r.prefix) r.n_pre = 0;
  r.tiles = max(1, r.n_pre + (r.nk + kKeys - 1) / kKeys);        // (rows that see nothing are still written)
  return r;
}

// What a block keeps of the step in shared memory: all[s], and offs[s] = work before request s, in places, for 0 <= s <= n_seqs.
__host__ __device__ __forceinline__ size_t work_bytes(int n_seqs) { return (size_t)n_seqs * sizeof(Lengths) + (size_t)(n_seqs + 1) * sizeof(int); }
template <int kKeys, int kItems, int kExtra>
__device__ __forceinline__ int work_of(const Request& r, int n_kv) {
  return n_kv * (r.tiles * r.items + kExtra * ((r.items + kItems - 1) / kItems));
}
// By all threads of the block (a multiple of 32, at most 1024).
template <int kKeys, int kItems, int kExtra>
__device__ __forceinline__ void add_up_work(const Args& a, int rows, Lengths* all, int* offs, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  if (a.n_seqs <= 32) {                          // one warp's work: no second pass through shared memory
    if (warp == 0) {
      Lengths l = {};
      int w = 0;
      if (lane < a.n_seqs) {
        l = lengths(a, lane, rows);
        w = work_of<kKeys, kItems, kExtra>(request<kKeys>(a, l), a.n_kv);
      }
      int x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane < a.n_seqs) {
        all[lane] = l;
        offs[lane] = x - w;
      }
      if (lane == 31) offs[a.n_seqs] = x;
    }
    __syncthreads();
    return;
  }
  const int per = (a.n_seqs + blockDim.x - 1) / blockDim.x;
  const int s0 = min(tid * per, a.n_seqs), s1 = min(s0 + per, a.n_seqs);
  int sum = 0;
  for (int s = s0; s < s1; ++s) {
    const Lengths l = lengths(a, s, rows);
    all[s] = l;
    offs[s] = sum;
    sum += work_of<kKeys, kItems, kExtra>(request<kKeys>(a, l), a.n_kv);
  }
  int x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  int base = x - sum;
  for (int w = 0; w < warp; ++w) base += scratch[w];
  for (int s = s0; s < s1; ++s) offs[s] += base;
  if (tid == 0) {
    int total = 0;
    for (int w = 0; w < nw; ++w) total += scratch[w];
    offs[a.n_seqs] = total;
  }
  __syncthreads();
}

// Blocks that take part in `work`: kExtra + 2 places each at the least, so that every share has a tile (it may begin with the last place of
// a unit of two items, whose tile belongs to the block before, and go on with the kExtra places of the next unit), and no share that lies
// inside a unit is without one.
template <int kExtra>
__device__ __forceinline__ int blocks_for(int work) { return min((int)gridDim.x, max(work / (kExtra + 2), 1)); }
// What this block takes of it: every block as much as every other, the first `work % blocks` one more.
template <int kExtra>
__device__ __forceinline__ void share_of_block(int work, int& begin, int& end) {
  const int b = blockIdx.x, blocks = blocks_for<kExtra>(work);
  begin = end = 0;
  if (b >= blocks) return;
  const int each = work / blocks, more = work - each * blocks;
  begin = b * each + min(b, more);
  end = begin + each + (b < more ? 1 : 0);
}
// The block whose share place p lies in.
template <int kExtra>
__device__ __forceinline__ int block_of(int work, int p) {
  const int blocks = blocks_for<kExtra>(work), each = work / blocks, more = work - each * blocks, edge = more * (each + 1);
  return p < edge ? p / (each + 1) : more + (p - edge) / each;
}

// The request that place p lies in (0 <= p < offs[n_seqs]).
__device__ __forceinline__ int request_at(const int* offs, int n_seqs, int p) {
  int lo = 0, hi = n_seqs;                                       // offs[lo] <= p < offs[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offs[mid] <= p) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A block's share of one unit of up to kItems items: tiles [t0, t1) of the unit's.  The unit has kExtra places and then those of its tiles: tile t of
// a unit of two items has two and belongs to the block that has the first of them.  next: the place behind the unit, or the block's
// end, also where the share ends before the first tile of the unit behind; last: the place that the unit's last tile is found by.  A share
// that begins with a unit's last place has no tile of it: t0 = t1.
struct Piece { int s, kvh, item, t0, t1, next, last; bool two; Request r; };
template <int kKeys, int kItems, int kExtra>
__device__ __forceinline__ Piece piece_at(const Args& a, const Lengths* all, const int* offs, int p, int end) {
  Piece x;
  x.s = request_at(offs, a.n_seqs, p);
  x.r = request<kKeys>(a, all[x.s]);
  const int rem = p - offs[x.s], whole = kItems * x.r.tiles + kExtra, units = (x.r.items + kItems - 1) / kItems;
  const int per_head = x.r.tiles * x.r.items + kExtra * units;
  x.kvh = rem / per_head;
  const int in_head = rem - x.kvh * per_head, unit = in_head / whole;
  x.item = unit * kItems;                                        // the unit's first item: its neighbours read the same keys
  x.two = kItems == 2 && x.item + 1 < x.r.items;
  const int off = in_head - unit * whole, size = (x.two ? 2 : 1) * x.r.tiles + kExtra, off_end = min(size, off + (end - p));
  const int from = max(off - kExtra, 0), to = max(off_end - kExtra, 0);
  x.t0 = x.two ? (from + 1) / 2 : from;
  x.t1 = x.two ? (to + 1) / 2 : to;
  x.next = p + (off_end - off);
  if (end - x.next <= kExtra) x.next = end;                      // no tile of the unit behind
  x.last = p - off + size - (x.two ? 2 : 1);
  return x;
}

// Partial number (2 block + which) * kItems + item: which = 0 for the unit that the block's share begins inside, 1 for the one that it ends
// inside.  Columns in fours: [hd / 4, rounded up][kRows][4], so that threads that own a row each write and read whole lines;
// then [kRows] maxima (in log2 units) and [kRows] sums.
// Its note, of which = 1 alone: x = request, or -1: none; y = kv head; z = first row among the request's rows of that kv head;
// w = rows | the last block that has a part of the unit << 8.
__host__ __device__ __forceinline__ size_t partial_floats(int rows, int hd) { return (size_t)rows * ((hd + 3) / 4 * 4 + 2); }

// Adds the partials of the units that were cut: block (b, y) of the grid acts if a unit begins in b's last piece and goes on; y is
// an item and 32 of its rows.  Lane = row, and a warp has every eighth group of four columns, so that partials are read in whole
// lines; the results pass through shared memory, so that rows are written in whole lines too.  All of a partial's values are
// requested before the first is used: with two or three partials a unit the kernel is one round trip to L2.
template <typename T, int kRows, int kItems, int kMaxHd>
__global__ void __launch_bounds__(256) join_kernel(Args a, bool wide) {
  constexpr int kGroups = kMaxHd / 32;           // groups of four columns of a thread
  __shared__ __align__(16) T tile[32][kMaxHd + 16 / sizeof(T)];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, item = blockIdx.y / (kRows / 32), row0 = (blockIdx.y % (kRows / 32)) * 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 note = a.notes[b * kItems + item];
  const int rows = min((note.w & 0xff) - row0, 32), last = note.w >> 8;
  if (note.x < 0 || rows <= 0) return;
  const int quads = (a.hd + 3) / 4, row = row0 + min(lane, rows - 1);
  const size_t stride = partial_floats(kRows, a.hd);
  auto part = [&](int i) { return a.partials + stride * ((size_t)(i == b ? 2 * b + 1 : 2 * i) * kItems + item); };
  const size_t at_m = (size_t)quads * 4 * kRows + row, at_l = at_m + kRows;
  const int start = min(max(a.cu_q[note.x], 0), a.n_rows);
  float m = -INFINITY, l = 0.f;
  float4 sum[kGroups] = {};
#pragma unroll 2
  for (int i = b; i <= last; ++i) {              // running maximum again: one pass over the partials
    const float* p = part(i);
    const float mi = p[at_m], li = p[at_l];
    float4 x[kGroups];
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
      if (warp + 8 * k < quads) x[k] = *reinterpret_cast<const float4*>(p + ((size_t)(warp + 8 * k) * kRows + row) * 4);
    const float now = fmaxf(m, mi), base = now == -INFINITY ? 0.f : now, keep = exp2f(m - base), w = exp2f(mi - base);
    m = now;
    l = l * keep + li * w;
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
      if (warp + 8 * k < quads) {
        sum[k].x = sum[k].x * keep + x[k].x * w;
        sum[k].y = sum[k].y * keep + x[k].y * w;
        sum[k].z = sum[k].z * keep + x[k].z * w;
        sum[k].w = sum[k].w * keep + x[k].w * w;
      }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < kGroups; ++k)
    if (warp + 8 * k < quads) {
      const float v[4] = {sum[k].x * inv, sum[k].y * inv, sum[k].z * inv, sum[k].w * inv};
      st4(&tile[lane][4 * (warp + 8 * k)], v);
    }
  __syncthreads();
  constexpr int kVec = 16 / sizeof(T);
  auto out_of = [&](int i) {
    const int r = note.z + row0 + i, node = r / a.group, head = note.y * a.group + r % a.group;
    return (T*)a.out + (start + node) * a.out_stride + (size_t)head * a.hd;
  };
  if (wide) {                                    // rows of the output, and the head size, in 16-byte words
    const int words = a.hd / kVec;
    for (int i = threadIdx.x; i < rows * words; i += 256) {
      const int r = i / words, c = (i % words) * kVec;
      *reinterpret_cast<uint4*>(out_of(r) + c) = *reinterpret_cast<const uint4*>(&tile[r][c]);
    }
  } else {
    for (int i = threadIdx.x; i < rows * a.hd; i += 256) out_of(i / a.hd)[i % a.hd] = tile[i / a.hd][i % a.hd];
  }
}

}  // namespace tree
}  // namespace lmsf
