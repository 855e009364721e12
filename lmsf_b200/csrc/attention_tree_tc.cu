// Attention of drafted trees on tcgen05 tensor cores: bfloat16, head sizes 64 to 128 (multiples of 16, -DLMSF_HEAD_DIM), pages of a
// power of two of at least 8 keys.  The mathematics is attention_tree.cuh's: one pass over the keys with the running maximum and sum of the softmax.
//
// What bounds it: a request's keys and values are read once for all its nodes and all heads of a group, so up to some 150 rows a
// kv head (nodes x heads of the group) the kernel is bound by their bytes, above by the tensor cores and the exponentials.  What holds it
// from both is the way of one tile: scores, their maximum, weights, the product with v and the next scores follow one another, some 3,100 cycles for a tile of two
// items where their products take 2,048, and the first tile of a block has its way from memory before it.
// Measured (captured in a graph, other inputs in every launch): 64 requests of 33..64 nodes behind 2,048..4,096 keys, 32 heads of 128 over 8: 225 us, 688 TFLOP/s
// (of 1,628 that a library product reaches); 2 of 48 behind 24,000..32,000: 80 us, 600 TFLOP/s and 3.1 TB/s; 8 of 32 behind 2,047: 27.7 us, 2.6 TB/s (of 6.55); 27 of 1..64 behind
// 130..2,300, 32 heads of 64 over 8: 40.9 us; one of 8 behind 97: 10.2 us.  A window that hides nothing takes 0.2 to 0.6 us more than
// none (the rows' positions are read for its edge), one that does takes tiles away: 8 of 32 behind 2,047 with a window of 64 13.0 us, of 1,024 23.8.
//
// An item is up to 128 rows: 128 / group nodes x the heads of the group, which one copy brings into shared memory node-major.  A
// block works on pieces of units (a request, a kv head, two items; see attention_tree.cuh) with 128 keys a tile:
//   * a unit of two items: both take every tile, each its own queries;
//   * a unit of one item: the two halves of the block take the tiles in turn with the same queries, each with an output and a maximum of
//     its own, and add up at the end, so that one half's products run beside the other's softmax here too.
// Warps: 0-3 and 4-7 softmax of half 0 and 1, a row per thread; 8 works out the pieces and brings queries and tiles of k by tensor-map copies (a
// box per page, or 32 rows of the step's own k for drafted tokens); 9 brings tiles of v; 11 goes over those that some row must not see
// all of: rows that nobody sees are cleared, and in a tile whose rows not every row sees (drafted tokens, the edge of a window)
// values that are no numbers are set to zero and remembered, since their zero weights would make NaN of them; the rows that do
// see them get them added at the end; 10 issues the products, the halves in turn, so that one half's products run beside the other's softmax
// (a warp for each half let both halves do the same at the same time).
// Tensor memory: S of half x (128 columns, P over the first 64 of them as bfloat16 pairs) at 128 x, its output at 256 + 128 x.  (Steps of
// 64 keys, whose scores would have two places to be in, were slower: a product of 64 columns takes the tensor cores as long as one
// of 128, whose left operand has as many rows to be read.  For heads of 64, P in columns of its own and the next scores issued as soon as the last ones
// are read was slower too, 45 us where this takes 41: one warp issues all products in one order, and a wait more a tile costs as much as the scores' time;
// so was a strict turn of the two halves at their exponentials, 44 us: they do not contend for the exponentials' unit, which is 44 % busy.)
// Weights are rounded to bfloat16 for P V (2^-8 relative, the operand type of the product); sums, maxima, outputs are float32.
// Every wait is bounded (the two halves meet at an mbarrier too); when one runs out the block raises the error word (code 3) and ends.
#include <cstring>

#include "attention_tree.cuh"
#include "tc_common.cuh"

#ifndef LMSF_HEAD_DIM
#error "compile with -DLMSF_HEAD_DIM=64, 80, 96, 112 or 128"
#endif

LMSF_DEFINE_LAST_ERROR(lmsf_attention_tree_tc)

namespace lmsf {
namespace tree {

using namespace lmsf::tc;

constexpr int HD = LMSF_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 64 && HD <= 128, "head sizes 64 to 128 in steps of 16");
constexpr int BM = 128, BN = 128;              // rows of an item, keys of a tile
constexpr int kHB = (HD + 63) / 64;            // 64-wide blocks of the head dimension
constexpr int kTileBytes = kHB * BN * 128;     // one tile of q, k or v
constexpr int kStages = HD > 64 ? 2 : 4;       // tiles of k in flight, and of v
constexpr int kOffK = 2 * kTileBytes, kOffV = kOffK + kStages * kTileBytes, kOffWork = kOffV + kStages * kTileBytes;
constexpr uint32_t kTmemCols = 512, kOCol = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.0f;               // the output is rescaled when the maximum grew by more than this (log2 units)
// What a unit costs beside its tiles, in places of the sharing: the first tile's way from memory, the queries, the end.  27 requests of 1..64 nodes behind
// 130..2,300 keys take 52 us with 0, 46 with 1, 43 with 2, 42 with 3 and 4; a request of 8 behind 1,000 18.5 with 2, 21 with 3, 23 with 4.
constexpr int kExtra = 2;
constexpr int kThreadsTotal = 384, kHalf = 128;
constexpr int kRegsSoftmax = 216, kRegsOther = 72;
constexpr int kRing = 16;                      // notes of tiles and of pieces that warps leave one another
static_assert(kStages + 4 <= kRing, "notes are read before they are written again");

struct TcArgs {
  Args a;
  int nodes_per_item, block_shift, rows_box;
  int wide_out;                                // rows of the output take 16-byte stores
  int* error_flag;
};

__device__ __forceinline__ float ex2_approx(float x) {      // 2^x, 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void tmem_ld8_issue(uint32_t taddr, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8_issue(uint32_t taddr, const float* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
               ::"r"(taddr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]) : "memory");
}
// Waits and arrivals are the kernel's pace: a wait that finds its barrier ready takes a warp 78 cycles (110 with a hint for how long to sleep, 250
// where one lane waits for the others), a signal from warp to warp 130.  So all lanes wait, and the one lane that arrives does so under a
// predicate, without a branch.
__device__ __forceinline__ void arrive_if(bool go, uint32_t bar) {
  asm volatile("{\n.reg .pred q;\n.reg .b64 st;\nsetp.ne.b32 q, %1, 0;\n@q mbarrier.arrive.shared::cta.b64 st, [%0];\n}\n" ::"r"(bar), "r"((uint32_t)go) : "memory");
}
__device__ __forceinline__ void tma_load_box_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(mbar) : "memory");
}
// bits [lo, hi) of a word
__device__ __forceinline__ uint32_t bits(int lo, int hi) {
  lo = min(max(lo, 0), 32);
  hi = min(max(hi, 0), 32);
  const uint32_t upto = hi >= 32 ? 0xffffffffu : (1u << hi) - 1u, below = lo >= 32 ? 0xffffffffu : (1u << lo) - 1u;
  return upto & ~below;
}

// What the warps of a block need to know of a piece, left in shared memory by warp 8 a piece ahead.  They read it where they need it:
// held in registers it would not fit beside a row's scores, nor into what the other warps keep.
// last: the block that ends the unit; edge: the cached key up to which some row of the piece does not see all (its window lies behind), -1: none
struct __align__(16) PieceNote { int s, kvh, item, t0, nt, start, n, nk, prefix, lo, edge, n_pre, tiles, two, last, next; };
typedef const volatile PieceNote* NotePtr;
// The unit's first tile begins with cached key `lo`, rounded down.
template <typename Note>
__device__ __forceinline__ int cached_key(const Note& u, int t) { return (u.lo / BN + t) * BN; }
// Rows [lo, hi) of a tile are seen by some row of the piece's request; none of the others is multiplied, but for those that share a step
// of 16 with them.
template <typename Note>
__device__ __forceinline__ void rows_seen(const Note& u, int t, int& key0, int& lo, int& hi) {
  const bool nodes = t >= u.n_pre;
  key0 = nodes ? (t - u.n_pre) * BN : cached_key(u, t);
  lo = nodes ? 0 : max(u.lo - key0, 0);
  hi = min((nodes ? u.nk : u.prefix) - key0, BN);
}
// What the warps need to know of a tile: boxes whose page is not there, which steps of 16 keys somebody sees (from, to), and whether every
// row sees every key.
constexpr uint32_t kAllSeen = 0x80000000u;
__device__ __forceinline__ int from16(uint32_t note) { return (note >> 16) & 15; }
__device__ __forceinline__ int to16(uint32_t note) { return (note >> 20) & 15; }
// Seen by some row, but perhaps not by every one: drafted tokens, and cached ones at the edge of a window or before it.
template <typename Note>
__device__ __forceinline__ bool seen_by_some(const Note& u, int t, int key0) { return t >= u.n_pre || key0 <= u.edge; }

__global__ void __launch_bounds__(kThreadsTotal, 1) attention_tree_tc_kernel(const TcArgs ta, const __grid_constant__ CUtensorMap q_map,
                                                                             const __grid_constant__ CUtensorMap k_map,
                                                                             const __grid_constant__ CUtensorMap v_map,
                                                                             const __grid_constant__ CUtensorMap cache_map) {
  const Args& a = ta.a;
  extern __shared__ unsigned char smem_raw[];
  // k_full[kStages], k_empty, v_full, v_fixed, v_empty [kStages each], s_full[2], p_full[2][half of P], o_done[2], q_full, q_free, met,
  // noted[kRing]
  __shared__ __align__(8) uint64_t bars[5 * kStages + 11 + kRing];
  __shared__ PieceNote notes[kRing];
  __shared__ uint32_t tmem_base_mem;
  __shared__ int failed_mem, scratch[32];
  __shared__ uint32_t tile_notes[2][kRing];              // of the tiles of k, and of v
  __shared__ int odd_values[kRing];                      // of a piece: values that are no numbers were set to zero
  __shared__ float2 stats[2][kHalf];                     // maximum and sum of a half's rows (a unit of one item)
  volatile int* failed = &failed_mem;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  Lengths* lens = (Lengths*)(smem_raw + (smem - smem_addr(smem_raw)) + kOffWork);
  int* offs = (int*)(lens + a.n_seqs);
  const uint32_t sQ = smem, sK = smem + kOffK, sV = smem + kOffV, bar0 = smem_addr(&bars[0]);
  auto k_full = [&](int s) { return bar0 + 8u * s; };
  auto k_empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto v_full = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
  auto v_fixed = [&](int s) { return bar0 + 8u * (3 * kStages + s); };
  auto v_empty = [&](int s) { return bar0 + 8u * (4 * kStages + s); };
  auto s_full = [&](int x) { return bar0 + 8u * (5 * kStages + x); };
  auto p_full = [&](int x, int h) { return bar0 + 8u * (5 * kStages + 2 + 2 * x + h); };
  auto o_done = [&](int x) { return bar0 + 8u * (5 * kStages + 6 + x); };
  const uint32_t q_full = bar0 + 8u * (5 * kStages + 8), q_free = q_full + 8u, met = q_full + 16u;
  auto noted = [&](int i) { return bar0 + 8u * (5 * kStages + 11 + i % kRing); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    // s_full and o_done take the products' completion and an arrival of the thread that issued them: what that thread had seen before (a
    // tile's note, odd values) is then seen by those who wait there.  p_full takes an arrival of every warp of the half.
    for (int s = 0; s < kStages; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_fixed(s), 1);
      mbar_init(v_empty(s), 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_full(x), 2);
      mbar_init(o_done(x), 2);
      mbar_init(p_full(x, 0), kHalf / 32);
      mbar_init(p_full(x, 1), kHalf / 32);
    }
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    for (int i = 0; i < kRing; ++i) mbar_init(noted(i), 1);
    mbar_init(met, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed_mem = 0;
  }
  if (warp == 8 && lane < 4) {
    const CUtensorMap* m = lane == 0 ? &q_map : lane == 1 ? &k_map : lane == 2 ? &v_map : &cache_map;
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  pdl_wait();
  // Tensor memory is claimed behind everything that ran before, and what comes behind is let in once all blocks have theirs: a block that waited for
  // a kernel while it held columns which that kernel's blocks still wait for would wait for good.
  if (warp == 11) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_mem)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int rows_item = ta.nodes_per_item * a.group;
  add_up_work<BN, 2, kExtra>(a, rows_item, lens, offs, scratch);
  if (tid < 2) a.notes[2 * blockIdx.x + tid] = make_int4(-1, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_mem;
  pdl_launch_dependents();
  int begin, end;
  const int work = offs[a.n_seqs];
  share_of_block<kExtra>(work, begin, end);
  // the note of the block's i-th piece; for the warps that bring tiles a copy of it
  auto note_of = [&](int i, bool& ok) -> NotePtr {
    if (ok) ok = mbar_wait_f(noted(i), (uint32_t)((i / kRing) & 1), failed);
    return &notes[i % kRing];
  };
  auto copy_of = [&](int i, bool& ok) {
    if (ok) ok = mbar_wait_f(noted(i), (uint32_t)((i / kRing) & 1), failed);
    return notes[i % kRing];
  };

  if (warp >= 8) {
    regs_dec<kRegsOther>();
    // The tiles of k or v of one piece after the other, by a whole warp.  Lane i brings box i of a tile of cached keys (a page, or 128 keys of
    // one), or 32 drafted tokens; the page of the tile behind is requested before this one's copies and looked at after them.
    const int n_box = BN / ta.rows_box;
    auto entry = [&](const auto& u, int t) {                         // what the block table says of this lane's box of tile t
      const int key = cached_key(u, t) + lane * ta.rows_box;
      return t < u.n_pre && lane < n_box && key < u.prefix ? a.block_table[(size_t)u.s * a.max_blocks + (key >> ta.block_shift)] : -1;
    };
    // The tile's note goes out with it: the barrier's arrival is behind it.
    auto bring = [&](const PieceNote& u, int t, int page, bool is_v, int g) {
      const uint32_t bar = is_v ? v_full(g % kStages) : k_full(g % kStages), dst = (is_v ? sV : sK) + (g % kStages) * kTileBytes;
      const bool nodes = t >= u.n_pre;
      int key0, lo, hi;
      rows_seen(u, t, key0, lo, hi);
      const int key = key0 + lane * ta.rows_box;
      const bool seen = !nodes && lane < n_box && key < u.prefix && key + ta.rows_box > u.lo, there = seen && page >= 0 && page < a.pages;
      const uint32_t here = __ballot_sync(0xffffffffu, there), missing = __ballot_sync(0xffffffffu, seen && !there);
      const int boxes = (hi + 31) / 32;                          // of drafted tokens
      if (lane == 0) {
        const bool all = lo == 0 && hi == BN && !missing && !seen_by_some(u, t, key0);
        *(volatile uint32_t*)&tile_notes[is_v][g % kRing] = missing | ((uint32_t)(lo / 16) << 16) | ((uint32_t)((hi + 15) / 16) << 20) | (all ? kAllSeen : 0u);
        mbar_arrive_expect_tx(bar, (uint32_t)((nodes ? boxes * 32 : __popc(here) * ta.rows_box) * 128 * kHB));
      }
      __syncwarp();
      if (nodes) {
        if (lane < boxes) {
#pragma unroll
          for (int hb = 0; hb < kHB; ++hb)
            tma_load_box_3d(dst + hb * (BN * 128) + lane * (32 * 128), is_v ? &v_map : &k_map, hb * 64, u.kvh, u.start + key0 + lane * 32, bar);
        }
      } else if (there) {
#pragma unroll
        for (int hb = 0; hb < kHB; ++hb)
          tma_load_box(dst + hb * (BN * 128) + lane * ta.rows_box * 128, &cache_map, hb * 64, key & (a.block_size - 1), (is_v ? a.n_kv : 0) + u.kvh, page, bar);
      }
    };
    if (warp == 8) {
      // ------------------------------------------------------------------ notes, queries, tiles of k
      int g = 0;                                                 // tiles of the block so far
      bool ok = true;
      auto note_at = [&](int p) {                                // (last: a place yet; edge: none yet)
        Piece u = piece_at<BN, 2, kExtra>(a, lens, offs, p, end);
        if (u.t0 == u.t1) u = piece_at<BN, 2, kExtra>(a, lens, offs, u.next, end);       // (the block's first place was a unit's last)
        return PieceNote{u.s, u.kvh, u.item, u.t0, u.t1 - u.t0, u.r.start, u.r.n, u.r.nk, u.r.prefix, u.r.lo, -1, u.r.n_pre, u.r.tiles, u.two, u.last, u.next};
      };
      auto leave_note = [&](int i, PieceNote& u) {
        u.last = u.t0 == 0 && u.nt < u.tiles ? block_of<kExtra>(work, u.last) : 0;
        if (a.window > 0) {                                      // by the rows' own positions: a caller's may lie anywhere behind the cached tokens
          const int from = u.item * ta.nodes_per_item, to = min(u.n, from + (u.two ? 2 : 1) * ta.nodes_per_item);
          int top = 0;
          for (int i = from + lane; i < to; i += 32) top = max(top, a.positions[u.start + i]);
          u.edge = __reduce_max_sync(0xffffffffu, top) - a.window;
        }
        if (lane == 0) {
          notes[i % kRing] = u;
          mbar_arrive(noted(i));
        }
        __syncwarp();
      };
      auto bring_q = [&](const PieceNote& u) {
        if (lane == 0) {
          const int items = u.two ? 2 : 1;
          mbar_arrive_expect_tx(q_full, (uint32_t)(items * rows_item * 128 * kHB));
          for (int x = 0; x < items; ++x)
#pragma unroll
            for (int hb = 0; hb < kHB; ++hb)
              tma_load_box_3d(sQ + x * kTileBytes + hb * (BM * 128), &q_map, hb * 64, u.kvh * a.group, u.start + (u.item + x) * ta.nodes_per_item, q_full);
        }
        __syncwarp();
      };
      PieceNote u = {}, behind = {};
      int page = -1;
      if (begin < end) {                                         // the way to the first keys is the block's start: nothing waits on it that can go beside it
        u = note_at(begin);
        page = entry(u, u.t0);
        leave_note(0, u);
        bring_q(u);
      }
      for (int i = 0, p = begin; p < end && ok; ++i, u = behind) {
        const int t0 = u.t0, nt = u.nt;
        if (i > 0) page = entry(u, t0);
        for (int t = t0; t < t0 + nt && ok; ++t, ++g) {
          const int s = g % kStages;
          if (g >= kStages && !mbar_wait_f(k_empty(s), (uint32_t)((g / kStages - 1) & 1), failed)) { ok = false; break; }
          const int next = t + 1 < t0 + nt ? entry(u, t + 1) : -1;
          bring(u, t, page, false, g);
          page = next;
          if (t == t0 && i > 0) {                                // the queries, as soon as the piece before has issued its last scores
            if (!mbar_wait_f(q_free, (uint32_t)((i - 1) & 1), failed)) { ok = false; ++g; break; }
            bring_q(u);
          }
          if (t == min(t0 + 1, t0 + nt - 1) && u.next < end) {   // (behind the first copies)
            behind = note_at(u.next);
            leave_note(i + 1, behind);
          }
        }
        p = u.next;
        if (p >= end && ok) {                                    // the last queries, and the arrival behind them
          mbar_wait_drain(q_full, (uint32_t)(i & 1));
          ok = mbar_wait_f(q_free, (uint32_t)(i & 1), failed);
        }
      }
      // no copy of this block may be in flight when it ends, nor an arrival on its barriers
      for (int i = max(0, g - kStages); i < g; ++i) mbar_wait_drain(k_full(i % kStages), (uint32_t)((i / kStages) & 1));
      for (int i = max(0, g - kStages); i < g && ok; ++i) ok = mbar_wait_f(k_empty(i % kStages), (uint32_t)((i / kStages) & 1), failed);
      if (!ok) mbar_wait_drain(q_full, 0u), mbar_wait_drain(q_full, 1u);
    } else if (warp == 9) {
      // ------------------------------------------------------------------ tiles of v
      int g = 0;
      bool ok = true;
      for (int i = 0, p = begin; p < end && ok; ++i) {
        const PieceNote u = copy_of(i, ok);
        if (!ok) break;
        const int t0 = u.t0, nt = u.nt;
        int page = entry(u, t0);
        for (int t = t0; t < t0 + nt; ++t, ++g) {
          const int s = g % kStages;
          if (g >= kStages && !mbar_wait_f(v_empty(s), (uint32_t)((g / kStages - 1) & 1), failed)) { ok = false; break; }
          const int next = t + 1 < t0 + nt ? entry(u, t + 1) : -1;
          bring(u, t, page, true, g);
          page = next;
        }
        p = u.next;
      }
      for (int i = max(0, g - kStages); i < g; ++i) mbar_wait_drain(v_full(i % kStages), (uint32_t)((i / kStages) & 1));
      for (int i = max(0, g - kStages); i < g && ok; ++i) ok = mbar_wait_f(v_empty(i % kStages), (uint32_t)((i / kStages) & 1), failed);
    } else if (warp == 11) {
      // ------------------------------------------------------------------ tiles of v that are not for everybody
      int g = 0;
      bool ok = true;
      for (int i = 0, p = begin; p < end && ok; ++i) {
        const PieceNote u = copy_of(i, ok);
        if (!ok) break;
        const int t0 = u.t0, nt = u.nt;
        if (lane == 0) odd_values[i % kRing] = 0;
        for (int t = t0; t < t0 + nt && ok; ++t, ++g) {
          const int s = g % kStages;
          ok = mbar_wait_f(v_full(s), (uint32_t)((g / kStages) & 1), failed);
          if (!ok) break;
          const uint32_t note = *(volatile uint32_t*)&tile_notes[1][g % kRing], missing = note & 0xffffu;
          if (!(note & kAllSeen)) {
            int key0, lo, hi;
            rows_seen(u, t, key0, lo, hi);
            const bool some = seen_by_some(u, t, key0);
            // eight lanes a row, four rows at a time, and the 64-wide blocks of the head one after the other
            const uint32_t v = sV + s * kTileBytes + (lane & 7) * 16;
            const int r_lane = lane >> 3;
            auto clear = [&](int from, int to) {
              for (int r = from + r_lane; r < to; r += 4)
#pragma unroll
                for (int hb = 0; hb < kHB; ++hb)
                  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v + (hb * BN + r) * 128), "r"(0) : "memory");
            };
            clear(lo & ~15, lo);
            clear(hi, (hi + 15) & ~15);
            for (uint32_t left = missing; left; left &= left - 1) {
              const int box = __ffs((int)left) - 1;
              clear(max(box * ta.rows_box, lo), min((box + 1) * ta.rows_box, hi));
            }
            __syncwarp();
            if (some) {
              // 0 x is 0 but for infinities and NaN: a sum of them says whether there is one among the values
              __nv_bfloat162 odd2 = __float2bfloat162_rn(0.f);
              const __nv_bfloat162 zero2 = odd2;
              for (int r = lo + r_lane; r < hi; r += 16) {
#pragma unroll
                for (int hb = 0; hb < kHB; ++hb) {
                  uint32_t w[4][4];
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[k][0]), "=r"(w[k][1]), "=r"(w[k][2]), "=r"(w[k][3])
                                 : "r"(v + (hb * BN + min(r + 4 * k, hi - 1)) * 128) : "memory");
#pragma unroll
                  for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd2 = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[k][e]), zero2, odd2);
                }
              }
              const bool odd = __hisnan(__low2bfloat16(odd2)) || __hisnan(__high2bfloat16(odd2));
              if (__any_sync(0xffffffffu, odd)) {
                if (lane == 0) odd_values[i % kRing] = 1;
                for (int r = lo + r_lane; r < hi; r += 4)
                  for (int hb = 0; hb < kHB; ++hb) {
                    const uint32_t at = v + (hb * BN + r) * 128;
                    uint32_t w[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
                      if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
                    }
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                  }
              }
            }
            fence_async_smem();
          }
          __syncwarp();
          arrive_if(lane == 0, v_fixed(s));
        }
        p = u.next;
      }
    } else if (warp == 10) {
      // ------------------------------------------------------------------ products
      constexpr uint32_t idesc_s = instr_desc(BM, BN, 0), idesc_o = instr_desc(BM, HD, 1);
      const bool leader = elect_one();
      const uint64_t dq0 = smem_desc(sQ, 16, 1024), dk0 = smem_desc(sK, 16, 1024), dv0 = smem_desc(sV, BN * 128, 1024);
      int g0 = 0, n_p[2] = {0, 0};                               // tiles of the block before the piece; P's of a half so far
      bool ok = true;
      for (int i = 0, p = begin; p < end && ok; ++i) {
        NotePtr u = note_of(i, ok);
        if (!ok) break;
        const bool two = u->two != 0;
        const int nt = u->nt, every = two ? 1 : 2;               // every: tiles between two of a half
        auto issue_s = [&](int x, int j) {
          const int s = (g0 + j) % kStages;
          const uint64_t dq = dq0 + (uint64_t)(((two ? x : 0) * kTileBytes) >> 4), dk = dk0 + (uint64_t)((s * kTileBytes) >> 4);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks / 4) * (BN * 128) + (ks % 4) * 32;
            umma(leader, tmem + x * BN, dq + (off >> 4), dk + (off >> 4), idesc_s, ks > 0);
          }
          umma_commit(leader, s_full(x));
          arrive_if(leader, s_full(x));
          if (!two || x == 1) {
            umma_commit(leader, k_empty(s));
            if (j == nt - 1) umma_commit(leader, q_free);        // (a tile's scores are issued in the tiles' order)
          }
        };
        int k_ready = -1;                                        // tiles of k up to this one are there
        auto k_wait = [&](int j) {
          if (k_ready >= j) return;
          const int g = g0 + j;
          ok = mbar_wait_f(k_full(g % kStages), (uint32_t)((g / kStages) & 1), failed);
          tc_fence_after();
          k_ready = j;
        };
        ok = mbar_wait_f(q_full, (uint32_t)(i & 1), failed);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int j = two ? 0 : x;
          if (ok && j < nt) k_wait(j);
          if (ok && j < nt) issue_s(x, j);
        }
        for (int j = 0; j < nt && ok; ++j) {
          const int g = g0 + j, s = g % kStages;
          const uint32_t note = *(volatile uint32_t*)&tile_notes[0][g % kRing];
          const uint64_t dv = dv0 + (uint64_t)((s * kTileBytes) >> 4);
          const int jn = j + every;
          // (v has landed and, where that was to be done, been gone over: warp 11 says so of every tile)
          ok = mbar_wait_f(v_fixed(s), (uint32_t)((g / kStages) & 1), failed);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!ok || (!two && x != (j & 1))) continue;
            const uint32_t phase = (uint32_t)(n_p[x] & 1);
            const bool first = j < every;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (ok) ok = mbar_wait_f(p_full(x, h), phase, failed);
              if (!ok) continue;
              tc_fence_after();
#pragma unroll
              for (int k4 = 0; k4 < BN / 32; ++k4) {             // of the steps of 16 keys those that somebody sees
                const int ks = h * (BN / 32) + k4;
                umma_ts(leader && ks >= from16(note) && ks < to16(note), tmem + kOCol + x * 128, tmem + x * BN + ks * 8, dv + ((ks * 16 * 128) >> 4), idesc_o,
                        (!first || ks > from16(note)) ? 1u : 0u);
              }
            }
            if (!ok) continue;
            ++n_p[x];
            if (!two || x == 1) umma_commit(leader, v_empty(s));
            if (jn < nt) {
              k_wait(jn);
              if (ok) issue_s(x, jn);
            } else {
              umma_commit(leader, o_done(x));
              arrive_if(leader, o_done(x));
            }
          }
        }
        g0 += nt;
        p = u->next;
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax of half x
    regs_inc<kRegsSoftmax>();
    const int x = warp >> 2, row = tid & 127;
    const uint32_t t_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * BN, t_o = t_s + kOCol;
    const float sl2 = a.scale * kLog2e;
    int n_s = 0, n_o = 0, n_met = 0, g0 = 0;                             // scores and outputs of this half so far, meetings of the two; tiles of the block
    bool ok = true;
    auto meet = [&]() {
      __syncwarp();
      arrive_if(lane == 0, met);
      ok = mbar_wait_f(met, (uint32_t)(n_met & 1), failed);
      ++n_met;
    };
    for (int i_piece = 0, p = begin; p < end; ++i_piece) {
      NotePtr u = note_of(i_piece, ok);
      if (!ok) break;
      const bool two = u->two != 0;
      int node = u->n;                                           // of this thread's row; the tree's size: none
      if (row < rows_item) node = (u->item + (two ? x : 0)) * ta.nodes_per_item + row / a.group;
      const bool mine = node < u->n, any_mine = __any_sync(0xffffffffu, mine);
      const int after = mine && a.window > 0 ? a.positions[u->start + node] - a.window : -1;
      auto mask_word = [&](int i) { return a.mask[(size_t)(u->start + node) * a.words + i]; };
      const int nt = u->nt, every = two ? 1 : 2;
      float m = -INFINITY, l = 0.f;
      const int j0 = two ? 0 : x;
      const bool have = j0 < nt;                                 // this half has a tile
      for (int j = j0; j < nt; j += every, ++n_s) {
        const int t = u->t0 + j;
        uint32_t sees[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (t >= u->n_pre) {                                     // what the row sees of the drafted tokens, requested before the scores are awaited
          const int w0 = (t - u->n_pre) * (BN / 32), n_words = (u->nk + 31) / 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) sees[i] = mine && w0 + i < n_words ? mask_word(w0 + i) : 0u;
        }
        // S of the tile is complete, and with it every product issued before it: P V of this half's tile before too
        ok = mbar_wait_f(s_full(x), (uint32_t)(n_s & 1), failed);
        if (!ok) break;
        if (!any_mine) {                                         // a warp without rows: its P is never looked at
          arrive_if(lane == 0, p_full(x, 0));
          arrive_if(lane == 0, p_full(x, 1));
          continue;
        }
        tc_fence_after();
        float sc[BN];
#pragma unroll
        for (int c = 0; c < BN; c += 32) tmem_ld32_issue(t_s + c, sc + c);
        const uint32_t note = *(volatile uint32_t*)&tile_notes[0][(g0 + j) % kRing];
        if (note & kAllSeen) {
          tmem_wait_ld();
        } else {                                                 // what the row sees of the tile's keys, as bits
          int key0, lo, hi;
          rows_seen(*u, t, key0, lo, hi);
          lo = max(lo, after + 1 - key0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sees[i] &= t >= u->n_pre ? bits(0, hi - 32 * i) : bits(lo - 32 * i, hi - 32 * i);
            for (uint32_t left = note & 0xffffu; left; left &= left - 1) {
              const int box = (__ffs((int)left) - 1) * ta.rows_box - 32 * i;
              sees[i] &= ~bits(box, box + ta.rows_box);
            }
          }
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < BN; ++i)
            if (!((sees[i >> 5] >> (i & 31)) & 1u)) sc[i] = -INFINITY;
        }
        float m0 = fmax3(sc[0], sc[1], sc[2]), m1 = fmax3(sc[3], sc[4], sc[5]), m2 = fmax3(sc[6], sc[7], sc[8]), m3 = fmax3(sc[9], sc[10], sc[11]);
#pragma unroll
        for (int i = 12; i + 7 < BN; i += 8) {
          m0 = fmax3(m0, sc[i], sc[i + 1]);
          m1 = fmax3(m1, sc[i + 2], sc[i + 3]);
          m2 = fmax3(m2, sc[i + 4], sc[i + 5]);
          m3 = fmax3(m3, sc[i + 6], sc[i + 7]);
        }
        float top = fmaxf(fmax3(m0, m1, m2), fmax3(m3, sc[BN - 4], sc[BN - 3]));
        top = fmax3(top, sc[BN - 2], sc[BN - 1]) * sl2;
        const bool grow = top > m + kRescale;                    // (and at the first key that a row sees)
        float alpha = 1.f;
        if (grow) {
          alpha = ex2_approx(m - top);
          m = top;
          l *= alpha;
        }
        if (j > j0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            float r[16];
            tmem_ld8_issue(t_o + c, r);
            tmem_ld8_issue(t_o + c + 8, r + 8);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] *= alpha;
            tmem_st8_issue(t_o + c, r);
            tmem_st8_issue(t_o + c + 8, r + 8);
          }
        }
        const float neg_m = m == -INFINITY ? 0.f : -m;
        const uint64_t scale2 = pk2(sl2, sl2), neg2 = pk2(neg_m, neg_m);
        uint64_t sum = pk2(0.f, 0.f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float x0, x1;
            upk2(fma2(pk2(sc[h * 64 + 2 * i], sc[h * 64 + 2 * i + 1]), scale2, neg2), x0, x1);
            x0 = ex2_approx(x0);
            x1 = ex2_approx(x1);
            sum = add2(sum, pk2(x0, x1));
            w[i] = pack_bf16(x0, x1);
          }
          tmem_st32_issue(t_s + h * 32, w);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          arrive_if(lane == 0, p_full(x, h));
        }
        float l0, l1;
        upk2(sum, l0, l1);
        l += l0 + l1;
      }
      if (ok && have) ok = mbar_wait_f(o_done(x), (uint32_t)(n_o & 1), failed);
      if (!ok) break;
      n_o += have;
      tc_fence_after();
      // rows of one item that lie in both halves are added up here: half x writes the columns [x HD / 2, + HD / 2)
      float w_own = 1.f, w_other = 0.f;
      if (!two) {
        stats[x][row] = make_float2(m, l);
        tc_fence_before();
        meet();
        if (!ok) break;
        tc_fence_after();                                        // the other half's output is read below, and o_done of this half says nothing of it
        const float2 o = stats[x ^ 1][row];
        const float m_all = fmaxf(m, o.x), base = m_all == -INFINITY ? 0.f : m_all;
        w_own = ex2_approx(m - base);
        w_other = ex2_approx(o.x - base);
        l = l * w_own + o.y * w_other;
        m = m_all;
      }
      const bool whole = nt == u->tiles;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int slot = (2 * (int)blockIdx.x + (u->t0 == 0 ? 1 : 0)) * 2 + (two ? x : 0);
      float* part = a.partials + slot * partial_floats(BM, HD) + row * 4;
      bf16* out = (bf16*)a.out + (u->start + node) * a.out_stride + (size_t)(u->kvh * a.group + row % a.group) * HD;
      // half a row's columns at a time, summed over this block's keys
      constexpr int kN = HD / 2;
      const bool other_has = !two && (x ^ 1) < nt;
      const int c_from = two ? 0 : x * kN, c_to = two ? HD : c_from + kN;
      if (any_mine) {
#pragma unroll 1
        for (int c0 = c_from; c0 < c_to; c0 += kN) {
          float o[kN];
#pragma unroll
          for (int c = 0; c < kN; c += 8) tmem_ld8_issue(t_o + c0 + c, o + c);
          if (two) {
            tmem_wait_ld();
          } else {
            float r[kN];
#pragma unroll
            for (int c = 0; c < kN; c += 8) tmem_ld8_issue((t_o ^ 128u) + c0 + c, r + c);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kN; ++c) o[c] = (have ? o[c] * w_own : 0.f) + (other_has ? r[c] * w_other : 0.f);
          }
          if (mine && whole) {
#pragma unroll
            for (int c = 0; c < kN; ++c) o[c] *= inv;
            if (ta.wide_out) {
#pragma unroll
              for (int c = 0; c < kN; c += 8) {
                uint4 w;
                w.x = pack_bf16(o[c], o[c + 1]);
                w.y = pack_bf16(o[c + 2], o[c + 3]);
                w.z = pack_bf16(o[c + 4], o[c + 5]);
                w.w = pack_bf16(o[c + 6], o[c + 7]);
                *reinterpret_cast<uint4*>(out + c0 + c) = w;
              }
            } else {
#pragma unroll
              for (int c = 0; c < kN; ++c) out[c0 + c] = __float2bfloat16_rn(o[c]);
            }
          } else if (mine) {
#pragma unroll
            for (int c = 0; c < kN; c += 4)
              *reinterpret_cast<float4*>(part + (size_t)(c0 + c) * BM) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
          }
          __syncwarp();                                          // (the next columns are read by the whole warp at once, with or without a row of its own)
        }
        if (odd_values[i_piece % kRing] && mine) {
          // Values that were set to zero, for the rows that see them: infinities and NaN only, so that it does not matter that what they are added to has been
          // divided and rounded already.  (Rare: nothing here is made to be fast.)
#pragma unroll 1
          for (int t = u->t0; t < u->t0 + nt; ++t) {
            int key0, lo, hi;
            rows_seen(*u, t, key0, lo, hi);
            if (!seen_by_some(*u, t, key0)) continue;
            const bool nodes = t >= u->n_pre;
#pragma unroll 1
            for (int k = key0 + lo; k < key0 + hi; ++k) {
              const bf16* src;
              if (nodes) {
                if (!((mask_word(k >> 5) >> (k & 31)) & 1u)) continue;
                src = (const bf16*)a.v + (u->start + k) * a.v_stride + (size_t)u->kvh * HD;
              } else {
                if (k <= after) continue;
                const int page = a.block_table[(size_t)u->s * a.max_blocks + (k >> ta.block_shift)];
                if (page < 0 || page >= a.pages) continue;
                src = (const bf16*)a.cache + page * a.page_stride + a.v_off + ((size_t)u->kvh * a.block_size + (k & (a.block_size - 1))) * HD;
              }
#pragma unroll 1
              for (int c = c_from; c < c_to; ++c) {
                const float v = __bfloat162float(src[c]);
                if (fabsf(v) <= 3.4e38f) continue;
                if (whole) out[c] = __float2bfloat16_rn(__bfloat162float(out[c]) + v);
                else part[(size_t)(c & ~3) * BM + (c & 3)] += v;
              }
            }
          }
        }
      }
      if (!whole && mine && (two || x == 0)) {
        part[(size_t)HD * BM - 3 * row] = m;
        part[(size_t)HD * BM + BM - 3 * row] = l;
        if (row == 0 && u->t0 == 0) {
          const int item = u->item + (two ? x : 0);
          a.notes[2 * blockIdx.x + (two ? x : 0)] = make_int4(u->s, u->kvh, item * rows_item, min(ta.nodes_per_item, u->n - item * ta.nodes_per_item) * a.group
                                                              | (u->last << 8));
        }
      }
      // the next piece's first P V overwrites the outputs, of both halves where they were added up
      tc_fence_before();
      if (!two) meet();
      if (!ok) break;
      p = u->next;
      g0 += nt;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*failed && tid == 0 && ta.error_flag) atomicExch(ta.error_flag, 3);
  if (warp == 11) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

// A map of [outer][middle][HD] bfloat16 with boxes of 64 x box_middle x box_outer.
static bool make_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  EncodeTiledFn encode = encode_tiled_fn();
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  return encode && encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tree
}  // namespace lmsf

LMSF_API long long lmsf_attention_tree_tc_workspace(int sms, int hd) {
  return sms * (4 * (long long)lmsf::tree::partial_floats(lmsf::tree::BM, hd) * 4 + 2 * 16);
}

// As lmsf_attention_tree, for bfloat16; all rows 16-byte aligned but out's.
LMSF_API int lmsf_attention_tree_tc(const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                    void* out, long long out_stride, const void* cache, long long page_stride, long long v_off, int pages,
                                    const int* block_table, int max_blocks, int block_size, const int* cu_q, const int* prefix_len,
                                    const unsigned* mask, int words, const int* positions, int window, float scale, int n_seqs, int n_rows,
                                    int n_q_heads, int n_kv_heads, int hd, void* workspace, int sms, int* error_flag, void* stream) {
  using namespace lmsf;
  using namespace lmsf::tree;
  if (n_seqs <= 0 || n_rows <= 0) return 0;
  if (hd != HD) LMSF_REFUSE("attention_tree: built for head size %d, called with %d", HD, hd);
  if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads) LMSF_REFUSE("attention_tree: %d query heads of %d kv heads", n_q_heads, n_kv_heads);
  if (n_seqs > kMaxSeqs) LMSF_REFUSE("attention_tree: %d requests are more than one launch takes (%d)", n_seqs, kMaxSeqs);
  if (words < 1 || max_blocks < 1 || block_size < 8 || (block_size & (block_size - 1)))
    LMSF_REFUSE("attention_tree: words=%d, max_blocks=%d, block_size=%d", words, max_blocks, block_size);
  if (window > 0 && !positions) LMSF_REFUSE("attention_tree: a window needs the nodes' positions");
  const int group = n_q_heads / n_kv_heads;
  if (group > BM || !(scale > 0.f) || pages < 1) LMSF_REFUSE("attention_tree: group of %d heads, scale %g, %d pages", group, scale, pages);
  if (((unsigned long long)q | (unsigned long long)k | (unsigned long long)v | (unsigned long long)cache) % 16 ||
      (q_stride | k_stride | v_stride | page_stride) % 8)
    LMSF_REFUSE("attention_tree: q, k, v and the cache need 16-byte aligned rows");
  const long long tiles = ((long long)max_blocks * block_size + BN - 1) / BN + (32ll * words + BN - 1) / BN + 1 + kExtra;
  TcArgs ta;
  ta.nodes_per_item = BM / group;
  const int rows_item = ta.nodes_per_item * group;
  if ((((long long)n_rows * group + rows_item - 1) / rows_item + n_seqs) * n_kv_heads * tiles > 0x7fffffffll)
    LMSF_REFUSE("attention_tree: %d rows of %d heads over %d pages are too much work for one launch", n_rows, n_q_heads, max_blocks);
  ta.a = Args{q, q_stride, k, k_stride, v, v_stride, out, out_stride, cache, page_stride, v_off, pages, block_table, max_blocks, block_size,
              cu_q, prefix_len, mask, words, positions, window, scale, n_seqs, n_rows, n_q_heads, n_kv_heads, group, hd, nullptr, nullptr};
  ta.a.notes = (int4*)workspace;
  ta.a.partials = (float*)(ta.a.notes + 2 * sms);
  ta.block_shift = 0;
  while ((1 << ta.block_shift) < block_size) ++ta.block_shift;
  ta.rows_box = block_size < BN ? block_size : BN;
  ta.wide_out = (unsigned long long)out % 16 == 0 && out_stride % 8 == 0;
  ta.error_flag = error_flag;
  CUtensorMap maps[4];
  const cuuint64_t e = 2, d = HD;
  {
    const cuuint64_t dims[3] = {d, (cuuint64_t)n_q_heads, (cuuint64_t)n_rows}, strides[2] = {d * e, (cuuint64_t)q_stride * e};
    const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)ta.nodes_per_item};
    if (!make_map(&maps[0], q, 3, dims, strides, box)) LMSF_REFUSE("attention_tree: no tensor map of the queries");
  }
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t dims[3] = {d, (cuuint64_t)n_kv_heads, (cuuint64_t)n_rows}, strides[2] = {d * e, (cuuint64_t)(i ? v_stride : k_stride) * e};
    const cuuint32_t box[3] = {64, 1, 32};
    if (!make_map(&maps[1 + i], i ? v : k, 3, dims, strides, box)) LMSF_REFUSE("attention_tree: no tensor map of the drafted tokens' keys");
  }
  {
    const cuuint64_t dims[4] = {d, (cuuint64_t)block_size, 2 * (cuuint64_t)n_kv_heads, (cuuint64_t)pages};
    const cuuint64_t strides[3] = {d * e, (cuuint64_t)block_size * d * e, (cuuint64_t)page_stride * e};
    const cuuint32_t box[4] = {64, (cuuint32_t)ta.rows_box, 1, 1};
    if (!make_map(&maps[3], cache, 4, dims, strides, box)) LMSF_REFUSE("attention_tree: no tensor map of the cache");
  }
  const size_t smem = kOffWork + work_bytes(n_seqs) + 1024;
  static bool raised[64] = {};
  int dev = 0;
  cudaError_t rc = cudaGetDevice(&dev);
  if (rc != cudaSuccess) return (int)rc;
  if (dev < 64 && !raised[dev]) {
    rc = cudaFuncSetAttribute(attention_tree_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kOffWork + work_bytes(kMaxSeqs) + 1024));
    if (rc != cudaSuccess) return (int)rc;
    raised[dev] = true;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int status = launch_pdl(attention_tree_tc_kernel, dim3(sms), dim3(kThreadsTotal), smem, st, ta, maps[0], maps[1], maps[2], maps[3]);
  if (status) return status;
  return launch_pdl(join_kernel<bf16, BM, 2, 128>, dim3(sms, 2 * BM / 32), dim3(256), 0, st, ta.a, (bool)ta.wide_out);
}
