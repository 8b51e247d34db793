// Attention of a tree of drafted tokens over the caches (rt_attn_tree) on the tensor cores: f16 caches whose
// rows TMA can read.
//
// The (node, query head) pairs of one kv head are the rows of 128-row MMA tiles, so that a key or a
// value comes from memory once for all of them.  The tiles of a (sequence, kv head), 64 cache rows each
// after one of the nodes' own keys, are one long line over all sequences and heads, which persistent streams cut
// into equal runs: ragged lengths and odd numbers of heads leave no SM waiting.  A run may begin or end inside a
// (sequence, kv head); such a part leaves (m, l, acc) in scratch and a second launch joins the parts.  Where the call is
// small the cuts are at the ends of heads, and there is no second launch.
//
// A block, one per SM, has two softmax warpgroups, a thread to a row, each with its own MMA issuer and half of tensor
// memory.  Up to 128 rows (what bounds that is the caches' bytes) each of them is a stream of its own: while one is at
// a part's end or beginning, the other goes on.  More rows are taken two tiles at a time by the two warpgroups of one
// stream, which share every K and V tile: read by a block each, they met the limit of the L2.  (One
// warpgroup after another on the tiles of one part, sharing the rows' reference points, the scheme of the prefill
// kernel, stopped at every part's end: 32 x 8190 rows, 25 tokens 200 us for 161; 65001 rows, 64 tokens 102 for 92, both with
// probabilities of one half.)
//
// What it takes with 32 heads on 8 of 128: 32 sequences of 8190 rows, 25 tokens 187 us, 4.5 TB/s (the caches' bytes at
// the copy rate: 128); 16 of 4096 at most, 16 tokens 56 us, 3.7 TB/s, of which some 9 pass before the first product and 6 in
// the joining launch; one of 65001, 64 tokens 110 us, 619 TFLOP/s counting each product once: a chain of scores, softmax and the
// product of the probabilities, whose place the next scores take.  (Probabilities of one half, 11 bits: 162, 53 and 92 us.)
// The smallest, 8 heads of 52, 190 rows and 7 tokens: 12 us, all of it latency.
//
// A producer warp for each stream fills rings of K and V tiles by TMA that run on across the parts' ends.  Scores have
// two buffers of 64 columns; the probabilities take their scores' place, each as two halves, its upper eleven bits and
// the rest, that are multiplied by the same values: one half alone made results half again as far off as
// their own rounding to f16 does.  A row's reference point moves only when its maximum has grown by more than seven
// binary orders, and O is rescaled then.
//
// What a row does not see has no part in its result, whatever it holds: values past the length, and values
// that are not finite in tiles that some rows see in part, are cleared in shared memory, and a row whose result
// is not finite, or that sees a cleared value, is computed again key by key at the block's end.
#include <algorithm>
#include <climits>

#include "speculate.cuh"
#include "sm100.cuh"
#include "tc_common.cuh"

namespace rt {
namespace {

using namespace sm100;
using namespace tc;

constexpr int kThreads = 384;
constexpr int BK = 64;                               // keys of a tile
static_assert(BK == RT_MAX_NODES, "the nodes' own keys are one tile");
constexpr float kLn2 = 0.6931471805599453f;
// A row's reference point is set kLift binary orders below its maximum and moves when the maximum is kTop above it: a
// probability, 2^(s - reference) in f32, is at most 2^15, and what two halves leave of it is 2^-22 of it or
// 2^-25, which is 2^-33 of the row's largest.  (kLift 10, 6 and 2: 65001 rows and 64 tokens 112, 110 and 108 us, with 8 111.)
constexpr float kLift = 8.f, kTop = 15.f;

template <int HD>
struct Cfg {
  static constexpr int Q_BYTES = BM * HD * 2;        // of a warpgroup
  static constexpr int SLOT_BYTES = BK * HD * 2;
  static constexpr int SLOTS = HD == 128 ? 10 : 20;  // of keys and values together
  // of each, in a stream alone and in each of two
  static constexpr int K1 = SLOTS / 2, V1 = SLOTS / 2, K2 = HD == 128 ? 3 : 5, V2 = HD == 128 ? 2 : 5;
  static_assert(K1 + V1 <= SLOTS && 2 * (K2 + V2) <= SLOTS, "rings");
  // Tensor memory of a warpgroup: two buffers of scores and the accumulator.
  static constexpr int S_COL = 0, O_COL = 2 * BK, WG_COLS = 256, TMEM_COLS = 512;
};
constexpr int kMaxSlots = 10;     // of keys or of values
constexpr int kFlags = 32;        // twice the parts (of a tile at least) that two warpgroups of a stream are apart at most
static_assert(kFlags / 2 >= kMaxSlots + 2, "a ring's length and the tiles in hand");

// A part of a stream's run: tiles [t0, t1) of (b, kvh).
struct Part {
  int b, kvh, t0, t1, rows, nodes, first, tiles;   // t0 == t1: a sequence without nodes; t0 < 0: no more; tiles: of the whole (b, kvh)
};

// What a block shares beside Q and the rings.  [2]: by stream or by warpgroup.
struct Shared {
  uint64_t kFull[kMaxSlots], kEmpty[kMaxSlots], vFull[kMaxSlots], vEmpty[kMaxSlots];
  uint64_t sFull[2][2], pReady[2][2], pvDone[2][2];   // of a warpgroup, by the tile's parity
  uint64_t partReady[2][2], partDone[2][2];           // ..., by the part's
  uint64_t qFull[2];
  uint64_t looked[2][2];                              // tiles of a stream that have been looked through, by their number's
  unsigned long long spoilt[2][kFlags];   // nodes whose values are not all finite, by the part's number
  int spoiltRow[2][kFlags];               // and the last such cache row among tiles that some rows see in part, or -1
  Part part[2][2];
  // Tiles of keys and of values that a stream has asked for, Qs of a warpgroup: what may be on its way when a block gives up.
  int asked[2][2], askedQ[2];
  uint64_t over[2];                                   // then: all products of a warpgroup are done
  int marked[2];                                      // whether rows of a warpgroup are to be computed again
  uint32_t tmem;
  int abort;
};
template <int HD>
constexpr int smem_bytes() { return 2 * Cfg<HD>::Q_BYTES + Cfg<HD>::SLOTS * Cfg<HD>::SLOT_BYTES + (int)sizeof(Shared); }
static_assert(smem_bytes<128>() <= 227 * 1024 && smem_bytes<64>() <= 227 * 1024, "shared memory of a block");

struct Plan {
  int32_t mTiles, groups;   // runs: one to a stream (pairs of row tiles share one)
  int32_t solo;             // one row tile: two streams to a block
  int32_t whole;            // cut at the ends of (sequence, kv head) only
  int32_t qNodes;           // nodes of a row tile where TMA fetches Q, or 0
  int32_t heads4;           // the maps have a dimension of heads: no neighbour's columns in a tile
  float* acc;               // [groups][2][mTiles][HD/4][128][4]
  float* ml;                // [groups][2][mTiles][128][2]
  int2* joins;              // [batch * kvHeads]: twice the run of its first part, plus that part's place (-1: it is the only
                            // one); the run of its last part.  Unwritten where the launch that writes it has given up
};

// Tiles of a sequence: one of the nodes' own keys, then the cache's from `first` on.
struct Sequence {
  int rows, nodes, first, tiles;
};
__device__ __forceinline__ Sequence sequence_of(const TreeParams& p, int b) {
  Sequence s;
  s.rows = p.kvLens ? p.kvLens[b] : p.kvLen;
  s.nodes = p.counts ? p.counts[b] : p.nodes;
  if (s.rows < 0 || s.rows > p.cacheRows || s.nodes < 0 || s.nodes > p.nodes) s.rows = s.nodes = 0;
  s.first = p.wl != RT_WINDOW_INF && s.rows > p.wl ? (s.rows - p.wl) / BK : 0;
  s.tiles = s.nodes > 0 ? 1 + max((s.rows + BK - 1) / BK - s.first, 0) : 0;
  return s;
}

// First tile of run g: total * g / groups (the division of 64 bits takes a microsecond, most calls do without).
__device__ __forceinline__ int64_t run_begin(int64_t total, int g, int groups) {
  const int64_t x = total * g;
  return x >> 32 ? x / groups : (int64_t)((uint32_t)x / (uint32_t)groups);
}

// A stream's run, part by part: tiles [t0, t1) of (b, kvh).  All lanes of a warp hold the same.
struct Walk {
  int b, kvh, t0, t1;
  Sequence s;
  int64_t left;     // tiles (or, cut at the ends of heads, (sequence, head) pairs) still to come
  int start;        // first tile of the next part

  __device__ __forceinline__ void begin(const TreeParams& p, const Plan& plan, int group) {
    const int lane = threadIdx.x & 31;
    start = 0;
    if (plan.whole) {
      const int64_t units = (int64_t)p.batch * p.kvHeads;
      const int64_t u0 = units * group / plan.groups;
      left = units * (group + 1) / plan.groups - u0;
      b = (int)(u0 / p.kvHeads);
      kvh = (int)(u0 - (int64_t)b * p.kvHeads);
      if (left > 0) s = sequence_of(p, b);
      return;
    }
    // Sums of tiles by sequence, 32 at a time: their total, then the sequence that holds this run's first tile.
    auto tiles_of = [&](int x) { return x < p.batch ? sequence_of(p, x).tiles : 0; };
    const int firsts = tiles_of(lane);
    int64_t total = firsts;
    for (int b0 = 32; b0 < p.batch; b0 += 32) total += tiles_of(b0 + lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= p.kvHeads;
    // (no run is empty: where there are fewer tiles than streams, as many runs as tiles)
    const int groups = (int)min((int64_t)plan.groups, total);
    left = 0;
    if (group >= groups) return;
    const int64_t at = run_begin(total, group, groups);
    left = run_begin(total, group + 1, groups) - at;
    int64_t before = 0;
    for (int b0 = 0;; b0 += 32) {
      const int64_t mine = (b0 == 0 ? firsts : tiles_of(b0 + lane)) * (int64_t)p.kvHeads;
      int64_t upTo = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upTo, o);
        if (lane >= o) upTo += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upTo > at);
      if (hit) {   // (`at` is below the total: some sequence holds it)
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        before += __shfl_sync(0xffffffffu, upTo - mine, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upTo, 31);
    }
    s = sequence_of(p, b);
    const int64_t in = at - before;
    kvh = (int)((uint32_t)in / (uint32_t)s.tiles);   // (a sequence has fewer than 2^31 tiles in all heads: see plan_of)
    start = (int)(in - (int64_t)kvh * s.tiles);
  }
  __device__ __forceinline__ Part part() const { return {b, kvh, t0, t1, s.rows, s.nodes, s.first, s.tiles}; }
  // The next part; false at the run's end.  (A part of no tiles is a sequence without nodes.)
  __device__ __forceinline__ bool next(const TreeParams& p, const Plan& plan) {
    if (left <= 0) return false;
    if (kvh == p.kvHeads) {
      kvh = 0;
      do {
        if (++b >= p.batch) return false;   // (not with lengths that stay as they are during the call)
        s = sequence_of(p, b);
      } while (!plan.whole && s.tiles == 0);
    }
    t0 = start;
    start = 0;
    if (plan.whole) {
      t1 = s.tiles;
      left--;
    } else {
      t1 = (int)min((int64_t)s.tiles, t0 + left);
      left -= t1 - t0;
    }
    return true;
  }
  __device__ __forceinline__ void advance() { kvh++; }
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int h, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(h), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Tile t of the walk's part into a slot: keys or values by the map.
template <int HD, bool PADDED>
__device__ __forceinline__ void load_tile(const CUtensorMap* map, const Plan& plan, int hd, const Walk& walk, int t, uint32_t dst,
                                          uint32_t bar) {
  const int x0 = plan.heads4 ? 0 : PADDED ? (walk.kvh * hd) & ~7 : walk.kvh * HD;
  const int h = plan.heads4 ? walk.kvh : 0, y = t == 0 ? 0 : (walk.s.first + t - 1) * BK;
  constexpr int chunkBytes = BK * 128;
  mbar_expect_tx(bar, HD / 64 * chunkBytes);
#pragma unroll
  for (int c = 0; c < HD / 64; c++) tma_load_4d(dst + c * chunkBytes, map, x0 + c * 64, h, y, walk.b, bar);
}

// After a failed wait, by all warps of the block: it does not end, and its shared memory is nobody else's, while copies into it
// and products that read it may be on their way, also those of a role that had come to its end before.  (Waits with a
// limit, too.)
__device__ __noinline__ void wait_for_what_is_asked(Shared& sh, int nK, int nV) {
  volatile int never = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto all = [&](uint64_t* full, int slots, int asked) {
    for (int q = max(asked - slots, 0); q < asked; q++) mbar_poll_warp(smem_u32(&full[q % slots]), (q / slots) & 1, &never);
  };
  if (warp == 8 || warp == 11) {
    const int s = warp == 11;
    all(sh.kFull + s * nK, nK, sh.asked[s][0]);
    all(sh.vFull + s * nV, nV, sh.asked[s][1]);
  } else if (warp == 9 || warp == 10) {
    const int g = warp - 9;
    all(&sh.qFull[g], 1, sh.askedQ[g]);
    if (lane == 0) {
      mbar_init(smem_u32(&sh.over[g]), 1);
      fence_barrier_init();
    }
    __syncwarp();
    if (elect_one()) tc_commit(smem_u32(&sh.over[g]));
    __syncwarp();
    mbar_poll_warp(smem_u32(&sh.over[g]), 0, &never);
  }
}

// One row over a part's tiles by one warp, a key to a lane for the scores: the result's columns (lane, lane + 32, ...), the
// maximum and the sum.
__device__ __forceinline__ void exact_tree_row(const TreeParams& p, const Part& s, int node, int head, const TreeRow& row,
                                               float (&acc)[4], float& m, float& l) {
  const int lane = threadIdx.x & 31, hd = p.hd;
  const __half* q = static_cast<const __half*>(p.q) + ((int64_t)s.b * p.nodes + node) * p.qStride + (int64_t)head * hd;
  // (rows of keys begin on 16-byte boundaries, heads and queries where hd and q's stride let them)
  const bool wide = hd % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  m = p.sinks && s.t0 == 0 ? fmaxf(p.sinks[head] * kLn2, kNegSeed) : kNegSeed;
  l = m > kNegSeed ? 1.f : 0.f;
#pragma unroll
  for (int c = 0; c < 4; c++) acc[c] = 0.f;
  for (int t = s.t0; t < s.t1; t++) {
    const bool own = t == 0;
    const int key0 = own ? 0 : (s.first + t - 1) * BK, end = own ? s.nodes : min(s.rows, key0 + BK);
    const int64_t stride = own ? p.kNewStride : (int64_t)p.kvHeads * hd, vStride = own ? p.vNewStride : stride;
    const int64_t column = (int64_t)s.kvh * hd;
    const __half* k = own ? static_cast<const __half*>(p.kNew) + (int64_t)s.b * p.nodes * p.kNewStride
                          : static_cast<const __half*>(p.kCache) + s.b * p.cacheSeqStride;
    const __half* v = own ? static_cast<const __half*>(p.vNew) + (int64_t)s.b * p.nodes * p.vNewStride
                          : static_cast<const __half*>(p.vCache) + s.b * p.cacheSeqStride;
    for (int j0 = key0; j0 < end; j0 += 32) {
      const int j = j0 + lane;
      const bool sees = j < end && (own ? (row.nodes >> j & 1) != 0 : j >= row.lo);
      if (!__any_sync(0xffffffffu, sees)) continue;
      float x = 0.f;
      if (sees) {
        const __half* kj = k + j * stride + column;
        if (wide) {
#pragma unroll 8
          for (int c = 0; c < hd; c += 8) {
            const uint4 a = *reinterpret_cast<const uint4*>(q + c), b = *reinterpret_cast<const uint4*>(kj + c);
            const __half2 *a2 = reinterpret_cast<const __half2*>(&a), *b2 = reinterpret_cast<const __half2*>(&b);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float2 u = __half22float2(a2[e]), w = __half22float2(b2[e]);
              x = fmaf(u.y, w.y, fmaf(u.x, w.x, x));
            }
          }
        } else {
#pragma unroll 8
          for (int c = 0; c < hd; c++) x = fmaf(__half2float(q[c]), __half2float(kj[c]), x);
        }
      }
      const float mNew = fmaxf(m, warp_max(sees ? x : -INFINITY)), f = fast_exp2((m - mNew) * kLog2e);
      const float mine = sees ? fast_exp2((x - mNew) * kLog2e) : 0.f;
      l = l * f + warp_sum(mine);
      m = mNew;
#pragma unroll
      for (int c = 0; c < 4; c++) acc[c] *= f;
      // (eight keys' values on their way at a time; those past the last key are the last key's, with no weight)
      const int keys = min(end - j0, 32);
#pragma unroll 1
      for (int i0 = 0; i0 < keys; i0 += 8) {
        __half x[8][4];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const __half* vi = v + (j0 + min(i0 + i, keys - 1)) * vStride + column;
#pragma unroll
          for (int c = 0; c < 4; c++) x[i][c] = lane + 32 * c < hd ? vi[lane + 32 * c] : __half(0.f);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float w = __shfl_sync(0xffffffffu, mine, i0 + i);
#pragma unroll
          for (int c = 0; c < 4; c++) acc[c] = w != 0.f ? fmaf(w, __half2float(x[i][c]), acc[c]) : acc[c];
        }
      }
    }
  }
}

// Q of a part into shared memory by one warp, in 16-byte units of the swizzled K-major layout, in the background where
// the rows' alignment allows that; the caller waits (cp.async.wait_all) and fences.
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool read, bool wide) {
  if (wide) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(read ? 8 : 0) : "memory");
}
template <int HD, bool PADDED>
__device__ __forceinline__ void stage_q(const TreeParams& p, int b, int kvh, int nodes, int mTile, int shift, uint32_t sQ) {
  constexpr int kUnits = HD / 8, kStep = 32 / kUnits;   // a lane keeps its columns and goes down the rows
  const int lane = threadIdx.x & 31, heads = p.qHeads / p.kvHeads, hd = PADDED ? p.hd : HD;
  const int rows = min(nodes * heads - mTile * BM, BM);
  const __half* qg = static_cast<const __half*>(p.q);
  const bool wide = shift == 0 && hd % 8 == 0 && p.qStride % 8 == 0 && (reinterpret_cast<uintptr_t>(qg) & 15) == 0;
  const bool quads = hd % 4 == 0 && p.qStride % 4 == 0 && (reinterpret_cast<uintptr_t>(qg) & 7) == 0;
  const int cu = lane % kUnits, c0 = cu * 8 - shift;
  int qr = lane / kUnits, node = (mTile * BM + qr) / heads, h = mTile * BM + qr - node * heads;
  const __half* src = qg + ((int64_t)b * p.nodes + node) * p.qStride + (int64_t)(kvh * heads + h) * hd;
  const int64_t nextNode = p.qStride - (int64_t)heads * hd;
  const uint32_t column = sQ + (cu >> 3) * (BM * 128);
#pragma unroll 1
  for (; qr < rows; qr += kStep) {
    const uint32_t dst = column + qr * 128 + (((cu & 7) ^ (qr & 7)) << 4);
    // (columns outside the head are zeros; their addresses are the row's start)
    if (wide) {
      const bool in = c0 < hd;
      copy_async(dst, src + (in ? c0 : 0), in, true);
    } else if (quads) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const bool in = c0 + e >= 0 && c0 + e < hd;
        copy_async(dst + 2 * e, src + (in ? c0 + e : 0), in, false);
      }
    } else {
      uint32_t e[8];
#pragma unroll
      for (int x = 0; x < 8; x++) e[x] = c0 + x >= 0 && c0 + x < hd ? __half_as_ushort(src[c0 + x]) : 0u;
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(e[0] | e[1] << 16), "r"(e[2] | e[3] << 16),
                   "r"(e[4] | e[5] << 16), "r"(e[6] | e[7] << 16)
                   : "memory");
    }
#pragma unroll
    for (int k = 0; k < kStep; k++) {
      src += hd;
      if (++h == heads) h = 0, src += nextNode;
    }
  }
}

// What this row sees of a part; and its sink, if this is the part that counts it, or the seed.
__device__ __forceinline__ TreeRow row_of_part(const TreeParams& p, const Part& part, int node, int head, float& seen) {
  TreeRow row;      // (rows without a node go along: what they make is not stored)
  row.nodes = 0;
  row.lo = 0;
  seen = kNegSeed;
  if (node < part.nodes) {
    if (part.t0 == 0 || p.wl != RT_WINDOW_INF) row = tree_row(p, part.b, node, part.rows, part.nodes);
    if (p.sinks && part.t0 == 0) seen = fmaxf(p.sinks[head] - kLift, kNegSeed);   // (in the log2 domain)
  }
  return row;
}

// A row's scores in tensor memory: -inf but for the node bits, or for the columns [c0, c1).
__device__ __noinline__ void hide_scores(uint32_t sCol, bool own, uint64_t nodes, int c0, int c1) {
#pragma unroll 1
  for (int u = 0; u < BK / 32; u++) {
    const int a = max(c0 - 32 * u, 0), z = min(c1 - 32 * u, 32);
    uint32_t bits = a < z ? (0xffffffffu >> (32 - z)) & (0xffffffffu << a) : 0u;
    if (own) bits = u == 0 ? (uint32_t)nodes : u == 1 ? (uint32_t)(nodes >> 32) : 0u;
    if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
    uint32_t x[32];
    tmem_ld32(sCol + 32 * u, x);
    tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < 32; c++) x[c] = bits >> c & 1u ? x[c] : 0xff800000u;
    tmem_st32(sCol + 32 * u, x);
  }
  tmem_wait_st();
}

// Part `which` of `of` of a tile of V in shared memory, by a warpgroup: rows from the live ones to the end of their step
// of 16 keys (later steps are not multiplied) are cleared, and, if looked through, values within them that are not
// finite, which are recorded.
template <int HD>
__device__ __noinline__ void clear_values(uint32_t tile, bool own, bool look, int key0, int liveRows, int which, int of,
                                          unsigned long long* spoilt, int* spoiltRow) {
  constexpr int kUnits = HD / 8;   // of 16 bytes in a row
  const int thread = (threadIdx.x & 127) + 128 * which, threads = 128 * of;
  auto place = [&](int u, int& r) {
    r = u / kUnits;
    const int c = u % kUnits;
    return tile + (c >> 3) * (BK * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  };
  const int end = (liveRows + 15) & ~15;
  int r;
#pragma unroll 1
  for (int u = liveRows * kUnits + thread; u < end * kUnits; u += threads)
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(place(u, r)), "r"(0u) : "memory");
  if (look)
#pragma unroll 1
    for (int u = thread; u < liveRows * kUnits; u += threads) {
      const uint32_t at = place(u, r);
      uint32_t x[4], odd = 0u;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
      // a half is infinite or NaN if its exponent is all ones: the addition carries into its sign's place
#pragma unroll
      for (int e = 0; e < 4; e++) odd |= ((x[e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
      if (odd) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] &= ~(((((x[e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u) >> 15) * 0xffffu);
        if (own) atomicOr(spoilt, 1ull << r);
        else atomicMax(spoiltRow, key0 + r);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
      }
    }
  fence_proxy_async();
}

// A row of a sequence without nodes is zeros; a length out of its bounds is recorded.
__device__ __noinline__ void no_nodes(const TreeParams& p, const Part& part, int node, int head, bool here, int hd) {
  if (part.kvh == 0 && (threadIdx.x & 127) == 0) {
    int a, c;
    tree_sequence(p, part.b, a, c);
  }
  if (!here) return;
  __half* out = static_cast<__half*>(p.out) + (((int64_t)part.b * p.nodes + node) * p.qHeads + head) * hd;
  for (int c = 0; c < hd; c++) out[c] = __float2half_rn(0.f);
}

// What a row that is to be computed again has in the place of its first column, or of its sum: NaNs that no arithmetic makes.
constexpr unsigned short kAgain = 0x7e01;
constexpr uint32_t kAgainSum = 0x7fc00001u;

// The results of a part's rows: to `out` where the part is a whole (sequence, kv head), else as (m, l, acc).  Returns whether
// the row has been marked: the `odd` ones and those that are not finite.  Where a row's scores are all its own (settled: no
// neighbour's columns were multiplied by zeros) a sum that is NaN comes from a score that it sees, and
// the row is NaN as it should be.
template <int HD, bool PADDED>
__device__ __forceinline__ bool store_rows(const TreeParams& p, const Part& part, int node, int head, bool here, int shift,
                                           uint32_t oCol, float m, float l, bool odd, bool settled, float* acc, float* ml) {
  const int rowInTile = threadIdx.x & 127, hd = PADDED ? p.hd : HD;
  const bool final = part.t0 == 0 && part.t1 == part.tiles;
  const bool valid = node < part.nodes;
  const float inv = 1.f / l;
  const uint32_t keep = valid && l != 0.f ? ~0u : 0u;   // rows without a node and rows that see nothing are zeros
  __half* out = static_cast<__half*>(p.out) + (((int64_t)part.b * p.nodes + node) * p.qHeads + head) * hd;
  const bool wide = !PADDED && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const bool quads = hd % 4 == 0 && shift % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
  float check = l * 0.f;   // NaN if anything is not finite
#pragma unroll 1
  for (int c = 0; c < HD; c += 32) {
    uint32_t o[32];
    tmem_ld32(oCol + c, o);
    tmem_wait_ld();
#pragma unroll
    for (int x = 0; x < 32; x++)
      if (!PADDED || (c + x >= shift && c + x < shift + hd)) check = fmaf(__uint_as_float(o[x]), 0.f, check);
    if (!here) continue;
    if (!final) {
#pragma unroll
      for (int x = 0; x < 32; x += 4)
        *reinterpret_cast<uint4*>(acc + ((c + x) / 4 * BM + rowInTile) * 4) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
      continue;
    }
#pragma unroll
    for (int x = 0; x < 16; x++) {
      const __half2 hp = __floats2half2_rn(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv);
      o[x] = *reinterpret_cast<const uint32_t*>(&hp) & keep;
    }
    if (wide) {
#pragma unroll
      for (int x = 0; x < 16; x += 4)
        *reinterpret_cast<uint4*>(out + c + 2 * x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
    } else if (quads) {   // (a quad of the tile is inside the head or outside as a whole)
#pragma unroll
      for (int x = 0; x < 32; x += 4)
        if (c + x >= shift && c + x < shift + hd) *reinterpret_cast<uint2*>(out + c + x - shift) = make_uint2(o[x / 2], o[x / 2 + 1]);
    } else {
#pragma unroll
      for (int x = 0; x < 32; x++)
        if (c + x >= shift && c + x < shift + hd)
          out[c + x - shift] = __ushort_as_half((unsigned short)(x & 1 ? o[x / 2] >> 16 : o[x / 2]));
    }
  }
  const bool again = (odd || check != 0.f) && here && valid && !(settled && l != l);
  if (!final && here)
    *reinterpret_cast<float2*>(ml + 2 * rowInTile) = make_float2(m * kLn2, again ? __uint_as_float(kAgainSum) : valid ? l : 0.f);
  if (final && again) *reinterpret_cast<unsigned short*>(out) = kAgain;
  return again;
}

// The marked rows of a run, key by key: at the block's end, by all of its warps and where nobody waits for them.  (Between a
// warpgroup's parts, by the warp whose rows they were, they took longer than the waits of its stream may.)  256 rows of 8 heads
// over 65001 keys: 18 ms.
__device__ __noinline__ void redo_rows(const TreeParams& p, const Plan& plan, int columns, int group, int mTile) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = p.qHeads / p.kvHeads;
  Walk walk;
  walk.begin(p, plan, group);
  for (int index = 0; walk.next(p, plan); walk.advance(), index++) {
    const Part part = walk.part();
    if (part.t0 == part.t1) continue;
    const bool final = part.t0 == 0 && part.t1 == part.tiles;
    const int shift = columns != p.hd && !plan.heads4 ? (part.kvh * p.hd) & 7 : 0;
    const int64_t place = ((int64_t)group * 2 + (index > 0 ? 1 : 0)) * plan.mTiles + mTile;
    float* const acc = plan.acc + place * (columns * BM);
    float* const ml = plan.ml + place * (2 * BM);
    for (int x = warp; x < BM; x += kThreads / 32) {
      const int r = mTile * BM + x, node = r / heads, head = part.kvh * heads + r - node * heads;
      if (node >= part.nodes) break;
      __half* out = static_cast<__half*>(p.out) + (((int64_t)part.b * p.nodes + node) * p.qHeads + head) * p.hd;
      if (final ? *reinterpret_cast<const unsigned short*>(out) != kAgain : __float_as_uint(ml[2 * x + 1]) != kAgainSum) continue;
      const TreeRow row = tree_row(p, part.b, node, part.rows, part.nodes);
      float a[4], m, l;
      exact_tree_row(p, part, node, head, row, a, m, l);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int col = lane + 32 * c;
        if (col >= p.hd) continue;
        if (final) out[col] = __float2half_rn(a[c] * inv);
        else acc[((col + shift) / 4 * BM + x) * 4 + (col + shift) % 4] = a[c];
      }
      if (!final && lane == 0) ml[2 * x] = m, ml[2 * x + 1] = l;
    }
  }
}

// HD: columns of the tile, 64 or 128.  PADDED: the head is narrower, at columns [shift, shift + p.hd) of it.
template <int HD, bool PADDED>
__global__ void __launch_bounds__(kThreads, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
               const __grid_constant__ CUtensorMap mapKNew, const __grid_constant__ CUtensorMap mapVNew,
               const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ TreeParams p, const __grid_constant__ Plan plan) {
  using C = Cfg<HD>;
  extern __shared__ __align__(1024) unsigned char smemRaw[];
  Shared& sh = *reinterpret_cast<Shared*>(smemRaw + 2 * C::Q_BYTES + C::SLOTS * C::SLOT_BYTES);
  const uint32_t sQ = smem_u32(smemRaw), sRing = sQ + 2 * C::Q_BYTES;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hd = PADDED ? p.hd : HD;
  // Warpgroup g: which stream of the block it belongs to, that stream's run, its row tile.
  const int pairs = (plan.mTiles + 1) / 2;
  auto stream_of = [&](int g) { return plan.solo ? g : 0; };
  auto run_of = [&](int g) { return plan.solo ? 2 * (int)blockIdx.x + g : (int)blockIdx.x / pairs; };
  auto tile_of = [&](int g) { return plan.solo ? 0 : 2 * ((int)blockIdx.x % pairs) + g; };
  auto active = [&](int g) { return run_of(g) < plan.groups && tile_of(g) < plan.mTiles; };
  const int consumers = plan.solo ? 1 : active(1) ? 2 : 1;       // warpgroups of a stream
  const int nK = plan.solo ? C::K2 : C::K1, nV = plan.solo ? C::V2 : C::V1;
  auto kSlot = [&](int s, int j) { return s * nK + j % nK; };
  auto vSlot = [&](int s, int j) { return s * nV + j % nV; };
  const uint32_t sV = sRing + (plan.solo ? 2 : 1) * nK * C::SLOT_BYTES;
  auto shift_of = [&](int kvh) { return PADDED && !plan.heads4 ? (kvh * hd) & 7 : 0; };
  auto bar = [](const uint64_t& b) { return smem_u32(&b); };

  if (tid == 0) {
    sh.abort = (sQ & 1023u) != 0;   // (there is no static shared memory before it)
    sh.marked[0] = sh.marked[1] = 0;
    for (int i = 0; i < kMaxSlots; i++) {
      mbar_init(bar(sh.kFull[i]), 1);
      mbar_init(bar(sh.kEmpty[i]), consumers);
      mbar_init(bar(sh.vFull[i]), 1);
      mbar_init(bar(sh.vEmpty[i]), consumers);
    }
    for (int g = 0; g < 2; g++) {
      mbar_init(bar(sh.qFull[g]), 1);
      for (int i = 0; i < 2; i++) {
        mbar_init(bar(sh.sFull[g][i]), 1);
        mbar_init(bar(sh.pReady[g][i]), 4);
        mbar_init(bar(sh.pvDone[g][i]), 1);
        mbar_init(bar(sh.partReady[g][i]), 1);
        mbar_init(bar(sh.partDone[g][i]), 4);
        mbar_init(bar(sh.looked[g][i]), 4 * consumers);
      }
      for (int i = 0; i < kFlags; i++) sh.spoilt[g][i] = 0, sh.spoiltRow[g][i] = -1;
    }
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tensormap(&mapK);
    prefetch_tensormap(&mapV);
    prefetch_tensormap(&mapKNew);
    prefetch_tensormap(&mapVNew);
    prefetch_tensormap(&mapQ);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&sh.tmem), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem;
  volatile int* const abortFlag = &sh.abort;
  auto wait = [&](const uint64_t& b, int parity) { return mbar_poll_warp(smem_u32(&b), (uint32_t)parity & 1u, abortFlag); };
  grid_dependency_wait();
  // The next launch's blocks may be set up meanwhile, but not those of the joining launch, which are many.
  if (plan.whole) grid_launch_dependents();

  // Every warp finds the beginning of its run, in one place: written out in each role the code took longer to arrive
  // than to run (16 x 4096 rows: 4.7 us of the issuers' 10 before their first product).
  const int mine = warp < 8 ? warp >> 2 : warp == 9 || warp == 10 ? warp - 9 : warp == 11;   // its warpgroup or stream
  Walk walk;
  walk.left = 0;
  if (warp >= 8 && (warp != 11 || plan.solo) && active(mine)) walk.begin(p, plan, run_of(mine));
  bool ok = !*abortFlag;
  // Tiles of which some rows see a part: their values are looked through for what others may not meet.
  auto looks = [&](int t, int key0, int rows) { return t == 0 || (p.wl != RT_WINDOW_INF && key0 < (int64_t)rows + RT_MAX_NODES - p.wl); };

  if (warp == 8 || warp == 11) {
    // ------------------------------ keys and values of a stream ------------------------------
    const int s = warp == 8 ? 0 : 1;
    int count[2] = {0, 0};
    if (ok && (s == 0 || plan.solo) && active(s)) {
      // The next tile of keys and the next one of values, each fetched when its slot is free.
      Walk walks[2] = {walk, walk};
      int at[2];
      bool more[2];
      auto forward = [&](Walk& w, int& t, bool& m) {
        while (m && t == w.t1) {
          w.advance();
          m = w.next(p, plan);
          if (m) t = w.t0;
        }
      };
#pragma unroll
      for (int x = 0; x < 2; x++) {
        more[x] = walks[x].next(p, plan);
        at[x] = more[x] ? walks[x].t0 : 0;
        forward(walks[x], at[x], more[x]);
      }
      uint32_t idle = 0;
      while (more[0] || more[1]) {
        bool moved = false;
#pragma unroll
        for (int x = 0; x < 2; x++) {
          if (!more[x]) continue;
          const int n = x ? nV : nK, slot = x ? vSlot(s, count[x]) : kSlot(s, count[x]);
          const uint64_t* empty = x ? sh.vEmpty : sh.kEmpty;
          const uint64_t* full = x ? sh.vFull : sh.kFull;
          if (count[x] >= n && !__all_sync(0xffffffffu, mbar_test_wait(bar(empty[slot]), (uint32_t)(count[x] / n - 1) & 1u))) continue;
          if (elect_one())
            load_tile<HD, PADDED>(at[x] == 0 ? (x ? &mapVNew : &mapKNew) : (x ? &mapV : &mapK), plan, hd, walks[x], at[x],
                                  (x ? sV : sRing) + slot * C::SLOT_BYTES, bar(full[slot]));
          __syncwarp();
          count[x]++;
          at[x]++;
          forward(walks[x], at[x], more[x]);
          moved = true;
        }
        if (moved) {
          idle = 0;
          continue;
        }
        // (the limit is that of the other waits, a second or two, by default; a limit of one poll does not wait at all)
        if (idle++ / 16 + 1 >= p.polls || (idle % 32 == 0 && *abortFlag)) {
          *abortFlag = 1;
          break;
        }
        __nanosleep(64);
        __syncwarp();
      }
    }
    if (lane == 0) sh.asked[s][0] = count[0], sh.asked[s][1] = count[1];
  } else if (warp == 9 || warp == 10) {
    // ------------------------------ MMA issuer of a warpgroup, and its parts' beginnings ------------------------------
    const int g = warp - 9, s = stream_of(g), mTile = tile_of(g);
    int qParts = 0;   // parts with a Q
    if (ok && active(g)) {
      constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // SBO, version, SW128
      constexpr uint32_t kLboK = (16u >> 4) << 16, kLboV = ((uint32_t)(BK * 128) >> 4) << 16;   // V: next 64 columns
      auto desc = [](uint32_t lo32) { return ((uint64_t)kDescHi << 32) | lo32; };
      const uint32_t myQ = sQ + g * C::Q_BYTES, aLo = ((myQ & 0x3ffffu) >> 4) | kLboK;
      const uint32_t sCol = tmem + g * C::WG_COLS + C::S_COL, oCol = tmem + g * C::WG_COLS + C::O_COL;
      int j = 0, index = 0, seen = 0;   // tiles, parts, tiles looked through
      for (; ok && walk.next(p, plan); walk.advance(), index++) {
        const int shift = shift_of(walk.kvh), n = walk.t1 - walk.t0;
        // (the part before last is over; the last one's scores are all there, so Q is read no more)
        if (index >= 2) ok = wait(sh.partDone[g][index & 1], index / 2 - 1);
        if (!ok) break;
        if (n > 0 && plan.qNodes) {
          if (elect_one()) {
            const uint32_t chunk = (p.qHeads / p.kvHeads) * plan.qNodes * 128;
            mbar_expect_tx(bar(sh.qFull[g]), HD / 64 * chunk);
#pragma unroll
            for (int c = 0; c < HD / 64; c++)
              tma_load_4d(myQ + c * (BM * 128), &mapQ, c * 64, walk.kvh * (p.qHeads / p.kvHeads), mTile * plan.qNodes, walk.b,
                          bar(sh.qFull[g]));
          }
          __syncwarp();
        } else if (n > 0) {
          stage_q<HD, PADDED>(p, walk.b, walk.kvh, walk.s.nodes, mTile, shift, myQ);
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async();
        }
        if (lane == 0) sh.part[g][index & 1] = walk.part();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(sh.partReady[g][index & 1]));
        const int kSteps = PADDED ? (shift + hd + 15) / 16 : HD / 16;  // K = 16 per instruction
        const uint32_t idescO = instr_desc(PADDED ? (shift + hd + 15) & ~15 : HD, true);
        auto scores = [&](int jj) {
          const int slot = kSlot(s, jj);
          ok = wait(sh.kFull[slot], jj / nK);
          if (!ok) return;
          tc_fence_after_sync();
          if (elect_one()) {
            const uint32_t bLo = (((sRing + slot * C::SLOT_BYTES) & 0x3ffffu) >> 4) | kLboK;
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
              if (PADDED && kk >= kSteps) break;
              const uint32_t off = (kk >> 2), low = (kk & 3) * 2;
              mma_f16_ss(sCol + (jj & 1) * BK, desc(aLo + off * ((BM * 128) >> 4) + low), desc(bLo + off * ((BK * 128) >> 4) + low),
                         instr_desc(BK, false), kk > 0);
            }
            tc_commit(bar(sh.kEmpty[slot]));
            tc_commit(bar(sh.sFull[g][jj & 1]));
          }
          __syncwarp();
        };
        // (P(j-2)'s buffer, and O: the last product of the part before is waited for below, and the part's first
        // probabilities come after its results have been read)
        if (n > 0 && plan.qNodes) {
          ok = wait(sh.qFull[g], qParts++);
          if (!ok) break;
        }
        if (n > 0) scores(j);
        for (int i = 0; ok && i < n; i++, j++) {
          // S(j+1) goes into the buffer that P(j-1) has left.
          if (j >= 1) ok = wait(sh.pvDone[g][(j - 1) & 1], (j - 1) >> 1);
          if (ok && i + 1 < n) scores(j + 1);
          const int t = walk.t0 + i, key0 = t == 0 ? 0 : (walk.s.first + t - 1) * BK, slot = vSlot(s, j);
          const int keys = t == 0 ? walk.s.nodes : min(walk.s.rows - key0, BK), steps = (keys + 15) / 16;
          if (ok) ok = wait(sh.vFull[slot], j / nV);
          if (ok && (looks(t, key0, walk.s.rows) || keys < BK)) {
            ok = wait(sh.looked[s][seen & 1], seen >> 1);
            seen++;
          }
          if (ok) ok = wait(sh.pReady[g][j & 1], j >> 1);
          if (!ok) break;
          tc_fence_after_sync();
          if (elect_one()) {
            const uint32_t bLo = (((sV + slot * C::SLOT_BYTES) & 0x3ffffu) >> 4) | kLboV;
            const uint32_t pCol = sCol + (j & 1) * BK;
            auto product = [&](int kk) {   // 16 keys, the probabilities' upper and lower halves
              const uint64_t v = desc(bLo + kk * (2048 >> 4));
              mma_f16_ts(oCol, pCol + kk * 8, v, idescO, (i > 0 || kk > 0) ? 1u : 0u);
              mma_f16_ts(oCol, pCol + BK / 2 + kk * 8, v, idescO, 1u);
            };
            if (steps == BK / 16) {
#pragma unroll
              for (int kk = 0; kk < BK / 16; kk++) product(kk);
            } else {
#pragma unroll 1
              for (int kk = 0; kk < steps; kk++) product(kk);
            }
            tc_commit(bar(sh.vEmpty[slot]));
            tc_commit(bar(sh.pvDone[g][j & 1]));
          }
          __syncwarp();
        }
      }
      if (ok && index >= 2) ok = wait(sh.partDone[g][index & 1], index / 2 - 1);
      if (ok && lane == 0) {
        sh.part[g][index & 1].t0 = -1;   // no more
        mbar_arrive(bar(sh.partReady[g][index & 1]));
      }
      if (!ok) *abortFlag = 1;
    }
    if (lane == 0) sh.askedQ[g] = qParts;
  } else {
    // ------------------------------ softmax and results of a warpgroup ------------------------------
    const int g = warp >> 2, s = stream_of(g), mTile = tile_of(g), rowInTile = tid & 127;
    const uint32_t laneBase = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t sCol = tmem + laneBase + g * C::WG_COLS + C::S_COL, oCol = tmem + laneBase + g * C::WG_COLS + C::O_COL;
    const int heads = p.qHeads / p.kvHeads, r = mTile * BM + rowInTile, node = r / heads, headIn = r - node * heads;
    const bool here = node < p.nodes;
    const bool warpLive = __any_sync(0xffffffffu, here);
    int j = 0, lookedAt = 0, live = 0;   // tiles, tiles looked through, parts with tiles so far
    for (int index = 0; ok && active(g); index++) {
      ok = wait(sh.partReady[g][index & 1], index / 2);
      if (!ok) break;
      const Part part = sh.part[g][index & 1];
      if (part.t0 < 0) break;   // no more
      const int n = part.t1 - part.t0, head = part.kvh * heads + headIn, shift = shift_of(part.kvh);
      if (n == 0) {   // a sequence without nodes (cut at the ends of heads: no other block has its rows)
        no_nodes(p, part, node, head, here, hd);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(sh.partDone[g][index & 1]));
        continue;
      }
      float seen;        // the row's reference point (log2 domain)
      const TreeRow row = row_of_part(p, part, node, head, seen);
      float l = seen != kNegSeed ? exp2f(kLift) : 0.f;      // the row's sink
      unsigned long long* const spoilt = &sh.spoilt[s][live % kFlags];
      int* const spoiltRow = &sh.spoiltRow[s][live % kFlags];
      if (rowInTile == 0 && (g == 0 || plan.solo))
        sh.spoilt[s][(live + kFlags / 2) % kFlags] = 0, sh.spoiltRow[s][(live + kFlags / 2) % kFlags] = -1;
      live++;

#pragma unroll 1
      for (int i = 0; i < n; i++, j++) {
        const int t = part.t0 + i, key0 = t == 0 ? 0 : (part.first + t - 1) * BK;
        const int keys = t == 0 ? part.nodes : min(part.rows - key0, BK);
        const bool look = looks(t, key0, part.rows);
        ok = wait(sh.sFull[g][j & 1], j >> 1);
        if (!ok) break;  // the whole warp leaves together
        tc_fence_after_sync();
        if (look || keys < BK) {
          // (S(j) was issued when P V(j-2) was done: the slot's phase before this one is over)
          const int slot = vSlot(s, j);
          ok = wait(sh.vFull[slot], j / nV);
          if (!ok) break;
          clear_values<HD>(sV + slot * C::SLOT_BYTES, t == 0, look, key0, keys, plan.solo ? 0 : g, consumers, spoilt, spoiltRow);
          __syncwarp();
          // (a tile of this kind cannot be two behind another: that one's product comes between)
          if (lane == 0) mbar_arrive(bar(sh.looked[s][lookedAt & 1]));
          lookedAt++;
        }
        const uint32_t sBuf = sCol + (j & 1) * BK;
        if (warpLive) {
          // Scores that their row does not see become -inf where they are, in tensor memory: on the way through the
          // registers the compiler made selections on every tile of it.
          if (__any_sync(0xffffffffu, t == 0 || row.lo > key0 || keys < BK))
            hide_scores(sBuf, t == 0, row.nodes, row.lo - key0, part.rows - key0);
          uint32_t sv[BK];
          tmem_ld32(sBuf, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
          tmem_ld32(sBuf + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
          tmem_wait_ld();
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < BK; c += 8)
#pragma unroll
            for (int u = 0; u < 4; u++) mx4[u] = max3(mx4[u], __uint_as_float(sv[c + 2 * u]), __uint_as_float(sv[c + 2 * u + 1]));
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * kLog2e;
          const bool grow = mx > seen + kTop;
          if (__any_sync(0xffffffffu, grow)) {
            // A row whose reference point is still the seed has met no key: its accumulator row is zero.
            const bool pass = i > 0 && __any_sync(0xffffffffu, grow && seen != kNegSeed);
            // (a row moves by itself: rows without a node, whose scores are whatever was there, move no other)
            const float mnew = grow || i == 0 || seen == kNegSeed ? fmaxf(seen, mx - kLift) : seen;
            const float f = fast_exp2(seen - mnew);
            if (pass) {
              // (S(j) is there: P V(j-2) is done, and the open phase of the other barrier is P V(j-1)'s)
              ok = wait(sh.pvDone[g][(j - 1) & 1], (j - 1) >> 1);
              if (!ok) break;
              tc_fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                tmem_ld32(oCol + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 32; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                tmem_st32(oCol + c, o);
              }
              tmem_wait_st();
            }
            l *= f;
            seen = mnew;
          }
          const float2 scale2 = make_float2(kLog2e, kLog2e), shift2 = make_float2(-seen, -seen);
          float2 sum2[4];
          uint32_t hi[32], lo[32];
#pragma unroll
          for (int u = 0; u < 4; u++) sum2[u] = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < BK; c += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), scale2, shift2);
            const float2 pe = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sum2[(c >> 1) & 3] = add2(sum2[(c >> 1) & 3], pe);
            // the upper eleven bits as they are, and what is left of it
            const float2 up = make_float2(__uint_as_float(__float_as_uint(pe.x) & 0xffffe000u), __uint_as_float(__float_as_uint(pe.y) & 0xffffe000u));
            const float2 rest = fma2(up, make_float2(-1.f, -1.f), pe);
            const __half2 hp = __floats2half2_rn(up.x, up.y), lp = __floats2half2_rn(rest.x, rest.y);
            hi[c / 2] = *reinterpret_cast<const uint32_t*>(&hp);
            lo[c / 2] = *reinterpret_cast<const uint32_t*>(&lp);
          }
          const float2 s01 = add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3]));
          l += s01.x + s01.y;
          tmem_st32(sBuf, hi);   // P in its scores' place
          tmem_st32(sBuf + BK / 2, lo);
          tmem_wait_st();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(sh.pReady[g][j & 1]));
      }
      if (!ok) break;

      // ---- the part's end ----
      ok = wait(sh.pvDone[g][(j - 1) & 1], (j - 1) >> 1);
      if (!ok) break;
      tc_fence_after_sync();
      if (warpLive) {
        // a run's first part goes to the first of its two places, its last to the second
        const int64_t place = ((int64_t)run_of(g) * 2 + (index > 0 ? 1 : 0)) * plan.mTiles + mTile;
        float* const acc = plan.acc + place * (HD * BM);
        float* const ml = plan.ml + place * (2 * BM);
        const bool odd = (*spoilt & row.nodes) || *spoiltRow >= row.lo;
        if (store_rows<HD, PADDED>(p, part, node, head, here, shift, oCol, seen, l, odd, !PADDED || plan.heads4, acc, ml))
          sh.marked[g] = 1;
      }
      if (!plan.whole && mTile == 0 && rowInTile == 0) {
        int2* const join = plan.joins + (int64_t)part.b * p.kvHeads + part.kvh;
        if (part.t0 == 0) join->x = part.t1 == part.tiles ? -1 : 2 * run_of(g) + (index > 0 ? 1 : 0);
        if (part.t1 == part.tiles) join->y = run_of(g);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(sh.partDone[g][index & 1]));
    }
    if (!ok) *abortFlag = 1;
  }

  // Common exit: every role arrives here, then the allocating warp frees tensor memory.
  tc_fence_before_sync();
  __syncthreads();
  if (*abortFlag) {
    wait_for_what_is_asked(sh, nK, nV);
    if (tid == 0) atomicOr(p.status, kStatusWaitTimeout);
    __syncthreads();
  } else if (sh.marked[0] | sh.marked[1]) {
    for (int g = 0; g < 2; g++)
      if (sh.marked[g]) redo_rows(p, plan, HD, run_of(g), tile_of(g));
  }
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// The parts of every (sequence, kv head) that lies in several runs, joined, COLS columns of a row to a thread: sixteen where
// that fills the GPU, else four (19 parts of 256 rows and 8 heads: 21 us with sixteen).  Heads that lie in one run
// have their results already.
template <int HD, int COLS>
__global__ void __launch_bounds__(256) tree_tc_merge_kernel(const TreeParams p, const Plan plan) {
  constexpr int kBlocks = HD / (2 * COLS);   // of a head
  const int mTile = blockIdx.z, kvh = blockIdx.y, b = blockIdx.x / kBlocks;
  const int row = threadIdx.x & 127, c0 = (blockIdx.x % kBlocks) * 2 * COLS + (threadIdx.x >> 7) * COLS;
  const int heads = p.qHeads / p.kvHeads, hd = p.hd, shift = HD != hd && !plan.heads4 ? (kvh * hd) & 7 : 0;
  const int r = mTile * BM + row, node = r / heads;
  grid_dependency_wait();
  const Sequence s = sequence_of(p, b);
  if (blockIdx.x % kBlocks == 0 && kvh == 0 && mTile == 0 && threadIdx.x == 0) {
    int a, c;
    tree_sequence(p, b, a, c);   // a length out of its bounds is recorded
  }
  if (node >= p.nodes) return;
  float sum[COLS];
#pragma unroll
  for (int c = 0; c < COLS; c++) sum[c] = 0.f;
  if (s.tiles > 0) {
    const int2 join = plan.joins[(int64_t)b * p.kvHeads + kvh];
    if (join.x < 0) return;
    // The runs after the first begin inside the head, so that it is their first part.
    const int g0 = join.x >> 1, g1 = join.y;
    // (a first launch that gave up has left the table unwritten, and in the scratch may be anything)
    if (g1 < g0 || g1 >= plan.groups) return;
    auto place = [&](int g) { return ((int64_t)g * 2 + (g == g0 ? join.x & 1 : 0)) * plan.mTiles + mTile; };
    float m = kNegSeed;
#pragma unroll 8
    for (int g = g0; g <= g1; g++) {
      const float2 ml = *reinterpret_cast<const float2*>(plan.ml + place(g) * (2 * BM) + 2 * row);
      if (ml.y != 0.f) m = fmaxf(m, ml.x);
    }
    float l = 0.f;
#pragma unroll (COLS == 4 ? 8 : 2)
    for (int g = g0; g <= g1; g++) {
      const float2 ml = *reinterpret_cast<const float2*>(plan.ml + place(g) * (2 * BM) + 2 * row);
      const float4* a = reinterpret_cast<const float4*>(plan.acc + place(g) * (HD * BM) + (c0 / 4 * BM + row) * 4);
      float4 v[COLS / 4];
#pragma unroll
      for (int c = 0; c < COLS / 4; c++) v[c] = a[c * BM];
      if (ml.y == 0.f) continue;   // (a part that this row sees nothing of: its columns may hold anything)
      const float w = fast_exp2((ml.x - m) * kLog2e);
      l = fmaf(w, ml.y, l);
#pragma unroll
      for (int c = 0; c < COLS / 4; c++) {
        sum[4 * c] = fmaf(w, v[c].x, sum[4 * c]);
        sum[4 * c + 1] = fmaf(w, v[c].y, sum[4 * c + 1]);
        sum[4 * c + 2] = fmaf(w, v[c].z, sum[4 * c + 2]);
        sum[4 * c + 3] = fmaf(w, v[c].w, sum[4 * c + 3]);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < COLS; c++) sum[c] *= inv;
  }
  __half* out = static_cast<__half*>(p.out) +
                (((int64_t)b * p.nodes + node) * p.qHeads + kvh * heads + r - node * heads) * hd + c0 - shift;
  const bool quads = hd % 4 == 0 && shift % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
#pragma unroll
  for (int c = 0; c < COLS; c += 4) {
    const __half2 lo = __floats2half2_rn(sum[c], sum[c + 1]), hi = __floats2half2_rn(sum[c + 2], sum[c + 3]);
    if (quads) {
      if (c0 + c >= shift && c0 + c < shift + hd)
        *reinterpret_cast<uint2*>(out + c) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      continue;
    }
    const __half v[4] = {__low2half(lo), __high2half(lo), __low2half(hi), __high2half(hi)};
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (c0 + c + e >= shift && c0 + c + e < shift + hd) out[c + e] = v[e];
  }
}

// Columns of the tile that holds every head: 64 or 128, 0 if none does.
int tile_columns(const TreeParams& p) {
  int most = p.hd;
  if (p.hd % 8 != 0)
    for (int h = 0; h < p.kvHeads && h < 8; h++) most = std::max(most, ((h * p.hd) & 7) + p.hd);
  return most <= 64 ? 64 : most <= 128 ? 128 : 0;
}

bool make_map4(CUtensorMap* map, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
               std::string* err) {
  auto fn = encode_fn();
  if (!fn) {
    *err = "cuTensorMapEncodeTiled is not available from the driver";
    return false;
  }
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    *err = "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r);
    return false;
  }
  return true;
}
// Rows of keys or values for all sequences, as columns of a head, heads, rows, sequences (heads4) or columns of the row,
// 1, rows, sequences; box = 64 columns x BK rows.
bool make_rows_map(CUtensorMap* map, const void* base, bool heads4, const TreeParams& p, int64_t rows, int64_t rowStride,
                   int64_t seqStride, std::string* err) {
  const cuuint64_t dims[4] = {(cuuint64_t)(heads4 ? p.hd : p.hd * p.kvHeads), (cuuint64_t)(heads4 ? p.kvHeads : 1),
                              (cuuint64_t)rows, (cuuint64_t)p.batch};
  const cuuint64_t strides[3] = {(cuuint64_t)(heads4 ? p.hd : rowStride) * 2, (cuuint64_t)rowStride * 2, (cuuint64_t)seqStride * 2};
  const cuuint32_t box[4] = {64, 1, BK, 1};
  return make_map4(map, base, dims, strides, box, err);
}

Plan plan_of(const TreeParams& p, int smCount, bool whole) {
  Plan plan{};
  const int64_t rows = (int64_t)p.nodes * (p.qHeads / p.kvHeads), units = (int64_t)p.batch * p.kvHeads;
  plan.mTiles = (int)((rows + BM - 1) / BM);
  plan.solo = plan.mTiles == 1;
  plan.groups = plan.solo ? 2 * smCount : std::max(smCount / ((plan.mTiles + 1) / 2), 1);
  plan.heads4 = p.hd % 8 == 0;
  const int64_t seen = p.wl != RT_WINDOW_INF && p.wl < p.kvLen ? p.wl : p.kvLen;
  const int64_t tiles = (seen + BK - 1) / BK + 1;
  // (a sequence's tiles in all heads are counted in 32 bits)
  whole = whole || p.kvHeads * tiles >= (1ll << 31);
  // Cut at the ends of heads unless an even cut saves more than the second launch takes, about four tiles' time.
  const int64_t turns = (units + plan.groups - 1) / plan.groups;
  plan.whole = whole || p.splits == 1 || (p.splits == 0 && turns * tiles <= units * tiles / plan.groups + 4);
  if (plan.whole) plan.groups = (int)std::min<int64_t>(plan.groups, units);
  else plan.groups = (int)std::min<int64_t>(plan.groups, units * tiles);
  return plan;
}

template <int HD, bool PADDED>
cudaError_t launch(const TreeParams& p, Plan& plan, int smCount, cudaStream_t s, std::string* err) {
  CUtensorMap k, v, kn, vn, q;
  // Q by TMA where its rows allow that and a row tile is whole nodes: heads of the group, then nodes, are its rows.
  const int heads = p.qHeads / p.kvHeads;
  plan.qNodes = 0;
  if (p.hd % 8 == 0 && p.qStride % 8 == 0 && (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && heads <= BM &&
      (plan.mTiles == 1 || BM % heads == 0))
    plan.qNodes = plan.mTiles == 1 ? p.nodes : BM / heads;
  if (plan.qNodes) {
    cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.qHeads, (cuuint64_t)p.nodes, (cuuint64_t)p.batch};
    cuuint64_t strides[3] = {(cuuint64_t)p.hd * 2, (cuuint64_t)p.qStride * 2, (cuuint64_t)p.nodes * p.qStride * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)heads, (cuuint32_t)plan.qNodes, 1};
    if (!make_map4(&q, p.q, dims, strides, box, err)) return cudaErrorInvalidValue;
  }
  const int64_t kvw = (int64_t)p.kvHeads * p.hd;
  if (!make_rows_map(&k, p.kCache, plan.heads4, p, p.cacheRows, kvw, p.cacheSeqStride, err) ||
      !make_rows_map(&v, p.vCache, plan.heads4, p, p.cacheRows, kvw, p.cacheSeqStride, err) ||
      !make_rows_map(&kn, p.kNew, plan.heads4, p, p.nodes, p.kNewStride, p.nodes * p.kNewStride, err) ||
      !make_rows_map(&vn, p.vNew, plan.heads4, p, p.nodes, p.vNewStride, p.nodes * p.vNewStride, err))
    return cudaErrorInvalidValue;
  if (!plan.qNodes) q = k;   // (not used; a valid map all the same)
  const int blocks = plan.solo ? (plan.groups + 1) / 2 : plan.groups * ((plan.mTiles + 1) / 2);
  auto kern = tree_tc_kernel<HD, PADDED>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_shared(reinterpret_cast<const void*>(kern), smem_bytes<HD>(), allowed);
  if (e != cudaSuccess) return e;
  e = launch_dependent(kern, dim3((unsigned)blocks), dim3(kThreads), smem_bytes<HD>(), s, k, v, kn, vn, q, p, plan);
  if (e != cudaSuccess || plan.whole) return e;
  const int64_t units = (int64_t)p.batch * p.kvHeads * plan.mTiles;
  const bool wide = units * (HD / 32) >= 2 * smCount;   // blocks of sixteen columns to a thread
  auto merge = wide ? tree_tc_merge_kernel<HD, 16> : tree_tc_merge_kernel<HD, 4>;
  return launch_dependent(merge, dim3((unsigned)p.batch * (HD / (wide ? 32 : 8)), (unsigned)p.kvHeads, (unsigned)plan.mTiles),
                          dim3(256), 0, s, p, plan);
}

}  // namespace

bool tree_tc_supported(const TreeParams& p, int dtype) {
  if (dtype != RT_F16 || tile_columns(p) == 0) return false;
  auto al = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  const int64_t kvw = (int64_t)p.kvHeads * p.hd;
  // TMA: 16-byte aligned bases, rows and sequences
  return al(p.kCache) && al(p.vCache) && al(p.kNew) && al(p.vNew) && kvw % 8 == 0 && p.cacheSeqStride % 8 == 0 &&
         p.kNewStride % 8 == 0 && p.vNewStride % 8 == 0 && encode_fn();
}

size_t tree_tc_scratch(const TreeParams& p, int smCount) {
  const Plan plan = plan_of(p, smCount, false);
  if (plan.whole) return 0;
  return (size_t)plan.groups * 2 * plan.mTiles * (tile_columns(p) * BM + 2 * BM) * sizeof(float) +
         (size_t)p.batch * p.kvHeads * sizeof(int2);
}

cudaError_t launch_tree_tc(const TreeParams& p, int smCount, bool whole, int* launches, cudaStream_t s, std::string* err) {
  Plan plan = plan_of(p, smCount, whole);
  const int hdt = tile_columns(p);
  plan.acc = p.scratch;
  plan.ml = p.scratch + (size_t)plan.groups * 2 * plan.mTiles * hdt * BM;
  plan.joins = reinterpret_cast<int2*>(plan.ml + (size_t)plan.groups * 2 * plan.mTiles * 2 * BM);
  *launches = plan.whole ? 1 : 2;
  if (hdt == 64) return p.hd == 64 ? launch<64, false>(p, plan, smCount, s, err) : launch<64, true>(p, plan, smCount, s, err);
  return p.hd == 128 ? launch<128, false>(p, plan, smCount, s, err) : launch<128, true>(p, plan, smCount, s, err);
}

}  // namespace rt
