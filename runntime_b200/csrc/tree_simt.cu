// Attention of a tree of drafted tokens over the caches (rt_attn_tree) on the FP32 pipes: f32, and f16
// where the tensor cores' copies cannot read the rows (tree_tc.cu).
//
// A row is one (node, query head) pair; the query heads that share a kv head are stacked with the nodes,
// so that a block reads each key and value once for BM of them.  Online softmax over tiles of 64 keys: the
// cache's tiles in turn, then one of the nodes' own keys, whose visibility is a bit of the row's mask.  Keys
// a row does not see have no part in its sums, whatever their values hold.
//
// Scores and outputs are blocked in registers, 4 x 4 and 4 x 8 per thread (half or a quarter of the rows for calls of
// up to 32 and 16), which makes shared memory and the FP32 pipes about equally busy.
// Splits of the key range leave (m, l, acc), which a second launch joins.
//
// Large calls are bound by the FP32 pipes and by shared memory: f32, 16 x 2000 rows, 32 tokens of 32 heads on 8 of 128,
// 536 us, 20 TFLOP/s.  Small ones are a chain of latencies, one tile to a block: f32, 4 sequences of 2000 rows, 12 tokens of
// 8 heads on 4 of 64 in a window of 512, 15.7 us, of which a block takes 5.4 (masks, Q and the lengths, asked for together,
// 0.8; the tile 1.4; scores, softmax and outputs 3.2) and the rest is the two launches, and the joining's own loads.
#include "speculate.cuh"
#include "sm100.cuh"

namespace rt {
namespace {

constexpr int kThreads = 256;
constexpr int BK = 64;
constexpr int kSplitMax = 64;
constexpr float kLn2 = 0.6931471805599453f;

// e^(x - m).  The difference comes first: it is exact next to the maximum, where the weights are, and a
// product with log2(e) before it would be off by as much as the score's own last bits.
__device__ __forceinline__ float exp_from(float x, float m) { return sm100::fast_exp2((x - m) * kLog2e); }

// Elements between rows of K in shared memory: 16-byte rows an odd number of them apart, so that eight
// threads on eight consecutive keys meet no bank twice.
__host__ __device__ constexpr int pitch_of(int hd4) { return (hd4 / 4) & 1 ? hd4 : hd4 + 4; }

template <int BM, int HDP>
constexpr int smem_bytes() {   // the probabilities take the keys' place
  const int k = BK * pitch_of(HDP), p = BM * (BK + 4);
  return (BM * HDP + BK * HDP + (k > p ? k : p)) * 4;
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* at) {   // (on a boundary of four elements)
  if constexpr (sizeof(T) == 2) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    return *reinterpret_cast<const float4*>(at);
  }
}

// Rows [0, BK) of a tile to shared memory as f32, zeros past `live` and past hd.  Zero, or a NaN where one of
// the thread's numbers is not finite.
template <typename T, int HDP, int PITCH, bool VECTOR>
__device__ __forceinline__ float stage(float* dst, const T* src, int64_t stride, int live, int hd) {
  constexpr int PER = VECTOR ? 4 : 1;
  constexpr int UNITS = HDP / PER;
  float odd = 0.f;
#pragma unroll 4
  for (int u = threadIdx.x; u < BK * UNITS; u += kThreads) {
    const int r = u / UNITS, c = (u - r * UNITS) * PER;
    if constexpr (VECTOR) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < live && c < hd) v = load4(src + r * stride + c);
      *reinterpret_cast<float4*>(dst + r * PITCH + c) = v;
      odd = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, odd))));
    } else {
      const float v = r < live && c < hd ? to_f32(src[r * stride + c]) : 0.f;
      dst[r * PITCH + c] = v;
      odd = fmaf(v, 0.f, odd);
    }
  }
  return odd;
}

template <typename T, int BM, int HDP, bool VECTOR>
__global__ void __launch_bounds__(kThreads, 2) tree_simt_kernel(const TreeParams p) {
  constexpr int TM = BM / 16;                 // rows of a thread
  constexpr int CG = (HDP + 63) / 64;         // groups of four columns of a thread
  constexpr int KP = pitch_of(HDP);
  extern __shared__ float smem[];
  float* sQ = smem;                           // [BM][HDP]
  float* sV = sQ + BM * HDP;                  // [BK][HDP]
  float* sK = sV + BK * HDP;                  // [BK][KP]
  float* sP = sK;                             // [BM][BK + 4], once the scores are there
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int group = p.qHeads / p.kvHeads, kvh = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % p.splits, mTile = blockIdx.x / p.splits;
  grid_dependency_wait();
  // (The joining launch is not let in early: 16.2 us for 15.7 at 4 sequences in a window of 512.)

  // What does not hang on the lengths is asked for beside them: the rows' masks and Q, whatever its rows past the
  // sequence's nodes hold.
  const uint64_t* masks = tree_masks(p, b);
  uint64_t mask[TM];
  int node[TM], head[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const int r = mTile * BM + ty * TM + i;
    node[i] = r / group;
    head[i] = kvh * group + (r - node[i] * group);
    mask[i] = node[i] < p.nodes ? masks[node[i]] : 0;
  }
  int len, nodes;
  tree_sequence(p, b, len, nodes);
  const bool qVector = VECTOR && p.qStride % 4 == 0 && reinterpret_cast<uintptr_t>(p.q) % (4 * sizeof(T)) == 0;
#pragma unroll 2
  for (int u = tid; u < BM * HDP / 4; u += kThreads) {
    const int i = u / (HDP / 4), c = (u - i * (HDP / 4)) * 4, r = mTile * BM + i;
    const int n = r / group, h = kvh * group + (r - n * group);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n < p.nodes && c < p.hd) {
      const T* at = static_cast<const T*>(p.q) + ((int64_t)b * p.nodes + n) * p.qStride + (int64_t)h * p.hd + c;
      if (qVector) {
        v = load4(at);
      } else {
        v.x = to_f32(at[0]);
        if (c + 1 < p.hd) v.y = to_f32(at[1]);
        if (c + 2 < p.hd) v.z = to_f32(at[2]);
        if (c + 3 < p.hd) v.w = to_f32(at[3]);
      }
    }
    *reinterpret_cast<float4*>(sQ + u * 4) = v;
  }
  TreeRow row[TM];
  bool live[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) {
    live[i] = node[i] < nodes;
    row[i].nodes = 0;
    row[i].lo = len;
    if (live[i]) row[i] = tree_row(p, masks, mask[i], len, nodes);
  }
  // The tiles of the cache from the first row that any node of the block sees (depths only grow from zero),
  // then the nodes' own; every split takes a run of them.
  int first = 0;
  if (p.wl != RT_WINDOW_INF && len > p.wl) first = (len - p.wl) / BK;
  const int cacheTiles = (len + BK - 1) / BK - first;
  const int tiles = nodes > 0 ? (cacheTiles > 0 ? cacheTiles : 0) + 1 : 0;
  const int t0 = (int)((int64_t)tiles * split / p.splits), t1 = (int)((int64_t)tiles * (split + 1) / p.splits);

  float m[TM], l[TM], acc[TM][CG][4];
#pragma unroll
  for (int i = 0; i < TM; i++) {
    // (sinks arrive in the log2 domain; the first split's block counts them)
    const bool sink = p.sinks && split == 0 && live[i];
    m[i] = sink ? fmaxf(p.sinks[head[i]] * kLn2, kNegSeed) : kNegSeed;
    l[i] = m[i] > kNegSeed ? 1.f : 0.f;
#pragma unroll
    for (int g = 0; g < CG; g++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[i][g][e] = 0.f;
  }

  for (int t = t0; t < t1; t++) {
    const bool own = t == tiles - 1;
    const int key0 = own ? 0 : (first + t) * BK;
    const int have = own ? nodes : min(len - key0, BK);
    const bool hides = own || (p.wl != RT_WINDOW_INF && key0 < (int64_t)len + RT_MAX_NODES - p.wl);   // from some rows
    __syncthreads();
    const T* k = own ? static_cast<const T*>(p.kNew) + (int64_t)b * p.nodes * p.kNewStride
                     : static_cast<const T*>(p.kCache) + b * p.cacheSeqStride + (int64_t)key0 * p.kvHeads * p.hd;
    const T* v = own ? static_cast<const T*>(p.vNew) + (int64_t)b * p.nodes * p.vNewStride
                     : static_cast<const T*>(p.vCache) + b * p.cacheSeqStride + (int64_t)key0 * p.kvHeads * p.hd;
    const int64_t kStride = own ? p.kNewStride : (int64_t)p.kvHeads * p.hd;
    const int64_t vStride = own ? p.vNewStride : (int64_t)p.kvHeads * p.hd;
    stage<T, HDP, KP, VECTOR>(sK, k + (int64_t)kvh * p.hd, kStride, have, p.hd);
    const float odd = stage<T, HDP, HDP, VECTOR>(sV, v + (int64_t)kvh * p.hd, vStride, have, p.hd);
    // A key that a row does not see may hold anything: where some of the tile's values are not finite they are
    // met key by key below.
    const bool apart = __syncthreads_or(hides && odd != 0.f);

    // Scores: rows ty*TM.., keys tx + 16 j.
    float s[TM][4];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll 8
    for (int c = 0; c < HDP; c += 4) {
      float4 qv[TM], kv[4];
#pragma unroll
      for (int i = 0; i < TM; i++) qv[i] = *reinterpret_cast<const float4*>(sQ + (ty * TM + i) * HDP + c);
#pragma unroll
      for (int j = 0; j < 4; j++) kv[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * KP + c);
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
          s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
          s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
          s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
        }
    }
    __syncthreads();
    // Softmax step.  A row's sixteen threads are neighbours.
#pragma unroll
    for (int i = 0; i < TM; i++) {
      float top = -INFINITY;
      bool sees[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int key = tx + 16 * j;
        sees[j] = key < have && (own ? (row[i].nodes >> key & 1) != 0 : key0 + key >= row[i].lo) && live[i];
        if (!sees[j]) s[i][j] = -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mNew = fmaxf(m[i], top);
      const float f = exp_from(m[i], mNew);
      m[i] = mNew;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float e = sees[j] ? exp_from(s[i][j], mNew) : 0.f;
        sum += e;
        sP[(ty * TM + i) * (BK + 4) + tx + 16 * j] = e;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = l[i] * f + sum;
#pragma unroll
      for (int g = 0; g < CG; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[i][g][e] *= f;
    }
    __syncwarp();   // (a warp reads only the rows that it has written)
    // Output: columns tx*4 + 64 g.
    const int keys = (have + 3) & ~3;
#pragma unroll 4
    for (int c = 0; c < keys; c += 4) {
      float4 pv[TM];
#pragma unroll
      for (int i = 0; i < TM; i++) pv[i] = *reinterpret_cast<const float4*>(sP + (ty * TM + i) * (BK + 4) + c);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int g = 0; g < CG; g++) {
          const int col = tx * 4 + 64 * g;
          if (HDP % 64 != 0 && col >= HDP) continue;
          const float4 vv = *reinterpret_cast<const float4*>(sV + (c + e) * HDP + col);
#pragma unroll
          for (int i = 0; i < TM; i++) {
            const float w = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
            if (apart && w == 0.f) continue;
            acc[i][g][0] = fmaf(w, vv.x, acc[i][g][0]);
            acc[i][g][1] = fmaf(w, vv.y, acc[i][g][1]);
            acc[i][g][2] = fmaf(w, vv.z, acc[i][g][2]);
            acc[i][g][3] = fmaf(w, vv.w, acc[i][g][3]);
          }
        }
    }
  }

#pragma unroll
  for (int i = 0; i < TM; i++) {
    if (node[i] >= p.nodes) continue;
    const int64_t at = ((int64_t)b * p.nodes + node[i]) * p.qHeads + head[i];
    if (p.splits == 1) {
      const float inv = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
      T* out = static_cast<T*>(p.out) + at * p.hd;
#pragma unroll
      for (int g = 0; g < CG; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int col = tx * 4 + 64 * g + e;
          if (col < p.hd) out[col] = from_f32<T>(l[i] == 0.f ? 0.f : acc[i][g][e] * inv);
        }
    } else {
      float* dst = p.scratch + (at * p.splits + split) * (2 + p.hd);
      if (tx == 0) dst[0] = m[i], dst[1] = l[i];
#pragma unroll
      for (int g = 0; g < CG; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int col = tx * 4 + 64 * g + e;
          if (col < p.hd) dst[2 + col] = acc[i][g][e];
        }
    }
  }
}

// One warp per (node, query head): weights of the splits, then the columns.
constexpr int kMergeWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(const TreeParams p) {
  __shared__ float weights[kMergeWarps][kSplitMax];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * kMergeWarps + warp;
  grid_dependency_wait();
  if (at >= (int64_t)p.batch * p.nodes * p.qHeads) return;
  const float* src = p.scratch + at * p.splits * (2 + p.hd);
  const int pitch = 2 + p.hd;
  float m0 = kNegSeed, m1 = kNegSeed, l0 = 0.f, l1 = 0.f;
  if (lane < p.splits) m0 = src[lane * pitch], l0 = src[lane * pitch + 1];
  if (lane + 32 < p.splits) m1 = src[(lane + 32) * pitch], l1 = src[(lane + 32) * pitch + 1];
  const float top = warp_max(fmaxf(l0 == 0.f ? kNegSeed : m0, l1 == 0.f ? kNegSeed : m1));
  const float f0 = l0 == 0.f ? 0.f : exp_from(m0, top), f1 = l1 == 0.f ? 0.f : exp_from(m1, top);
  const float l = warp_sum(l0 * f0 + l1 * f1);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane < p.splits) weights[warp][lane] = f0 * inv;
  if (lane + 32 < p.splits) weights[warp][lane + 32] = f1 * inv;
  __syncwarp();
  T* out = static_cast<T*>(p.out) + at * p.hd;
  for (int c = lane; c < p.hd; c += 32) {
    float sum = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.splits; s++) {
      const float w = weights[warp][s];
      if (w != 0.f) sum = fmaf(w, src[s * pitch + 2 + c], sum);   // (a split without keys has left no columns)
    }
    out[c] = from_f32<T>(sum);
  }
}

template <typename T, int BM, int HDP>
cudaError_t launch_hd(const TreeParams& p, bool vector, cudaStream_t s) {
  auto kern = vector ? tree_simt_kernel<T, BM, HDP, true> : tree_simt_kernel<T, BM, HDP, false>;
  constexpr int smem = smem_bytes<BM, HDP>();
  static std::atomic<uint64_t> allowed[2];
  const cudaError_t e = allow_shared(reinterpret_cast<const void*>(kern), smem, allowed[vector]);
  if (e != cudaSuccess) return e;
  const int rows = p.nodes * (p.qHeads / p.kvHeads);
  return launch_dependent(kern, dim3((unsigned)((rows + BM - 1) / BM * p.splits), (unsigned)p.kvHeads, (unsigned)p.batch),
                          dim3(kThreads), smem, s, p);
}

template <typename T, int BM>
cudaError_t launch_bm(const TreeParams& p, cudaStream_t s) {
  // Rows read four elements at a time where every one starts on a multiple of them.
  auto al = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % (4 * sizeof(T)) == 0; };
  const bool vector = p.hd % 4 == 0 && p.cacheSeqStride % 4 == 0 && p.kNewStride % 4 == 0 && p.vNewStride % 4 == 0 &&
                      al(p.kCache) && al(p.vCache) && al(p.kNew) && al(p.vNew);
  if (p.hd <= 32) return launch_hd<T, BM, 32>(p, vector, s);
  if (p.hd <= 64) return launch_hd<T, BM, 64>(p, vector, s);
  if (p.hd <= 96) return launch_hd<T, BM, 96>(p, vector, s);
  return launch_hd<T, BM, 128>(p, vector, s);
}

// Rows of a block: the fewest of 16, 32 and 64 that hold a kv head's, or 64.
int rows_of(const TreeParams& p) {
  const int rows = p.nodes * (p.qHeads / p.kvHeads);
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

}  // namespace

void plan_tree_simt(TreeParams& p, int smCount) {
  if (p.splits > 0) return;
  const int bm = rows_of(p), rows = p.nodes * (p.qHeads / p.kvHeads);
  const int64_t units = (int64_t)p.batch * p.kvHeads * ((rows + bm - 1) / bm);
  const int seen = p.wl != RT_WINDOW_INF && p.wl < p.kvLen ? p.wl : p.kvLen;
  const int tiles = (seen + BK - 1) / BK + 1;
  // Two blocks to an SM, or four of the few rows that a block has registers and shared memory to spare with, one tile at
  // least to a split.  (A tile takes longer than the joining of its part: 4 x 2000 rows
  // in a window of 512, 24 rows and 4 kv heads of 64, 28.2 us with two tiles at least.)
  int64_t splits = (bm == 16 && p.hd <= 64 ? 4 : 2) * smCount / units;
  if (splits > tiles) splits = tiles;
  p.splits = splits < 1 ? 1 : splits > kSplitMax ? kSplitMax : (int)splits;
}

cudaError_t launch_tree_simt(const TreeParams& p, int dtype, cudaStream_t s) {
  const int bm = rows_of(p);
  if (dtype == RT_F16)
    return bm == 16 ? launch_bm<__half, 16>(p, s) : bm == 32 ? launch_bm<__half, 32>(p, s) : launch_bm<__half, 64>(p, s);
  return bm == 16 ? launch_bm<float, 16>(p, s) : bm == 32 ? launch_bm<float, 32>(p, s) : launch_bm<float, 64>(p, s);
}

cudaError_t launch_tree_merge(const TreeParams& p, int dtype, cudaStream_t s) {
  const int64_t rows = (int64_t)p.batch * p.nodes * p.qHeads;
  const dim3 grid((unsigned)((rows + kMergeWarps - 1) / kMergeWarps));
  auto kern = dtype == RT_F16 ? tree_merge_kernel<__half> : tree_merge_kernel<float>;
  return launch_dependent(kern, grid, dim3(kMergeWarps * 32), 0, s, p);
}

}  // namespace rt
