// The operators of a speculative decode step: parameters, launchers and what their kernels share.
#pragma once

#include <atomic>

#include "common.cuh"

namespace rt {

// Lets a kernel have `bytes` of shared memory on the current device; asked for once on each (`done` is the kernel's own: a
// bit for each device; the call takes 0.4 us).
inline cudaError_t allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (e != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// ---- attention of a tree of drafted tokens (rt_attn_tree) ----------------------------------------
struct TreeParams {
  const void* q;
  void* out;
  const void* kCache;
  const void* vCache;
  const void* kNew;
  const void* vNew;
  const int32_t* kvLens;
  const int32_t* counts;
  const uint64_t* masks;
  const float* sinks;
  float* scratch;       // FP32 pipes, splits > 1: [batch*nodes*qHeads][splits][2+hd] f32 (m, l, acc); tensor cores, cut inside heads:
                        // the accumulators, (m, l) and joins of tree_tc.cu's Plan
  int* status;
  int64_t cacheSeqStride, qStride, kNewStride, vNewStride;   // elements
  int32_t batch, nodes, cacheRows, kvLen, qHeads, kvHeads, hd, wl, sharedMasks, splits;
  uint32_t polls;       // for a free place in a ring of tiles before the kernel gives up
};

#ifdef __CUDACC__
// Rows in the cache and nodes of sequence b; a length outside its bounds is recorded and leaves nothing.
__device__ __forceinline__ void tree_sequence(const TreeParams& p, int b, int& rows, int& nodes) {
  rows = p.kvLens ? p.kvLens[b] : p.kvLen;
  nodes = p.counts ? p.counts[b] : p.nodes;
  if (rows < 0 || rows > p.cacheRows || nodes < 0 || nodes > p.nodes) {
    atomicOr(p.status, kStatusBadState);
    rows = nodes = 0;
  }
}

// What node i of sequence b sees: nodes (a bit each) and cache rows from lo on.
struct TreeRow {
  uint64_t nodes;
  int lo;
};
__device__ __forceinline__ const uint64_t* tree_masks(const TreeParams& p, int b) {
  return p.masks + (p.sharedMasks ? 0 : (int64_t)b * p.nodes);
}
__device__ __forceinline__ TreeRow tree_row(const TreeParams& p, const uint64_t* m, uint64_t mask, int rows, int nodes) {
  const uint64_t live = nodes >= 64 ? ~0ull : (1ull << nodes) - 1;
  TreeRow r;
  r.nodes = mask & live;
  r.lo = 0;
  if (p.wl != RT_WINDOW_INF) {
    const int depth = max(__popcll(r.nodes) - 1, 0);
    const int64_t lo = (int64_t)rows + depth - p.wl;
    r.lo = lo > 0 ? (int)min(lo, (int64_t)rows) : 0;
    if (depth > p.wl)   // (nodes further up than the window reaches)
      for (int j = 0; j < nodes; j++)
        if ((r.nodes >> j & 1) && depth - max(__popcll(m[j] & live) - 1, 0) > p.wl) r.nodes &= ~(1ull << j);
  }
  return r;
}
__device__ __forceinline__ TreeRow tree_row(const TreeParams& p, int b, int i, int rows, int nodes) {
  const uint64_t* m = tree_masks(p, b);
  return tree_row(p, m, m[i], rows, nodes);
}
#endif

// How the FP32-pipe kernel cuts the call: fills splits where they are 0.
void plan_tree_simt(TreeParams& p, int smCount);
cudaError_t launch_tree_simt(const TreeParams& p, int dtype, cudaStream_t s);
// The splits' partials into out, a second launch.
cudaError_t launch_tree_merge(const TreeParams& p, int dtype, cudaStream_t s);

// On the tensor cores (f16, rows that TMA can read): scratch that the call wants (0: none), and the call; whole: cut
// at the ends of heads, with no scratch.
bool tree_tc_supported(const TreeParams& p, int dtype);
size_t tree_tc_scratch(const TreeParams& p, int smCount);
cudaError_t launch_tree_tc(const TreeParams& p, int smCount, bool whole, int* launches, cudaStream_t s, std::string* err);

cudaError_t launch_rotary(const rt_rotary_args& a, int smCount, cudaStream_t s);
cudaError_t launch_verify(const rt_verify_args& a, int* status, int smCount, cudaStream_t s);
// committed (or NULL): the rows that each sequence got.
cudaError_t launch_commit(const rt_commit_args& a, int32_t* committed, int* status, int smCount, int* launches, cudaStream_t s);

}  // namespace rt
