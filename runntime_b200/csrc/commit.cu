// Commit of accepted rows to the ends of the caches (rt_commit_rows): a gather of a few rows per sequence
// for the K and V of all layers in one launch.
//
// A copy, so bandwidth-bound where it is large and bound by three dependent loads (length and count,
// index, row) where it is small.  A block takes one tensor and sequence, checks the sequence's
// indices once, and walks (row, column) pairs; where that leaves most SMs idle the rows are dealt out
// to several blocks.  64 sequences of up to 16 rows of 1024 f16, 16 tensors: 6.3 us for 29 MB read and written (4.6 TB/s,
// part of it from L2); one sequence of 7 rows of 288, 12 tensors: 1.7 us.
#include "speculate.cuh"

namespace rt {
namespace {

constexpr int kThreads = 256;
// Tensors of one launch: their addresses are its parameters, which a launch of few copies in a smaller structure.
constexpr int kFew = 16, kTensors = 128;

template <int N>
struct Params {
  void* caches[N];
  const void* fresh[N];
  const int32_t* index;
  const int32_t* counts;
  const int32_t* kvLens;
  int64_t cacheSeqStride, freshSeqStride, freshRowStride, width;   // in units of the copies
  int32_t* committed;
  int* status;
  int32_t nodes, cacheRows, lead, indexStride;
};

template <typename V, int N>
__global__ void __launch_bounds__(kThreads) commit_kernel(const __grid_constant__ Params<N> p) {
  __shared__ int from[RT_MAX_NODES];
  const int b = blockIdx.y;
  grid_dependency_wait();
  const int length = p.kvLens[b], count = p.counts[b];
  // (the index of a row is asked for beside the count that says whether it is one)
  const int j = threadIdx.x;
  int pick = j;
  if (j >= p.lead && j < p.nodes) pick = p.index[(int64_t)b * p.indexStride + j - p.lead];
  const int64_t n = (int64_t)count + p.lead;
  bool bad = count < 0 || n > p.nodes || length < 0 || length + n > p.cacheRows;
  if (!bad && j >= p.lead && j < n) {
    bad = pick < 0 || pick >= p.nodes - p.lead;
    pick += p.lead;
  }
  if (j < p.nodes) from[j] = pick;
  const bool refused = __syncthreads_or(bad);
  if (p.committed && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) p.committed[b] = refused ? 0 : (int32_t)n;
  if (refused) {
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadState);
    return;
  }
  V* cache = static_cast<V*>(p.caches[blockIdx.x]) + b * p.cacheSeqStride + length * p.width;
  const V* fresh = static_cast<const V*>(p.fresh[blockIdx.x]) + b * p.freshSeqStride;
  const int64_t rowsPerTurn = gridDim.z;
  if (p.width >= kThreads) {
    for (int64_t r = blockIdx.z; r < n; r += rowsPerTurn)
      for (int64_t c = threadIdx.x; c < p.width; c += kThreads) cache[r * p.width + c] = fresh[from[r] * p.freshRowStride + c];
  } else {
    const int w = (int)p.width, all = w * (int)((n - blockIdx.z + rowsPerTurn - 1) / rowsPerTurn);
    for (int i = threadIdx.x; i < all; i += kThreads) {
      const int k = i / w, c = i - k * w;
      const int64_t r = blockIdx.z + k * rowsPerTurn;
      cache[r * w + c] = fresh[from[r] * p.freshRowStride + c];
    }
  }
}

template <typename V, int N>
cudaError_t launch_n(const rt_commit_args& a, int32_t* committed, int elems, int* status, int smCount, int* launches,
                     cudaStream_t s) {
  const int64_t rowStride = a.freshRowStride ? a.freshRowStride : a.width;
  for (int first = 0; first < a.tensors; first += N) {
    const int count = a.tensors - first < N ? a.tensors - first : N;
    Params<N> p;
    for (int t = 0; t < count; t++) {
      p.caches[t] = a.caches[first + t];
      p.fresh[t] = a.fresh[first + t];
    }
    p.index = a.index;
    p.counts = a.counts;
    p.kvLens = a.kvLens;
    p.cacheSeqStride = a.cacheSeqStride / elems;
    p.freshSeqStride = a.nodes * rowStride / elems;
    p.freshRowStride = rowStride / elems;
    p.width = a.width / elems;
    p.committed = committed;
    p.status = status;
    p.nodes = a.nodes;
    p.cacheRows = a.cacheRows;
    p.lead = a.lead;
    p.indexStride = a.indexStride ? a.indexStride : a.nodes;
    // Rows dealt out to as many blocks as put two on every SM.
    const int64_t blocks = (int64_t)count * a.batch;
    int64_t turns = (2 * smCount + blocks - 1) / blocks;
    turns = turns > a.nodes ? a.nodes : turns;
    const cudaError_t e = launch_dependent(commit_kernel<V, N>, dim3((unsigned)count, (unsigned)a.batch, (unsigned)turns),
                                           dim3(kThreads), 0, s, p);
    if (e != cudaSuccess) return e;
    ++*launches;
  }
  return cudaSuccess;
}

template <typename V>
cudaError_t launch(const rt_commit_args& a, int32_t* committed, int elems, int* status, int smCount, int* launches,
                   cudaStream_t s) {
  return a.tensors <= kFew ? launch_n<V, kFew>(a, committed, elems, status, smCount, launches, s)
                           : launch_n<V, kTensors>(a, committed, elems, status, smCount, launches, s);
}

}  // namespace

cudaError_t launch_commit(const rt_commit_args& a, int32_t* committed, int* status, int smCount, int* launches, cudaStream_t s) {
  const int es = a.dtype == RT_F16 ? 2 : 4;
  // The widest copies that every address and stride is a multiple of.
  uintptr_t all = 16 | (uintptr_t)(a.width * es) | (uintptr_t)(a.freshRowStride * es) | (uintptr_t)(a.cacheSeqStride * es);
  for (int t = 0; t < a.tensors; t++)
    all |= reinterpret_cast<uintptr_t>(a.caches[t]) | reinterpret_cast<uintptr_t>(a.fresh[t]);
  const int bytes = (int)(all & (~all + 1));
  if (bytes == 16) return launch<uint4>(a, committed, 16 / es, status, smCount, launches, s);
  if (bytes == 8) return launch<uint2>(a, committed, 8 / es, status, smCount, launches, s);
  if (bytes == 4) return launch<uint32_t>(a, committed, 4 / es, status, smCount, launches, s);
  return launch<uint16_t>(a, committed, 1, status, smCount, launches, s);
}

}  // namespace rt
