// What the speculative-decoding kernels share: a sequence's context length and the shape of its
// drafted tree, checked on the device (they are inputs of a captured graph, the host never sees them).
#pragma once

#include "common.cuh"

namespace ns {

constexpr int kTreeMax = NS_TREE_MAX_NODES;

// Context length of sequence b, or -1 (flagged) when it is no length of a cache of max_ctx slots.
__device__ __forceinline__ int tree_len(const int32_t* lens, int b, int max_ctx) {
  const int n = lens[b];
  return n >= 0 && n <= max_ctx ? n : -1;
}

// Ancestors of node t of a chain, itself included: bits 0..t.
__device__ __forceinline__ uint64_t chain_mask(int t) { return t >= 63 ? ~0ull : (1ull << (t + 1)) - 1; }

// Ancestors of node t, itself included, as bits; 0: an unused node.  `par(i)` gives the parent of
// node i (-1: the context).  Parents precede their children, so the walk ends; a parent out of order,
// below -2 or unused makes the node unused and sets *bad.
template <typename ParentFn>
__device__ __forceinline__ uint64_t tree_mask(int t, ParentFn par, bool* bad) {
  uint64_t m = 0;
  int at = t;
  while (true) {
    const int up = par(at);
    if (up == -2 && at == t) return 0;
    if (up >= at || up < -1) {
      *bad = true;
      return 0;
    }
    m |= 1ull << at;
    if (up < 0) return m;
    at = up;
  }
}

// Host-side launch of a kernel with programmatic dependent launch (the kernel waits with
// griddep_wait before it reads anything another kernel writes) and, for cluster > 1, clusters.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, ns_stream_t stream,
                              int cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
inline bool strides_multiple(const int64_t* s, int n, int64_t of) {
  for (int i = 0; i < n; ++i)
    if (s[i] % of) return false;
  return true;
}

}  // namespace ns
