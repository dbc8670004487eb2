// What the paged-cache kernels share: argument checks of a pool and the
// lookup in prefix sums.
#pragma once

#include "tw_common.cuh"

namespace tw {

constexpr int kPagedAlign = 8;  // strides are multiples of 8 elements (16 bytes)

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline bool paged_stride_ok(int64_t s) { return s > 0 && s % kPagedAlign == 0; }

// Status of a pool's fields (TW_OK: usable).
inline int check_paged_pool(const tw_paged_pool& p) {
  if (p.head_dim != kHeadDim) return TW_ERR_UNSUPPORTED;
  if (p.dtype != TW_F16 && p.dtype != TW_BF16) return TW_ERR_UNSUPPORTED;
  if (!p.k_pages || !p.v_pages || p.num_pages <= 0 || p.num_pages > INT32_MAX ||
      p.page_size <= 0 || p.kv_heads <= 0)
    return TW_ERR_BAD_ARG;
  if (!aligned16(p.k_pages) || !aligned16(p.v_pages) || !paged_stride_ok(p.page_stride) ||
      !paged_stride_ok(p.head_stride) || !paged_stride_ok(p.token_stride))
    return TW_ERR_BAD_ARG;
  return TW_OK;
}

// First index i of [0, n) with ends[i] > x, ends ascending; n when there is none.
template <typename Index>
__device__ __forceinline__ int first_above(const Index* ends, int n, Index x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// The error flag keeps the largest code, whatever order the threads run in.
__device__ __forceinline__ void raise_error(int32_t* flag, int code) {
  if (flag) atomicMax(flag, code);
}

// launch_pdl with clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
inline int launch_pdl_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, int cluster,
                              size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see pdl_wait
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  if (err != cudaSuccess) {
    set_last_cuda_error(err);
    return TW_ERR_CUDA;
  }
  return check_launch();
}

}  // namespace tw
