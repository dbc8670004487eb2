// Asynchronous copies and barriers of sm_100a: mbarriers with bounded waits,
// tiled TMA loads, proxy fences, tensor maps of a paged pool.
#pragma once

#include <cuda.h>

#include "tw_common.cuh"

namespace tw {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// True in one thread of a converged warp.  Copies and products take their operands
// from uniform registers: under this test the compiler knows that one thread issues
// them, under `lane == 0` it would emit a loop over the warp's values for each.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count)
               : "memory");
}
// Makes initialised barriers visible to the copy engine.
__device__ __forceinline__ void mbar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)),
               "r"(bytes)
               : "memory");
}
// One look at a barrier's phase.  kSuspend: the thread may sleep for a while first,
// which spares power (what bounds a kernel of products) but wakes later.
template <bool kSuspend>
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  if constexpr (kSuspend)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
  return done != 0;
}
__device__ __forceinline__ unsigned long long global_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// A wait ends after two seconds whatever happens; the caller then gives up.
constexpr unsigned long long kWaitLimitNs = 2000000000ull;

// Waits for the phase of this parity to complete.  False: the wait ran out, or
// another thread's did (abort_flag, in shared memory, tells the others).
// Inlined, like all of a kernel that splits its registers by setmaxnreg: a call
// would hold the whole kernel to one register count.
template <typename Look>
__device__ __forceinline__ bool wait_until(Look look, volatile int* abort_flag) {
  unsigned long long start = 0;
#pragma unroll 1
  for (unsigned i = 1;; ++i) {
    if (look()) return true;
    if ((i & 63) == 0) {
      if (*abort_flag) return false;
      const unsigned long long now = global_ns();
      if (start == 0) start = now;
      if (now - start > kWaitLimitNs) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
template <bool kSuspend = true>
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity,
                                          volatile int* abort_flag) {
  return wait_until([&] { return mbar_try<kSuspend>(bar, parity); }, abort_flag);
}

// Orders this thread's shared-memory accesses before later ones of the copy
// engine or the tensor cores.
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint32_t dst, uint64_t* bar,
                                            int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint32_t dst, uint64_t* bar,
                                            int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// The driver's tensor-map encoder, looked up once (nullptr: unavailable).
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// A map of 16-bit rows whose first dimension is head_dim contiguous elements,
// copied in boxes of 64 elements (one 128-byte swizzle row) by `box[1..]`.
// Out-of-range coordinates read zeros.
inline int encode_rows_map(CUtensorMap* map, int dtype, int rank, const void* base,
                           const cuuint64_t* dims, const cuuint64_t* strides_bytes,
                           const cuuint32_t* box) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return TW_ERR_UNSUPPORTED;
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult rc = encode(
      map, dtype == TW_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
      (cuuint32_t)rank, const_cast<void*>(base), dims, strides_bytes, box, one,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? TW_OK : TW_ERR_BAD_ARG;
}

}  // namespace tw
