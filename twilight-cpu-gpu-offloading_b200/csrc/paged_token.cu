// Paged attention of calls in which every request has few new rows: a CTA per item.
#include "paged_token.cuh"

namespace tw {

constexpr int kTokSmem = kTokRing + 1024;  // + alignment of the swizzle

template <typename T, typename Out>
__global__ void __launch_bounds__(kTokThreads, 2)
paged_token_kernel(const __grid_constant__ PagedWork w, const __grid_constant__ PagedMaps maps) {
  extern __shared__ char s_raw[];
  __shared__ TokShared sh;
  if (threadIdx.x == 0) token_init(sh);
  if (threadIdx.x == kTokWarps * 32) {
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  pdl_wait();
  pdl_launch_dependents();
  // the first CTAs, which are done at once
  if (blockIdx.x < kPadCtas) {
    paged_clear_padding<Out>(w.a, blockIdx.x);
    return;
  }
  char* smem = (char*)(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);
  token_item<T, Out>(w, maps, smem, sh, blockIdx.x - kPadCtas, 0, threadIdx.x);
}

template <typename T, typename Out>
static int launch(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream) {
  static DynSmemOptIn opt_in;
  const auto kernel = paged_token_kernel<T, Out>;
  const int rc = ensure_dyn_smem((const void*)kernel, opt_in, kTokSmem);
  if (rc != TW_OK) return rc;
  const int64_t ctas = (int64_t)w.a.requests * w.a.pool.kv_heads * w.few.splits + kPadCtas;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(kTokThreads), (size_t)kTokSmem, stream, w,
                    maps);
}

int launch_paged_token(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream) {
  if (w.a.pool.dtype == TW_F16)
    return w.a.out_dtype == TW_F32 ? launch<__half, float>(w, maps, stream)
                                   : launch<__half, __half>(w, maps, stream);
  return w.a.out_dtype == TW_F32 ? launch<__nv_bfloat16, float>(w, maps, stream)
                                 : launch<__nv_bfloat16, __nv_bfloat16>(w, maps, stream);
}

}  // namespace tw
