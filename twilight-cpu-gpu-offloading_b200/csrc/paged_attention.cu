// Attention of new tokens over a paged KV cache.
//
// Row (t, h): token t of request b at position p sees the keys [lo, p];
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale * q . k_j,
// with the running maximum m and sum of one pass over the keys.
#include <math_constants.h>

#include "paged.cuh"

namespace tw {

constexpr int kRowWarps = 8;  // rows per CTA of the row kernel

struct PagedRows {
  const int32_t* table;  // the request's row of the block table
  int first;             // first row of q of the request
  int n;                 // its new tokens
  int kv;                // its tokens, the new ones included
};

template <typename T, typename Out>
__global__ void __launch_bounds__(kRowWarps * 32)
paged_row_kernel(tw_paged_attention_args a, float scale_log2) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (row >= (int64_t)a.tokens * a.q_heads) return;
  const int t = (int)(row / a.q_heads);
  const int h = (int)(row - (int64_t)t * a.q_heads);
  const int g = h / (a.q_heads / a.pool.kv_heads);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  float m = -CUDART_INF_F, l = 0.f;
  const int b = first_above(a.cu_q + 1, a.requests, t);
  if (b < a.requests) {
    const int n = a.cu_q[b + 1] - a.cu_q[b];
    const int64_t cap = (int64_t)a.table_width * a.pool.page_size;
    int kv = a.kv_lens[b];
    if (kv > cap) {
      kv = (int)cap;
      raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
    }
    const int p = kv - n + (t - a.cu_q[b]);
    const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const T* q = (const T*)a.q + (int64_t)t * a.q_token_stride + (int64_t)h * a.q_head_stride;
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(q[lane * 4 + i]) * scale_log2;
    const int32_t* table = a.block_table + (int64_t)b * a.table_stride;
    for (int j = lo; j <= p; ++j) {
      const int i = j / a.pool.page_size;
      const int page = table[i];
      const bool ok = page >= 0 && page < a.pool.num_pages;
      if (!ok) raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
      const int64_t at = (int64_t)page * a.pool.page_stride + (int64_t)g * a.pool.head_stride +
                         (int64_t)(j - i * a.pool.page_size) * a.pool.token_stride + lane * 4;
      float s = 0.f, v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s = fmaf(x[c], ok ? to_f32<T>(((const T*)a.pool.k_pages)[at + c]) : 0.f, s);
        v[c] = ok ? to_f32<T>(((const T*)a.pool.v_pages)[at + c]) : 0.f;
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      const float m_new = fmaxf(m, s);
      const float m_use = m_new == -CUDART_INF_F ? 0.f : m_new;
      const float keep = exp2f(m - m_use);
      const float e = exp2f(s - m_use);
      m = m_new;
      l = fmaf(l, keep, e);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] = fmaf(acc[c], keep, e * v[c]);
    }
  }
  Out* out = (Out*)a.out + (int64_t)t * a.out_token_stride + (int64_t)h * a.out_head_stride;
#pragma unroll
  for (int c = 0; c < 4; ++c) out[lane * 4 + c] = from_f32<Out>(l == 0.f ? 0.f : acc[c] / l);
  if (a.lse && lane == 0)
    a.lse[row] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename T, typename Out>
int launch_paged_rows(const tw_paged_attention_args& a, float scale_log2, cudaStream_t stream) {
  const int64_t rows = (int64_t)a.tokens * a.q_heads;
  const int64_t ctas = (rows + kRowWarps - 1) / kRowWarps;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  return launch_pdl(paged_row_kernel<T, Out>, dim3((unsigned)ctas), dim3(kRowWarps * 32), 0,
                    stream, a, scale_log2);
}

}  // namespace tw

using namespace tw;

extern "C" size_t tw_paged_attention_args_size(void) { return sizeof(tw_paged_attention_args); }

extern "C" size_t tw_paged_attention_workspace_size(int requests, int tokens, int q_heads,
                                                    int kv_heads, int max_q_len, int max_kv_len,
                                                    int head_dim) {
  return 0;
}

extern "C" int tw_paged_attention(const tw_paged_attention_args* args, void* stream) {
  if (!args) return TW_ERR_BAD_ARG;
  const tw_paged_attention_args& a = *args;
  const int rc = check_paged_pool(a.pool);
  if (rc != TW_OK) return rc;
  if (a.pool.page_size % 8 != 0) return TW_ERR_UNSUPPORTED;
  if (a.tokens < 0 || a.requests < 0) return TW_ERR_BAD_ARG;
  if (a.tokens == 0) return TW_OK;
  if (!a.q || !a.block_table || !a.cu_q || !a.kv_lens || !a.out || a.requests <= 0 ||
      a.q_heads <= 0 || a.q_heads % a.pool.kv_heads != 0 || a.table_width <= 0 ||
      a.table_stride < a.table_width || a.max_q_len < 0 || a.max_kv_len < 0 || a.window < 0 ||
      a.reserved != 0 || !(a.softmax_scale > 0.f))
    return TW_ERR_BAD_ARG;
  if (a.q_heads / a.pool.kv_heads > 64) return TW_ERR_UNSUPPORTED;
  if (a.out_dtype != a.pool.dtype && a.out_dtype != TW_F32) return TW_ERR_BAD_ARG;
  if (!aligned16(a.q) || !aligned16(a.out) || !paged_stride_ok(a.q_token_stride) ||
      !paged_stride_ok(a.q_head_stride) || !paged_stride_ok(a.out_token_stride) ||
      !paged_stride_ok(a.out_head_stride))
    return TW_ERR_BAD_ARG;
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.pool.dtype == TW_F16)
    return a.out_dtype == TW_F32 ? launch_paged_rows<__half, float>(a, scale_log2, st)
                                 : launch_paged_rows<__half, __half>(a, scale_log2, st);
  return a.out_dtype == TW_F32
             ? launch_paged_rows<__nv_bfloat16, float>(a, scale_log2, st)
             : launch_paged_rows<__nv_bfloat16, __nv_bfloat16>(a, scale_log2, st);
}
