// Paged KV cache, the bookkeeping of a step: block tables and slot map from
// the requests' lengths (paged_step_kernel) and the write of the new rows to
// their slots (paged_write_kernel).
#include "paged.cuh"

namespace tw {

// ---- step plan ----------------------------------------------------------------
// Every page a request gives back or takes has a place on the stack that three
// prefix sums over the requests fix: new tokens, pages wanted, pages returned.
// A CTA needs nothing but those sums and the *inputs* (pages that a token gets
// are looked up where they lie before the step: in the table, on the stack, or
// in the table row of a request that ended), so each CTA scans the lengths
// itself and then works on its share of tokens and pages; nothing is exchanged
// and the step is one launch.
//
// Bound: latency.  The bytes are a few per token; the time is the launch plus
// three dependent loads (lengths -> table or stack -> slot).  Measured: 5 us for
// 16 requests with a token each, 7 us for 256 requests with 12 600 tokens (a
// thread per token; with four tokens a thread: 12 us).
constexpr int kStepThreads = 512;
constexpr int kStepMaxRequests = 8192;
constexpr int kStepTokensPerCta = kStepThreads;

struct StepSums {
  long long tokens, wanted, returned;
};

__device__ __forceinline__ StepSums add(const StepSums& a, const StepSums& b) {
  return {a.tokens + b.tokens, a.wanted + b.wanted, a.returned + b.returned};
}

__device__ __forceinline__ StepSums shfl_up(const StepSums& a, int off) {
  return {__shfl_up_sync(0xffffffffu, a.tokens, off), __shfl_up_sync(0xffffffffu, a.wanted, off),
          __shfl_up_sync(0xffffffffu, a.returned, off)};
}

__device__ __forceinline__ int saturate(long long x) {
  return (int)(x < INT32_MAX ? x : INT32_MAX);
}

// The request's lengths in pages.
struct StepRequest {
  int len, add;          // tokens held, tokens to add (0 when it ended)
  int have, want, give;  // pages held, pages wanted, pages returned
  bool wide;             // its pages would not fit the table's width
};

__device__ __forceinline__ StepRequest step_request(int len, int fresh, int page_size, int width) {
  StepRequest r;
  r.len = max(len, 0);
  r.add = max(fresh, 0);
  const unsigned s = (unsigned)page_size;
  const unsigned have = ((unsigned)r.len + s - 1) / s;  // < 2^32: len < 2^31, s < 2^31
  const unsigned long long after = (unsigned long long)r.len + r.add;
  const long long need = (long long)((after + s - 1) / s) - (long long)have;
  r.wide = (long long)have + need > width;
  r.have = (int)min(have, (unsigned)width);
  r.want = (fresh < 0 || r.wide) ? 0 : (int)need;
  r.give = fresh < 0 ? r.have : 0;
  return r;
}

__global__ void __launch_bounds__(kStepThreads) paged_step_kernel(tw_paged_step_args a) {
  extern __shared__ int s_sums[];
  int* s_tokens = s_sums;                // inclusive prefix sums per request
  int* s_wanted = s_tokens + a.requests;
  int* s_returned = s_wanted + a.requests;
  __shared__ StepSums s_warp[kStepThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.requests;
  const int count = (int)max(0ll, min((long long)*a.free_count, (long long)a.num_pages));

  StepSums base = {0, 0, 0};
  for (int b0 = 0; b0 < B; b0 += kStepThreads) {
    const int b = b0 + tid;
    StepSums x = {0, 0, 0};
    if (b < B) {
      const StepRequest r = step_request(a.lens[b], a.new_lens[b], a.page_size, a.table_width);
      x = {r.add, r.want, r.give};
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const StepSums y = shfl_up(x, off);
      if (lane >= off) x = add(x, y);
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    StepSums before = base;
    StepSums total = base;
    for (int w = 0; w < kStepThreads / 32; ++w) {
      if (w < warp) before = add(before, s_warp[w]);
      total = add(total, s_warp[w]);
    }
    x = add(x, before);
    if (b < B) {
      s_tokens[b] = saturate(x.tokens);
      s_wanted[b] = saturate(x.wanted);
      s_returned[b] = saturate(x.returned);
    }
    base = total;
    __syncthreads();
  }
  const int total = saturate(base.tokens);
  const int returned = saturate(base.returned);
  const long long top = (long long)count + base.returned;

  // The page at place p of the stack once the ended requests' pages are on it.
  auto stack_page = [&](long long p) -> int {
    if (p < count) return a.free_pages[p];
    const int k = (int)(p - count);
    const int r = first_above(s_returned, B, k);
    const int first = r > 0 ? s_returned[r - 1] : 0;
    return a.block_table[(int64_t)r * a.table_stride + (k - first)];
  };
  auto served = [&](int b, const StepRequest& r) {
    return !r.wide && (r.want == 0 || (long long)s_wanted[b] <= top);
  };

  // (unsigned counters: a signed one would overflow past counts near 2^31)
  const unsigned step = gridDim.x * kStepThreads;
  const unsigned first = blockIdx.x * kStepThreads + tid;
  for (unsigned t = first; t < (unsigned)a.tokens_cap; t += step) {
    int64_t slot = -1;
    int position = 0;
    if (t < (unsigned)total) {
      const int b = first_above(s_tokens, B, (int)t);
      const StepRequest r = step_request(a.lens[b], a.new_lens[b], a.page_size, a.table_width);
      position = r.len + ((int)t - (b > 0 ? s_tokens[b - 1] : 0));
      if (served(b, r)) {
        const int i = position / a.page_size;
        const int page = i < r.have
                             ? a.block_table[(int64_t)b * a.table_stride + i]
                             : stack_page(top - 1 - (s_wanted[b] - r.want + (i - r.have)));
        if (page >= 0 && page < a.num_pages)
          slot = (int64_t)page * a.page_size + (position - i * a.page_size);
        else
          raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
      }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
  // pages returned, at their places on the stack
  for (unsigned k = first; k < (unsigned)returned; k += step) {
    if ((long long)count + k < a.num_pages)
      a.free_pages[(long long)count + k] = stack_page((long long)count + k);
    else
      raise_error(a.error_flag, TW_ERR_CAPACITY);
  }
  // per request: lengths and the pages it takes
  for (unsigned b = first; b < (unsigned)B; b += step) {
    const StepRequest r = step_request(a.lens[b], a.new_lens[b], a.page_size, a.table_width);
    const bool ok = served(b, r);
    if (!ok) raise_error(a.error_flag, TW_ERR_CAPACITY);
    a.kv_lens[b] = a.new_lens[b] < 0 ? 0 : ok ? r.len + r.add : r.len;
    a.cu_q[b + 1] = s_tokens[b];
  }
  const int wanted = saturate(base.wanted);
  for (unsigned k = first; k < (unsigned)wanted && (long long)k < top; k += step) {
    const int b = first_above(s_wanted, B, (int)k);
    if ((long long)s_wanted[b] > top) break;  // refused, and so are all after it
    const StepRequest r = step_request(a.lens[b], a.new_lens[b], a.page_size, a.table_width);
    const int i = r.have + ((int)k - (s_wanted[b] - r.want));
    a.block_table[(int64_t)b * a.table_stride + i] = stack_page(top - 1 - k);
  }
  if (blockIdx.x == 0 && tid == 0) {
    // requests are served up to the first whose pages the stack does not hold
    const int n = first_above(s_wanted, B, saturate(top));
    const long long taken_end = n > 0 ? s_wanted[n - 1] : 0;
    a.cu_q[0] = 0;
    *a.free_count_out = (int)min(top - taken_end, (long long)a.num_pages);
    if (total > a.tokens_cap) raise_error(a.error_flag, TW_ERR_CAPACITY);
  }
}

// ---- row write ------------------------------------------------------------------
// One 16-byte vector of K and the same of V per thread; the 16 threads of a row
// write 256 contiguous bytes.  Bound: HBM (each byte read and written once).
// Measured: 8192 tokens x 8 heads out of a fused projection: 12.7 us, 5.3 TB/s;
// 64 tokens: 3.0 us from call to call, a launch.
constexpr int kWriteThreads = 256;

__global__ void __launch_bounds__(kWriteThreads)
paged_write_kernel(const __grid_constant__ tw_paged_pool pool, const uint4* __restrict__ k,
                   int64_t k_token, int64_t k_head, const uint4* __restrict__ v, int64_t v_token,
                   int64_t v_head, const int64_t* __restrict__ slots, int64_t rows,
                   int32_t* error_flag) {
  pdl_wait();
  pdl_launch_dependents();
  const int c = threadIdx.x & (kVecPerRow16 - 1);
  const int64_t row = (int64_t)blockIdx.x * (kWriteThreads / kVecPerRow16) +
                      threadIdx.x / kVecPerRow16;
  if (row >= rows) return;
  int64_t t, h;
  if (rows <= INT32_MAX) {  // a 64-bit division takes as long as a load
    t = (unsigned)row / (unsigned)pool.kv_heads;
    h = row - t * pool.kv_heads;
  } else {
    t = row / pool.kv_heads;
    h = row - t * pool.kv_heads;
  }
  const uint4 kv = __ldcs(k + (t * k_token + h * k_head) / kPagedAlign + c);
  const uint4 vv = __ldcs(v + (t * v_token + h * v_head) / kPagedAlign + c);
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= pool.num_pages * pool.page_size) {
    if (slot != -1) raise_error(error_flag, TW_ERR_INVALID_INDEX);
    return;
  }
  const int64_t page = slot <= INT32_MAX ? (unsigned)slot / (unsigned)pool.page_size
                                         : slot / pool.page_size;
  const int64_t o = slot - page * pool.page_size;
  const int64_t to = (page * pool.page_stride + h * pool.head_stride + o * pool.token_stride) /
                         kPagedAlign + c;
  reinterpret_cast<uint4*>(pool.k_pages)[to] = kv;
  reinterpret_cast<uint4*>(pool.v_pages)[to] = vv;
}

}  // namespace tw

using namespace tw;

extern "C" size_t tw_paged_pool_size(void) { return sizeof(tw_paged_pool); }
extern "C" size_t tw_paged_step_args_size(void) { return sizeof(tw_paged_step_args); }

extern "C" int tw_paged_step(const tw_paged_step_args* args, void* stream) {
  if (!args) return TW_ERR_BAD_ARG;
  const tw_paged_step_args& a = *args;
  if (!a.lens || !a.new_lens || !a.block_table || !a.free_pages || !a.free_count || !a.kv_lens ||
      !a.cu_q || !a.free_count_out || a.requests <= 0 || a.page_size <= 0 || a.table_width <= 0 ||
      a.table_stride < a.table_width || a.num_pages <= 0 || a.num_pages > INT32_MAX ||
      a.tokens_cap < 0 || (a.tokens_cap > 0 && (!a.slots || !a.positions)))
    return TW_ERR_BAD_ARG;
  if (a.kv_lens == a.lens || a.kv_lens == a.new_lens || a.free_count_out == a.free_count)
    return TW_ERR_BAD_ARG;
  if (a.requests > kStepMaxRequests) return TW_ERR_UNSUPPORTED;
  static DynSmemOptIn opt_in;
  const int smem = 3 * a.requests * (int)sizeof(int);
  const int rc = ensure_dyn_smem((const void*)paged_step_kernel, opt_in, smem);
  if (rc != TW_OK) return rc;
  const int ctas = min(148, max(1, (a.tokens_cap + kStepTokensPerCta - 1) / kStepTokensPerCta));
  return launch_pdl(paged_step_kernel, dim3(ctas), dim3(kStepThreads), (size_t)smem,
                    (cudaStream_t)stream, a);
}

extern "C" int tw_paged_write(const tw_paged_pool* pool, const void* k, int64_t k_token_stride,
                              int64_t k_head_stride, const void* v, int64_t v_token_stride,
                              int64_t v_head_stride, const int64_t* slots, int64_t tokens,
                              int32_t* error_flag, void* stream) {
  if (!pool) return TW_ERR_BAD_ARG;
  const int rc = check_paged_pool(*pool);
  if (rc != TW_OK) return rc;
  if (tokens < 0) return TW_ERR_BAD_ARG;
  if (tokens == 0) return TW_OK;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v) || !paged_stride_ok(k_token_stride) ||
      !paged_stride_ok(k_head_stride) || !paged_stride_ok(v_token_stride) ||
      !paged_stride_ok(v_head_stride))
    return TW_ERR_BAD_ARG;
  const int64_t rows = tokens * pool->kv_heads;
  const int64_t ctas = (rows * kVecPerRow16 + kWriteThreads - 1) / kWriteThreads;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  return launch_pdl(paged_write_kernel, dim3((unsigned)ctas), dim3(kWriteThreads), 0,
                    (cudaStream_t)stream, *pool, (const uint4*)k, k_token_stride, k_head_stride,
                    (const uint4*)v, v_token_stride, v_head_stride, slots, rows, error_flag);
}
