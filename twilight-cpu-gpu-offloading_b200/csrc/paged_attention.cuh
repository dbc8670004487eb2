// What the kernels of the paged attention share: a call's work, a request's
// rows and keys, the split of the keys, and values that are not finite.
#pragma once

#include <math_constants.h>

#include "async.cuh"
#include "paged.cuh"

namespace tw {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTileKeys = 128;  // splits begin at multiples of this

// How one kernel of the call divides a request's keys: ranges of `chunk` keys
// (a multiple of kTileKeys), `splits` of them at most.  A request of the call
// that is longer than max_kv_len said gets its rest in the last range.
struct PagedSplit {
  int chunk;
  int splits;
  float* part_o;    // [rows][splits][D], each range's softmax-weighted mean of V
  float* part_lse;  // [rows][splits], its log2 sum of exponentials
};

struct PagedWork {
  tw_paged_attention_args a;
  float scale_log2;  // softmax_scale * log2(e)
  int group;         // query heads per KV head
  int few_tokens;    // requests with at most this many new tokens: token kernel (0: none)
  int few_rows;      // few_tokens * group
  int box;           // token rows of one TMA box
  PagedSplit few;    // rows: (request * kv_heads + head) * few_rows + row
  PagedSplit many;   // rows: token * q_heads + head
};

struct PagedRequest {
  int first, n;  // its rows of q: [first, first + n)
  int kv;        // its tokens, the new ones included
};

// Lengths as the call gives them, cut to what its buffers hold.  A request with rows that
// q does not have is not computed: cut, the rest would be at wrong positions.
__device__ __forceinline__ PagedRequest paged_request(const tw_paged_attention_args& a, int b) {
  PagedRequest r;
  const int first = a.cu_q[b], end = a.cu_q[b + 1];
  r.kv = max(a.kv_lens[b], 0);  // read with them, before a branch
  const bool held = first >= 0 && end <= a.tokens;
  if (!held) raise_error(a.error_flag, TW_ERR_BAD_ARG);
  r.first = min(max(first, 0), a.tokens);
  r.n = held ? max(end - first, 0) : 0;
  // 2^30: positions are 32-bit, and a tile or range past the last key must be one too
  const long long cap = min((long long)a.table_width * a.pool.page_size, 1ll << 30);
  if (r.kv > cap) {
    r.kv = (int)cap;
    raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
  }
  return r;
}

// Keys that the row at position p sees: [low(p), p].
__device__ __forceinline__ int paged_low(const tw_paged_attention_args& a, int p) {
  return a.window > 0 ? max(0, p - a.window + 1) : 0;
}

// 2^x by the special-function unit (relative error 2^-22; 2^-inf = 0).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct PagedRange {
  int begin, end;  // keys
  int parts;       // ranges that [low, high) is divided into
};

// Range `part` of the keys [low, high).
__device__ __forceinline__ PagedRange paged_range(const PagedSplit& sp, int low, int high,
                                                  int part) {
  low = low / kTileKeys * kTileKeys;
  PagedRange x;
  x.parts = min(max((high - low + sp.chunk - 1) / sp.chunk, 1), sp.splits);
  x.begin = low + part * sp.chunk;
  x.end = part == x.parts - 1 ? high : min(high, x.begin + sp.chunk);
  return x;
}

// Keys that some of the rows [i, i + n) of a request see.
struct PagedKeys {
  int low, high;
};
__device__ __forceinline__ PagedKeys paged_keys(const tw_paged_attention_args& a,
                                                const PagedRequest& r, int i, int n) {
  const int p = r.kv - r.n + i;
  return {paged_low(a, max(p, 0)), max(p + n, 0)};
}

// Weights stand this much above the reference, in log2 units: an fp16 weight below 2^-25
// is nothing in the product with V, and 1e5 keys of little weight each can be a share of
// a result.  The reference moves when a score exceeds it by 8, so weights stay within
// 2^15, and what is lost lies below 2^-32 of the row's largest.  (bf16 has the range.)
template <typename T> constexpr float kLift = 0.f;
template <> constexpr float kLift<__half> = 7.f;

// The infinities and NaN of a pair of 16-bit values (exponent all ones): bit 15, bit 31.
template <typename T>
__device__ __forceinline__ uint32_t odd_halves(uint32_t two);
template <>
__device__ __forceinline__ uint32_t odd_halves<__half>(uint32_t two) {
  return ((two & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
template <>
__device__ __forceinline__ uint32_t odd_halves<__nv_bfloat16>(uint32_t two) {
  return ((two & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t clear_odd(uint32_t& two) {
  const uint32_t odd = odd_halves<T>(two);
  two &= ~((odd >> 15) * 0xffffu);
  return odd;
}
// Clears them in eight values; true: there were some.
template <typename T>
__device__ __forceinline__ bool clear_odd(uint4& x) {
  return (clear_odd<T>(x.x) | clear_odd<T>(x.y) | clear_odd<T>(x.z) | clear_odd<T>(x.w)) != 0;
}

// V of key k of request b, KV head g; nullptr: its page is none.
template <typename T>
__device__ __forceinline__ const T* paged_value(const tw_paged_attention_args& a, int b, int g,
                                                int k) {
  const int i = k / a.pool.page_size;
  const int page = a.block_table[(int64_t)b * a.table_stride + i];
  if (page < 0 || page >= a.pool.num_pages) return nullptr;
  return (const T*)a.pool.v_pages + (int64_t)page * a.pool.page_stride +
         (int64_t)g * a.pool.head_stride +
         (int64_t)(k - i * a.pool.page_size) * a.pool.token_stride;
}

// Log-sum-exp of a row with reference m (log2 units) and sum l, and the same in log2
// units for the merge.  Rounded once: log2(l) is small beside m, and m + log2(l) times ln 2
// would round at m's size twice.
__device__ __forceinline__ float paged_lse(float m, float l) {
  return l == 0.f ? -CUDART_INF_F : fmaf(m, kLn2, log2f(l) * kLn2);
}
__device__ __forceinline__ float paged_lse2(float m, float l) {
  return l == 0.f ? -CUDART_INF_F : m + log2f(l);
}

// Result of a row whose keys are one range: out and lse.  `n` consecutive
// dimensions from d0; lse by the thread with d0 == 0.
template <typename Out, int N>
__device__ __forceinline__ void paged_store_row(const tw_paged_attention_args& a, int t, int h,
                                                int d0, const float (&o)[N], float lse) {
  Out* out = (Out*)a.out + (int64_t)t * a.out_token_stride + (int64_t)h * a.out_head_stride + d0;
  constexpr int kVec = 16 / sizeof(Out);
  if constexpr (N % kVec == 0) {
#pragma unroll
    for (int c = 0; c < N; c += kVec) {
      __align__(16) Out x[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) x[i] = from_f32<Out>(o[c + i]);
      *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<uint4*>(x);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) out[c] = from_f32<Out>(o[c]);
  }
  if (a.lse && d0 == 0)
    a.lse[(int64_t)t * a.q_heads + h] = lse;
}

// A range's result of a row, for the merge.
template <int N>
__device__ __forceinline__ void paged_store_part(const PagedSplit& sp, int64_t row, int s, int d0,
                                                 const float (&o)[N], float lse2) {
  float* to = sp.part_o + (row * sp.splits + s) * kHeadDim + d0;
#pragma unroll
  for (int c = 0; c < N; c += 4)
    *reinterpret_cast<float4*>(to + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
  if (d0 == 0) sp.part_lse[row * sp.splits + s] = lse2;
}

// The maps of the pool's K and V: [page][head][row][D] boxes of `box` rows of
// one head of one page, 64 elements wide.
struct PagedMaps {
  CUtensorMap k, v;
};

// Rows past the last token: out 0, lse -inf.  For CTA `cta` of kPadCtas.
constexpr int kPadCtas = 8;
template <typename Out>
__device__ __forceinline__ void paged_clear_padding(const tw_paged_attention_args& a, int cta) {
  const int end = min(max(a.cu_q[a.requests], 0), a.tokens);
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  const int64_t rows = (int64_t)(a.tokens - end) * a.q_heads;
  for (int64_t i = (int64_t)cta * blockDim.x + threadIdx.x; i < rows * 32;
       i += (int64_t)kPadCtas * blockDim.x) {
    const int64_t row = i >> 5;
    paged_store_row<Out, 4>(a, end + (int)(row / a.q_heads), (int)(row % a.q_heads),
                            (int)(i & 31) * 4, zero, -CUDART_INF_F);
  }
}

// New tokens that a CTA of the chunk kernel takes: 2 x 128 rows.
__host__ __device__ __forceinline__ int paged_chunk_tokens(int group) { return 2 * (128 / group); }

int launch_paged_token(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream);
int launch_paged_chunk(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream);

}  // namespace tw
