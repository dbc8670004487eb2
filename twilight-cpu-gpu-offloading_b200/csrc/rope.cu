// Rotary positions: rows by themselves, and fused with the write of new rows to
// the paged cache.
//
// Pair n of a row at position p, of dimensions (i, j): (i, j) = (n, n + pairs) in the half
// layout, (2n, 2n + 1) in the interleaved one;
//   (x_i, x_j) -> scale * (x_i cos - x_j sin, x_j cos + x_i sin), angle = p * frequency_n.
// Dimensions from 2 * pairs on pass.
#include "paged.cuh"

namespace tw {

// Bound: HBM (each row read and written once).  16 threads take a row, 16 bytes each; a CTA
// takes a token's rows (or those of several tokens when they are few), so that an angle is
// worked out once for all heads.  The product p * frequency is 64-bit (at position 10^6 a
// 32-bit one is off by 0.06), then reduced to a part of a turn, of which sine and cosine are
// 32-bit; the rotation is 32-bit and rounded once.
constexpr int kRopeThreads = 256;
constexpr int kRopeRows = kRopeThreads / kVecPerRow16;  // rows of the CTA at a time
constexpr int kRopeAhead = 4;                           // rows of a thread on their way
constexpr int kRopePairs = kHeadDim / 2;
constexpr int kRopeTokens = 16;                         // of a CTA at most

enum RopeMode {
  kRopeInterleaved,  // both of a pair are in one thread's 16 bytes
  kRopeHalf,         // pairs is a multiple of 8: the others are in another thread's 16 bytes
  kRopeHalfOdd       // they are in two other threads' (or in this one's): by shared memory
};

struct RopeWork {
  tw_rope rope;
  const int32_t* positions;
  const uint4 *x, *k, *v;
  uint4* out;
  // strides in 16-byte vectors
  int64_t x_token, x_head, k_token, k_head, v_token, v_head, out_token, out_head;
  int64_t tokens;
  int heads;             // rows of x
  int rows;              // of a token: x, then (kWrite) K and V
  int tokens_per_cta;
  // kWrite
  tw_paged_pool pool;
  const int64_t* slots;
  float* row_weights;
  int32_t* row_positions;
  int32_t* error_flag;
};

// Eight values of a row, turned: y = x * c + s * partner, s negative for the first of a pair.
template <typename T, int kMode>
__device__ __forceinline__ uint4 rotate(uint4 x, int c, int pairs, const float2 (&cs)[8],
                                        char* stage) {
  const T* v = reinterpret_cast<const T*>(&x);
  __align__(16) T other[8];
  if constexpr (kMode == kRopeInterleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = v[e ^ 1];
  } else if constexpr (kMode == kRopeHalf) {
    const int n = pairs / 8;
    const int from = c < n ? c + n : c < 2 * n ? c - n : c;
    uint4 y;
    y.x = __shfl_sync(0xffffffffu, x.x, from, kVecPerRow16);
    y.y = __shfl_sync(0xffffffffu, x.y, from, kVecPerRow16);
    y.z = __shfl_sync(0xffffffffu, x.z, from, kVecPerRow16);
    y.w = __shfl_sync(0xffffffffu, x.w, from, kVecPerRow16);
    *reinterpret_cast<uint4*>(other) = y;
  } else {
    __syncwarp();
    reinterpret_cast<uint4*>(stage)[c] = x;
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = c * 8 + e;
      const int from = d < pairs ? d + pairs : d < 2 * pairs ? d - pairs : d;
      other[e] = reinterpret_cast<const T*>(stage)[from];
    }
  }
  __align__(16) T y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    y[e] = c * 8 + e < 2 * pairs
               ? from_f32<T>(fmaf(to_f32<T>(v[e]), cs[e].x, to_f32<T>(other[e]) * cs[e].y))
               : v[e];
  return *reinterpret_cast<uint4*>(y);
}

template <typename T, int kMode, bool kWrite>
__global__ void __launch_bounds__(kRopeThreads)
rope_kernel(const __grid_constant__ RopeWork w) {
  __shared__ float2 s_turn[kRopeTokens][kRopePairs];  // scale * (cos, sin)
  __shared__ __align__(16) char s_stage[kMode == kRopeHalfOdd ? kRopeRows * kHeadDim * 2 : 16];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, c = tid % kVecPerRow16, lane_row = tid / kVecPerRow16;
  const int pairs = w.rope.pairs;
  const int64_t t0 = (int64_t)blockIdx.x * w.tokens_per_cta;
  const int here = (int)min((int64_t)w.tokens_per_cta, w.tokens - t0);
  const int items = here * w.rows;

  // item: (token of the CTA, row of the token)
  auto load = [&](int item) -> uint4 {
    if (item >= items) return make_uint4(0u, 0u, 0u, 0u);
    const int ti = w.tokens_per_cta == 1 ? 0 : item / w.rows;
    int r = item - ti * w.rows;
    const int64_t t = t0 + ti;
    if (!kWrite || r < w.heads) return __ldcs(w.x + t * w.x_token + r * w.x_head + c);
    r -= w.heads;
    if (r < w.pool.kv_heads) return __ldcs(w.k + t * w.k_token + r * w.k_head + c);
    return __ldcs(w.v + t * w.v_token + (r - w.pool.kv_heads) * w.v_head + c);
  };
  uint4 x[kRopeAhead];
#pragma unroll
  for (int i = 0; i < kRopeAhead; ++i) x[i] = load(lane_row + i * kRopeRows);

  for (int i = tid; i < here * pairs; i += kRopeThreads) {
    const int ti = i / pairs, n = i - ti * pairs;
    const double turns = (double)w.positions[t0 + ti] * w.rope.frequencies[n] *
                         0.15915494309189533577;  // 1 / (2 pi)
    float sin, cos;
    sincospif(2.f * (float)(turns - rint(turns)), &sin, &cos);
    if (w.rope.inverse) sin = -sin;
    s_turn[ti][n] = make_float2(cos * w.rope.scale, sin * w.rope.scale);
  }
  __syncthreads();

  float2 cs[8];
  int64_t page = -1, offset = 0;
  int of = -1;  // the token they are of
  for (int first = lane_row; (first & ~1) < items; first += kRopeAhead * kRopeRows) {
#pragma unroll
    for (int i = 0; i < kRopeAhead; ++i) {
      const int item = first + i * kRopeRows;
      if ((item & ~1) >= items) break;  // (a warp's two rows together: it exchanges values)
      const bool real = item < items;
      const int ti = w.tokens_per_cta == 1 ? 0 : min(item, items - 1) / w.rows;
      if (ti != of) {
        of = ti;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = c * 8 + e;
          int n = kMode == kRopeInterleaved ? d >> 1 : d < pairs ? d : d - pairs;
          const bool second = kMode == kRopeInterleaved ? d & 1 : d >= pairs;
          cs[e] = s_turn[ti][min(n, kRopePairs - 1)];
          if (!second) cs[e].y = -cs[e].y;
        }
        if constexpr (kWrite) {
          const int64_t slot = w.slots[t0 + ti];
          page = -1;
          if (slot >= 0 && slot < w.pool.num_pages * w.pool.page_size) {
            page = slot <= INT32_MAX ? (unsigned)slot / (unsigned)w.pool.page_size
                                     : slot / w.pool.page_size;
            offset = slot - page * w.pool.page_size;
          } else if (slot != -1) {
            raise_error(w.error_flag, TW_ERR_INVALID_INDEX);
          }
        }
      }
      int r = item - ti * w.rows;
      const uint4 y = rotate<T, kMode>(x[i], c, pairs, cs, s_stage + lane_row * kHeadDim * 2);
      if (!real) continue;
      if (!kWrite || r < w.heads) {
        w.out[(t0 + ti) * w.out_token + r * w.out_head + c] = y;
        continue;
      }
      if (page < 0) continue;
      r -= w.heads;
      const bool value = r >= w.pool.kv_heads;
      if (value) r -= w.pool.kv_heads;
      const int64_t to = (page * w.pool.page_stride + r * w.pool.head_stride +
                          offset * w.pool.token_stride) / kPagedAlign + c;
      reinterpret_cast<uint4*>(value ? w.pool.v_pages : w.pool.k_pages)[to] = value ? x[i] : y;
      if (!value && c == 0) {
        const int64_t at = (page * w.pool.kv_heads + r) * w.pool.page_size + offset;
        if (w.row_weights) w.row_weights[at] = 0.f;
        if (w.row_positions) w.row_positions[at] = w.positions[t0 + ti];
      }
    }
#pragma unroll
    for (int i = 0; i < kRopeAhead; ++i) x[i] = load(first + (i + kRopeAhead) * kRopeRows);
  }
}

static int check_rope(const tw_rope& r, int head_dim, int dtype) {
  if (head_dim != kHeadDim || (dtype != TW_F16 && dtype != TW_BF16)) return TW_ERR_UNSUPPORTED;
  if (r.pairs < 0 || r.pairs > kRopePairs || (r.pairs > 0 && !r.frequencies) ||
      (r.interleaved != 0 && r.interleaved != 1) || (r.inverse != 0 && r.inverse != 1) ||
      !(fabsf(r.scale) < INFINITY))
    return TW_ERR_BAD_ARG;
  return TW_OK;
}

static bool rows_ok(const void* p, int64_t token, int64_t head) {
  return p && aligned16(p) && paged_stride_ok(token) && paged_stride_ok(head);
}

template <typename T, bool kWrite>
static int launch_rope(RopeWork& w, cudaStream_t stream) {
  // few rows a token: several tokens fill the CTA's 16 rows at a time
  w.tokens_per_cta = w.rows >= kRopeRows ? 1 : kRopeRows / w.rows;
  const int64_t ctas = (w.tokens + w.tokens_per_cta - 1) / w.tokens_per_cta;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  const auto kernel = w.rope.interleaved       ? rope_kernel<T, kRopeInterleaved, kWrite>
                      : w.rope.pairs % 8 == 0 ? rope_kernel<T, kRopeHalf, kWrite>
                                              : rope_kernel<T, kRopeHalfOdd, kWrite>;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(kRopeThreads), 0, stream, w);
}

}  // namespace tw

using namespace tw;

extern "C" size_t tw_rope_size(void) { return sizeof(tw_rope); }
extern "C" size_t tw_paged_rope_write_args_size(void) { return sizeof(tw_paged_rope_write_args); }

extern "C" int tw_rope_rows(const tw_rope* rope, const void* x, int64_t x_token_stride,
                            int64_t x_head_stride, const int32_t* positions, int64_t tokens,
                            int heads, int head_dim, int dtype, void* out,
                            int64_t out_token_stride, int64_t out_head_stride, void* stream) {
  if (!rope) return TW_ERR_BAD_ARG;
  const int rc = check_rope(*rope, head_dim, dtype);
  if (rc != TW_OK) return rc;
  if (tokens < 0 || heads < 0) return TW_ERR_BAD_ARG;
  if (tokens == 0 || heads == 0) return TW_OK;
  if (!positions || !rows_ok(x, x_token_stride, x_head_stride) ||
      !rows_ok(out, out_token_stride, out_head_stride))
    return TW_ERR_BAD_ARG;
  RopeWork w = {};
  w.rope = *rope;
  w.positions = positions;
  w.x = (const uint4*)x;
  w.x_token = x_token_stride / kPagedAlign;
  w.x_head = x_head_stride / kPagedAlign;
  w.out = (uint4*)out;
  w.out_token = out_token_stride / kPagedAlign;
  w.out_head = out_head_stride / kPagedAlign;
  w.tokens = tokens;
  w.heads = w.rows = heads;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == TW_F16 ? launch_rope<__half, false>(w, s)
                         : launch_rope<__nv_bfloat16, false>(w, s);
}

extern "C" int tw_paged_rope_write(const tw_paged_rope_write_args* args, void* stream) {
  if (!args) return TW_ERR_BAD_ARG;
  const tw_paged_rope_write_args& a = *args;
  int rc = check_paged_pool(a.pool);
  if (rc == TW_OK) rc = check_rope(a.rope, a.pool.head_dim, a.pool.dtype);
  if (rc != TW_OK) return rc;
  if (a.tokens < 0 || a.q_heads < 0 || a.q_heads > (1 << 20) || a.pool.kv_heads > (1 << 20) ||
      a.reserved != 0)
    return TW_ERR_BAD_ARG;
  if (a.tokens == 0) return TW_OK;
  if (!a.positions || !a.slots || !rows_ok(a.k, a.k_token_stride, a.k_head_stride) ||
      !rows_ok(a.v, a.v_token_stride, a.v_head_stride) ||
      (a.q_heads > 0 && (!rows_ok(a.q, a.q_token_stride, a.q_head_stride) ||
                         !rows_ok(a.q_out, a.q_out_token_stride, a.q_out_head_stride))))
    return TW_ERR_BAD_ARG;
  RopeWork w = {};
  w.rope = a.rope;
  w.positions = a.positions;
  w.x = (const uint4*)a.q;
  w.x_token = a.q_token_stride / kPagedAlign;
  w.x_head = a.q_head_stride / kPagedAlign;
  w.k = (const uint4*)a.k;
  w.k_token = a.k_token_stride / kPagedAlign;
  w.k_head = a.k_head_stride / kPagedAlign;
  w.v = (const uint4*)a.v;
  w.v_token = a.v_token_stride / kPagedAlign;
  w.v_head = a.v_head_stride / kPagedAlign;
  w.out = (uint4*)a.q_out;
  w.out_token = a.q_out_token_stride / kPagedAlign;
  w.out_head = a.q_out_head_stride / kPagedAlign;
  w.tokens = a.tokens;
  w.heads = a.q_heads;
  w.rows = a.q_heads + 2 * a.pool.kv_heads;
  w.pool = a.pool;
  w.slots = a.slots;
  w.row_weights = a.row_weights;
  w.row_positions = a.row_positions;
  w.error_flag = a.error_flag;
  cudaStream_t s = (cudaStream_t)stream;
  return a.pool.dtype == TW_F16 ? launch_rope<__half, true>(w, s)
                                : launch_rope<__nv_bfloat16, true>(w, s);
}
