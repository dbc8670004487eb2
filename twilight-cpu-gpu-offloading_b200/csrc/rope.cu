// Rotary positions: rows by themselves, and fused with the write of new rows to
// the paged cache.
//
// Pair n of a row at position p, of dimensions (i, j): (i, j) = (n, n + pairs) in the half
// layout, (2n, 2n + 1) in the interleaved one;
//   (x_i, x_j) -> scale * (x_i cos - x_j sin, x_j cos + x_i sin), angle = p * frequency_n.
// Dimensions from 2 * pairs on pass.
#include "paged.cuh"
#include "tensor.cuh"

namespace tw {

// Bound: HBM (each row read and written once).  A warp takes up to 16 rows of a token, 16
// threads a row and 16 bytes each, all on their way before it works out the token's angles,
// two a thread; so nothing waits for another warp.  (A CTA a token, whose threads share the
// angles through a barrier: 77 us for 8192 tokens of 48 rows, now 36, 5.6 TB/s; without the
// write, 8192 of 32 rows half of which turns: 18.4 us.)  The product p * frequency is 64-bit
// (at position 10^6 a 32-bit one is off by 0.06), then reduced to a part of a turn; sine and
// cosine of it are the special-function unit's, whose error on [-pi, pi] (2^-21.19 at most, by
// CUDA's documents) is far below the 16-bit rounding; the rotation is 32-bit and rounded once.
constexpr int kRopeThreads = 256, kRopeWarps = kRopeThreads / 32;
constexpr int kRopeFew = 148 * 64, kRopeMany = 148 * 512;  // rows of a call
constexpr int kRopePairs = kHeadDim / 2;

enum RopeMode {
  kRopeInterleaved,  // both of a pair are in one thread's 16 bytes
  kRopeHalf,         // pairs is a multiple of 8: the others are in another thread's 16 bytes
  kRopeHalfOdd       // they are in two other threads' (or in this one's): by shared memory
};

// Place of pair n in shared memory: 16 bytes more for every eight, so that threads that
// read eight each meet no bank conflicts.
__device__ __forceinline__ int turn_at(int n) { return n + n / 8 * 2; }
constexpr int kRopeTurns = kRopePairs + kRopePairs / 8 * 2;

struct RopeWork {
  tw_rope rope;
  const int32_t* positions;
  const uint4 *x, *k, *v;
  uint4* out;
  // strides in 16-byte vectors
  int64_t x_token, x_head, k_token, k_head, v_token, v_head, out_token, out_head;
  int64_t tokens;
  int heads;             // rows of x
  int parts;             // warps of a token: those of x, then (kWrite) of K and of V
  int x_parts, k_parts;
  // kWrite
  tw_paged_pool pool;
  const int64_t* slots;
  float* row_weights;
  int32_t* row_positions;
  int32_t* error_flag;
};

// The 32-bit values of two 16-bit ones, and back (rounded to nearest).
template <typename T> struct Two;
template <> struct Two<__half> {
  static __device__ __forceinline__ uint64_t wide(uint32_t x) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
    return pair(f.x, f.y);
  }
  static __device__ __forceinline__ uint32_t narrow(uint64_t x) {
    float a, b;
    unpair(x, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Two<__nv_bfloat16> {
  static __device__ __forceinline__ uint64_t wide(uint32_t x) {
    return pair(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t narrow(uint64_t x) {
    float a, b;
    unpair(x, a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Eight values of a row, turned: x * cos + partner * sin, sin negative for the first of a pair.
// `turned`: how many of the eight are (the others pass as they are).
template <typename T, int kMode>
__device__ __forceinline__ uint4 rotate(uint4 x, int c, int pairs, int turned,
                                        const uint64_t (&cos)[4], const uint64_t (&sin)[4],
                                        char* stage) {
  uint4 other;
  if constexpr (kMode == kRopeInterleaved) {
    other = make_uint4(__byte_perm(x.x, 0, 0x1032), __byte_perm(x.y, 0, 0x1032),
                       __byte_perm(x.z, 0, 0x1032), __byte_perm(x.w, 0, 0x1032));
  } else if constexpr (kMode == kRopeHalf) {
    const int n = pairs / 8;
    const int from = c < n ? c + n : c < 2 * n ? c - n : c;
    other.x = __shfl_sync(0xffffffffu, x.x, from, kVecPerRow16);
    other.y = __shfl_sync(0xffffffffu, x.y, from, kVecPerRow16);
    other.z = __shfl_sync(0xffffffffu, x.z, from, kVecPerRow16);
    other.w = __shfl_sync(0xffffffffu, x.w, from, kVecPerRow16);
  } else {
    __syncwarp();
    reinterpret_cast<uint4*>(stage)[c] = x;
    __syncwarp();
    __align__(16) uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = c * 8 + e;
      const int from = d < pairs ? d + pairs : d < 2 * pairs ? d - pairs : d;
      v[e] = reinterpret_cast<const uint16_t*>(stage)[from];
    }
    other = *reinterpret_cast<uint4*>(v);
  }
  const auto turn = [&](uint32_t a, uint32_t b, int i) {
    return Two<T>::narrow(fma2(Two<T>::wide(a), cos[i], mul2(Two<T>::wide(b), sin[i])));
  };
  uint4 y = make_uint4(turn(x.x, other.x, 0), turn(x.y, other.y, 1), turn(x.z, other.z, 2),
                       turn(x.w, other.w, 3));
  if (turned < 8) {
    // (2 * pairs is even: a pair of values turns or passes as a whole)
    if (turned < 2) y.x = x.x;
    if (turned < 4) y.y = x.y;
    if (turned < 6) y.z = x.z;
    y.w = x.w;
  }
  return y;
}

template <typename T, int kMode, bool kWrite, int kRows>
__global__ void __launch_bounds__(kRopeThreads)
rope_kernel(const __grid_constant__ RopeWork w) {
  __shared__ __align__(16) float2 s_turns[kRopeWarps][kRopeTurns];  // scale * (cos, sin)
  __shared__ __align__(16) char s_stage[kMode == kRopeHalfOdd ? kRopeThreads * 16 : 16];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % kVecPerRow16, second = lane / kVecPerRow16;
  const int64_t unit = (int64_t)blockIdx.x * kRopeWarps + warp;
  const int64_t t = unit <= INT32_MAX ? (unsigned)unit / (unsigned)w.parts : unit / w.parts;
  if (t >= w.tokens) return;
  // the warp's rows are all of x, all of K or all of V
  int part = (int)(unit - t * w.parts), rows = w.heads;
  const uint4* from = w.x + t * w.x_token;
  int64_t step = w.x_head;
  bool key = false, value = false;
  if (kWrite && part >= w.x_parts) {
    part -= w.x_parts;
    rows = w.pool.kv_heads;
    value = part >= w.k_parts;
    key = !value;
    if (value) part -= w.k_parts;
    from = value ? w.v + t * w.v_token : w.k + t * w.k_token;
    step = value ? w.v_head : w.k_head;
  }
  const int first = part * kRows + second;
  const int mine = (rows - first + 1) / 2;       // of this half of the warp, from `first` on
  const int both = (rows - part * kRows + 1) / 2;  // of either: a warp exchanges values
  from += first * step + c;
  uint4 x[kRows / 2];
#pragma unroll
  for (int i = 0; i < kRows / 2; ++i) {
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (i < mine) x[i] = __ldcs(from);
    from += 2 * step;
  }
  const int position = w.positions[t];
  uint4* to = w.out + t * w.out_token + first * w.out_head + c;
  step = w.out_head;
  if (kWrite && (key || value)) {
    const int64_t slot = w.slots[t];
    if (slot < 0 || slot >= w.pool.num_pages * w.pool.page_size) {
      if (slot != -1 && lane == 0) raise_error(w.error_flag, TW_ERR_INVALID_INDEX);
      return;
    }
    const int64_t page = slot <= INT32_MAX ? (unsigned)slot / (unsigned)w.pool.page_size
                                           : slot / w.pool.page_size;
    const int64_t offset = slot - page * w.pool.page_size;
    step = w.pool.head_stride / kPagedAlign;
    to = reinterpret_cast<uint4*>(value ? w.pool.v_pages : w.pool.k_pages) +
         (page * w.pool.page_stride + offset * w.pool.token_stride) / kPagedAlign + first * step +
         c;
    if (value) {
#pragma unroll
      for (int i = 0; i < kRows / 2; ++i)
        if (i < mine) to[2 * i * step] = x[i];
      return;
    }
    const int head = part * kRows + lane;
    if (lane < kRows && head < rows) {
      const int64_t at = (page * w.pool.kv_heads + head) * w.pool.page_size + offset;
      if (w.row_weights) w.row_weights[at] = 0.f;
      if (w.row_positions) w.row_positions[at] = position;
    }
  }

  const int pairs = w.rope.pairs;
  float2* s_turn = s_turns[warp];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = lane * 2 + i;
    if (n < pairs) {
      const double turns = (double)position * w.rope.frequencies[n] *
                           0.15915494309189533577;  // 1 / (2 pi)
      const float angle = 6.283185307179586f * (float)(turns - rint(turns));
      const float sin = w.rope.inverse ? -__sinf(angle) : __sinf(angle);
      s_turn[turn_at(n)] = make_float2(__cosf(angle) * w.rope.scale, sin * w.rope.scale);
    }
  }
  __syncwarp();
  uint64_t cos[4], sin[4];  // of the thread's eight dimensions
  const int turned = min(max(2 * pairs - c * 8, 0), 8);
  if constexpr (kMode == kRopeInterleaved) {
    // (read in twos: what lies behind the last pair is not used)
    const float4* s = reinterpret_cast<const float4*>(&s_turn[turn_at(c * 4)]);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float4 y = s[e / 2];
      cos[e] = pair(y.x, y.x);
      sin[e] = pair(-y.y, y.y);
      cos[e + 1] = pair(y.z, y.z);
      sin[e + 1] = pair(-y.w, y.w);
    }
  } else if constexpr (kMode == kRopeHalf) {
    const int n = c * 8 < pairs ? c * 8 : min(c * 8 - pairs, kRopePairs - 8);
    const float4* s = reinterpret_cast<const float4*>(&s_turn[turn_at(n)]);
    const float sign = c * 8 < pairs ? -1.f : 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 y = s[e];
      cos[e] = pair(y.x, y.z);
      sin[e] = pair(sign * y.y, sign * y.w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float2 cs[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = c * 8 + e + i;
        cs[i] = s_turn[turn_at(min(d < pairs ? d : d - pairs, kRopePairs - 1))];
        if (d < pairs) cs[i].y = -cs[i].y;
      }
      cos[e / 2] = pair(cs[0].x, cs[1].x);
      sin[e / 2] = pair(cs[0].y, cs[1].y);
    }
  }

#pragma unroll
  for (int i = 0; i < kRows / 2; ++i) {
    if (i >= both) break;
    const uint4 y = rotate<T, kMode>(x[i], c, pairs, turned, cos, sin,
                                     s_stage + (warp * 2 + second) * kHeadDim * 2);
    if (i < mine) to[2 * i * step] = y;
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

template <typename T, bool kWrite, int kRows>
static int launch_rope(RopeWork& w, cudaStream_t stream) {
  w.x_parts = (w.heads + kRows - 1) / kRows;
  w.k_parts = kWrite ? (w.pool.kv_heads + kRows - 1) / kRows : 0;
  w.parts = w.x_parts + 2 * w.k_parts;
  const int64_t ctas = (w.tokens * w.parts + kRopeWarps - 1) / kRopeWarps;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  const auto kernel = w.rope.interleaved       ? rope_kernel<T, kRopeInterleaved, kWrite, kRows>
                      : w.rope.pairs % 8 == 0 ? rope_kernel<T, kRopeHalf, kWrite, kRows>
                                              : rope_kernel<T, kRopeHalfOdd, kWrite, kRows>;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(kRopeThreads), 0, stream, w);
}

// Few rows: four a warp, so that they spread over more SMs; many: 16 a warp, which share its
// angles.  us with four, eight, 16 a warp, in a graph of calls (up to 150k rows mostly in L2):
//   rows         2.4k         9.4k         38k          75k          110k           300k
//   40 a token   1.9 2.1 2.7  2.2 2.3 2.8  5.0 4.3 4.3  8.5 6.8 7.7  12  9.1  9.8   33 26 26
//   48, written  2.1 2.2 2.4  2.4 2.3 2.5  5.1 4.3 3.8  9.3 7.6 7.6  13 10.2 10.3   36 27 27
// 8192 tokens of 32 rows (262k), half of each turned: 19.8 with eight, 18.4 with 16, 21.1 with
// 32, which is what 16 are for.
template <typename T, bool kWrite>
static int launch_rope(RopeWork& w, cudaStream_t stream) {
  const int64_t rows = w.tokens * (w.heads + (kWrite ? 2 * w.pool.kv_heads : 0));
  return rows <= kRopeFew    ? launch_rope<T, kWrite, 4>(w, stream)
         : rows <= kRopeMany ? launch_rope<T, kWrite, 8>(w, stream)
                             : launch_rope<T, kWrite, 16>(w, stream);
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
  w.heads = heads;
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
  w.pool = a.pool;
  w.slots = a.slots;
  w.row_weights = a.row_weights;
  w.row_positions = a.row_positions;
  w.error_flag = a.error_flag;
  cudaStream_t s = (cudaStream_t)stream;
  return a.pool.dtype == TW_F16 ? launch_rope<__half, true>(w, s)
                                : launch_rope<__nv_bfloat16, true>(w, s);
}
