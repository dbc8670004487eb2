// Paged attention of requests with few new rows per KV head (a token each, as
// in decoding, or a few): at most 16 rows (tokens x query heads of the group).
//
// Mathematics: for each range of keys, one pass with a running reference m and
// sum l per row: p_j = 2^(s_j - m), l += p_j, O += p_j v_j, both scaled when m
// moves.  m moves only when a score exceeds it by more than 8 (fp16: 15, see kLift;
// p stays below 2^8 or 2^15, far from overflow), so the accumulators are rarely
// rescaled.  A range leaves O / l and m + log2 l; ranges are joined by weights
// 2^(lse_s - max).
//
// Bound: HBM, every K / V row of the visible keys read once per KV head
// (512 bytes a key); the 16-row products are 4 % of what the tensor cores
// could do in that time, so the warp-level mma.sync (one 16 x 8 x 16 product
// per instruction, operands and results in registers) is enough and needs no
// round trip through tensor memory.
//
// Layout: six warps take an item: one KV head of one request and one range of its keys.
// Two warps fetch 64-key tiles (K and V, 32 KB) into a ring of three stages by
// TMA, a box for each page piece; four warps take 16 keys of every tile
// each, keep m, l and O of all 16 rows in registers, and join at the end
// through shared memory.  Two items are resident per SM: up to 192 KB in flight.  They
// are two CTAs in a call of such requests alone.  In a mixed call they are the halves of
// a CTA of the chunk kernel, which takes items after its chunks: the SMs that the last
// chunks leave idle get them, with no second kernel that would have to wait for the end
// of the first.
//
// Measured: 16 requests from 8k to 131k, 32 / 8 heads: 708 us, 6.48 TB/s (99 %
// of the measured copy rate); 256 requests up to 2k, 64 / 8 heads: 185 us, 5.7
// TB/s; one request at 32k: 29 us with the merge, 4.6 TB/s (3 us pass before the
// first tile, and nothing is read while the warps join).
#pragma once

#include "paged_attention.cuh"

namespace tw {

constexpr int kTokRows = 16;
constexpr int kTokTile = 64;       // keys per stage
constexpr int kTokStages = 3;
constexpr int kTokWarps = 4;       // consumers
constexpr int kTokThreads = (kTokWarps + 2) * 32;  // and a warp that copies K, one V
constexpr int kTokHalf = kTokTile * 128;          // 64 of the 128 dimensions of a tile
constexpr int kTokStageBytes = 4 * kTokHalf;      // K lo, K hi, V lo, V hi
constexpr int kTokRowPad = kHeadDim + 4;          // floats per row of the join
constexpr int kTokRing = kTokStages * kTokStageBytes;
constexpr float kMoveBy = 8.0f;    // log2 units

template <typename T> struct MmaType;
template <> struct MmaType<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct MmaType<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Offset of element (row, d) of a [64 rows][128] tile stored as two halves of
// 128-byte rows with the 16-byte columns of each row XORed by row % 8.
__device__ __forceinline__ uint32_t tok_offset(int row, int d) {
  return (uint32_t)((d >> 6) * kTokHalf + row * 128 + (((d & 63) * 2) ^ ((row & 7) << 4)));
}

// Barriers of an item's threads and of its consumers (0 and 1 are the chunk kernel's).
__device__ __forceinline__ void item_sync(int half) {
  asm volatile("bar.sync %0, %1;" ::"r"(2 + half), "n"(kTokThreads) : "memory");
}
__device__ __forceinline__ void consumer_sync(int half) {
  asm volatile("bar.sync %0, %1;" ::"r"(4 + half), "n"(kTokWarps * 32) : "memory");
}

struct TokShared {
  uint64_t full[kTokStages], empty[kTokStages];
  float m[kTokWarps][kTokRows], l[kTokWarps][kTokRows];
  volatile int abort;
  // Keys with a V value that is not finite and that some row does not see, a bit each:
  // 1..15: later than the first token by so much; 16..30: before the last token's
  // window, so much (less 16) after the first key.
  unsigned odd;
};

// By one of the item's threads, before any is in token_item.
__device__ __forceinline__ void token_init(TokShared& sh) {
  for (int i = 0; i < kTokStages; ++i) {
    mbar_init(&sh.full[i], 2);
    mbar_init(&sh.empty[i], kTokWarps);
  }
  sh.abort = 0;
  sh.odd = 0;
  mbar_init_fence();
}

inline int64_t paged_token_items(const PagedWork& w) {
  return (int64_t)w.a.requests * w.a.pool.kv_heads * w.few.splits;
}

// Item `item` (request, KV head, range) by kTokThreads threads, tid being the caller's
// among them, thread 0 of which has called token_init; `smem`: kTokRing bytes on a
// 1024-byte boundary; `half`: which of the CTA's groups of so many threads they are.  The
// caller's grid has waited.
template <typename T, typename Out>
__device__ __forceinline__ void token_item(const PagedWork& w, const PagedMaps& maps, char* smem,
                                           TokShared& sh, int64_t item, int half, int tid) {
  const tw_paged_attention_args& a = w.a;
  const int lane = tid & 31, warp = tid >> 5;
  const int kv_heads = a.pool.kv_heads;
  const int split = (int)(item % w.few.splits);
  const int unit = (int)(item / w.few.splits);
  const int b = unit / kv_heads;
  const int g = unit - b * kv_heads;
  // Lane l < boxes of a copying warp knows the page of box l of the next tile; the
  // first, where it has to be without a window, is read together with the lengths:
  // one round trip less before the first copy.
  const int boxes = kTokTile / w.box;
  const int box = lane % boxes;
  const int32_t* table = a.block_table + (int64_t)b * a.table_stride;
  const int guess = split * w.few.chunk + box * w.box;
  int page = 0;
  if (warp >= kTokWarps && a.window == 0 && guess / a.pool.page_size < a.table_width)
    page = table[guess / a.pool.page_size];
  const PagedRequest rq = paged_request(a, b);
  if (rq.n == 0) return;
  if (rq.n > w.few_tokens || rq.n > a.max_q_len) {
    if (rq.n > a.max_q_len && tid == 0) raise_error(a.error_flag, TW_ERR_BAD_ARG);
    return;
  }
  const PagedKeys keys = paged_keys(a, rq, 0, rq.n);
  const PagedRange range = paged_range(w.few, keys.low, keys.high, split);
  if (split >= range.parts) return;
  const int R = w.group;
  const int rows = rq.n * R;
  const int low = max(range.begin, keys.low);  // first key that some row sees, in this range
  const int tile0 = low / kTokTile * kTokTile;
  const int tiles = range.end > low ? (range.end - tile0 + kTokTile - 1) / kTokTile : 0;

  const uint32_t ring = smem_addr(smem);
  item_sync(half);

  if (warp >= kTokWarps) {
    // ---- copies: a warp those of K, a warp those of V
    const int matrix = warp - kTokWarps;
    const CUtensorMap* map = matrix == 0 ? &maps.k : &maps.v;
    const uint32_t box_bytes = (uint32_t)w.box * 128;  // of 64 dimensions
    int key = tile0 + box * w.box;
    // boxes wholly before the first visible key are not read: a page that slid out
    // of the window may be gone
    const int skipped = (low - tile0) / w.box;
    if (key != guess || a.window != 0)
      page = key < range.end && box >= skipped ? table[key / a.pool.page_size] : 0;
    int i = 0;
    for (; i < tiles; ++i) {
      const int stage = i % kTokStages;
      int p = page;
      if (lane < boxes && key < range.end && (i > 0 || box >= skipped) &&
          (p < 0 || p >= a.pool.num_pages)) {
        raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
        p = (int)a.pool.num_pages;  // out of the map's range: zeros
      }
      key += kTokTile;
      if (i + 1 < tiles && key < range.end) page = table[key / a.pool.page_size];
      if (i >= kTokStages &&
          !__all_sync(0xffffffffu, mbar_wait<false>(&sh.empty[stage],
                                                    (uint32_t)((i / kTokStages - 1) & 1), &sh.abort)))
        break;
      const int first = tile0 + i * kTokTile;
      const int from = i == 0 ? skipped : 0;
      const int to = (min(range.end - first, kTokTile) + w.box - 1) / w.box;
      int row = (first + from * w.box) % a.pool.page_size;  // of the next box in its page
      uint32_t dst = ring + stage * kTokStageBytes + matrix * 2 * kTokHalf + from * box_bytes;
      if (elect_one()) mbar_arrive_expect(&sh.full[stage], (uint32_t)(to - from) * box_bytes * 2);
      for (int x = from; x < to; x += 4) {  // four boxes a turn: their pages at once
        int px[4], rx[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          px[y] = __shfl_sync(0xffffffffu, p, x + y);
          rx[y] = row;
          row += w.box;
          if (row == a.pool.page_size) row = 0;
        }
        if (elect_one()) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (x + y < to) {
              tma_load_4d(map, dst + y * box_bytes, &sh.full[stage], 0, rx[y], g, px[y]);
              tma_load_4d(map, dst + kTokHalf + y * box_bytes, &sh.full[stage], 64, rx[y], g, px[y]);
            }
        }
        dst += 4 * box_bytes;
      }
    }
    if (sh.abort) {
      // give up: wait (with the same limit) for the copies in flight
      volatile int never = 0;
      for (int j = max(0, i - kTokStages); j < i; ++j)
        mbar_wait<false>(&sh.full[j % kTokStages], (uint32_t)((j / kTokStages) & 1), &never);
    }
    return;
  }

  // ---- consumers: fragments of the 16 query rows, row r = token * R + head
  uint32_t qf[8][4];
  const int r0 = lane >> 2, r1 = r0 + 8;
  const int c0 = (lane & 3) * 2;
  {
    const T* q0 = (const T*)a.q + (int64_t)(rq.first + r0 / R) * a.q_token_stride +
                  (int64_t)(g * R + r0 % R) * a.q_head_stride + c0;
    const T* q1 = (const T*)a.q + (int64_t)(rq.first + r1 / R) * a.q_token_stride +
                  (int64_t)(g * R + r1 % R) * a.q_head_stride + c0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      qf[k][0] = r0 < rows ? *reinterpret_cast<const uint32_t*>(q0 + k * 16) : 0u;
      qf[k][1] = r1 < rows ? *reinterpret_cast<const uint32_t*>(q1 + k * 16) : 0u;
      qf[k][2] = r0 < rows ? *reinterpret_cast<const uint32_t*>(q0 + k * 16 + 8) : 0u;
      qf[k][3] = r1 < rows ? *reinterpret_cast<const uint32_t*>(q1 + k * 16 + 8) : 0u;
    }
  }
  // visible keys of the thread's two rows (rows past the last see what row 0 sees)
  const int p0 = rq.kv - rq.n + (r0 < rows ? r0 / R : 0);
  const int p1 = rq.kv - rq.n + (r1 < rows ? r1 / R : 0);
  const int low0 = paged_low(a, p0), low1 = paged_low(a, p1);
  // keys that every row sees: tiles inside need no mask
  const int all_low = paged_low(a, rq.kv - 1), all_high = rq.kv - rq.n + 1;

  float acc[16][4];
#pragma unroll
  for (int d = 0; d < 16; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[d][c] = 0.f;
  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
  const int wrow = warp * 16;  // the warp's keys of a tile
  const uint32_t k_at = ring + tok_offset(wrow + (lane >> 4) * 8 + (lane & 7), 0);
  const int k_col = ((lane >> 3) & 1) * 16;  // bytes
  const int k_xor = (lane & 7) << 4;
  const uint32_t v_at = ring + 2 * kTokHalf + (wrow + ((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
  const int v_col = (lane >> 4) * 16;

  for (int i = 0; i < tiles; ++i) {
    const int stage = i % kTokStages;
    const uint32_t base = stage * kTokStageBytes;
    const int key0 = tile0 + i * kTokTile + wrow;  // the warp's first key
    if (!__all_sync(0xffffffffu,
                    mbar_wait<false>(&sh.full[stage], (uint32_t)((i / kTokStages) & 1), &sh.abort)))
      break;
    if (key0 < range.end && key0 + 16 > low) {
      const bool edge = key0 < all_low || key0 + 16 > all_high || key0 < low ||
                        key0 + 16 > range.end;
      float s[2][4];
#pragma unroll
      for (int c = 0; c < 4; ++c) s[0][c] = s[1][c] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t kb[4];
        ldmatrix4(kb, k_at - (((lane & 7) << 4)) + base + (k >> 2) * kTokHalf +
                          ((((k & 3) * 32) + k_col) ^ k_xor));
        MmaType<T>::mma(s[0], qf[k], kb[0], kb[1]);
        MmaType<T>::mma(s[1], qf[k], kb[2], kb[3]);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[n][c] *= w.scale_log2;
      if (edge) {
        // hide what a row does not see, and clear V rows that none sees and what is not
        // finite in those that some row does not see: that must not meet a weight of
        // zero (the rows that do see such a value get it added at the end)
        const int first = key0 + c0;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int j = first + n * 8 + (c & 1);
            const bool seen = c < 2 ? (j >= low0 && j <= p0) : (j >= low1 && j <= p1);
            if (!seen || j < range.begin || j >= range.end) s[n][c] = -CUDART_INF_F;
          }
        const int row = lane >> 1;
        const int j = key0 + row;
        uint4* z = reinterpret_cast<uint4*>(smem + base + 2 * kTokHalf + (lane & 1) * kTokHalf +
                                            (wrow + row) * 128);
        if (j < low || j >= range.end) {
#pragma unroll
          for (int c = 0; c < 8; ++c) z[c] = make_uint4(0u, 0u, 0u, 0u);
        } else if (j >= all_high || j < all_low) {
          bool odd = false;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint4 x = z[c];
            if (clear_odd<T>(x)) {
              z[c] = x;
              odd = true;
            }
          }
          if (odd) atomicOr(&sh.odd, 1u << (j >= all_high ? j - all_high + 1 : j - keys.low + 16));
        }
        __syncwarp();
      }
      float t0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float t1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, off));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
      }
      const bool move0 = t0 - m0 > kMoveBy + kLift<T>, move1 = t1 - m1 > kMoveBy + kLift<T>;
      if (__any_sync(0xffffffffu, move0 || move1)) {
        const float n0 = move0 ? t0 - kLift<T> : m0, n1 = move1 ? t1 - kLift<T> : m1;
        // an unmoved reference keeps its sums (-inf - -inf would be NaN)
        const float f0 = move0 ? ex2(m0 - n0) : 1.f, f1 = move1 ? ex2(m1 - n1) : 1.f;
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int d = 0; d < 16; ++d) {
          acc[d][0] *= f0;
          acc[d][1] *= f0;
          acc[d][2] *= f1;
          acc[d][3] *= f1;
        }
      }
      const float u0 = m0 == -CUDART_INF_F ? 0.f : m0, u1 = m1 == -CUDART_INF_F ? 0.f : m1;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][0] = ex2(s[n][0] - u0);
        s[n][1] = ex2(s[n][1] - u0);
        s[n][2] = ex2(s[n][2] - u1);
        s[n][3] = ex2(s[n][3] - u1);
        l0 += s[n][0] + s[n][1];
        l1 += s[n][2] + s[n][3];
      }
      // weights rounded to the 16-bit type for the product (the sum l keeps them
      // in 32 bits): half a unit each, of either sign
      const uint32_t pf[4] = {MmaType<T>::pack(s[0][0], s[0][1]), MmaType<T>::pack(s[0][2], s[0][3]),
                              MmaType<T>::pack(s[1][0], s[1][1]), MmaType<T>::pack(s[1][2], s[1][3])};
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        uint32_t vb[4];
        ldmatrix4_trans(vb, v_at + base + (d >> 2) * kTokHalf +
                                ((((d & 3) * 32) + v_col) ^ k_xor));
        MmaType<T>::mma(acc[2 * d], pf, vb[0], vb[1]);
        MmaType<T>::mma(acc[2 * d + 1], pf, vb[2], vb[3]);
      }
      if (edge) fence_async_smem();  // the cleared rows, before the next copy into them
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[stage]);
  }

  // ---- join the four warps
  if (sh.abort && lane == 0) raise_error(a.error_flag, TW_ERR_TIMEOUT);
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, off);
    l1 += __shfl_xor_sync(0xffffffffu, l1, off);
  }
  consumer_sync(half);  // the ring is free: every tile has been read
  float* s_o = reinterpret_cast<float*>(smem);  // [warps][rows][kTokRowPad]
#pragma unroll
  for (int d = 0; d < 16; ++d) {
    float* o = s_o + (warp * kTokRows + r0) * kTokRowPad + d * 8 + c0;
    *reinterpret_cast<float2*>(o) = make_float2(acc[d][0], acc[d][1]);
    *reinterpret_cast<float2*>(o + 8 * kTokRowPad) = make_float2(acc[d][2], acc[d][3]);
  }
  if ((lane & 3) == 0) {
    sh.m[warp][r0] = m0;
    sh.m[warp][r1] = m1;
    sh.l[warp][r0] = l0;
    sh.l[warp][r1] = l1;
  }
  consumer_sync(half);
  const bool joined = range.parts == 1;
  {
    const int r = tid >> 3, d0 = (tid & 7) * 16;
    float m = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < kTokWarps; ++k) m = fmaxf(m, sh.m[k][r]);
    const float u = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f, o[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] = 0.f;
#pragma unroll
    for (int k = 0; k < kTokWarps; ++k) {
      const float f = ex2(sh.m[k][r] - u);
      l = fmaf(sh.l[k][r], f, l);
      const float* x = s_o + (k * kTokRows + r) * kTokRowPad + d0;
#pragma unroll
      for (int c = 0; c < 16; ++c) o[c] = fmaf(x[c], f, o[c]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] *= inv;
    // what was cleared before the product and this row does see
#pragma unroll 1
    for (unsigned bits = r < rows ? sh.odd : 0u; bits; bits &= bits - 1) {
      const int bit = __ffs(bits) - 1, p = rq.kv - rq.n + r / R;
      const int k = bit < 16 ? all_high + bit - 1 : keys.low + bit - 16;
      const T* v = k >= paged_low(a, p) && k <= p ? paged_value<T>(a, b, g, k) : nullptr;
      if (!v) continue;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float y = to_f32<T>(v[d0 + c]);
        if (!(fabsf(y) < CUDART_INF_F)) o[c] += y;
      }
    }
    if (r < rows) {
      const int t = rq.first + r / R, h = g * R + r % R;
      if (joined)
        paged_store_row<Out, 16>(a, t, h, d0, o, paged_lse(m, l));
      else
        paged_store_part<16>(w.few, (int64_t)unit * w.few_rows + r, split, d0, o,
                             paged_lse2(m, l));
    }
  }
}

}  // namespace tw
