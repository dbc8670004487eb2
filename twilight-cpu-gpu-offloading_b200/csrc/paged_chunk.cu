// Paged attention of requests with many new tokens: chunks of prompts.
//
// Mathematics as in the token kernel (reference m that moves only when a score
// exceeds it by more than 8 in log2 units, sum l, O), on 128 x 128 products.
//
// Bound: the tensor cores, 4 D flops per visible (row, key): S = Q K^T and
// O += P V.  Next to them the special-function unit, one 2^x per pair, which
// takes as long as the two products (16 a clock against 8192 flops a clock).
//
// Layout: a CTA takes 2 x 128 rows of one KV head, a row being a (token, query
// head of the group) pair, so K and V are read once for all heads of the group
// and each tile of 128 keys once for both halves.  One thread issues all
// products; two warps copy Q, and K and V tiles by TMA into a ring of five 32 KB
// slots, page piece by page piece; one warp looks over the V tiles that hold keys
// which some row does not see; two warpgroups take one half each, a thread one
// row: it reads its row of S from tensor memory, writes the weights P back over it
// in 16 bits, and the product with V takes P from there.  The halves alternate:
// while one computes its weights, the tensor cores work for the other.  (Two
// threads a row, or two issuing threads, measured slower.)
//
// Measured: 4096 tokens over a 32k context, 64 / 8 heads: 3.57 ms, 1.15
// PFLOP/s, at the board's power limit (1.5 to 1.6 GHz); 2048 tokens, 32 / 8
// heads: 1.0 ms there, 47 us as a prompt of their own.  The tensor pipe is busy
// 67 % of a busy SM's cycles; a tile takes 1.8 us, and each CTA 6 us more.  The
// looking warp costs a prompt of 2048 tokens 1.5 us, a windowed call 3 of 76.
#include "paged_token.cuh"
#include "tensor.cuh"

#include <type_traits>

namespace tw {

constexpr int kChRows = 128;                      // rows of a half
constexpr int kChSoftmax = 256;                   // threads 0..255: the halves' rows
constexpr int kChMmaWarp = 8, kChKeyWarp = 9, kChValueWarp = 10, kChLookWarp = 11;
constexpr int kChThreads = 384;
// Registers: the launch gives 168 to each of 384 threads; the warpgroups of the
// rows take from the third: 216 + 216 + 72 = 3 * 168.
constexpr int kChRowRegs = 216, kChIssueRegs = 72;
constexpr int kChHalfTile = 128 * 128;            // bytes: 128 rows of 64 elements
constexpr int kChTileBytes = 2 * kChHalfTile;
constexpr int kChSlots = 5;
constexpr int kChSmem = (2 + kChSlots) * kChTileBytes + 1024;
constexpr int kChColumns = 512;                   // S0, S1, O0, O1: 128 columns each
constexpr float kChMoveBy = 8.0f;                 // log2 units
constexpr float kChNear = 1048576.0f;             // log2 units
constexpr int kChFma = 8;                         // one pair in this many on the FMA pipe

template <typename T> struct Pack16;
template <> struct Pack16<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t add_zero_times(uint32_t two, uint32_t sum) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(two), "r"(0u), "r"(sum));
    return r;
  }
};
template <> struct Pack16<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t add_zero_times(uint32_t two, uint32_t sum) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(two), "r"(0u), "r"(sum));
    return r;
  }
};

// The lowest n bits (n <= 0: none, n >= 32: all).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}

// The looking warp is done; the rows' threads wait for that.
__device__ __forceinline__ void looked_arrive() {
  asm volatile("bar.arrive 1, %0;" ::"n"(kChSoftmax + 32) : "memory");
}
__device__ __forceinline__ void looked_wait() {
  asm volatile("bar.sync 1, %0;" ::"n"(kChSoftmax + 32) : "memory");
}

// The warp's 32 rows on their way out: 16-byte columns XORed by row % 8.
template <typename Out>
__device__ __forceinline__ void stage_row(char* smem, int warp, int row, int quarter,
                                          const float (&o)[32]) {
  constexpr int kVec = 16 / sizeof(Out);  // elements of a column
  char* base = smem + (warp * 32 + row) * (kHeadDim * (int)sizeof(Out));
#pragma unroll
  for (int c = 0; c < 32 / kVec; ++c) {
    __align__(16) Out x[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = from_f32<Out>(o[c * kVec + e]);
    const int column = (quarter * (32 / kVec) + c) ^ (row & 7);
    *reinterpret_cast<uint4*>(base + column * 16) = *reinterpret_cast<uint4*>(x);
  }
}
template <typename Out, typename Place>
__device__ __forceinline__ void write_rows(const char* smem, int warp, int lane, Place place) {
  constexpr int kColumns = kHeadDim * (int)sizeof(Out) / 16;  // 16 or 32
  constexpr int kRows = 32 / kColumns;                        // rows a turn
  const int column = lane % kColumns;
#pragma unroll 4
  for (int x = 0; x < 32; x += kRows) {
    const int row = x + lane / kColumns;
    Out* to = place(row);
    if (to)
      reinterpret_cast<uint4*>(to)[column] = *reinterpret_cast<const uint4*>(
          smem + (warp * 32 + row) * (kHeadDim * (int)sizeof(Out)) + ((column ^ (row & 7)) * 16));
  }
}

// Adds what is not finite in a V row, of which the lane holds dimensions 4l .. 4l + 3 in
// `x`, to the warp's staged rows in `rows` (a bit each), four rows at a time.
template <typename T, typename Out>
__device__ __forceinline__ void add_odd_staged(char* smem, int warp, int lane, uint2 x,
                                               unsigned rows) {
  constexpr int kVec = 16 / sizeof(Out);
  struct __align__(4 * sizeof(Out)) Four {
    Out v[4];
  };
  if (!(odd_halves<T>(x.x) | odd_halves<T>(x.y))) return;
  const T* v = reinterpret_cast<const T*>(&x);
  float y[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) y[c] = to_f32<T>(v[c]);
#pragma unroll 1
  for (int first = 0; first < 32; first += 4, rows >>= 4) {
    if (!(rows & 15)) continue;
    Four* at[4];
    Four o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = first + r;
      at[r] = reinterpret_cast<Four*>(
          reinterpret_cast<Out*>(smem + (warp * 32 + row) * (kHeadDim * (int)sizeof(Out))) +
          ((lane * 4 / kVec) ^ (row & 7)) * kVec + lane * 4 % kVec);
      o[r] = *at[r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (!(fabsf(y[c]) < CUDART_INF_F)) o[r].v[c] = from_f32<Out>(to_f32<Out>(o[r].v[c]) + y[c]);
      if (rows >> r & 1) *at[r] = o[r];
    }
  }
}

// Keys of the CTA that hold a V value that is not finite and that some row does not see,
// a bit each: [0]: later than the first token, by distance from it; [1]: before the last
// token's window, by distance from the first key.
struct ChunkOdd {
  unsigned bits[2][8];  // at most 255 each: the CTA has at most 256 tokens
  int any;
};

struct ChunkShared {
  uint64_t full[kChSlots], empty[kChSlots];
  uint64_t loaded[kChSlots];    // a V tile that has to be looked over is there
  uint64_t q_full;
  uint64_t s_full[2];           // scores of a half
  uint64_t p_full[2][2];        // weights of a half: keys 0..63, 64..127 of the tile
  uint64_t o_full, drain;
  uint32_t tmem;
  volatile int abort;
  ChunkOdd odd;
};

// kMixed: some requests may have few tokens, whose items the grid takes too.  (A kernel of
// its own: with the items' code in it a call of one short chunk takes 0.3 us longer.)
template <typename T, typename Out, bool kMixed>
__global__ void __launch_bounds__(kChThreads, 1)
paged_chunk_kernel(const __grid_constant__ PagedWork w, const __grid_constant__ PagedMaps maps,
                   const __grid_constant__ CUtensorMap q_map) {
  extern __shared__ char s_raw[];
  __shared__ ChunkShared sh;
  const tw_paged_attention_args& a = w.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kv_heads = a.pool.kv_heads;
  const int R = w.group;
  const int tokens = paged_chunk_tokens(R), half_tokens = tokens / 2;
  char* smem = (char*)(((uintptr_t)s_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t q_at = smem_addr(smem);
  const uint32_t ring = q_at + 2 * kChTileBytes;
  if (tid == 0) {
    for (int i = 0; i < kChSlots; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
      mbar_init(&sh.loaded[i], 1);
    }
    mbar_init(&sh.q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i][0], 4);
      mbar_init(&sh.p_full[i][1], 4);
    }
    mbar_init(&sh.o_full, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    mbar_init_fence();
  }
  if (tid < 16) sh.odd.bits[tid >> 3][tid & 7] = 0;
  if (tid == 16) sh.odd.any = 0;
  pdl_wait();
  pdl_launch_dependents();

  // The CTA's request: a request with rows [c, d) owns the slots from
  // c / tokens + b on, one per `tokens` rows, and no two requests share one.
  // The last slots come first: within a request they see the most keys.
  const int64_t cta = blockIdx.x;
  const int split = (int)(cta % w.many.splits);
  const int g = (int)(cta / w.many.splits % kv_heads);
  const int slots = a.tokens / tokens + a.requests;
  const int64_t ctas = (int64_t)slots * kv_heads * w.many.splits;
  if constexpr (kMixed) {
    if (cta >= ctas + kPadCtas) {  // two items
      static_assert(kChThreads == 2 * kTokThreads);
      __shared__ TokShared tok[2];
      const int half = tid >= kTokThreads, at = tid - half * kTokThreads;
      const int64_t item = (cta - ctas - kPadCtas) * 2 + half;
      if (item >= (int64_t)a.requests * kv_heads * w.few.splits) return;
      if (at == 0) token_init(tok[half]);
      token_item<T, Out>(w, maps, smem + half * kTokRing, tok[half], item, half, at);
      return;
    }
  }
  if (cta >= ctas) {
    paged_clear_padding<Out>(a, (int)(cta - ctas));
    return;
  }
  const int slot = slots - 1 - (int)(cta / w.many.splits / kv_heads);
  // last b whose first slot is <= slot: 32 candidates a round
  int b = 0;
  for (int n = a.requests; n > 1;) {
    const int stride = (n + 31) / 32;
    const int i = lane * stride;
    const bool at_most = i < n && a.cu_q[b + i] / tokens + b + i <= slot;
    const int k = max(__popc(__ballot_sync(0xffffffffu, at_most)) - 1, 0);
    b += k * stride;
    n = min(stride, n - k * stride);
  }
  // Lane l < boxes of a copying warp knows the page of box l of the next tile; the
  // first, where it has to be without a window, is read together with the lengths.
  const int boxes = kTileKeys / w.box;
  const int32_t* table = a.block_table + (int64_t)b * a.table_stride;
  const bool copies = (warp == kChKeyWarp || warp == kChValueWarp) && lane < boxes;
  const int guess = split * w.many.chunk + lane * w.box;
  int page = 0;
  if (copies && a.window == 0 && guess / a.pool.page_size < a.table_width)
    page = table[guess / a.pool.page_size];
  const PagedRequest rq = paged_request(a, b);
  const int begin = (slot - (rq.first / tokens + b)) * tokens;  // first token of the CTA
  if (rq.n <= w.few_tokens || begin >= rq.n || begin < 0) return;
  if (rq.n > a.max_q_len) {
    if (tid == 0) raise_error(a.error_flag, TW_ERR_BAD_ARG);
    return;
  }
  const int here = min(rq.n - begin, tokens);    // tokens of the CTA
  const PagedKeys keys = paged_keys(a, rq, begin, here);
  const PagedRange range = paged_range(w.many, keys.low, keys.high, split);
  if (split >= range.parts) return;
  const int halves = here > half_tokens ? 2 : 1;
  const int p_first = rq.kv - rq.n + begin;      // position of the first token
  const int low = max(range.begin, keys.low), high = range.end;
  const int key0 = low / kTileKeys * kTileKeys;
  const int tiles = high > low ? (high - key0 + kTileKeys - 1) / kTileKeys : 0;

  // Tiles of V with rows that are not of the range, or that not all tokens see.  What
  // those hold must not meet a weight of zero in the product (0 x NaN, 0 x infinity):
  // the looking warp clears them and what is not finite in them before it hands a tile
  // on, and the rows that do see such a value get it added at the end.
  const int see_last = paged_low(a, max(p_first + here - 1, 0));
  const auto look = [&](int first) {
    return first < max(low, see_last) || first + kTileKeys > min(high, p_first + 1);
  };

  // Boxes wholly before the first visible key are not read: a page that slid out
  // of the window may be gone.
  const int skipped = (low - key0) / w.box;
  int key = key0 + lane * w.box;
  if (copies && (key != guess || a.window != 0))
    page = key < high && lane >= skipped ? table[key / a.pool.page_size] : 0;
  if (warp == kChMmaWarp) tmem_alloc(&sh.tmem, kChColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = sh.tmem;

  // (the register split inside the branches: past a join the smaller number holds)
  if (warp >= kChMmaWarp) {
    shrink_registers<kChIssueRegs>();
    if (warp == kChKeyWarp || warp == kChValueWarp) {
      // ---- copies: one warp those of Q and K, one those of V.  Ring slot n % kChSlots:
      // n = 2j is K tile j, n = 2j + 1 is V tile j.
      const bool values = warp == kChValueWarp;
      const CUtensorMap* map = values ? &maps.v : &maps.k;
      if (elect_one()) {
        prefetch_map(map);
        if (!values) {
          mbar_arrive_expect(&sh.q_full, (uint32_t)(halves * R * half_tokens * kHeadDim * 2));
          for (int i = 0; i < halves && tiles > 0; ++i)
            for (int d = 0; d < 2; ++d)
              tma_load_3d(&q_map, q_at + i * kChTileBytes + d * kChHalfTile, &sh.q_full, d * 64,
                          g * R, rq.first + begin + i * half_tokens);
        }
      }
      __syncwarp();
      const uint32_t box_bytes = (uint32_t)w.box * 128;  // of 64 dimensions
      int n = values ? 1 : 0;
      uint32_t looked = 0, turn = 0;  // a bit per slot: its last tile gets looked over; phase
      bool ok = true;
      for (int j = 0; j < tiles; ++j, n += 2) {
        int p = page;
        if (lane < boxes && key < high && (j > 0 || lane >= skipped) &&
            (p < 0 || p >= a.pool.num_pages)) {
          raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
          p = (int)a.pool.num_pages;  // out of the map's range: zeros
        }
        key += kTileKeys;
        if (lane < boxes && j + 1 < tiles && key < high) page = table[key / a.pool.page_size];
        const int first = key0 + j * kTileKeys;
        const int valid = min(high - first, kTileKeys);
        const int from = j == 0 ? skipped : 0, to = (valid + w.box - 1) / w.box;
        const int s = n % kChSlots;
        if (n >= kChSlots) {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[s], (uint32_t)((n / kChSlots - 1) & 1),
                                                 &sh.abort));
          if (!ok) break;
        }
        const bool passes = values && look(first);  // by the looking warp
        uint64_t* bar = passes ? &sh.loaded[s] : &sh.full[s];
        looked = passes ? looked | 1u << s : looked & ~(1u << s);
        turn ^= (uint32_t)passes << s;
        if (elect_one()) mbar_arrive_expect(bar, (uint32_t)(to - from) * box_bytes * 2);
        uint32_t dst = ring + s * kChTileBytes + from * box_bytes;
        int row = (first + from * w.box) % a.pool.page_size;  // of the next box in its page
        for (int x = from; x < to; x += 4) {  // four boxes a turn: their pages at once
          int px[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) px[y] = __shfl_sync(0xffffffffu, p, x + y);
          int rx[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            rx[y] = row;
            row += w.box;
            if (row == a.pool.page_size) row = 0;
          }
          if (elect_one()) {
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (x + y < to) {
                tma_load_4d(map, dst + y * box_bytes, bar, 0, rx[y], g, px[y]);
                tma_load_4d(map, dst + kChHalfTile + y * box_bytes, bar, 64, rx[y], g, px[y]);
              }
          }
          dst += 4 * box_bytes;
        }
      }
      if (!ok || sh.abort) {
        // give up: wait (with the same limit) for the copies in flight
        volatile int never = 0;
        mbar_wait(&sh.q_full, 0, &never);
        for (int i = n - 2; i >= 0 && i > n - 2 - kChSlots; i -= 2) {
          const int s = i % kChSlots;
          if (looked >> s & 1)
            mbar_wait(&sh.loaded[s], ~(turn >> s) & 1, &never);
          else
            mbar_wait(&sh.full[s], (uint32_t)((i / kChSlots) & 1), &never);
        }
      }
    } else if (warp == kChLookWarp) {
      // ---- V tiles with keys that some row does not see
      uint32_t turn = 0;
      bool ok = true;
      for (int j = 0; j < tiles && ok; ++j) {
        const int first = key0 + j * kTileKeys;
        if (!look(first)) continue;
        const int s = (2 * j + 1) % kChSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.loaded[s], turn >> s & 1, &sh.abort));
        if (!ok) break;
        turn ^= 1u << s;
        char* tile = smem + (2 + s) * kChTileBytes;
        auto at = [&](int i) {  // 16-byte vector i of the tile's rows
          return reinterpret_cast<uint4*>(tile + ((i >> 3) & 1) * kChHalfTile + (i >> 4) * 128) +
                 (i & 7);
        };
        // rows [0, c0) and [c1, 128) are not of the range; [c0, before): not all tokens'
        // windows begin so early; [after, c1): later than the first token
        const int c0 = max(low - first, 0), c1 = min(high - first, kTileKeys);
        const int after = min(max(p_first + 1 - first, c0), c1);
        const int before = min(max(see_last - first, c0), after);
        for (int i = lane; i < c0 * 16; i += 32) *at(i) = make_uint4(0u, 0u, 0u, 0u);
        for (int i = c1 * 16 + lane; i < kTileKeys * 16; i += 32)
          *at(i) = make_uint4(0u, 0u, 0u, 0u);
        // is there any (0 times it is NaN): eight vectors on their way at a time
        uint32_t sum[4] = {0u, 0u, 0u, 0u};
        auto find = [&](int from, int to) {
#pragma unroll 8
          for (int i = from * 16 + lane; i < to * 16; i += 32) {
            const uint4 x = *at(i);
            sum[0] = Pack16<T>::add_zero_times(x.x, sum[0]);
            sum[1] = Pack16<T>::add_zero_times(x.y, sum[1]);
            sum[2] = Pack16<T>::add_zero_times(x.z, sum[2]);
            sum[3] = Pack16<T>::add_zero_times(x.w, sum[3]);
          }
        };
        find(c0, before);
        find(after, c1);
        const uint32_t odd = odd_halves<T>(sum[0]) | odd_halves<T>(sum[1]) |
                             odd_halves<T>(sum[2]) | odd_halves<T>(sum[3]);
        if (__any_sync(0xffffffffu, odd != 0)) {
          if (lane == 0) sh.odd.any = 1;
          for (int r0 = c0; r0 < c1; r0 += 2) {  // two rows of 16 vectors
            const int r = r0 + (lane >> 4);
            bool found = false;
            if (r < c1 && (r < before || r >= after)) {
              uint4 x = *at(r * 16 + (lane & 15));
              found = clear_odd<T>(x);
              if (found) *at(r * 16 + (lane & 15)) = x;
            }
            if ((__ballot_sync(0xffffffffu, found) >> (lane & 16) & 0xffff) && (lane & 15) == 0) {
              const int kind = r >= after ? 0 : 1;
              const int bit = first + r - (kind == 0 ? p_first : keys.low);
              atomicOr(&sh.odd.bits[kind][bit >> 5], 1u << (bit & 31));
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.full[s]);
      }
      looked_arrive();
    } else if (warp == kChMmaWarp) {
      // ---- products, all issued by one thread
      if (tiles > 0 && elect_one()) {
        constexpr uint32_t desc_s = product_desc(Pack16<T>::kBf16, kTileKeys, false);
        constexpr uint32_t desc_o = product_desc(Pack16<T>::kBf16, kHeadDim, true);
        // S of half i from Q_i and the K tile in ring slot s
        auto scores = [&](int i, int s) {
          const uint32_t qa = q_at + i * kChTileBytes, ka = ring + s * kChTileBytes;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t off = (k >> 2) * kChHalfTile + (k & 3) * 32;
            mma_smem(tmem + i * 128, operand_desc(qa + off, 16, 1024),
                     operand_desc(ka + off, 16, 1024), desc_s, k > 0);
          }
          mma_commit(&sh.s_full[i]);
        };
        auto values = [&](int i, int s, int part, bool add) {
          const uint32_t va = ring + s * kChTileBytes;
#pragma unroll
          for (int k = part * 4; k < part * 4 + 4; ++k)
            mma_tmem(tmem + 256 + i * 128, tmem + i * 128 + k * 8,
                     operand_desc(va + k * 2048, kChHalfTile, 1024), desc_o, add || k > 0);
        };
        auto wait_slot = [&](int n) {
          return mbar_wait(&sh.full[n % kChSlots], (uint32_t)((n / kChSlots) & 1), &sh.abort);
        };
        bool ok = mbar_wait(&sh.q_full, 0, &sh.abort) && wait_slot(0);
        if (ok) {
          tmem_fence_after();
          for (int i = 0; i < halves; ++i) scores(i, 0);
          mma_commit(&sh.empty[0]);
        }
        for (int j = 0; j < tiles && ok; ++j) {
          const int nv = 2 * j + 1, nk = 2 * j + 2;
          if (!wait_slot(nv)) break;
          if (j + 1 < tiles && !wait_slot(nk)) break;
          for (int i = 0; i < halves; ++i) {
            ok = mbar_wait(&sh.p_full[i][0], (uint32_t)(j & 1), &sh.abort);
            if (!ok) break;
            tmem_fence_after();
            values(i, nv % kChSlots, 0, j > 0);
            ok = mbar_wait(&sh.p_full[i][1], (uint32_t)(j & 1), &sh.abort);
            if (!ok) break;
            tmem_fence_after();
            values(i, nv % kChSlots, 1, true);
            if (i == halves - 1) mma_commit(&sh.empty[nv % kChSlots]);
            if (j + 1 < tiles) scores(i, nk % kChSlots);
          }
          if (ok && j + 1 < tiles) mma_commit(&sh.empty[nk % kChSlots]);
        }
        if (!sh.abort) {
          mma_commit(&sh.o_full);
        } else {
          volatile int never = 0;
          mma_commit(&sh.drain);
          mbar_wait(&sh.drain, 0, &never);
        }
      }
    }
  } else {
    grow_registers<kChRowRegs>();
    // ---- weights: a thread per row
    const int i = warp >> 2;              // half
    const int r = tid & (kChRows - 1);    // row of the half
    const int token = r / R, head = r - token * R;
    const int ti = i * half_tokens + token;  // token of the CTA
    const bool live = token < half_tokens && ti < here;
    const int p = p_first + ti;           // keys [see, p] (rows that are not live: any)
    const int see = paged_low(a, p);
    // keys that all rows of the half see: tiles inside need no mask
    const int p_half = p_first + i * half_tokens;
    const int all_low = paged_low(a, p_half + half_tokens - 1), all_high = p_half + 1;
    const uint32_t my = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = my + i * 128, o_col = my + 256 + i * 128;
    // the reference scaled (and lowered: weights stand above it), as a score, and the
    // score beyond which it moves (rounded down: no weight exceeds 2^(kChMoveBy + kLift))
    float m = -CUDART_INF_F, top_s = -CUDART_INF_F, move_at = -CUDART_INF_F;
    const float move_by = fminf(kChMoveBy / w.scale_log2, 1e38f);
    float l = 0.f;
    const uint64_t scale2 = pair(w.scale_log2, w.scale_log2);
    bool ok = true;
    if (i < halves) {
      for (int j = 0; j < tiles; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[i], (uint32_t)(j & 1), &sh.abort));
        if (!ok) break;
        tmem_fence_after();
        float s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s[c], s_col + c * 32);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld(s[c]);
        const int first = key0 + j * kTileKeys;
        const bool edge = first < all_low || first < low || first + kTileKeys > min(all_high, high);
        if (edge) {
          // a bit per key, which predicates take eight at a time
          const int from = max(see, low) - first, to = min(p + 1, high) - first;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t seen = low_bits(to - c * 32) & ~low_bits(from - c * 32);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!(seen >> x & 1)) s[c][x] = -CUDART_INF_F;
          }
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          top[c] = max3(s[c][0], s[c][1], s[c][2]);
#pragma unroll
          for (int x = 3; x < 31; x += 2) top[c] = max3(top[c], s[c][x], s[c][x + 1]);
          top[c] = max3(top[c], s[c][31], s[c][31]);
        }
        const float t = max3(max3(top[0], top[1], top[2]), top[3], top[3]);
        const bool move = t > move_at;
        if (__any_sync(0xffffffffu, move)) {
          float f = 1.f;
          if (move) {
            const float m_new = t * w.scale_log2 - kLift<T>;
            f = ex2(fabsf(m_new) < kChNear ? m - m_new : (top_s - t) * w.scale_log2);
            m = m_new;
            top_s = t;
            move_at = __fadd_rd(t, move_by);
          }
          l *= f;
          if (j > 0) {  // O of the tiles so far is complete: S of this one came after it
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float o[32];
              tmem_ld32(o, o_col + c * 32);
              tmem_wait_ld(o);
              uint32_t u[32];
#pragma unroll
              for (int x = 0; x < 32; ++x) u[x] = __float_as_uint(o[x] * f);
              tmem_st32(o_col + c * 32, u);
            }
          }
        }
        // An exponent is s * scale - m in one operation, whose product is not rounded, but
        // m is: by up to 2^-5 while |m| < 2^20, the same for all weights, which the sum
        // makes good.  Beyond that it would carry them out of range; there it is
        // (s - top_s) * scale.
        const bool near = fabsf(m) < kChNear;
        const float u = near ? -m : kLift<T>;
        const uint64_t u2 = pair(u, u);
        // Weights, rounded to the 16-bit type for the product (the sum l keeps them
        // in 32 bits): half a unit each, of either sign.  Where all is finite, one
        // pair in kChFma goes through the FMA pipe instead of the special-function
        // unit, which alone would take as long as the products.
        // A tile's weights are summed by themselves first: beside a large l each alone
        // could be less than its last bit.
        auto weights = [&](auto plain) {
          uint64_t l2[2] = {0ull, 0ull};
          // an operand of its own for each form, or the compiler computes all 64
          // products before it branches and spills them
          uint64_t by = scale2;
          asm volatile("// form %1" : "+l"(by) : "n"((int)decltype(plain)::value));
          const float less = near || m == -CUDART_INF_F ? 0.f : -top_s;
          const uint64_t less2 = pair(less, less);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t packed[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              uint64_t y = pair(s[c][x], s[c][x + 1]);
              if (!decltype(plain)::value) y = add2(y, less2);
              y = fma2(y, by, u2);
              float e0, e1;
              if (decltype(plain)::value && (x >> 1) % kChFma == kChFma - 1) {
                ex2_fma(y, e0, e1);
              } else {
                unpair(y, e0, e1);
                e0 = ex2(e0);
                e1 = ex2(e1);
              }
              l2[(x >> 1) & 1] = add2(l2[(x >> 1) & 1], pair(e0, e1));
              packed[x >> 1] = Pack16<T>::pack(e0, e1);
            }
            tmem_st16(s_col + c * 16, packed);
            if (c & 1) {  // the product with V takes 64 keys at a time
              tmem_wait_st();
              tmem_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh.p_full[i][c >> 1]);
            }
          }
          float x0, x1;
          unpair(add2(l2[0], l2[1]), x0, x1);
          l += x0 + x1;
        };
        // Rows that are not live have no say: theirs are another request's or padding
        // rows of q, or (groups that do not divide 128) what an earlier kernel left in
        // shared memory, and a result's bits must not depend on those.
        if (__all_sync(0xffffffffu, !edge && (!live || near)))
          weights(std::true_type{});
        else
          weights(std::false_type{});
      }
    }
    if (tiles > 0 && ok)
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_full, 0, &sh.abort));
    tmem_fence_after();
    if (!ok && lane == 0) raise_error(a.error_flag, TW_ERR_TIMEOUT);
    const int t = rq.first + begin + ti, h = g * R + head;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const bool joined = range.parts == 1;
    looked_wait();
    if (i < halves) {
      // Rows go through shared memory (Q and the ring are free: all products are
      // done), so that a warp writes whole rows to memory: a thread writing its own
      // row 16 bytes at a time took 3.5 us for the 256 rows.
      const uint64_t inv2 = pair(inv, inv);
      {
        float o[4][32];
        if (tiles > 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(o[c], o_col + c * 32);
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_wait_ld(o[c]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int x = 0; x < 32; ++x) o[c][x] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const uint64_t y = mul2(pair(o[c][x], o[c][x + 1]), inv2);
            unpair(y, o[c][x], o[c][x + 1]);
          }
          if (joined)
            stage_row<Out>(smem, warp, lane, c, o[c]);
          else
            stage_row<float>(smem, warp, lane, c, o[c]);
        }
      }
      // what was cleared before the product, for the rows that do see it
      if (sh.odd.any) {
        __syncwarp();
#pragma unroll 1
        for (int x = 0; x < 16; ++x) {
#pragma unroll 1
          for (unsigned bits = sh.odd.bits[x >> 3][x & 7]; bits; bits &= bits - 1) {
            const int k = (x & 7) * 32 + __ffs(bits) - 1 + (x < 8 ? p_first : keys.low);
            const unsigned rows = __ballot_sync(0xffffffffu, live && k >= see && k <= p);
            const T* v = paged_value<T>(a, b, g, k);
            if (!v) continue;
            const uint2 mine = reinterpret_cast<const uint2*>(v)[lane];
            if (joined)
              add_odd_staged<T, Out>(smem, warp, lane, mine, rows);
            else
              add_odd_staged<T, float>(smem, warp, lane, mine, rows);
            __syncwarp();
          }
        }
      }
      if (live) {
        const int64_t row = (int64_t)t * a.q_heads + h;
        if (!joined)
          w.many.part_lse[row * w.many.splits + split] = paged_lse2(m, l);
        else if (a.lse)
          a.lse[row] = paged_lse(m, l);
      }
      __syncwarp();
      // row x of the warp: token y / R by multiplication (exact for y < 128, R <= 64)
      const unsigned by_r = (65536u + R - 1) / R;
      const int y0 = (warp & 3) * 32, t0 = rq.first + begin + i * half_tokens;
      const int rows = min(half_tokens, here - i * half_tokens) * R;
      if (joined) {
        Out* to = (Out*)a.out + (int64_t)t0 * a.out_token_stride +
                  (int64_t)(g * R) * a.out_head_stride;
        write_rows<Out>(smem, warp, lane, [&](int x) -> Out* {
          const int y = y0 + x, k = (int)(y * by_r >> 16);
          return y < rows ? to + (int64_t)k * a.out_token_stride + (y - k * R) * a.out_head_stride
                          : nullptr;
        });
      } else {
        float* to = w.many.part_o +
                    (((int64_t)t0 * a.q_heads + g * R) * w.many.splits + split) * kHeadDim;
        write_rows<float>(smem, warp, lane, [&](int x) -> float* {
          const int y = y0 + x, k = (int)(y * by_r >> 16);
          return y < rows ? to + ((int64_t)k * a.q_heads + (y - k * R)) * w.many.splits * kHeadDim
                          : nullptr;
        });
      }
    }
    tmem_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == kChMmaWarp) {
    tmem_fence_after();
    tmem_free(tmem, kChColumns);
  }
}

template <typename T, typename Out, bool kMixed>
static int launch_chunk(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream) {
  const int tokens = paged_chunk_tokens(w.group);
  CUtensorMap q_map;
  const cuuint64_t dims[3] = {(cuuint64_t)kHeadDim, (cuuint64_t)w.a.q_heads,
                              (cuuint64_t)w.a.tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)w.a.q_head_stride * 2,
                                 (cuuint64_t)w.a.q_token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)w.group, (cuuint32_t)tokens / 2};
  int rc = encode_rows_map(&q_map, w.a.pool.dtype, 3, w.a.q, dims, strides, box);
  if (rc != TW_OK) return rc;
  static DynSmemOptIn opt_in;
  const auto kernel = paged_chunk_kernel<T, Out, kMixed>;
  rc = ensure_dyn_smem((const void*)kernel, opt_in, kChSmem);
  if (rc != TW_OK) return rc;
  const int64_t ctas = ((int64_t)w.a.tokens / tokens + w.a.requests) * w.a.pool.kv_heads *
                           w.many.splits +
                       kPadCtas + (paged_token_items(w) + 1) / 2;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(kChThreads), (size_t)kChSmem, stream, w,
                    maps, q_map);
}

template <typename T, typename Out>
static int launch_chunk(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream) {
  return w.few.splits > 0 ? launch_chunk<T, Out, true>(w, maps, stream)
                          : launch_chunk<T, Out, false>(w, maps, stream);
}

int launch_paged_chunk(const PagedWork& w, const PagedMaps& maps, cudaStream_t stream) {
  if (w.a.pool.dtype == TW_F16)
    return w.a.out_dtype == TW_F32 ? launch_chunk<__half, float>(w, maps, stream)
                                   : launch_chunk<__half, __half>(w, maps, stream);
  return w.a.out_dtype == TW_F32 ? launch_chunk<__nv_bfloat16, float>(w, maps, stream)
                                 : launch_chunk<__nv_bfloat16, __nv_bfloat16>(w, maps, stream);
}

}  // namespace tw
