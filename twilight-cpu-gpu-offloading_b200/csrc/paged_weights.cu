// Attention weights that the cached rows of a paged cache are given.
//
// weight[slot of key j][g] += sum over counted rows i that see j and heads r of group g of
// exp(scale * q_ir . k_j - lse_ir), with the log-sum-exp that the attention left.
//
// Bound: for single tokens HBM (K is read once, 256 bytes a key and head); for chunks the
// special-function unit (one 2^x a pair, 16 a clock and SM, but for the pairs in six whose 2^x
// the FMA pipe works out where all of a piece is seen), then the tensor cores (2 D flops a
// pair) and the board's power limit.
//
// Layout: an item is 256 keys of a request and KV head.  The product is taken with keys
// along the rows of tensor memory, S^T = K Q^T, so that a thread owns a key and the sum over
// rows needs no exchange.  Sixteen warps sum, in two groups that take tiles of 128 (token,
// head) rows in turn: while a group reads its keys' scores and adds up their exponentials, the
// tensor cores make the next tile's for the other.  (Of tiles of 16 rows one group takes all:
// eight warps more that wait cost power, 405 us instead of 399 below.)  One warp issues the
// products, one copies tiles of q and reads their log-sum-exps, two copy K, page piece by page
// piece, with the next items' on its way while one is worked on, so that single tokens stream.
// Clusters of one CTA take every n-th item of all requests', back and forth; each warp finds
// them from the lengths by itself.  Where a call has few items, larger clusters take them, each
// CTA every n-th tile, and the first CTA adds their sums in order: a result does not depend on
// scheduling.
//
// Measured: 16 requests of 8k to 131k, a token each, 32 / 8 heads: 398 us in a run of a
// second, 5.9 TB/s, at 1005 W and 1.73 GHz, and 355 to 367 in a few calls by themselves, 6.4
// to 6.7 TB/s (reads alone; a copy moves 6.55); one at 32k: 17.4 us, of which 10.6 are its
// bytes' and the rest the way to the first tile (lengths, page, K) and from the last; 2048
// tokens at 32k: 665 us in a run of a second, 0.80 PFLOP/s, at 1.78 GHz, and 597 to 638 in a
// few calls (a tile takes 2.4k clocks, of which its exponentials are 1.7k); a prompt of 2048:
// 37.5 us, of which 8 come before the first tile and 16 tiles a CTA take 1.5 each.
// Tried: 8 warps that sum (880 us for the last but one), 64 columns of a tile for each group
// (680 us), products of 64 columns that follow each other sooner (960 us: the tensor cores read
// K again for each), two warps that issue (613 us, and 469 instead of 394 for single tokens).
#include "paged_attention.cuh"
#include "tensor.cuh"

#include <type_traits>

namespace tw {

constexpr int kWtKeys = 256, kWtCols = 128;
constexpr int kWtAhead = 2;                // tiles whose log-sum-exps are read at a time
constexpr int kWtHalfTile = 128 * 128;     // bytes: 128 rows of 64 elements
constexpr int kWtTile = 2 * kWtHalfTile;
constexpr int kWtSlots = 7;                // of shared memory, a tile each

// How a call's items are done.
enum WeightMode {
  kWtWhole,  // a CTA takes an item; K of two items and three tiles of q in shared memory
  kWtSplit,  // a cluster takes one; K of one, four tiles of q, and the sums of the other CTAs
  kWtFew     // at most 16 (token, head) rows a request: K of three, eight tiles of 16 rows
             // (the first kernel, K of two: 16 requests of 8k to 131k in 545 us; K of three
             // and a second warp that copies it: 427)
};
template <int kMode> struct WeightLayout {
  static constexpr int kKeySlots = kMode == kWtFew ? 3 : kMode == kWtSplit ? 1 : 2;
  static constexpr int kRowSlots = kMode == kWtFew ? 8 : kMode == kWtSplit ? 4 : 3;
  static constexpr int kCols = kMode == kWtFew ? 16 : kWtCols;   // rows of a tile of q
  static constexpr int kRowHalf = kCols * 128;                   // bytes: 64 dimensions of them
  static constexpr int kRowTile = 2 * kRowHalf;
  static constexpr int kGroups = kMode == kWtFew ? 1 : 2;        // of 256 threads that sum
  static constexpr int kMmaWarp = 8 * kGroups, kRowWarp = kMmaWarp + 1;
  static constexpr int kKeyWarp = kMmaWarp + 2;                  // and the next
  static constexpr int kThreads = (kMmaWarp + 4) * 32;
};
constexpr int kWtLseSlots = 3;
// One pair in this many on the FMA pipe.  2048 tokens at 32k, in a run of a second: none 671
// us, 12: 671, 8: 666, 6: 664, 4: 698; in a few calls (two runs each): 641 and 645, 652 and
// 616, 596 and 613, 638 and 638, 675 and 640.  A prompt of 2048: 38.6, 37.9, 38.0, 37.5, 38.0.
constexpr int kWtFma = 6;
constexpr int kWtColumns = 512;            // S^T: 2 halves of the keys, 2 tiles, 128 columns
constexpr int kWtMaxCluster = 8;
static_assert((kWtMaxCluster - 1) * kWtKeys * 4 <= kWtTile);

struct WeightWork {
  tw_paged_weights_args a;
  tw_paged_attention_args lens;  // what paged_request and paged_low read
  int group;                     // query heads per KV head
  int box;                       // rows of one box of K
  int tile_tokens;               // tokens of 128 columns
  int few_tokens;                // tokens of 16 columns (or one): a box of their own
};

struct WeightItem {
  int request, head;
  int row0, tokens;       // counted rows of q: [row0, row0 + tokens)
  int p0;                 // position of the first
  int key0, begin, end;   // keys [begin, end) of the block from key0 on
  int from, tiles;        // tokens that see any of them: from `from` on, so many tiles
  int upto;
};

// Items are numbered through the requests: every warp walks over them in the same way, 32
// requests at a time.
struct WeightWalk {
  int base = -32;
  long long before = 0, end = 0;     // items of the requests before these 32; with them
  // of request base + lane
  int row0, tokens, p0, low, high;
  long long upto, items;

  __device__ __forceinline__ void load(const WeightWork& w, int lane) {
    const int b = base + lane;
    row0 = tokens = p0 = low = high = 0;
    items = 0;
    if (b < w.a.requests) {
      const PagedRequest r = paged_request(w.lens, b);
      if (r.n > w.a.max_q_len) {
        raise_error(w.a.error_flag, TW_ERR_BAD_ARG);
      } else if (r.n > 0) {
        const int skip = w.a.last > 0 ? max(0, r.n - w.a.last) : 0;
        row0 = r.first + skip;
        tokens = r.n - skip;
        p0 = r.kv - tokens;
        const PagedKeys keys = paged_keys(w.lens, r, skip, tokens);
        low = keys.low;
        high = keys.high;
        if (high > low)
          items = (long long)((high - low / kWtKeys * kWtKeys + kWtKeys - 1) / kWtKeys) *
                  w.a.pool.kv_heads;
      }
    }
    upto = items;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += y;
    }
    upto += before;
    end = __shfl_sync(0xffffffffu, upto, 31);
  }

  // Item `n`; false: there are not so many.  (n never goes down.)
  __device__ __forceinline__ bool find(const WeightWork& w, int lane, long long n, WeightItem& x) {
    while (n >= end) {
      base += 32;
      if (base >= w.a.requests) return false;
      before = end;
      load(w, lane);
    }
    const int l = __ffs(__ballot_sync(0xffffffffu, n < upto)) - 1;
    const long long of = n - (__shfl_sync(0xffffffffu, upto - items, l));
    x.request = base + l;
    x.row0 = __shfl_sync(0xffffffffu, row0, l);
    x.tokens = __shfl_sync(0xffffffffu, tokens, l);
    x.p0 = __shfl_sync(0xffffffffu, p0, l);
    const int lo = __shfl_sync(0xffffffffu, low, l), hi = __shfl_sync(0xffffffffu, high, l);
    // heads of a block follow one another: blocks that most rows see come first
    const int block = (int)(of / w.a.pool.kv_heads);
    x.head = (int)(of - (long long)block * w.a.pool.kv_heads);
    x.key0 = lo / kWtKeys * kWtKeys + block * kWtKeys;
    x.begin = max(lo, x.key0);
    x.end = min(hi, x.key0 + kWtKeys);
    x.from = max(0, x.begin - x.p0);
    x.upto = x.tokens;
    if (w.a.window > 0)
      x.upto = (int)min((long long)x.tokens, (long long)x.end + w.a.window - 1 - x.p0);
    x.tiles = (max(x.upto - x.from, 0) + w.tile_tokens - 1) / w.tile_tokens;
    return true;
  }
};

struct WeightShared {
  uint64_t k_full[3], k_empty[3];
  uint64_t q_full[8], q_empty[8];
  uint64_t lse_full[kWtLseSlots], lse_empty[kWtLseSlots];
  uint64_t s_full[2][2], s_free[2][2];  // [half][tile]
  uint64_t sums_full, sums_free, part_full, part_free, drain;
  uint32_t tmem;
  volatile int abort;
  float sums[kWtKeys];                          // of the second group's
  alignas(16) float lse[kWtLseSlots][kWtCols];  // minus the log-sum-exps
};

// No static shared memory beside it: the tiles begin on a boundary of 1024 bytes.
constexpr int kWtSmem = kWtSlots * kWtTile + (int)sizeof(WeightShared);
static_assert(kWtSmem <= 232448);

// Barriers and memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t remote(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void remote_arrive(uint64_t* bar, int rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                   remote(smem_addr(bar), rank))
               : "memory");
}
__device__ __forceinline__ void remote_store(float* p, int rank, float x) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(smem_addr(p), rank)), "f"(x)
               : "memory");
}
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return wait_until(
      [&] {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_addr(bar)), "r"(parity)
            : "memory");
        return done != 0;
      },
      abort);
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// 2^x of a pair on the FMA pipe, for all x (below -126.5: 0, from 127.5 on: infinity, NaN:
// NaN): n = x rounded to a whole number by adding 1.5 * 2^23, 2^(x - n) on [-1/2, 1/2] by the
// polynomial of degree 5 with the smallest largest relative error there (Remez exchange;
// 2.2e-7 with its roundings, as the special-function unit's), times 2^n put together from
// its bits.
__device__ __forceinline__ void ex2_five(uint64_t x2, float& e0, float& e1) {
  float x0, x1;
  unpair(x2, x0, x1);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(-127.f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(128.f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(128.f));
  x2 = pair(x0, x1);
  const uint64_t round = pair(12582912.f, 12582912.f), back = pair(-12582912.f, -12582912.f);
  const uint64_t r = add2(x2, round);
  const uint64_t f = fma2(add2(r, back), pair(-1.f, -1.f), x2);
  uint64_t p = pair(0x1.5c08e6p-10f, 0x1.5c08e6p-10f);
  p = fma2(p, f, pair(0x1.3d0c52p-7f, 0x1.3d0c52p-7f));
  p = fma2(p, f, pair(0x1.c6b6e4p-5f, 0x1.c6b6e4p-5f));
  p = fma2(p, f, pair(0x1.ebf918p-3f, 0x1.ebf918p-3f));
  p = fma2(p, f, pair(0x1.62e428p-1f, 0x1.62e428p-1f));
  p = fma2(p, f, pair(0x1.000002p+0f, 0x1.000002p+0f));
  float r0, r1;
  unpair(r, r0, r1);
  p = mul2(p, pair(__int_as_float((__float_as_int(r0) << 23) + 0x3f800000),
                   __int_as_float((__float_as_int(r1) << 23) + 0x3f800000)));
  unpair(p, e0, e1);
}

// The lowest n bits (n <= 0: none, n >= 32: all).
__device__ __forceinline__ uint32_t first_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}

template <bool kBf16, int kMode>
__global__ void __launch_bounds__(WeightLayout<kMode>::kThreads, 1)
paged_weights_kernel(const __grid_constant__ WeightWork w,
                     const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap q_map,
                     const __grid_constant__ CUtensorMap few_map) {
  extern __shared__ __align__(1024) char smem[];
  WeightShared& sh = *reinterpret_cast<WeightShared*>(smem + kWtSlots * kWtTile);
  const tw_paged_weights_args& a = w.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = w.group, T = w.tile_tokens;
  uint32_t cluster_rank, cluster_ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cluster_rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster_ctas));
  constexpr bool kSplit = kMode == kWtSplit;
  const int rank = kSplit ? (int)cluster_rank : 0, S = kSplit ? (int)cluster_ctas : 1;
  using Layout = WeightLayout<kMode>;
  constexpr int kKeySlots = Layout::kKeySlots, kRowSlots = Layout::kRowSlots;
  constexpr int kMmaWarp = Layout::kMmaWarp, kKeyWarp = Layout::kKeyWarp;
  constexpr int kCols = Layout::kCols, kRowHalf = Layout::kRowHalf, kRowTile = Layout::kRowTile;
  static_assert(2 * kKeySlots * kWtTile + kRowSlots * kRowTile <=
                (kSplit ? kWtSlots - 1 : kWtSlots) * kWtTile);
  const uint32_t keys_at = smem_addr(smem), rows_at = keys_at + 2 * kKeySlots * kWtTile;
  // kSplit: the other CTAs' sums, [rank - 1][key]
  float* s_part = reinterpret_cast<float*>(smem + (kWtSlots - 1) * kWtTile);
  if (tid == 0) {
    for (int i = 0; i < kKeySlots; ++i) {
      mbar_init(&sh.k_full[i], 2);
      mbar_init(&sh.k_empty[i], 1);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_empty[i], 1);
    }
    for (int i = 0; i < kWtLseSlots; ++i) {
      mbar_init(&sh.lse_full[i], 1);
      mbar_init(&sh.lse_empty[i], kWtKeys / 32);
    }
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sh.s_full[i][j], 1);
        mbar_init(&sh.s_free[i][j], 4);
      }
    mbar_init(&sh.sums_full, kWtKeys / 32);
    mbar_init(&sh.sums_free, kWtKeys / 32);
    if (kSplit) {
      mbar_init(&sh.part_full, (uint32_t)((S - 1) * (kWtKeys / 32)));
      mbar_init(&sh.part_free, kWtKeys / 32);
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    mbar_init_fence();
  }
  // columns that no token fills (groups that do not divide 128) stay zero rows
  const int spare = (kCols - T * R) * 8;  // 16-byte vectors of 64 dimensions
  for (int i = tid; i < kRowSlots * 2 * spare; i += Layout::kThreads)
    *reinterpret_cast<uint4*>(smem + 2 * kKeySlots * kWtTile + i / spare * kRowHalf + T * R * 128 +
                              i % spare * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  if (warp == kMmaWarp) tmem_alloc(&sh.tmem, kWtColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if constexpr (kSplit) cluster_barrier();  // all barriers are there
  const uint32_t tmem = sh.tmem;
  // (so far nothing but shared and tensor memory: while the kernel before this one ends)
  pdl_wait();
  pdl_launch_dependents();

  // Its items: back and forth through them, so that the long ones at the beginning (keys that
  // most rows see) and the short ones at the end come together.
  const long long mine = blockIdx.x / S, others = gridDim.x / S;
  const auto item = [&](int round) {
    return round * others + (round & 1 ? others - 1 - mine : mine);
  };
  WeightWalk walk;
  WeightItem x;
  bool ok = true;
  if (keys_at & 1023) {  // (what the layout of the products rests on)
    if (tid == 0) raise_error(a.error_flag, TW_ERR_UNSUPPORTED);
  } else if (warp >= kKeyWarp) {
    // ---- K of the items: a warp for each 128 keys
    const int h = warp - kKeyWarp;
    if (elect_one()) prefetch_map(&k_map);
    __syncwarp();
    const uint32_t box_bytes = (uint32_t)w.box * 128;  // of 64 dimensions
    const int boxes = 128 / w.box;                     // at most 16
    // lane l < boxes knows the page of box l, and looks the next item's up before it waits
    int p = 0, row = 0;
    bool wanted = false;
    const auto look_up = [&](const WeightItem& x, bool known, int page) {
      const int key = x.key0 + h * 128 + lane * w.box;
      wanted = lane < boxes && key < x.end && key + w.box > x.begin;
      if (wanted) {
        const int i = key / a.pool.page_size;
        row = key - i * a.pool.page_size;
        p = known ? page : a.block_table[(int64_t)x.request * a.table_stride + i];
      }
    };
    int n = 0, round = 0;
    // a single request's first pages are read together with its lengths
    const long long guess = item(0) / a.pool.kv_heads * kWtKeys + h * 128 + lane * w.box;
    const bool guesses = a.requests == 1 && a.window == 0 && lane < boxes &&
                         guess / a.pool.page_size < a.table_width;
    const int first_page = guesses ? a.block_table[guess / a.pool.page_size] : 0;
    bool more = walk.find(w, lane, item(0), x);
    if (more) look_up(x, guesses, first_page);
    while (more) {
      const bool skip = rank >= x.tiles;
      const int head = x.head, now_row = row;
      int now = p;
      const uint32_t all = __ballot_sync(0xffffffffu, wanted);
      if (wanted && (now < 0 || now >= a.pool.num_pages)) {
        raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
        now = (int)a.pool.num_pages;  // out of the map's range: zeros
      }
      more = walk.find(w, lane, item(++round), x);
      if (more) look_up(x, false, 0);
      if (skip) continue;
      const int s = n % kKeySlots;
      const int from = all ? __ffs(all) - 1 : 0, to = 32 - __clz(all);
      if (n >= kKeySlots) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.k_empty[s],
                                               (uint32_t)((n / kKeySlots - 1) & 1), &sh.abort));
        if (!ok) break;
      }
      if (elect_one())
        mbar_arrive_expect(&sh.k_full[s], (uint32_t)(to - from) * box_bytes * 2);
      for (int y0 = from; y0 < to; y0 += 4) {
        int px[4], rx[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          px[y] = __shfl_sync(0xffffffffu, now, y0 + y);
          rx[y] = __shfl_sync(0xffffffffu, now_row, y0 + y);
        }
        if (elect_one()) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (y0 + y < to) {
              const uint32_t dst = keys_at + (uint32_t)(s * 2 + h) * kWtTile +
                                   (uint32_t)((y0 + y) * w.box) * 128;
              tma_load_4d(&k_map, dst, &sh.k_full[s], 0, rx[y], head, px[y]);
              tma_load_4d(&k_map, dst + kWtHalfTile, &sh.k_full[s], 64, rx[y], head, px[y]);
            }
        }
        __syncwarp();
      }
      ++n;
    }
    if (!ok || sh.abort) {  // give up: wait (with the same limit) for the copies in flight
      volatile int never = 0;
      for (int i = max(n - kKeySlots, 0); i < n; ++i)
        mbar_wait(&sh.k_full[i % kKeySlots], (uint32_t)((i / kKeySlots) & 1), &never);
    }
  } else if (warp == Layout::kRowWarp) {
    // ---- tiles of q and their rows' log-sum-exps
    if (elect_one()) {
      prefetch_map(&q_map);
      prefetch_map(&few_map);
    }
    __syncwarp();
    int n = 0, nl = 0;  // tiles copied; with their log-sum-exps
    constexpr int kParts = (kCols + 31) / 32;
    int64_t place[kParts];  // of the lane's columns in a.lse
#pragma unroll
    for (int c = 0; c < kParts; ++c) {
      const int col = c * 32 + lane, token = col / R;
      place[c] = (int64_t)token * a.q_heads + (col - token * R);
    }
    for (int round = 0; ok && walk.find(w, lane, item(round), x); ++round) {
      for (int t0 = rank; ok && t0 < x.tiles; t0 += kWtAhead * S) {
        for (int y = 0; y < kWtAhead && t0 + y * S < x.tiles; ++y, ++n) {
          const int s = n % kRowSlots;
          if (n >= kRowSlots) {
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.q_empty[s],
                                                   (uint32_t)((n / kRowSlots - 1) & 1), &sh.abort));
            if (!ok) break;
          }
          const int i = x.from + (t0 + y * S) * T, here = min(T, x.upto - i);
          if (elect_one()) {
            const uint32_t dst = rows_at + (uint32_t)s * kRowTile;
            // rows past the last are masked
            const bool few = kMode == kWtFew || here <= w.few_tokens;
            const CUtensorMap* map = few ? &few_map : &q_map;
            mbar_arrive_expect(&sh.q_full[s], (uint32_t)((few ? w.few_tokens : T) * R) * 256);
            tma_load_3d(map, dst, &sh.q_full[s], 0, x.head * R, x.row0 + i);
            tma_load_3d(map, dst + kRowHalf, &sh.q_full[s], 64, x.head * R, x.row0 + i);
          }
          __syncwarp();
        }
        if (!ok) break;
        float z[kWtAhead][kParts];
#pragma unroll
        for (int y = 0; y < kWtAhead; ++y) {
          const int i = x.from + (t0 + y * S) * T, cols = min(T, x.upto - i) * R;
          const float* lse = a.lse + (int64_t)(x.row0 + i) * a.q_heads + x.head * R;
#pragma unroll
          for (int c = 0; c < kParts; ++c)
            z[y][c] = c * 32 + lane < cols ? -lse[place[c]] : -CUDART_INF_F;
        }
#pragma unroll
        for (int y = 0; y < kWtAhead; ++y) {
          if (t0 + y * S >= x.tiles) break;
          const int s = nl % kWtLseSlots;
          if (nl >= kWtLseSlots) {
            ok = __all_sync(0xffffffffu,
                            mbar_wait(&sh.lse_empty[s], (uint32_t)((nl / kWtLseSlots - 1) & 1),
                                      &sh.abort));
            if (!ok) break;
          }
          // (a row that saw nothing: no weight; its score less -infinity would be infinite)
#pragma unroll
          for (int c = 0; c < kParts; ++c)
            sh.lse[s][c * 32 + lane] = z[y][c] == CUDART_INF_F ? -CUDART_INF_F : z[y][c];
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.lse_full[s]);
          ++nl;
        }
      }
    }
    if (!ok || sh.abort) {
      volatile int never = 0;
      for (int i = max(n - kRowSlots, 0); i < n; ++i)
        mbar_wait(&sh.q_full[i % kRowSlots], (uint32_t)((i / kRowSlots) & 1), &never);
    }
  } else if (warp == kMmaWarp) {
    // ---- products
    const uint64_t k_desc = operand_desc(keys_at, 16, 1024);
    const uint64_t q_desc = operand_desc(rows_at, 16, 1024);
    int nk = 0, nq = 0;
    uint32_t used = 0, turn = 0;  // a bit per buffer of scores: used before; its phase
    for (int round = 0; ok && walk.find(w, lane, item(round), x); ++round) {
      if (rank >= x.tiles) continue;
      const int ks = nk % kKeySlots;
      const int halves = x.end - x.key0 > 128 ? 2 : 1;
      const bool first_half = x.begin < x.key0 + 128;
      ok = __all_sync(0xffffffffu,
                      mbar_wait(&sh.k_full[ks], (uint32_t)((nk / kKeySlots) & 1), &sh.abort));
      for (int t = rank; ok && t < x.tiles; t += S, ++nq) {
        const int qs = nq % kRowSlots;
        const int cols = min(T, x.upto - x.from - t * T) * R;
        const uint32_t desc = product_desc(kBf16, (cols + 15) / 16 * 16, false);
        // q and both places of scores, before the first product: a wait between them would come
        // to more than the products take
        const int buf = nq & 1;
        bool there = mbar_wait(&sh.q_full[qs], (uint32_t)((nq / kRowSlots) & 1), &sh.abort);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int bit = h * 2 + buf;
          if (h < (first_half ? 0 : 1) || h >= halves) continue;
          if (there && (used >> bit & 1))
            there = mbar_wait(&sh.s_free[h][buf], ~(turn >> bit) & 1, &sh.abort);
          used |= 1u << bit;
          turn ^= 1u << bit;
        }
        ok = __all_sync(0xffffffffu, there);
        if (!ok) break;
        tmem_fence_after();
        if (elect_one()) {
          // (addresses count in 16 bytes in the low bits of a descriptor)
          const uint64_t qa = q_desc + (uint64_t)(qs * (kRowTile >> 4));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h < (first_half ? 0 : 1) || h >= halves) continue;
            const uint64_t ka = k_desc + (uint64_t)((ks * 2 + h) * (kWtTile >> 4));
            const uint32_t d = tmem + (h * 2 + buf) * 128;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_smem(d, ka + (k >> 2) * (kWtHalfTile >> 4) + (k & 3) * 2,
                       qa + (k >> 2) * (kRowHalf >> 4) + (k & 3) * 2, desc, k > 0);
            mma_commit(&sh.s_full[h][buf]);
          }
          mma_commit(&sh.q_empty[qs]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) mma_commit(&sh.k_empty[ks]);
      __syncwarp();
      ++nk;
    }
    // The last arrival of the tensor cores at a barrier is waited for, or it could come when the
    // shared memory is another block's: those at q_empty and k_empty nobody else waits for.
    // (Waiting for each slot's own instead: 11 looks, 18.0 us for a single token at 32k, not 17.3.)
    volatile int never = 0;
    if (elect_one()) mma_commit(&sh.drain);
    __syncwarp();
    mbar_wait(&sh.drain, 0, &never);
  } else {
    // ---- sums: a thread per key and group; the groups take tiles in turn
    constexpr bool kFew = kMode == kWtFew;
    const int group = warp >> 3, h = (warp >> 2) & 1, key = tid & (kWtKeys - 1);
    const uint32_t my = tmem + ((uint32_t)((warp & 3) * 32) << 16) + h * 256;
    const uint64_t scale2 = pair(a.softmax_scale, a.softmax_scale);
    const uint64_t log2e2 = pair(1.4426950408889634f, 1.4426950408889634f);
    int nl = 0, joins = 0;  // tiles so far; items whose sums the groups joined
    uint32_t turn = 0;      // a bit per buffer of scores: its phase
    for (int round = 0; ok && walk.find(w, lane, item(round), x); ++round) {
      // This CTA's tiles of the item; which group goes on with the sums, and whether the other
      // has some for it.  Of a single tile it is the one that has it; with a cluster always the
      // first, which so sees every phase of the barriers between CTAs (a group that left one out
      // would take an older phase for the one it waits for).
      const int tiles = x.tiles > rank ? (x.tiles - rank - 1) / S + 1 : 0;
      const int last = kSplit || kFew || tiles != 1 ? 0 : nl & 1;
      const bool both = !kFew && (tiles > 1 || (tiles == 1 && (nl & 1) != last));
      const bool adds = group == last;
      const int j = x.key0 + key;
      const bool held = j >= x.begin && j < x.end;
      int page = -1;
      if (held && rank == 0 && adds)
        page = a.block_table[(int64_t)x.request * a.table_stride + j / a.pool.page_size];
      const bool mine = h == 0 ? x.begin < x.key0 + 128 : x.end > x.key0 + 128;
      float sum = 0.f;
      for (int t = rank; t < x.tiles; t += S, ++nl) {
        const int buf = nl & 1;
        if (!kFew && buf != group) continue;
        const int ls = nl % kWtLseSlots;
        // (also by warps with no keys: they must not hand a slot back twice in a phase)
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.lse_full[ls],
                                               (uint32_t)((nl / kWtLseSlots) & 1), &sh.abort));
        if (!ok) break;
        if (mine) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&sh.s_full[h][buf], turn >> buf & 1, &sh.abort));
          if (!ok) break;
          turn ^= 1u << buf;
          tmem_fence_after();
          const int i = x.from + t * T, here = min(T, x.upto - i);
          const int cols = here * R, p = x.p0 + i;  // position of the tile's first token
          const int kh = x.key0 + h * 128;
          // columns of the tokens that see this key: [from, to)
          const bool plain = here == T && kh >= x.begin && kh + 128 <= x.end && p >= kh + 127 &&
                             (a.window <= 0 || (long long)p + T - a.window <= kh);
          int from = 0, to = cols;
          if (!plain) {
            from = held ? max(j - p, 0) * R : 0;
            to = held ? cols : 0;
            if (held && a.window > 0)
              to = (int)max(min((long long)here, (long long)j + a.window - p), 0ll) * R;
          }
          const uint32_t at = my + buf * 128;
          uint64_t sum2[2] = {0ull, 0ull};
          // the columns [c0, c0 + N) of the tile, in s
          const auto add_columns = [&](const auto& s, int c0, auto n, auto some) {
            constexpr int N = decltype(n)::value;
            constexpr bool masked = decltype(some)::value;
            const uint32_t seen = first_bits(to - c0) & ~first_bits(from - c0);
            const float4* z = reinterpret_cast<const float4*>(&sh.lse[ls][c0]);
#pragma unroll
            for (int y = 0; y < N; y += 4) {
              const float4 l = z[y / 4];
              const uint64_t d0 = mul2(fma2(pair(s[y], s[y + 1]), scale2, pair(l.x, l.y)), log2e2);
              const uint64_t d1 =
                  mul2(fma2(pair(s[y + 2], s[y + 3]), scale2, pair(l.z, l.w)), log2e2);
              float e0, e1, e2, e3;
              const auto weigh = [&](uint64_t d, int number, float& u, float& v) {
                if (!masked && number % kWtFma == kWtFma - 1) {
                  ex2_five(d, u, v);
                } else {
                  unpair(d, u, v);
                  u = ex2(u);
                  v = ex2(v);
                }
              };
              weigh(d0, y / 2, e0, e1);
              weigh(d1, y / 2 + 1, e2, e3);
              if (masked) {
                e0 = seen >> y & 1 ? e0 : 0.f;
                e1 = seen >> (y + 1) & 1 ? e1 : 0.f;
                e2 = seen >> (y + 2) & 1 ? e2 : 0.f;
                e3 = seen >> (y + 3) & 1 ? e3 : 0.f;
              }
              sum2[0] = add2(sum2[0], pair(e0, e1));
              sum2[1] = add2(sum2[1], pair(e2, e3));
            }
          };
          // (two pieces of code: in one, the compiler masks always)
          const auto add = [&](const auto& s, int c0, auto n) {
            // (columns that no token fills are zero rows: an infinite key would make them NaN)
            if (plain && c0 + decltype(n)::value <= cols)
              add_columns(s, c0, n, std::false_type{});
            else
              add_columns(s, c0, n, std::true_type{});
          };
          const auto read_all = [&] {  // the scores are in registers: the next tile's may come
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_free[h][buf]);
          };
          if constexpr (kFew) {
            // (no more columns than there are: 417 us instead of 424 in a run of a second)
            if (cols <= 4) {
              float s[4];
              tmem_ld4(s, at);
              tmem_wait_ld(s);
              read_all();
              add(s, 0, std::integral_constant<int, 4>{});
            } else if (cols <= 8) {
              float s[8];
              tmem_ld8(s, at);
              tmem_wait_ld(s);
              read_all();
              add(s, 0, std::integral_constant<int, 8>{});
            } else {
              float s[16];
              tmem_ld16(s, at);
              tmem_wait_ld(s);
              read_all();
              add(s, 0, std::integral_constant<int, 16>{});
            }
          } else {
            // (each read is followed by its wait: a branch between them, and the compiler
            // may move the registers before they hold anything)
#pragma unroll 1
            for (int c0 = 0; c0 < cols; c0 += 32) {
              float s[32];
              tmem_ld32(s, at + c0);
              tmem_wait_ld(s);
              if (c0 + 32 >= cols) read_all();
              add(s, c0, std::integral_constant<int, 32>{});
            }
          }
          float y0, y1;
          unpair(add2(sum2[0], sum2[1]), y0, y1);
          sum += y0 + y1;  // a tile's by itself first: beside a large sum each could be nothing
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.lse_empty[ls]);
      }
      if (!ok) break;
      if (both) {
        if (group == 1) {
          if (joins > 0)
            ok = __all_sync(0xffffffffu,
                            mbar_wait(&sh.sums_free, (uint32_t)((joins - 1) & 1), &sh.abort));
          if (!ok) break;
          sh.sums[key] = sum;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.sums_full);
        } else {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&sh.sums_full, (uint32_t)(joins & 1), &sh.abort));
          if (!ok) break;
          sum += sh.sums[key];
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.sums_free);
        }
        ++joins;
      }
      if (!adds) continue;
      if constexpr (kSplit) {
        if (rank != 0) {
          if (round > 0)
            ok = __all_sync(0xffffffffu,
                            cluster_wait(&sh.part_free, (uint32_t)((round - 1) & 1), &sh.abort));
          if (!ok) break;
          remote_store(s_part + (rank - 1) * kWtKeys + key, 0, sum);
          __syncwarp();
          if (lane == 0) remote_arrive(&sh.part_full, 0);
        } else {
          ok = __all_sync(0xffffffffu,
                          cluster_wait(&sh.part_full, (uint32_t)(round & 1), &sh.abort));
          if (!ok) break;
          for (int r = 1; r < S; ++r) sum += s_part[(r - 1) * kWtKeys + key];
          __syncwarp();
          if (lane == 0)
            for (int r = 1; r < S; ++r) remote_arrive(&sh.part_free, r);
        }
      }
      // no other thread of the call adds to this slot, unless requests share its page
      if (page >= 0 && page < a.pool.num_pages)
        atomicAdd(a.row_weights + ((int64_t)page * a.pool.kv_heads + x.head) * a.pool.page_size +
                      j % a.pool.page_size,
                  sum);
    }
    if (!ok && lane == 0) raise_error(a.error_flag, TW_ERR_TIMEOUT);
    tmem_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == kMmaWarp) {
    tmem_fence_after();
    tmem_free(tmem, kWtColumns);
  }
  if constexpr (kSplit) cluster_barrier();  // no CTA is gone while another writes to it
}

// Clusters of `cluster` CTAs that the device holds at once, asked once per device.
template <bool kBf16, int kMode>
static int resident_clusters(int cluster, int& n) {
  static int known[kMaxDevices][4] = {};
  static std::mutex mu;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const int i = cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3;
  if (err == cudaSuccess && dev < kMaxDevices) {
    std::lock_guard<std::mutex> lk(mu);
    if (known[dev][i] > 0) {
      n = known[dev][i];
      return TW_OK;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(WeightLayout<kMode>::kThreads);
  cfg.dynamicSmemBytes = kWtSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (err == cudaSuccess)
    err = cudaOccupancyMaxActiveClusters(&n, paged_weights_kernel<kBf16, kMode>, &cfg);
  if (err != cudaSuccess) {
    set_last_cuda_error(err);
    return TW_ERR_CUDA;
  }
  if (n < 1) n = 1;
  if (dev < kMaxDevices) {
    std::lock_guard<std::mutex> lk(mu);
    known[dev][i] = n;
  }
  return TW_OK;
}

template <bool kBf16, int kMode>
static int launch_weights(const WeightWork& w, int cluster, int64_t items, cudaStream_t stream) {
  const tw_paged_weights_args& a = w.a;
  CUtensorMap k_map, q_map, few_map;
  const cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)a.pool.page_size,
                              (cuuint64_t)a.pool.kv_heads, (cuuint64_t)a.pool.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)a.pool.token_stride * 2,
                                 (cuuint64_t)a.pool.head_stride * 2,
                                 (cuuint64_t)a.pool.page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)w.box, 1, 1};
  int rc = encode_rows_map(&k_map, a.pool.dtype, 4, a.pool.k_pages, dims, strides, box);
  const cuuint64_t q_dims[3] = {(cuuint64_t)kHeadDim, (cuuint64_t)a.q_heads, (cuuint64_t)a.tokens};
  const cuuint64_t q_strides[2] = {(cuuint64_t)a.q_head_stride * 2,
                                   (cuuint64_t)a.q_token_stride * 2};
  const cuuint32_t q_box[3] = {64, (cuuint32_t)w.group, (cuuint32_t)w.tile_tokens};
  const cuuint32_t few_box[3] = {64, (cuuint32_t)w.group, (cuuint32_t)w.few_tokens};
  if (rc == TW_OK) rc = encode_rows_map(&q_map, a.pool.dtype, 3, a.q, q_dims, q_strides, q_box);
  if (rc == TW_OK) rc = encode_rows_map(&few_map, a.pool.dtype, 3, a.q, q_dims, q_strides, few_box);
  if (rc != TW_OK) return rc;
  static DynSmemOptIn opt_in;
  const auto kernel = paged_weights_kernel<kBf16, kMode>;
  rc = ensure_dyn_smem((const void*)kernel, opt_in, kWtSmem);
  int most = 0;
  if (rc == TW_OK) rc = resident_clusters<kBf16, kMode>(cluster, most);
  if (rc != TW_OK) return rc;
  const int64_t clusters = items < most ? items : most;
  return launch_pdl_cluster(kernel, dim3((unsigned)(clusters * cluster)),
                            dim3(WeightLayout<kMode>::kThreads), cluster,
                            (size_t)kWtSmem, stream, w, k_map, q_map, few_map);
}

}  // namespace tw

using namespace tw;

extern "C" size_t tw_paged_weights_args_size(void) { return sizeof(tw_paged_weights_args); }

extern "C" int tw_paged_weights(const tw_paged_weights_args* args, void* stream) {
  if (!args) return TW_ERR_BAD_ARG;
  const tw_paged_weights_args& a = *args;
  const int rc = check_paged_pool(a.pool);
  if (rc != TW_OK) return rc;
  if (a.pool.page_size % 8 != 0) return TW_ERR_UNSUPPORTED;
  if (a.tokens < 0 || a.requests < 0) return TW_ERR_BAD_ARG;
  if (a.tokens == 0) return TW_OK;
  if (!a.q || !a.block_table || !a.cu_q || !a.kv_lens || !a.lse || !a.row_weights ||
      a.requests <= 0 || a.q_heads <= 0 || a.q_heads % a.pool.kv_heads != 0 ||
      a.table_width <= 0 || a.table_stride < a.table_width || a.max_q_len < 0 ||
      a.max_kv_len < 0 || a.window < 0 || a.last < 0 || a.reserved != 0 ||
      !(a.softmax_scale > 0.f) || !(a.softmax_scale < INFINITY))
    return TW_ERR_BAD_ARG;
  if (a.q_heads / a.pool.kv_heads > 64) return TW_ERR_UNSUPPORTED;
  if (!aligned16(a.q) || !paged_stride_ok(a.q_token_stride) || !paged_stride_ok(a.q_head_stride))
    return TW_ERR_BAD_ARG;
  WeightWork w = {};
  w.a = a;
  w.lens.pool = a.pool;
  w.lens.cu_q = a.cu_q;
  w.lens.kv_lens = a.kv_lens;
  w.lens.tokens = a.tokens;
  w.lens.table_width = a.table_width;
  w.lens.window = a.window;
  w.lens.error_flag = a.error_flag;
  w.group = a.q_heads / a.pool.kv_heads;
  w.tile_tokens = kWtCols / w.group;
  w.few_tokens = w.group < 16 ? 16 / w.group : 1;
  w.box = 64;
  while (a.pool.page_size % w.box != 0) w.box /= 2;
  // Bounds of the items and of a request's tiles: a cluster an item where CTAs would idle.
  // Prompts, us with clusters of two, four, eight (of which the device holds 15):
  //   heads    256             512             1024            2048            4096 tokens
  //   32 / 8   14  11 *11      19  14 *16      29  20 *25      52 *37  50     *95 110 137
  //   16 / 4   13  11 *10      19  13 *11      29  19 *16      50  31 *30      93 *58  74
  //   64 / 8   19  14 *12      30  19 *20      51  31 *33      96 *62  78    *180 206 231
  // * what the rule takes.  It does not ask how many clusters the device holds, and where
  // those of eight come in more than one round it loses (512 and 1024 tokens of 32 / 8 heads);
  // single CTAs take 1.3 to 2 times as long as clusters of two.
  int64_t most = a.max_q_len < a.tokens ? a.max_q_len : a.tokens;
  if (a.last > 0 && a.last < most) most = a.last;
  int64_t keys = a.max_kv_len;
  if (a.window > 0 && a.window + most < keys) keys = a.window + most;
  const int64_t items =
      ((keys + kWtKeys - 1) / kWtKeys + (a.window > 0)) * a.requests * a.pool.kv_heads;
  const int64_t tiles = (most + w.tile_tokens - 1) / w.tile_tokens;
  int cluster = 1;
  while (cluster < kWtMaxCluster && 2 * cluster <= tiles && cluster * items < 148) cluster *= 2;
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t some = items > 0 ? items : 1;
  if (w.group <= 16 && most <= w.few_tokens) {
    w.tile_tokens = w.few_tokens;
    return a.pool.dtype == TW_F16 ? launch_weights<false, kWtFew>(w, 1, some, s)
                                  : launch_weights<true, kWtFew>(w, 1, some, s);
  }
  if (a.pool.dtype == TW_F16)
    return cluster > 1 ? launch_weights<false, kWtSplit>(w, cluster, some, s)
                       : launch_weights<false, kWtWhole>(w, 1, some, s);
  return cluster > 1 ? launch_weights<true, kWtSplit>(w, cluster, some, s)
                     : launch_weights<true, kWtWhole>(w, 1, some, s);
}
