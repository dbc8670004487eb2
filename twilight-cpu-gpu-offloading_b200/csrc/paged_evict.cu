// Eviction from the paged cache by accumulated attention weight.
//
// Of a request with more rows than `keep`, in every layer and KV head by itself: rows are
// ranked, protected ones (first and most recent positions) first, then by weight, then by
// row; the first `keep` stay.  The i-th row at or past `keep` that stays moves to the i-th
// place below `keep` that has become free, with its weight and position, so m rows evicted
// move m rows at most (in the order they had, nearly all rows would move).
//
// Bound: latency for one layer (launch, lengths -> table -> records, up to three histogram
// rounds, the copy: a chain of about 17 us, half of it in up to seven cluster barriers and
// what surrounds them), HBM for many: 8 bytes a row and 1 KB a row that moves.
//
// Layout: a cluster takes a (request, layer, head), its CTAs consecutive rows of it, whose
// keys (32 bits that order as the ranking does) stay in shared memory.  The keep-th largest
// key is found by a radix select of 11, 11 and 10 bits on histograms that all CTAs read from
// each other; a round whose bin is taken whole is the last.  Rows that move and free places
// are ranked by counting bits; their list goes to the cluster's shared memory, and each CTA
// copies its part.  One more cluster does the lengths and the pages.  No order of execution
// shows in a result.
//
// Measured: 64 of 4160 rows, 8 heads: 17 us; three requests of 2603 to 12859 rows cut to 2048
// in four layers: 44 us, 2.6 TB/s of rows and records (the longest request's clusters take
// 40, of which 14 are the copy).  A model's 32 layers of 8 heads: one request of 4160 rows cut
// to 4096 in 37 us (26 MB), of 40000 to 2048 in 224 (599 MB, 2.7 TB/s), of 40000 to 30000 in
// 494 (2.1 GB, 4.2 TB/s); seven idle slots beside it add 1 to 5.  Ranking the keys of the last
// bin one by one (10 us more than the rounds it saved), and 64-bit places worked out for each
// row by the whole warp (twice the copy), were left out.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace tw {

constexpr int kEvThreads = 512, kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 2048, kEvRounds = 3;
constexpr int kEvMaxCluster = 8;
constexpr int kEvMaxRequests = 8192;
// A cluster is as large as this many rows a CTA ask for, if the device holds them all at once;
// in any case so large that a CTA has no more than kEvMostRows.  (4160 rows: one CTA 19 us, two
// 17, four 18, eight 22; the four layers above, 128 clusters: two CTAs 44 us, four, of which
// the device holds about half at once, 51, eight 93.)
constexpr int kEvRowsPerCta = 4096, kEvCtas = 2 * 148, kEvMostRows = 16384;
constexpr int kEvMaxRows = 1 << 21;        // of a request: 8 CTAs' bits of its rows
constexpr int kEvSmem = 160 << 10;         // besides the histograms
constexpr int kEvAhead = 8;                // rows whose records a thread reads at a time
constexpr int kEvBatch = 8;                // rows that a warp copies at a time
constexpr uint32_t kEvProtected = 0xffffffffu;

struct EvictTask {
  int request, layer, head;
  int len, keep;
  int more;        // tasks that may follow it
  long long next;  // the position after the request's last
};

struct EvictShared {
  alignas(16) uint32_t hist[kEvRounds][kEvBins];
  uint32_t warp_sum[kEvWarps];
  unsigned long long warp_sums[kEvWarps];
  EvictTask task, own;      // the cluster's is that of its first CTA; a copy of it
  uint32_t bin, above, in;  // where a round's bins reach the rank; keys above it, in it
  uint32_t ties;            // of the CTA
  uint32_t holes, movers;   // of the CTA
};

struct EvictWork {
  tw_paged_evict_args a;
  int words;     // of 32 rows: a CTA's at most
  int held;      // keys that shared memory holds
  int units;     // layers * kv_heads
};

// Rows that stay of a request with `len`; len: nothing is evicted.
__device__ __forceinline__ int evict_kept(const tw_paged_evict_args& a, int len, int keep) {
  const bool held = len <= a.max_len && len <= (long long)a.table_width * a.pool.page_size;
  return held && keep >= 0 && keep < len ? keep : len;
}

// Where row j is: page and row of the page; page -1: its page is none.  (Nor has a row beyond
// the request one: what a call that changes weights meanwhile could leave in the list stays
// inside the buffers.)
struct EvictRow {
  int page, row;
};
__device__ __forceinline__ EvictRow evict_row(const tw_paged_evict_args& a, const EvictTask& t,
                                              int j) {
  if ((unsigned)j >= (unsigned)t.len) return {-1, 0};
  const unsigned i = (unsigned)j / (unsigned)a.pool.page_size;
  const int page = a.block_table[(int64_t)t.request * a.table_stride + i];
  if (page < 0 || page >= a.pool.num_pages) {
    raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
    return {-1, 0};
  }
  return {page, j - (int)(i * (unsigned)a.pool.page_size)};
}
// In a layer and head's records, and its K or V (in 16-byte vectors).
__device__ __forceinline__ int64_t evict_record(const tw_paged_evict_args& a, const EvictTask& t,
                                                EvictRow r) {
  return (int64_t)t.layer * a.record_layer_stride +
         ((int64_t)r.page * a.pool.kv_heads + t.head) * a.pool.page_size + r.row;
}
__device__ __forceinline__ int64_t evict_vector(const tw_paged_evict_args& a, const EvictTask& t,
                                                EvictRow r) {
  return ((int64_t)t.layer * a.layer_stride + (int64_t)r.page * a.pool.page_stride +
          (int64_t)t.head * a.pool.head_stride + (int64_t)r.row * a.pool.token_stride) /
         kPagedAlign;
}

// 32 bits that order as the ranking: a NaN weight above all others, -0 as 0.
__device__ __forceinline__ uint32_t evict_order(const tw_paged_evict_args& a, const EvictTask& t,
                                                float w, long long p) {
  if (p < a.sink || p >= t.next - a.recent) return kEvProtected;
  if (w != w) return kEvProtected - 1;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
// N rows `step` apart: all their pages are read at once, then all their records (without
// branches between, or each read would wait for the one before; a row past the end reads the
// last one's, a page that is none the first record).
template <int N>
__device__ __forceinline__ void evict_keys(const tw_paged_evict_args& a, const EvictTask& t, int j,
                                           int step, int end, uint32_t (&key)[N]) {
  const int32_t* table = a.block_table + (int64_t)t.request * a.table_stride;
  const unsigned size = (unsigned)a.pool.page_size;
  int page[N];
  float w[N];
  int p[N];
  bool bad = false;
#pragma unroll
  for (int y = 0; y < N; ++y) page[y] = table[(unsigned)min(j + y * step, end - 1) / size];
#pragma unroll
  for (int y = 0; y < N; ++y) {
    const bool real = (unsigned)page[y] < (unsigned)a.pool.num_pages;
    const int row = (int)((unsigned)min(j + y * step, end - 1) % size);
    const int64_t at = real ? evict_record(a, t, {page[y], row}) : 0;
    w[y] = a.row_weights[at];
    p[y] = a.row_positions[at];
    bad |= !real;
  }
#pragma unroll
  for (int y = 0; y < N; ++y)
    key[y] = (unsigned)page[y] < (unsigned)a.pool.num_pages ? evict_order(a, t, w[y], p[y]) : 0u;
  if (bad) raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
}

// Sum of x over the threads before this one; total: over all.
__device__ __forceinline__ uint32_t block_before(uint32_t x, uint32_t* s_warp, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t sum = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += y;
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kEvWarps; ++i) {
    const uint32_t y = s_warp[i];
    if (i < warp) before += y;
    total += y;
  }
  __syncthreads();
  return before + sum - x;
}

// The same for two counts of less than 2^31 in all.
__device__ __forceinline__ unsigned long long block_before(unsigned long long x,
                                                           unsigned long long* s_warp,
                                                           unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long sum = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += y;
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kEvWarps; ++i) {
    const unsigned long long y = s_warp[i];
    if (i < warp) before += y;
    total += y;
  }
  __syncthreads();
  return before + sum - x;
}

// Lengths, offsets, pages past the last row: by the CTAs of one cluster, each of which adds
// up all requests' pages itself.  Reads the table and what it ends on, writes neither.
__device__ void evict_lengths(const tw_paged_evict_args& a, uint32_t* s_back,
                              uint32_t* s_warp, int rank, int ctas) {
  const int tid = threadIdx.x;
  const int page = a.pool.page_size;
  const auto pages = [&](int n) {
    return (int)(((unsigned)n + (unsigned)page - 1) / (unsigned)page);
  };
  long long base = 0;
  for (int b0 = 0; b0 < a.requests; b0 += kEvThreads) {
    const int b = b0 + tid;
    uint32_t give = 0;
    if (b < a.requests) {
      const int len = max(a.lens[b], 0), kept = evict_kept(a, len, a.keep[b]);
      give = (uint32_t)(pages(len) - pages(kept));
      if (rank == 0) {
        if (len > a.max_len) raise_error(a.error_flag, TW_ERR_BAD_ARG);
        if (len > (long long)a.table_width * page) raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
        a.lens_out[b] = kept;
        const long long gone = (long long)a.offsets[b] + (len - kept);
        a.offsets_out[b] = (int)min(gone, (long long)INT32_MAX);
      }
    }
    uint32_t total;
    const uint32_t before = block_before(give, s_warp, total);
    if (b < a.requests) s_back[b] = (uint32_t)min(base + before + give, (long long)INT32_MAX);
    base += total;
  }
  __syncthreads();
  if (!a.free_pages) return;
  const int count = (int)max(0ll, min((long long)*a.free_count, (long long)a.pool.num_pages));
  const uint32_t returned = (uint32_t)min(base, (long long)INT32_MAX);
  for (uint32_t k = rank * kEvThreads + tid; k < returned; k += ctas * kEvThreads) {
    if ((long long)count + k >= a.pool.num_pages) {
      raise_error(a.error_flag, TW_ERR_CAPACITY);
      break;
    }
    const int b = first_above(s_back, a.requests, k);
    const int i = pages(max(a.lens[b], 0)) - (int)(s_back[b] - k);
    const int page_id = a.block_table[(int64_t)b * a.table_stride + i];
    if (page_id < 0 || page_id >= a.pool.num_pages) raise_error(a.error_flag, TW_ERR_INVALID_INDEX);
    a.free_pages[(long long)count + k] = page_id;
  }
  if (rank == 0 && tid == 0)
    *a.free_count_out = (int)min(count + base, (long long)a.pool.num_pages);
}

__global__ void __launch_bounds__(kEvThreads, 2)
paged_evict_kernel(const __grid_constant__ EvictWork w) {
  extern __shared__ __align__(16) uint32_t s_dyn[];
  __shared__ EvictShared sh;
  for (int i = threadIdx.x; i < kEvRounds * kEvBins; i += kEvThreads) (&sh.hist[0][0])[i] = 0;
  pdl_wait();
  pdl_launch_dependents();
  const tw_paged_evict_args& a = w.a;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int clusters = (int)(gridDim.x / C) - 1, mine = (int)(blockIdx.x / C);
  if (mine == clusters) {  // the last one
    evict_lengths(a, s_dyn, sh.warp_sum, rank, C);
    return;
  }
  uint32_t* s_keep = s_dyn;               // a bit per row: it stays
  uint32_t* s_eq = s_keep + w.words;      // its key is the keep-th largest
  uint32_t* s_holes = s_eq + w.words;     // free places before a word of rows, of all CTAs
  uint32_t* s_movers = s_holes + w.words; // rows that move before it
  uint32_t* s_key = s_movers + w.words;   // keys; then free places and the rows that move there
  const uint32_t pairs_held = (uint32_t)w.held / 2;

  const int64_t tasks = (int64_t)a.requests * w.units;
  int64_t at = mine;  // first task that may be next
  for (;;) {
    // ---- the next task that evicts anything: found by the first CTA, so that all of the
    // cluster do the same whatever becomes of the lengths meanwhile
    if (rank == 0 && warp == 0) {
      EvictTask t = {-1, 0, 0, 0, 0, 0, 0};
      while (at < tasks) {
        const int64_t x = at + (int64_t)lane * clusters;
        int len = 0, kept = 0, gone = 0;
        if (x < tasks) {
          const int b = (int)(x / w.units);
          len = max(a.lens[b], 0);
          kept = evict_kept(a, len, a.keep[b]);
          gone = a.offsets[b];
        }
        const unsigned found = __ballot_sync(0xffffffffu, kept < len);
        if (!found) {
          at += 32ll * clusters;
          continue;
        }
        const int first = __ffs(found) - 1;
        at += (int64_t)first * clusters;
        t.request = (int)(at / w.units);
        const int unit = (int)(at - (int64_t)t.request * w.units);
        t.layer = unit / a.pool.kv_heads;
        t.head = unit - t.layer * a.pool.kv_heads;
        t.len = __shfl_sync(0xffffffffu, len, first);
        t.keep = __shfl_sync(0xffffffffu, kept, first);
        t.next = (long long)t.len + __shfl_sync(0xffffffffu, gone, first);
        at += clusters;
        t.more = at < tasks;
        break;
      }
      if (lane == 0) sh.task = t;
    }
    cluster.sync();
    if (tid == 0) sh.own = *cluster.map_shared_rank(&sh.task, 0);
    __syncthreads();
    const EvictTask& t = sh.own;
    if (t.request < 0) break;

    const int seg = ((t.len + C - 1) / C + 31) / 32 * 32;
    const int row0 = min(rank * seg, t.len), n = min(seg, t.len - row0);
    const int words = (n + 31) / 32;
    const auto key = [&](int i) {
      if (i < w.held) return s_key[i];
      uint32_t k[1];
      evict_keys(a, t, row0 + i, 1, row0 + n, k);
      return k[0];
    };

    // ---- the keep-th largest key
    uint32_t prefix = 0;              // its bits found so far
    uint32_t need = (uint32_t)t.keep; // its rank among the keys with these
    uint32_t same = 0;                // keys that equal it in these
    int low = 0;                      // bits that were not needed
#pragma unroll 1
    for (int round = 0; round < kEvRounds; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
      const int bits = round == 2 ? 10 : 11;
      if (round == 0) {
        for (int i = tid; i < n; i += kEvAhead * kEvThreads) {
          uint32_t k[kEvAhead];
          evict_keys(a, t, row0 + i, kEvThreads, row0 + n, k);
#pragma unroll
          for (int y = 0; y < kEvAhead; ++y) {
            const int at = i + y * kEvThreads;
            if (at >= n) break;
            if (at < w.held) s_key[at] = k[y];
            atomicAdd(&sh.hist[0][k[y] >> shift], 1u);
          }
        }
      } else {
        const int top = shift + bits;
        for (int i = tid; i < n; i += kEvThreads) {
          const uint32_t k = key(i);
          if (k >> top == prefix >> top)
            atomicAdd(&sh.hist[round][k >> shift & ((1u << bits) - 1)], 1u);
        }
      }
      cluster.sync();
      // this thread's bins of all CTAs, the highest first
      constexpr int kEach = kEvBins / kEvThreads;
      uint32_t bin[kEach] = {};
      const int first = kEvBins - kEach * (tid + 1);
#pragma unroll
      for (int r = 0; r < kEvMaxCluster; ++r) {
        if (r >= C) break;
        const uint4 x = *reinterpret_cast<const uint4*>(
            cluster.map_shared_rank(&sh.hist[round][first], r));
        bin[0] += x.w;
        bin[1] += x.z;
        bin[2] += x.y;
        bin[3] += x.x;
      }
      static_assert(kEach == 4);
      uint32_t total;
      uint32_t before = block_before(bin[0] + bin[1] + bin[2] + bin[3], sh.warp_sum, total);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (before < need && need <= before + bin[i]) {
          sh.bin = (uint32_t)(first + kEach - 1 - i);
          sh.above = before;
          sh.in = bin[i];
        }
        before += bin[i];
      }
      __syncthreads();
      if (need > 0) {
        prefix |= sh.bin << shift;
        need -= sh.above;
        same = sh.in;
      }
      __syncthreads();
      low = shift;
      if (need == same) break;
    }
    const bool all = need == same;  // all that equal it stay (nothing at all: keep is 0)
    prefix >>= low;

    // ---- which rows stay
    uint32_t ties = 0;
    for (int x = warp; x < words; x += kEvWarps) {
      const int i = x * 32 + lane;
      const uint32_t k = i < n ? key(i) >> low : 0u;
      const unsigned above = __ballot_sync(0xffffffffu, i < n && t.keep > 0 && k > prefix);
      const unsigned equal = __ballot_sync(0xffffffffu, i < n && t.keep > 0 && k == prefix);
      if (lane == 0) {
        s_keep[x] = all ? above | equal : above;
        s_eq[x] = equal;
      }
      ties += __popc(equal);
    }
    if (!all) {  // of those that equal it the first `need` rows
      if (tid == 0) sh.ties = 0;
      __syncthreads();
      if (lane == 0) atomicAdd(&sh.ties, ties);
      cluster.sync();
      uint32_t before = 0;
      for (int r = 0; r < rank; ++r) before += *cluster.map_shared_rank(&sh.ties, r);
      for (int x0 = 0; x0 < words; x0 += kEvThreads) {
        const int x = x0 + tid;
        const uint32_t equal = x < words ? s_eq[x] : 0u;
        uint32_t total;
        const uint32_t first = before + block_before(__popc(equal), sh.warp_sum, total);
        before += total;
        int stay = (int)min(max((long long)need - first, 0ll), 32ll);
        if (stay >= __popc(equal)) {
          if (equal) s_keep[x] |= equal;
        } else {
          uint32_t left = equal, taken = 0;
          for (; stay > 0; --stay) {
            taken |= left & (0u - left);
            left &= left - 1;
          }
          if (x < words) s_keep[x] |= taken;
        }
      }
    }
    __syncthreads();

    // ---- free places (rows below keep that go) and rows that move (from keep on, that stay)
    const auto holes_of = [&](int x) {
      const int first = row0 + x * 32, end = min(min(t.keep, t.len) - first, min(32, n - x * 32));
      return end <= 0 ? 0u : ~s_keep[x] & (end >= 32 ? 0xffffffffu : (1u << end) - 1);
    };
    const auto movers_of = [&](int x) {
      const int from = t.keep - (row0 + x * 32);
      return from >= 32 ? 0u : from <= 0 ? s_keep[x] : s_keep[x] & ~((1u << from) - 1);
    };
    uint32_t holes = 0, movers = 0;
    for (int x0 = 0; x0 < words; x0 += kEvThreads) {
      const int x = x0 + tid;
      const uint32_t h = x < words ? __popc(holes_of(x)) : 0u;
      const uint32_t m = x < words ? __popc(movers_of(x)) : 0u;
      unsigned long long total;
      const unsigned long long before =
          block_before((unsigned long long)m << 32 | h, sh.warp_sums, total);
      if (x < words) {
        s_holes[x] = holes + (uint32_t)before;
        s_movers[x] = movers + (uint32_t)(before >> 32);
      }
      holes += (uint32_t)total;
      movers += (uint32_t)(total >> 32);
    }
    if (tid == 0) {
      sh.holes = holes;
      sh.movers = movers;
    }
    cluster.sync();  // (also: all CTAs are done with their keys)
    uint32_t holes_before = 0, movers_before = 0, pairs = 0;
    for (int r = 0; r < C; ++r) {
      const uint32_t h = *cluster.map_shared_rank(&sh.holes, r);
      const uint32_t m = *cluster.map_shared_rank(&sh.movers, r);
      if (r < rank) {
        holes_before += h;
        movers_before += m;
      }
      pairs += m;
    }

    // ---- pair k: place and row k, with CTA k % C; as many at a time as the CTAs hold
    for (uint32_t done = 0; done < pairs; done += pairs_held * C) {
      const auto put = [&](uint32_t list, uint32_t k, int row) {
        if (k < done || k - done >= pairs_held * C) return;
        const uint32_t i = k - done;
        *cluster.map_shared_rank(&s_key[list * pairs_held + i / C], i % C) = (uint32_t)row;
      };
      for (int x = warp; x < words; x += kEvWarps) {
        const uint32_t h = holes_of(x), m = movers_of(x), below = (1u << lane) - 1;
        const int row = row0 + x * 32 + lane;
        if (h >> lane & 1) put(0, holes_before + s_holes[x] + __popc(h & below), row);
        if (m >> lane & 1) put(1, movers_before + s_movers[x] + __popc(m & below), row);
      }
      cluster.sync();
      const uint32_t here = min(pairs - done, pairs_held * C);  // of all CTAs
      const int count = (int)((here + C - 1 - rank) / C);       // of this one
      // A warp takes up to 32 rows: a thread finds where one comes from and goes to and moves
      // its record, then the warp copies them, half of it K and half V.  (64-bit products for
      // each row by the whole warp took longer than the copies.)
      uint4* const pages = reinterpret_cast<uint4*>(lane < kVecPerRow16 ? a.pool.k_pages
                                                                        : a.pool.v_pages) +
                           lane % kVecPerRow16;
      const int per = min((count + kEvWarps - 1) / kEvWarps, 32);
      for (int first = warp * per; first < count; first += kEvWarps * per) {
        const int rows = min(per, count - first);
        int64_t source = 0, place = -1;  // -1: not to move; it reads the pool's first row
        if (lane < rows) {
          const EvictRow to = evict_row(a, t, (int)s_key[first + lane]);
          const EvictRow from = evict_row(a, t, (int)s_key[pairs_held + first + lane]);
          if (to.page >= 0 && from.page >= 0) {
            source = evict_vector(a, t, from);
            place = evict_vector(a, t, to);
            const int64_t i = evict_record(a, t, from), o = evict_record(a, t, to);
            const float weight = a.row_weights[i];
            const int position = a.row_positions[i];
            a.row_weights[o] = weight;
            a.row_positions[o] = position;
          }
        }
        for (int y0 = 0; y0 < rows; y0 += kEvBatch) {
          uint4 x[kEvBatch];
#pragma unroll
          for (int y = 0; y < kEvBatch; ++y)
            x[y] = __ldcs(pages + __shfl_sync(0xffffffffu, (long long)source, y0 + y));
#pragma unroll
          for (int y = 0; y < kEvBatch; ++y) {
            const long long to = __shfl_sync(0xffffffffu, (long long)place, y0 + y);
            if (to >= 0) pages[to] = x[y];
          }
        }
      }
      if (pairs - done > pairs_held * C) cluster.sync();
    }
    if (!t.more) {
      // (with pairs, a barrier has come after the last access to another CTA's memory)
      if (pairs == 0) cluster.sync();
      return;
    }
    for (int i = tid; i < kEvRounds * kEvBins; i += kEvThreads) (&sh.hist[0][0])[i] = 0;
  }
  cluster.sync();  // the first CTA's memory has been read
}

}  // namespace tw

using namespace tw;

extern "C" size_t tw_paged_evict_args_size(void) { return sizeof(tw_paged_evict_args); }

static bool apart(const void* p, size_t n, const void* q, size_t m) {
  return !p || !q || (uintptr_t)p + n <= (uintptr_t)q || (uintptr_t)q + m <= (uintptr_t)p;
}

extern "C" int tw_paged_evict(const tw_paged_evict_args* args, void* stream) {
  if (!args) return TW_ERR_BAD_ARG;
  const tw_paged_evict_args& a = *args;
  const int rc = check_paged_pool(a.pool);
  if (rc != TW_OK) return rc;
  if (a.requests < 0) return TW_ERR_BAD_ARG;
  if (a.requests == 0) return TW_OK;
  if (!a.row_weights || !a.row_positions || !a.block_table || !a.lens || !a.keep || !a.offsets ||
      !a.lens_out || !a.offsets_out || a.layers <= 0 || a.layer_stride < 0 ||
      a.layer_stride % kPagedAlign != 0 || a.record_layer_stride < 0 || a.table_width <= 0 ||
      a.table_stride < a.table_width || a.max_len < 0 || a.sink < 0 || a.recent < 0 ||
      (a.layers > 1 && (a.layer_stride == 0 || a.record_layer_stride == 0)))
    return TW_ERR_BAD_ARG;
  if ((a.free_pages == nullptr) != (a.free_count == nullptr) ||
      (a.free_pages == nullptr) != (a.free_count_out == nullptr))
    return TW_ERR_BAD_ARG;
  if (a.requests > kEvMaxRequests || a.max_len > kEvMaxRows ||
      (int64_t)a.layers * a.pool.kv_heads > INT32_MAX)
    return TW_ERR_UNSUPPORTED;
  const size_t n = (size_t)a.requests * 4;
  const struct { const void* p; size_t n; } in[] = {{a.lens, n}, {a.keep, n}, {a.offsets, n},
                                                    {a.free_count, 4}},
      out[] = {{a.lens_out, n}, {a.offsets_out, n}, {a.free_count_out, 4},
               {a.free_pages, (size_t)a.pool.num_pages * 4}};
  for (const auto& o : out) {
    for (const auto& i : in)
      if (!apart(o.p, o.n, i.p, i.n)) return TW_ERR_BAD_ARG;
    for (const auto& p : out)
      if (&p != &o && !apart(o.p, o.n, p.p, p.n)) return TW_ERR_BAD_ARG;
  }
  EvictWork w = {};
  w.a = a;
  w.units = a.layers * a.pool.kv_heads;
  const int64_t tasks = (int64_t)a.requests * w.units;
  int C = 1;
  while (C < kEvMaxCluster && a.max_len > C * kEvRowsPerCta &&
         (2 * C * tasks <= kEvCtas || a.max_len > C * kEvMostRows))
    C *= 2;
  const int seg = max(((a.max_len + C - 1) / C + 31) / 32 * 32, 128);
  w.words = seg / 32;
  w.held = min(seg, (kEvSmem - 16 * w.words) / 4);
  const int smem = max(16 * w.words + 4 * w.held, 4 * a.requests);
  static DynSmemOptIn opt_in;
  const int st = ensure_dyn_smem((const void*)paged_evict_kernel, opt_in, smem);
  if (st != TW_OK) return st;
  // (one more for the lengths)
  const int clusters = (int)min(tasks, (int64_t)(2 * kEvCtas / C)) + 1;
  return launch_pdl_cluster(paged_evict_kernel, dim3((unsigned)(clusters * C)), dim3(kEvThreads),
                            C, (size_t)smem, (cudaStream_t)stream, w);
}
