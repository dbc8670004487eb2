// Attention of new tokens over a paged KV cache: argument checks, how the call
// is divided, and the merge of split rows.
//
// Row (t, h): token t of request b at position p sees the keys [low, p];
// out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = scale * log2(e) * q . k_j.
#include "paged_attention.cuh"

namespace tw {

constexpr int kMergeWarps = 4;   // of a CTA
constexpr int kMergeAhead = 10;  // ranges that a warp reads before it knows the maximum

// Joins the ranges of split rows: out = sum_s 2^(lse_s - M) o_s / sum_s 2^(lse_s - M).
// Rows of few-token requests have many ranges: four warps a row take every fourth,
// so that a row's loads are in flight together; the others get a warp each.  The
// ranges are added in an order that does not depend on which was ready first.
// Bound: latency; 32 rows of 37 ranges cost about 4 us after the token kernel (one of
// them for the lengths, read when that has ended), 1.6 us less than with loads that wait
// for the maximum and 5 us less than with one warp a row.
template <typename Out, bool kFew>
__global__ void __launch_bounds__(kMergeWarps * 32)
paged_merge_kernel(const __grid_constant__ PagedWork w) {
  const tw_paged_attention_args& a = w.a;
  const PagedSplit& sp = kFew ? w.few : w.many;
  constexpr int kWarps = kFew ? kMergeWarps : 1;  // of a row
  // Every CTA waits, also one without work: what follows in the stream takes the end
  // of this kernel for the end of the one before it.
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = kFew ? threadIdx.x >> 5 : 0;
  const int64_t row = kFew ? blockIdx.x
                           : (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  int t, h;
  PagedRequest rq;
  PagedKeys keys;
  if (kFew) {
    const int r = (int)(row % w.few_rows);
    const int unit = (int)(row / w.few_rows);
    const int b = unit / a.pool.kv_heads;
    rq = paged_request(a, b);
    if (rq.n > w.few_tokens || rq.n > a.max_q_len || r >= rq.n * w.group) return;
    t = rq.first + r / w.group;
    h = (unit - b * a.pool.kv_heads) * w.group + r % w.group;
    keys = paged_keys(a, rq, 0, rq.n);
  } else {
    t = (int)(row / a.q_heads);
    h = (int)(row - (int64_t)t * a.q_heads);
    const int b = t < a.tokens ? first_above(a.cu_q + 1, a.requests, t) : a.requests;
    if (b >= a.requests) return;
    rq = paged_request(a, b);
    if (rq.n <= w.few_tokens || rq.n > a.max_q_len) return;
    const int tokens = paged_chunk_tokens(w.group);
    const int begin = (t - rq.first) / tokens * tokens;
    keys = paged_keys(a, rq, begin, min(rq.n - begin, tokens));
  }
  const int parts = paged_range(sp, keys.low, keys.high, 0).parts;
  if (parts == 1) return;  // the range wrote the result itself
  const float* lse = sp.part_lse + row * sp.splits;
  const float* po = sp.part_o + row * sp.splits * kHeadDim + lane * 4;
  // the first ranges of the warp are under way while the maximum is worked out
  float4 x[kMergeAhead];
  float z[kMergeAhead];
#pragma unroll
  for (int k = 0; k < kMergeAhead; ++k) {
    const int s = warp + k * kWarps;
    x[k] = s < parts ? *reinterpret_cast<const float4*>(po + (int64_t)s * kHeadDim)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
    z[k] = s < parts ? lse[s] : -CUDART_INF_F;
  }
  float m = -CUDART_INF_F;
  for (int s = lane; s < parts; s += 32) m = fmaxf(m, lse[s]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float u = m == -CUDART_INF_F ? 0.f : m;
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  auto take = [&](const float4& y, float lse_s) {
    const float f = ex2(lse_s - u);
    l += f;
    o[0] = fmaf(y.x, f, o[0]);
    o[1] = fmaf(y.y, f, o[1]);
    o[2] = fmaf(y.z, f, o[2]);
    o[3] = fmaf(y.w, f, o[3]);
  };
#pragma unroll
  for (int k = 0; k < kMergeAhead; ++k) take(x[k], z[k]);
#pragma unroll 8
  for (int s = warp + kMergeAhead * kWarps; s < parts; s += kWarps)
    take(*reinterpret_cast<const float4*>(po + (int64_t)s * kHeadDim), lse[s]);
  if constexpr (kFew) {
    __shared__ float s_l[kMergeWarps];
    __shared__ float4 s_o[kMergeWarps][32];
    if (lane == 0) s_l[warp] = l;
    s_o[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 1; k < kMergeWarps; ++k) {
      const float4 y = s_o[k][lane];
      l += s_l[k];
      o[0] += y.x;
      o[1] += y.y;
      o[2] += y.z;
      o[3] += y.w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] *= inv;
  paged_store_row<Out, 4>(a, t, h, lane * 4, o, paged_lse(m, l));
}

template <bool kFew>
static int launch_merge(const PagedWork& w, int64_t rows, cudaStream_t stream) {
  const int64_t ctas = kFew ? rows : (rows + kMergeWarps - 1) / kMergeWarps;
  if (ctas > INT32_MAX) return TW_ERR_UNSUPPORTED;
  const auto kernel = w.a.out_dtype == TW_F32   ? paged_merge_kernel<float, kFew>
                      : w.a.out_dtype == TW_F16 ? paged_merge_kernel<__half, kFew>
                                                : paged_merge_kernel<__nv_bfloat16, kFew>;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(kMergeWarps * 32), 0, stream, w);
}

// ---- division of a call -----------------------------------------------------------
constexpr int kFewRows = 16;  // rows of one warp-level product

static int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// `keys` keys in ranges of at least `chunk`, whole tiles, kMaxSplits at most.
constexpr int kMaxSplits = 256;
static PagedSplit cut(int64_t keys, int64_t chunk) {
  chunk = chunk * kMaxSplits < keys ? div_up(keys, kMaxSplits) : chunk;
  PagedSplit sp = {};
  sp.chunk = (int)(div_up(chunk, kTileKeys) * kTileKeys);
  sp.splits = (int)div_up(keys, sp.chunk);
  return sp;
}

constexpr int64_t kRowBytes = (kHeadDim + 4) * sizeof(float);  // of a row's partial result
static size_t part_bytes(int64_t rows, const PagedSplit& sp) {
  return sp.splits > 1 ? (size_t)rows * sp.splits * kRowBytes : 0;
}

// Ranges of the token kernel.  Its 2 CTAs per SM share the device; one request
// (or a few) is cut so that all of them get a range, no shorter than 256 keys
// (the pipeline's fill and the merge cost about that); many requests are cut
// into twice the CTAs, because their lengths differ; and no range is longer
// than 4096 keys, so that one long request among many short ones does not
// leave the others waiting, unless the partial results, which every request has a
// place for in each range, would take more than kFewBytes (256 requests with up to 4
// tokens each, one at 131k: 15 ranges of 8832 keys instead of 32).
constexpr int64_t kFewBytes = 256 << 20;
static PagedSplit split_few(int requests, int kv_heads, int rows, int64_t max_keys) {
  const int64_t units = (int64_t)requests * kv_heads;
  const int64_t ctas = 2 * 148 * (requests > 1 ? 2 : 1);
  int64_t chunk = div_up(units * max_keys, ctas);
  chunk = chunk < 256 ? 256 : chunk > 4096 ? 4096 : chunk;
  const int64_t most = kFewBytes / (units * rows * kRowBytes);
  if (chunk * most < max_keys) chunk = most > 1 ? div_up(max_keys, most) : max_keys;
  return cut(max_keys, chunk);
}

// Ranges of the chunk kernel: one, unless its CTAs would leave SMs idle.  A single
// request's CTAs are known: its keys are cut so that about all SMs get one, into
// ranges of 768 keys or more (a range costs 6 us besides its tiles, and the merge;
// 511 tokens at 3k, 14 heads: 47 us whole, 37, 31, 28 us in two, three, four ranges).
// Of several requests, those with few tokens get no chunk CTA, but how many that are
// the host does not know: the keys are cut for twice the SMs, into ranges of 1536
// keys or more (13 requests of 5k to 14k, five of them with up to 8 tokens: 184 us
// whole, 112 us in two ranges, 103 us in three).  Cutting does not pay where all have a
// CTA (6 requests of 5k to 7k, 645 tokens, 64 heads: 172 us whole, 183, 197 us in two,
// three ranges), nor does evening out the last wave of a single request (256 CTAs at
// 32k: 0.99 ms whole, 1.06 ms in four): the partial results' traffic costs more.
static PagedSplit split_many(int requests, int64_t units, int64_t keys) {
  const int64_t ctas = (requests > 1 ? 2 : 1) * 148;
  int64_t n = units < ctas ? ctas / units : 1;
  const int64_t least = requests > 1 ? 1536 : 768;
  n = keys / least < n ? keys / least : n;
  return cut(keys, n > 1 ? div_up(keys, n) : keys);
}

struct PagedPlan {
  int64_t few_rows, many_rows;  // rows with partial results
  size_t bytes;                 // of the workspace
};

// Divides a call by its sizes.
static PagedPlan plan_paged(PagedWork& w, int requests, int tokens, int q_heads, int kv_heads,
                            int max_q_len, int max_kv_len, int window) {
  w.group = q_heads / kv_heads;
  const int most = max_q_len < 1 ? 1 : max_q_len < tokens ? max_q_len : tokens;
  w.few_tokens = kFewRows / w.group < most ? kFewRows / w.group : most;
  if (requests == 1 && most > w.few_tokens) w.few_tokens = 0;  // one request: one kernel
  w.few_rows = w.few_tokens * w.group;
  // keys that a CTA's rows see, from a tile's begin on (1: there may be none)
  const int64_t cap = max_kv_len < 1 ? 1 : max_kv_len < (1 << 30) ? max_kv_len : 1 << 30;
  auto seen = [&](int64_t rows) {
    const int64_t x = (int64_t)window + rows + kTileKeys;
    return window > 0 && x < cap ? x : cap;
  };
  PagedPlan plan = {};
  if (w.few_tokens > 0) {
    w.few = split_few(requests, kv_heads, w.few_rows, seen(w.few_tokens));
    plan.few_rows = (int64_t)requests * kv_heads * w.few_rows;
  }
  if (most > w.few_tokens) {
    const int each = paged_chunk_tokens(w.group);
    const int64_t slots =
        requests == 1 ? div_up(tokens, each) : (int64_t)tokens / each + requests;
    w.many = split_many(requests, slots * kv_heads, seen(each));
    plan.many_rows = (int64_t)tokens * q_heads;
  }
  plan.bytes = part_bytes(plan.few_rows, w.few) + part_bytes(plan.many_rows, w.many);
  return plan;
}

static void place_parts(PagedSplit& sp, int64_t rows, float*& at) {
  if (sp.splits <= 1) return;
  sp.part_o = at;
  sp.part_lse = at + rows * sp.splits * kHeadDim;
  at += part_bytes(rows, sp) / sizeof(float);
}

}  // namespace tw

using namespace tw;

extern "C" size_t tw_paged_attention_args_size(void) { return sizeof(tw_paged_attention_args); }

extern "C" size_t tw_paged_attention_workspace_size(int requests, int tokens, int q_heads,
                                                    int kv_heads, int max_q_len, int max_kv_len,
                                                    int window, int head_dim) {
  if (requests <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 ||
      q_heads / kv_heads > 64 || max_q_len < 0 || max_kv_len < 0 || window < 0 ||
      head_dim != kHeadDim)
    return 0;
  PagedWork w = {};
  return plan_paged(w, requests, tokens, q_heads, kv_heads, max_q_len, max_kv_len, window).bytes;
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
  PagedWork w = {};
  w.a = a;
  w.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const PagedPlan plan = plan_paged(w, a.requests, a.tokens, a.q_heads, a.pool.kv_heads,
                                    a.max_q_len, a.max_kv_len, a.window);
  if (plan.bytes > 0) {
    if (!a.workspace || a.workspace_bytes < plan.bytes) return TW_ERR_CAPACITY;
    if (!aligned16(a.workspace)) return TW_ERR_BAD_ARG;
    float* at = (float*)a.workspace;
    place_parts(w.few, plan.few_rows, at);
    place_parts(w.many, plan.many_rows, at);
  }
  // one box: the rows that a page and a tile of 64 keys have in common
  w.box = 64;
  while (a.pool.page_size % w.box != 0) w.box /= 2;
  PagedMaps maps;
  const cuuint64_t dims[4] = {(cuuint64_t)kHeadDim, (cuuint64_t)a.pool.page_size,
                              (cuuint64_t)a.pool.kv_heads, (cuuint64_t)a.pool.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)a.pool.token_stride * 2,
                                 (cuuint64_t)a.pool.head_stride * 2,
                                 (cuuint64_t)a.pool.page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)w.box, 1, 1};
  int st = encode_rows_map(&maps.k, a.pool.dtype, 4, a.pool.k_pages, dims, strides, box);
  if (st == TW_OK) st = encode_rows_map(&maps.v, a.pool.dtype, 4, a.pool.v_pages, dims, strides, box);
  if (st != TW_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  // a mixed call is one launch too: the chunk kernel takes the token kernel's items
  st = w.many.splits > 0 ? launch_paged_chunk(w, maps, s) : launch_paged_token(w, maps, s);
  if (st == TW_OK && w.few.splits > 1) st = launch_merge<true>(w, plan.few_rows, s);
  if (st == TW_OK && w.many.splits > 1) st = launch_merge<false>(w, plan.many_rows, s);
  return st;
}
