// Which pages of a paged cache a query block reads: the mean key of every full
// page, and the choice by it.
//
// Page p of a sequence has the mean key m_p = sum_rows k / page_size, kept per
// pool page in fp32 (pages are shared, moved and copied with their means). A query
// block is up to query_block consecutive new rows of a sequence times the heads of
// a KV head's group; its list holds, ascending,
//   the pages of the first `prefix` tokens,
//   those with a key at most `window` before one of its queries, its own included,
//   and of the others the topk best by s_p = (sum of its queries) . m_p,
// as far as they are present. Only full pages are scored: every page that is
// partly filled holds a query's own position.
//
// Both the queries' sum and s_p are summed in 64 bits and s_p is rounded once to
// fp32: the order of the sums then changes a score, and so a list, only for values
// that lie within 2^-50 or so of a border, where 32 bits would make the lists
// depend on the order of every sum.
namespace sabre {
namespace paged {

// ---------------------------------------------------------------------------
// mean keys: reads 256 bytes a row and head once. A warp takes one page of one
// head, half of it the even rows and half the odd ones, 16 bytes a lane and
// eight loads in flight; the sums are fp32 in row order.
// ---------------------------------------------------------------------------
namespace means {

constexpr int kMaxWarps = 8;

struct Params {
  Cache c;  // k strides only
  const void* k;
  float* means;
  const int32_t* starts;
  long long m_sp, m_sh;
  int rows, heads;
};

template <typename T>
__global__ void __launch_bounds__(kMaxWarps * 32) paged_key_means_kernel(const Params p) {
  __shared__ int scratch[16];
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  if (tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // The page of this CTA: the blockIdx.x-th that the new rows fill. Warp 0 looks
  // for it, 32 sequences at a time.
  if (tid < 32) {
    int left = blockIdx.x, found = -1, page = -1;
    for (int b0 = 0; b0 < p.c.batch && found < 0; b0 += 32) {
      const int b = b0 + lane;
      int first = 0, full = 0;
      if (b < p.c.batch) {
        const int len = max(row_start(p.starts, b + 1, p.rows) - row_start(p.starts, b, p.rows), 0);
        const int n = p.c.length(b);
        // The rows before the new ones; lengths reach to the ends of int32.
        const int old = max(min(static_cast<long long>(p.c.seq_lens[b]) - len, static_cast<long long>(n)), 0ll);
        first = old >> p.c.page_shift;
        full = (n >> p.c.page_shift) - first;
      }
      int incl = full;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, s);
        if (lane >= s) incl += up;
      }
      const uint32_t here = __ballot_sync(0xffffffffu, left < incl);
      if (here != 0u) {
        found = __ffs(here) - 1;
        if (lane == found) page = p.c.page_of(b, (first + left - (incl - full)) << p.c.page_shift);
        page = __shfl_sync(0xffffffffu, page, found);
      }
      left -= __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) scratch[0] = page;
  }
  __syncthreads();
  const int page = scratch[0];
  if (page < 0) return;
  const int half = lane >> 4, ch = lane & 15;
  const int pairs = 1 << (p.c.page_shift - 1);
  for (int h = blockIdx.y * (blockDim.x >> 5) + (tid >> 5); h < p.heads; h += gridDim.y * (blockDim.x >> 5)) {
    const T* src = static_cast<const T*>(p.k) + page * p.c.k_sp + h * p.c.k_sh + half * p.c.k_st + ch * 8;
    float sum[8] = {};
    for (int r = 0; r < pairs; r += 8) {
      uint4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const uint4*>(src + (r + u) * 2 * p.c.k_st);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const T* e = reinterpret_cast<const T*>(&x[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += DT<T>::to_f(e[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = (sum[i] + __shfl_xor_sync(0xffffffffu, sum[i], 16)) * (0.5f / pairs);
    float* dst = p.means + page * p.m_sp + h * p.m_sh + ch * 8 + half * 4;
    *reinterpret_cast<float4*>(dst) = half ? make_float4(sum[4], sum[5], sum[6], sum[7])
                                           : make_float4(sum[0], sum[1], sum[2], sum[3]);
  }
}

}  // namespace means

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
namespace sel {

constexpr int kThreads = 256;
constexpr int kMaxPages = 32768;  // of a sequence: their keys are kept in shared memory

struct Params {
  Cache c;  // no pools
  const void* q;
  const float* means;
  const int32_t* starts;
  int32_t* lists;
  int32_t* counts;
  long long q_sr, q_sh, m_sp, m_sh;
  int rows, heads_kv, group, tokens, topk, window, prefix, cap;
};

// Scores as whole numbers in the same order: 0 is no candidate, 1 a NaN (taken
// last), numbers lie above, kAlways above them all.
constexpr uint32_t kAlways = 0xffffffffu;
__device__ __forceinline__ uint32_t order_key(float s) {
  if (s != s) return 1u;
  const uint32_t u = __float_as_uint(s + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) paged_select_kernel(const Params p) {
  extern __shared__ uint32_t s_key[];  // [pages]
  __shared__ int scratch[16];
  __shared__ double s_part[4][kD];
  __shared__ int s_hist[256];
  __shared__ int s_pick[4];
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int warp = tid >> 5;
  const int hk = blockIdx.y;
  if (tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int32_t* const out = p.lists + (static_cast<long long>(blockIdx.x) * p.heads_kv + hk) * p.cap;
  RowTile t{static_cast<int>(blockIdx.x), 0, static_cast<int>(blockIdx.x), 1, 0};
  bool some = true;
  if (p.starts)
    some = find_rows<kThreads>(p.c, p.starts, p.rows, p.tokens, blockIdx.x, scratch, t);
  else
    t.length = p.c.seq_lens[t.b];
  // Positions [i0, i1] of the block's rows; lengths reach to the ends of int32.
  const int count = min(p.tokens, t.len - t.r);
  const long long i0 = some ? static_cast<long long>(t.length) - t.len + t.r : -1;
  const long long i1 = i0 + count - 1;
  const int n = some ? static_cast<int>(max(min(static_cast<long long>(p.c.length(t.b)), i1 + 1), 0ll)) : 0;
  const int pages = (n + (1 << p.c.page_shift) - 1) >> p.c.page_shift;
  // Pages from `low` on, or that begin before the prefix's end, are always read.
  const int low = static_cast<int>(min(max(i0 - p.window, 0ll) >> p.c.page_shift, static_cast<long long>(pages)));
  const int head = static_cast<int>((static_cast<long long>(p.prefix) + (1 << p.c.page_shift) - 1) >> p.c.page_shift);

  // The queries' sum: 64 threads a row, two columns each.
  {
    double a = 0.0, b = 0.0;
    const T* q = static_cast<const T*>(p.q) + (tid & 63) * 2;
    for (int i = tid >> 6; some && i < count * p.group; i += 4) {
      const int row = t.first + t.r + i / p.group;
      const uint32_t x = *reinterpret_cast<const uint32_t*>(q + row * p.q_sr + (hk * p.group + i % p.group) * p.q_sh);
      const T* e = reinterpret_cast<const T*>(&x);
      a += static_cast<double>(DT<T>::to_f(e[0]));
      b += static_cast<double>(DT<T>::to_f(e[1]));
    }
    s_part[tid >> 6][(tid & 63) * 2] = a;
    s_part[tid >> 6][(tid & 63) * 2 + 1] = b;
  }
  __syncthreads();
  if (tid < kD) s_part[0][tid] = (s_part[0][tid] + s_part[1][tid]) + (s_part[2][tid] + s_part[3][tid]);
  __syncthreads();

  // Scores: eight lanes a page, 16 columns each (four of every 32).
  const int sub = lane & 7;
  double qs[16];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) qs[4 * j + e] = s_part[0][32 * j + 4 * sub + e];
  int scored = 0;
  for (int g = warp * 4; g < pages; g += kThreads / 8) {
    const int pg = g + (lane >> 3);
    const int page = pg < pages ? p.c.page_of(t.b, pg << p.c.page_shift) : -1;
    const bool always = pg >= low || pg < head;
    double s = 0.0;
    if (page >= 0 && !always) {
      const float* m = p.means + page * p.m_sp + hk * p.m_sh + 4 * sub;
      float4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const float4*>(m + 32 * j);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s = fma(qs[4 * j], static_cast<double>(x[j].x), s);
        s = fma(qs[4 * j + 1], static_cast<double>(x[j].y), s);
        s = fma(qs[4 * j + 2], static_cast<double>(x[j].z), s);
        s = fma(qs[4 * j + 3], static_cast<double>(x[j].w), s);
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (sub == 0 && pg < pages) {
      s_key[pg] = page < 0 ? 0u : always ? kAlways : order_key(static_cast<float>(s));
      scored += page >= 0 && !always ? 1 : 0;
    }
  }
  scored = __reduce_add_sync(0xffffffffu, scored);
  if (lane == 0) scratch[warp] = scored;
  __syncthreads();
  int candidates = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) candidates += scratch[w];

  // The topk-th largest of the candidates' keys, eight bits at a time from the top;
  // `want`: how many of those equal to it are taken.
  uint32_t limit = 1u;
  int want = candidates;
  if (p.topk == 0) {
    limit = kAlways - 1;
    want = 0;
  } else if (candidates > p.topk) {
    want = p.topk;
    limit = 0u;
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < pages; i += kThreads) {
        const uint32_t key = s_key[i];
        if (key != 0u && key != kAlways && (shift == 24 || key >> (shift + 8) == limit >> (shift + 8)))
          atomicAdd(&s_hist[key >> shift & 255u], 1);
      }
      __syncthreads();
      // Warp 0 finds the bin that the want-th largest is in: lane l holds bins
      // 255 - 8 l down to 248 - 8 l.
      if (warp == 0) {
        int bins[8], mine = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) mine += bins[u] = s_hist[255 - 8 * lane - u];
        int incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, incl, s);
          if (lane >= s) incl += up;
        }
        int above = incl - mine;
        if (above < want && want <= incl) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (above < want && want <= above + bins[u]) {
              s_pick[0] = 255 - 8 * lane - u;
              s_pick[1] = want - above;
            }
            above += bins[u];
          }
        }
      }
      __syncthreads();
      limit |= static_cast<uint32_t>(s_pick[0]) << shift;
      want = s_pick[1];
    }
  }

  // The list: a thread takes a run of pages; places by prefix sums of what is taken
  // above the limit and of what is equal to it.
  const int per = (pages + kThreads - 1) / kThreads;
  const int p0 = min(tid * per, pages), p1 = min(p0 + per, pages);
  int above = 0, equal = 0;
  for (int i = p0; i < p1; ++i) {
    above += s_key[i] > limit ? 1 : 0;
    equal += s_key[i] == limit ? 1 : 0;
  }
  int all_above = 0, all_equal = 0;
  above = prefix_sum<kThreads>(above, scratch, all_above);
  equal = prefix_sum<kThreads>(equal, scratch, all_equal);
  for (int i = p0; i < p1; ++i) {
    const uint32_t key = s_key[i];
    const bool take = key > limit || (key == limit && equal < want);
    const int place = above + min(equal, want);
    if (take && place < p.cap) out[place] = i;
    above += key > limit ? 1 : 0;
    equal += key == limit ? 1 : 0;
  }
  const int total = min(all_above + min(all_equal, want), p.cap);
  for (int i = total + tid; i < p.cap; i += kThreads) out[i] = -1;
  if (tid == 0) p.counts[static_cast<long long>(blockIdx.x) * p.heads_kv + hk] = total;
}

}  // namespace sel

// Checks of the tables of an entry point that has no K and V pools.
static int make_tables(Cache* c, const char* fn, const int32_t* page_table, const int32_t* seq_lens, int batch,
                       int heads_kv, int head_dim, int num_pages, int page_size, int max_pages, int64_t table_stride,
                       int dtype) {
  const int64_t st[3] = {kD, kD, kD};
  const void* none = reinterpret_cast<const void*>(16);  // aligned, never read
  return make_cache(c, fn, none, none, page_table, seq_lens, batch, heads_kv, head_dim, num_pages, page_size,
                    max_pages, st, st, table_stride, dtype);
}

static int check_means(const char* fn, const void* means, const int64_t* m) {
  if (!means || !m) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  if (!aligned16(means) || m[0] % 4 != 0 || m[1] % 4 != 0 || m[0] <= 0 || m[1] <= 0)
    return sabre_fail(SABRE_ERR_ALIGNMENT,
                      "%s: key_means must be 16-byte aligned with strides that are positive multiples of 4", fn);
  return SABRE_OK;
}

// Row tiles that `rows` rows of `batch` sequences need at most: a sequence of
// l > 0 rows takes (l - 1) / tokens + 1.
static inline long long row_slots(int rows, int batch, int tokens) {
  const int k = rows < batch ? rows : batch;
  return static_cast<long long>(rows - k) / tokens + k;
}

}  // namespace paged
}  // namespace sabre

extern "C" {

int sabre_paged_key_means(const void* k_pages, float* key_means, const int32_t* page_table, const int32_t* seq_lens,
                          const int32_t* q_start, int rows, int batch, int heads_kv, int head_dim, int num_pages,
                          int page_size, int max_pages, const int64_t* kp_strides, const int64_t* km_strides,
                          int64_t table_stride, int dtype, void* stream) {
  using namespace sabre::paged;
  const char* fn = "sabre_paged_key_means";
  means::Params p;
  int st = make_cache(&p.c, fn, k_pages, k_pages, page_table, seq_lens, batch, heads_kv, head_dim, num_pages,
                      page_size, max_pages, kp_strides, kp_strides, table_stride, dtype);
  if (st == SABRE_OK) st = check_means(fn, key_means, km_strides);
  if (st != SABRE_OK) return st;
  if (rows <= 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: rows must be positive", fn);
  if (!q_start && rows != batch)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: %d rows for %d sequences need q_start", fn, rows, batch);
  p.k = k_pages;
  p.means = key_means;
  p.starts = q_start;
  p.m_sp = km_strides[0];
  p.m_sh = km_strides[1];
  p.rows = rows;
  p.heads = heads_kv;
  // l new rows fill at most (l - 1) / page_size + 1 pages.
  const int warps = heads_kv < means::kMaxWarps ? heads_kv : means::kMaxWarps;
  const dim3 grid(static_cast<unsigned>(row_slots(rows, batch, page_size)), (heads_kv + warps - 1) / warps);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      dtype == SABRE_BF16
          ? launch_dependent(grid, warps * 32, 0, s, means::paged_key_means_kernel<__nv_bfloat16>, p)
          : launch_dependent(grid, warps * 32, 0, s, means::paged_key_means_kernel<__half>, p);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

int sabre_paged_select_width(int page_size, int max_pages, int topk, int query_block, int window,
                             int num_prefix_tokens) {
  if (page_size <= 0 || max_pages <= 0 || topk < 0 || query_block <= 0 || window < 0 || num_prefix_tokens < 0)
    return 0;
  const long long ps = page_size;
  // A span of s tokens touches (s + ps - 2) / ps + 1 pages at most.
  const long long width = topk + (num_prefix_tokens + ps - 1) / ps + (0ll + window + query_block + ps - 2) / ps + 1;
  return static_cast<int>(width < max_pages ? width : max_pages);
}

int sabre_paged_query_blocks(int rows, int batch, int query_block) {
  if (rows <= 0 || batch <= 0 || query_block <= 0) return 0;
  return static_cast<int>(sabre::paged::row_slots(rows, batch, query_block));
}

int sabre_paged_select(const void* q, const float* key_means, const int32_t* page_table, const int32_t* seq_lens,
                       const int32_t* q_start, int32_t* lists, int32_t* counts, int rows, int batch, int heads_q,
                       int heads_kv, int head_dim, int num_pages, int page_size, int max_pages, int topk,
                       int query_block, int window, int num_prefix_tokens, const int64_t* q_strides,
                       const int64_t* km_strides, int64_t table_stride, int dtype, void* stream) {
  using namespace sabre::paged;
  const char* fn = "sabre_paged_select";
  sel::Params p;
  int st = make_tables(&p.c, fn, page_table, seq_lens, batch, heads_kv, head_dim, num_pages, page_size, max_pages,
                       table_stride, dtype);
  if (st == SABRE_OK) st = check_means(fn, key_means, km_strides);
  if (st != SABRE_OK) return st;
  if (!q || !lists || !counts || !q_strides) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  if (rows <= 0 || heads_q <= 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: sizes must be positive", fn);
  if (heads_q % heads_kv != 0)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: heads_q/heads_kv must be an integer", fn);
  if (topk < 0 || query_block <= 0 || query_block > 1024 || window < 0 || num_prefix_tokens < 0)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: topk %d, query_block %d, window %d, num_prefix_tokens %d", fn, topk,
                      query_block, window, num_prefix_tokens);
  if (!q_start && (rows != batch || query_block != 1))
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: %d rows for %d sequences in blocks of %d need q_start", fn, rows,
                      batch, query_block);
  if (max_pages > sel::kMaxPages)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: a table of %d columns (at most %d)", fn, max_pages, sel::kMaxPages);
  if (!aligned16(q) || q_strides[0] % 8 != 0 || q_strides[1] % 8 != 0)
    return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: q must be 16-byte aligned with strides in multiples of 8 elements",
                      fn);
  p.q = q;
  p.means = key_means;
  p.starts = q_start;
  p.lists = lists;
  p.counts = counts;
  p.q_sr = q_strides[0];
  p.q_sh = q_strides[1];
  p.m_sp = km_strides[0];
  p.m_sh = km_strides[1];
  p.rows = rows;
  p.heads_kv = heads_kv;
  p.group = heads_q / heads_kv;
  p.tokens = query_block;
  p.topk = topk;
  p.window = window;
  p.prefix = num_prefix_tokens;
  p.cap = sabre_paged_select_width(page_size, max_pages, topk, query_block, window, num_prefix_tokens);
  const int smem = max_pages * static_cast<int>(sizeof(uint32_t));
  const auto kernel =
      dtype == SABRE_BF16 ? sel::paged_select_kernel<__nv_bfloat16> : sel::paged_select_kernel<__half>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       sel::kMaxPages * static_cast<int>(sizeof(uint32_t)));
  if (e != cudaSuccess) return sabre_cuda_fail(e, fn);
  e = launch_dependent(dim3(static_cast<unsigned>(row_slots(rows, batch, query_block)), heads_kv), sel::kThreads, smem,
                       static_cast<cudaStream_t>(stream), kernel, p);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

}  // extern "C"
