// Paged K/V cache: the layout every paged kernel shares, the store of new
// rows into pages, and copies of whole pages.
//
// A pool holds num_pages pages of page_size rows for each KV head,
// [num_pages, Hkv, page_size, D] with any strides; row t of sequence b lives in
// page page_table[b][t / page_size] at row t % page_size. A table entry of -1
// means the page is absent: its rows are not stored and not visible. Any other
// entry outside [0, num_pages) is treated the same way and recorded as
// SABRE_DEV_BAD_PAGE. Included by sabre_capi.cu after its host helpers.

namespace sabre {
namespace paged {

constexpr int kD = 128;
constexpr int kMaxRows = 1 << 30;  // page_size * max_pages: positions stay in int32

// The pool and the sequences' page tables, as the kernels see them. Page
// sizes are powers of two, so a position splits with a shift and a mask.
struct Cache {
  const int32_t* table;
  const int32_t* seq_lens;
  long long table_sb;
  long long k_sp, k_sh, k_st;  // element strides {page, head, row}
  long long v_sp, v_sh, v_st;
  int batch, num_pages, max_pages, page_shift;

  __device__ __forceinline__ int capacity() const { return max_pages << page_shift; }
  __device__ __forceinline__ int length(int b) const { return min(max(seq_lens[b], 0), capacity()); }
  // Table entry of a position below capacity().
  __device__ __forceinline__ int entry(int b, int pos) const { return table[b * table_sb + (pos >> page_shift)]; }
  // The entry as a page of the pool, or -1: absent.
  __device__ __forceinline__ int checked(int page) const {
    if (page < -1 || page >= num_pages) record_status(SABRE_DEV_BAD_PAGE);
    return page >= 0 && page < num_pages ? page : -1;
  }
  __device__ __forceinline__ int page_of(int b, int pos) const { return checked(entry(b, pos)); }
};

// Key j < n is visible to the query at position i when j <= i and (no window,
// i - j <= window, or j < prefix).
struct Window {
  int window, prefix;  // window < 0: none
  // First position inside the window of query i (0 for a row before its sequence,
  // i < 0, which sees nothing: i - window could pass the end of int32).
  __device__ __forceinline__ int first(int i) const { return window < 0 ? 0 : max(0, max(i, 0) - window); }
};

// First row of sequence b in a ragged batch of `rows` rows (one row each
// without starts). Clamped, so that no start reaches past the rows.
__device__ __forceinline__ int row_start(const int32_t* starts, int b, int rows) {
  return starts ? min(max(starts[b], 0), rows) : min(b, rows);
}

// ---------------------------------------------------------------------------
// store
//
// Moves 512 bytes per KV head and row, no arithmetic: bound by HBM, and by the
// launch and three dependent loads (starts, length, page) for a few rows. A
// warp finds the sequence of one row by counting the starts at or before it,
// 32 at a time; a thread then moves the same 16 bytes of eight rows, all eight
// loads in flight.
// ---------------------------------------------------------------------------
constexpr int kStoreThreads = 256;
constexpr int kStoreBatch = 8;                                // rows of a thread at a time
constexpr int kStoreMaxRows = kStoreBatch * kStoreThreads / 32;  // of a CTA, one KV head

struct StoreParams {
  Cache c;
  const uint4* k;
  const uint4* v;
  uint4* kp;
  uint4* vp;
  const int32_t* starts;
  long long k_sr, k_sh, v_sr, v_sh;  // strides of the rows, in 16-byte units
  int rows, heads, cta_rows;
};

__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const StoreParams p) {
  __shared__ int s_page[kStoreMaxRows], s_off[kStoreMaxRows];
  const int r0 = blockIdx.x * p.cta_rows;
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  // The next kernel (a decode over these pages, say) may start its set-up now;
  // it waits for this grid before touching memory.
  if (tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // a programmatic dependent launch: inputs are ready from here on
  for (int r = tid >> 5; r < p.cta_rows; r += kStoreThreads / 32) {
    const int row = r0 + r;
    int page = -1, off = 0;
    // Sequence b: start(b) <= row < start(b + 1).
    int b = -1;
    if (row < p.rows) {
      if (!p.starts) {
        b = row;
      } else {
        int before = 0;  // starts at or before the row
        for (int i = lane; i <= p.c.batch; i += 32) before += p.starts[i] <= row ? 1 : 0;
        before = __reduce_add_sync(0xffffffffu, before);
        b = before <= p.c.batch ? before - 1 : -1;
      }
    }
    if (b >= 0) {
      const int pos = p.c.seq_lens[b] - (row_start(p.starts, b + 1, p.rows) - row);
      if (pos >= 0 && pos < p.c.capacity()) {
        page = p.c.page_of(b, pos);
        off = pos & ((1 << p.c.page_shift) - 1);
      } else {
        record_status(SABRE_DEV_BAD_PAGE);
      }
    }
    if (lane == 0) {
      s_page[r] = page;
      s_off[r] = off;
    }
  }
  __syncthreads();
  // 16 threads move one head's row of K or V (256 bytes).
  const int units = p.heads * 32;
  for (int i = tid; i < units * (p.cta_rows / kStoreBatch); i += kStoreThreads) {
    const int rb = i / units * kStoreBatch;
    const int u = i % units;
    const int h = u >> 5;
    const int ch = u & 15;
    const bool is_v = (u & 16) != 0;
    const uint4* src = (is_v ? p.v + h * p.v_sh : p.k + h * p.k_sh) + ch;
    uint4* dst = (is_v ? p.vp + h * p.c.v_sh : p.kp + h * p.c.k_sh) + ch;
    const long long sr = is_v ? p.v_sr : p.k_sr;
    const long long sp = is_v ? p.c.v_sp : p.c.k_sp;
    const long long st = is_v ? p.c.v_st : p.c.k_st;
    uint4 x[kStoreBatch];
#pragma unroll
    for (int r = 0; r < kStoreBatch; ++r)
      if (s_page[rb + r] >= 0) x[r] = src[(r0 + rb + r) * sr];
#pragma unroll
    for (int r = 0; r < kStoreBatch; ++r)
      if (s_page[rb + r] >= 0) dst[s_page[rb + r] * sp + s_off[rb + r] * st] = x[r];
  }
}

// ---------------------------------------------------------------------------
// copy of whole pages
// ---------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyMoves = 480;  // pairs carried in one launch's arguments

struct CopyParams {
  uint4* base;
  long long buffer_stride, page_stride, page_units;  // in 16-byte units
  int32_t src[kCopyMoves];
  int32_t dst[kCopyMoves];
};

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  const int m = blockIdx.y;
  uint4* buf = p.base + blockIdx.z * p.buffer_stride;
  const uint4* src = buf + p.src[m] * p.page_stride;
  uint4* dst = buf + p.dst[m] * p.page_stride;
  const long long i0 = static_cast<long long>(blockIdx.x) * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  uint4 x[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i0 + u * kCopyThreads < p.page_units) x[u] = src[i0 + u * kCopyThreads];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i0 + u * kCopyThreads < p.page_units) dst[i0 + u * kCopyThreads] = x[u];
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Launches a programmatic dependent of the stream's previous kernel: its
// set-up may overlap that kernel's tail; it must execute griddepcontrol.wait
// before it touches memory.
template <typename K, typename... A>
static cudaError_t launch_dependent(dim3 grid, int threads, int smem, cudaStream_t s, K kernel, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Checks shared by the paged entry points; fills c. `kp` / `vp` strides are
// {page, head, row} in elements.
static int make_cache(Cache* c, const char* fn, const void* k_pages, const void* v_pages, const int32_t* page_table,
                      const int32_t* seq_lens, int batch, int heads_kv, int head_dim, int num_pages, int page_size,
                      int max_pages, const int64_t* kp, const int64_t* vp, int64_t table_stride, int dtype) {
  if (!k_pages || !v_pages || !page_table || !seq_lens || !kp || !vp)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  if (batch <= 0 || heads_kv <= 0 || num_pages <= 0 || page_size <= 0 || max_pages <= 0)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: sizes must be positive", fn);
  if (head_dim != kD) return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: head_dim %d (only 128)", fn, head_dim);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: page_size %d (a power of two from 16 to 1024)", fn, page_size);
  if (static_cast<long long>(page_size) * max_pages > kMaxRows)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: page_size * max_pages exceeds 2^30 rows", fn);
  if (heads_kv > 4096) return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: heads_kv %d > 4096", fn, heads_kv);
  if (dtype != SABRE_BF16 && dtype != SABRE_F16) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: dtype %d", fn, dtype);
  if (!aligned16(k_pages) || !aligned16(v_pages))
    return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: k_pages/v_pages must be 16-byte aligned", fn);
  for (int i = 0; i < 3; ++i)
    if (kp[i] <= 0 || vp[i] <= 0 || kp[i] % 8 != 0 || vp[i] % 8 != 0)
      return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: page strides must be positive multiples of 8 elements", fn);
  if (table_stride < (batch > 1 ? max_pages : 0))
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: page_table rows overlap (stride %lld < %d)", fn,
                      static_cast<long long>(table_stride), max_pages);
  c->table = page_table;
  c->seq_lens = seq_lens;
  c->table_sb = table_stride;
  c->k_sp = kp[0];
  c->k_sh = kp[1];
  c->k_st = kp[2];
  c->v_sp = vp[0];
  c->v_sh = vp[1];
  c->v_st = vp[2];
  c->batch = batch;
  c->num_pages = num_pages;
  c->max_pages = max_pages;
  c->page_shift = 0;
  while ((1 << c->page_shift) < page_size) ++c->page_shift;
  return SABRE_OK;
}

}  // namespace paged
}  // namespace sabre

extern "C" {

int sabre_paged_store(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* page_table,
                      const int32_t* seq_lens, const int32_t* q_start, int rows, int batch, int heads_kv,
                      int head_dim, int num_pages, int page_size, int max_pages, const int64_t* k_strides,
                      const int64_t* v_strides, const int64_t* kp_strides, const int64_t* vp_strides,
                      int64_t table_stride, int dtype, void* stream) {
  using namespace sabre::paged;
  if (!k || !v || !k_strides || !v_strides)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_paged_store: null pointer argument");
  StoreParams p;
  const int st = make_cache(&p.c, "sabre_paged_store", k_pages, v_pages, page_table, seq_lens, batch, heads_kv,
                            head_dim, num_pages, page_size, max_pages, kp_strides, vp_strides, table_stride, dtype);
  if (st != SABRE_OK) return st;
  if (rows <= 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_paged_store: rows must be positive");
  if (!q_start && rows != batch)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_paged_store: %d rows for %d sequences need q_start", rows, batch);
  if (!aligned16(k) || !aligned16(v))
    return sabre_fail(SABRE_ERR_ALIGNMENT, "sabre_paged_store: k/v must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return sabre_fail(SABRE_ERR_ALIGNMENT, "sabre_paged_store: k/v strides must be multiples of 8 elements");
  long long* s[6] = {&p.c.k_sp, &p.c.k_sh, &p.c.k_st, &p.c.v_sp, &p.c.v_sh, &p.c.v_st};
  for (int i = 0; i < 6; ++i) *s[i] /= 8;
  p.k = static_cast<const uint4*>(k);
  p.v = static_cast<const uint4*>(v);
  p.kp = static_cast<uint4*>(k_pages);
  p.vp = static_cast<uint4*>(v_pages);
  p.starts = q_start;
  p.k_sr = k_strides[0] / 8;
  p.k_sh = k_strides[1] / 8;
  p.v_sr = v_strides[0] / 8;
  p.v_sh = v_strides[1] / 8;
  p.rows = rows;
  p.heads = heads_kv;
  // Eight rows of every head fill the threads from eight heads on; with fewer
  // a CTA takes more rows.
  p.cta_rows = kStoreBatch * (heads_kv < 8 ? 8 / heads_kv : 1);
  const cudaError_t e = launch_dependent(dim3((rows + p.cta_rows - 1) / p.cta_rows), kStoreThreads, 0,
                                         static_cast<cudaStream_t>(stream), paged_store_kernel, p);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, "sabre_paged_store launch");
}

int sabre_copy_pages(void* pages, int buffers, int64_t buffer_stride, int num_pages, int64_t page_stride,
                     int64_t page_bytes, const int32_t* src, const int32_t* dst, int moves, void* stream) {
  using namespace sabre::paged;
  if (!pages || (moves > 0 && (!src || !dst)))
    return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_copy_pages: null pointer argument");
  if (buffers <= 0 || num_pages <= 0 || page_bytes <= 0 || moves < 0)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_copy_pages: sizes must be positive");
  if (buffers > 65535) return sabre_fail(SABRE_ERR_UNSUPPORTED, "sabre_copy_pages: buffers %d > 65535", buffers);
  if (!aligned16(pages) || page_bytes % 16 != 0 || page_stride % 16 != 0 || buffer_stride % 16 != 0)
    return sabre_fail(SABRE_ERR_ALIGNMENT, "sabre_copy_pages: pages and their strides must be 16-byte multiples");
  if ((num_pages > 1 && page_stride < page_bytes) || (buffers > 1 && buffer_stride < page_bytes))
    return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_copy_pages: pages overlap");
  // Pages are copied in no order, so none may be written twice or be written
  // while another move reads it.
  unsigned char* use = static_cast<unsigned char*>(calloc(num_pages, 1));
  if (!use) return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_copy_pages: out of host memory");
  const char* bad = nullptr;
  int at = 0;
  for (int i = 0; i < moves && !bad; ++i) {
    at = i;
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
      bad = "outside the pool";
    else if (use[dst[i]] & 2)
      bad = "written twice";
    else
      use[src[i]] |= 1, use[dst[i]] |= 2;
  }
  for (int i = 0; i < moves && !bad; ++i) {
    at = i;
    if (use[src[i]] & 2) bad = "read and written";
  }
  free(use);
  if (bad)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_copy_pages: move %d (%d -> %d): a page is %s", at, src[at],
                      dst[at], bad);
  CopyParams p;
  p.base = static_cast<uint4*>(pages);
  p.buffer_stride = buffer_stride / 16;
  p.page_stride = page_stride / 16;
  p.page_units = page_bytes / 16;
  const long long chunks = (p.page_units + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll);
  if (chunks > 0x7fffffffll) return sabre_fail(SABRE_ERR_UNSUPPORTED, "sabre_copy_pages: page too large");
  for (int m0 = 0; m0 < moves; m0 += kCopyMoves) {
    const int n = moves - m0 < kCopyMoves ? moves - m0 : kCopyMoves;
    memcpy(p.src, src + m0, n * sizeof(int32_t));
    memcpy(p.dst, dst + m0, n * sizeof(int32_t));
    copy_pages_kernel<<<dim3(static_cast<unsigned>(chunks), n, buffers), kCopyThreads, 0,
                        static_cast<cudaStream_t>(stream)>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return sabre_cuda_fail(e, "sabre_copy_pages launch");
  }
  return SABRE_OK;
}

}  // extern "C"
