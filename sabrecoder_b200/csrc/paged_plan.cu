// Block tables and slot maps of a paged cache, built on the device from request
// lengths: a step that makes room for its own rows can be captured whole.
//
// Sequence b goes from len_b to len_b + new_b rows and owns ceil(. / page_size)
// pages before and after; the i-th page that the batch needs (by sequence, then
// position) is free_pages[free_count - 1 - i]. Row r of sequence b (its rows
// follow those of the sequences before it) is at position pos = len_b + r -
// q_start[b], in slot table[b][pos / page_size] * page_size + pos % page_size.
//
// Reads 8 bytes a sequence and writes 16 a row: a call is bound by its launch and by
// the chain lengths -> prefix sums -> table or free page -> slot. One CTA plans: it sums
// the batch (in shared memory, so that rows and pages find their sequence by
// bisection), hands out the pages and, when they are few, places the rows. Many rows
// are placed by a second kernel over the whole card, from the new tables and lengths:
// 62600 rows of 16 sequences take 10.9 us in a cluster of eight CTAs, which writes 125
// KB an SM, and 7.2 so; 64 rows 3.7 in the cluster, 2.8 in one CTA.
namespace sabre {
namespace paged {
namespace plan {

constexpr int kThreads = 1024;    // 256 for small calls, which start and scan sooner
constexpr int kMaxBatch = 16384;  // three ints of shared memory a sequence
constexpr int kOwnRows = 2048;    // rows that the planning CTA places itself
constexpr int kRowThreads = 256;
constexpr int kRowFlight = 4;     // rows of a thread, their look-ups on the way together

struct Params {
  const int32_t* fresh;  // new rows of each sequence
  const int32_t* lens;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* table;
  int32_t* lens_out;
  int32_t* count_out;
  int32_t* q_start;
  long long* slots;
  long long* positions;
  long long table_sb;
  int batch, page_shift, num_pages, free_size, rows;
  int limit;  // rows of a sequence at most

  __device__ __forceinline__ int page(int id) const {  // a page of the pool, or -1
    if (id < -1 || id >= num_pages) record_status(SABRE_DEV_BAD_PAGE);
    return id >= 0 && id < num_pages ? id : -1;
  }
};

// Inclusive sums over the CTA of two counts at once, and their totals. scratch: two
// counts a warp.
__device__ __forceinline__ void scan2(long long& a, long long& b, longlong2* scratch, long long& all_a,
                                      long long& all_b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  auto scan = [&](long long& x, long long& y) {
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long ux = __shfl_up_sync(0xffffffffu, x, s), uy = __shfl_up_sync(0xffffffffu, y, s);
      if (lane >= s) x += ux, y += uy;
    }
  };
  scan(a, b);
  if (lane == 31) scratch[warp] = make_longlong2(a, b);
  __syncthreads();
  longlong2 sum = lane < warps ? scratch[lane] : make_longlong2(0, 0);
  scan(sum.x, sum.y);
  all_a = __shfl_sync(0xffffffffu, sum.x, 31);
  all_b = __shfl_sync(0xffffffffu, sum.y, 31);
  const long long before_a = __shfl_sync(0xffffffffu, sum.x, max(warp - 1, 0));
  const long long before_b = __shfl_sync(0xffffffffu, sum.y, max(warp - 1, 0));
  if (warp > 0) a += before_a, b += before_b;
}

// The last i in [0, n) with first[i] <= x; first ascends from first[0] <= x.
__device__ __forceinline__ int last_at(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (first[mid] <= x ? lo : hi) = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) paged_extend_kernel(const Params p) {
  extern __shared__ int s_seq[];  // [3][batch]: rows and pages before the sequence, its old length
  __shared__ longlong2 s_scan[kThreads / 32];
  int* const s_rows = s_seq;
  int* const s_pages = s_seq + p.batch;
  int* const s_len = s_seq + 2 * p.batch;
  const int tid = threadIdx.x;
  if (tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int ps1 = (1 << p.page_shift) - 1;
  auto have = [&](int len) -> int { return (len + ps1) >> p.page_shift; };

  const int threads = blockDim.x;
  const int per = (p.batch + threads - 1) / threads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  const int count = *p.free_count;
  long long rows = 0, pages = 0;
  bool bad = count < 0 || count > p.free_size;
  for (int b = b0; b < b1; ++b) {
    const int len = p.lens[b], fresh = p.fresh[b];
    // Refused below, with nothing of it used.
    if (len < 0 || fresh < 0 || static_cast<long long>(len) + fresh > p.limit) {
      bad = true;
      continue;
    }
    s_len[b] = len;
    s_rows[b] = fresh;
    rows += fresh;
    pages += have(len + fresh) - have(len);
  }
  long long row = rows, pg = pages, all_rows, all_pages;
  scan2(row, pg, s_scan, all_rows, all_pages);
  bad = __syncthreads_or(bad) != 0;
  // A call that does not fit changes nothing and has no rows.
  bad = bad || all_pages > count || all_rows > p.rows;
  const int total = bad ? 0 : static_cast<int>(all_rows), need = bad ? 0 : static_cast<int>(all_pages);
  row -= rows;
  pg -= pages;
  for (int b = b0; b < b1; ++b) {
    const int fresh = bad ? 0 : s_rows[b];
    const int len = bad ? p.lens[b] : s_len[b];
    p.q_start[b] = bad ? 0 : static_cast<int>(row);
    p.lens_out[b] = len + fresh;
    if (bad) continue;
    s_rows[b] = static_cast<int>(row);
    s_pages[b] = static_cast<int>(pg);
    row += fresh;
    pg += have(len + fresh) - have(len);
  }
  if (tid == 0) {
    if (bad) record_status(SABRE_DEV_NO_ROOM);
    p.q_start[p.batch] = total;
    *p.count_out = count - need;  // every thread has read it: barriers above
  }
  __syncthreads();
  if (p.rows <= kOwnRows)
    for (int r = tid; r < p.rows; r += threads) {
      long long slot = -1, pos = 0;
      if (r < total) {
        const int b = last_at(s_rows, p.batch, r);
        const int at = s_len[b] + r - s_rows[b];
        const int col = at >> p.page_shift, new_col = col - have(s_len[b]);
        const int id =
            p.page(new_col < 0 ? p.table[b * p.table_sb + col] : p.free_pages[count - 1 - s_pages[b] - new_col]);
        pos = at;
        if (id >= 0) slot = (static_cast<long long>(id) << p.page_shift) + (at & ps1);
      }
      p.slots[r] = slot;
      p.positions[r] = pos;
    }
  // Columns that no row's look-up above reads.
  for (int i0 = tid; i0 < need; i0 += 4 * threads) {
    int id[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) id[u] = i0 + u * threads < need ? p.free_pages[count - 1 - i0 - u * threads] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * threads;
      if (i >= need) break;
      const int b = last_at(s_pages, p.batch, i);
      p.table[b * p.table_sb + have(s_len[b]) + i - s_pages[b]] = p.page(id[u]);
    }
  }
}

// Slots and positions of a plan's rows.
__global__ void __launch_bounds__(kRowThreads) paged_slots_kernel(const Params p) {
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int total = p.q_start[p.batch];
  const int r0 = blockIdx.x * (kRowThreads * kRowFlight) + threadIdx.x;
  int id[kRowFlight], at[kRowFlight];
#pragma unroll
  for (int u = 0; u < kRowFlight; ++u) {
    const int r = r0 + u * kRowThreads;
    id[u] = -1;
    at[u] = 0;
    if (r < total) {
      const int b = last_at(p.q_start, p.batch, r);
      at[u] = p.lens_out[b] - (p.q_start[b + 1] - r);
      id[u] = p.table[b * p.table_sb + (at[u] >> p.page_shift)];
    }
  }
#pragma unroll
  for (int u = 0; u < kRowFlight; ++u) {
    const int r = r0 + u * kRowThreads;
    if (r >= p.rows) break;
    const int pg = p.page(id[u]);
    p.slots[r] = pg < 0 ? -1 : (static_cast<long long>(pg) << p.page_shift) + (at[u] & ((1 << p.page_shift) - 1));
    p.positions[r] = at[u];
  }
}

}  // namespace plan

// Both entries; max_len: rows of a sequence at most, or -1: as many as its table row holds.
static int extend_call(const char* fn, const int32_t* new_rows, int32_t* page_table, const int32_t* seq_lens,
                       int32_t* seq_lens_out, const int32_t* free_pages, const int32_t* free_count,
                       int32_t* free_count_out, int32_t* q_start, int64_t* slots, int64_t* positions, int rows,
                       int batch, int num_pages, int page_size, int max_pages, int free_size, int max_len,
                       int64_t table_stride, void* stream) {
  if (!new_rows || !page_table || !seq_lens || !seq_lens_out || !free_count || !free_count_out || !q_start ||
      (free_size > 0 && !free_pages) || (rows > 0 && (!slots || !positions)))
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  if (new_rows == seq_lens_out)  // the rows are placed by both
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: new_rows and seq_lens_out are the same", fn);
  if (rows < 0 || batch <= 0 || num_pages <= 0 || max_pages <= 0 || free_size < 0)
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: sizes must be positive", fn);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: page_size %d (a power of two from 16 to 1024)", fn, page_size);
  if (static_cast<long long>(page_size) * max_pages > kMaxRows)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: page_size * max_pages exceeds 2^30 rows", fn);
  if (batch > plan::kMaxBatch)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: %d sequences (at most %d)", fn, batch, plan::kMaxBatch);
  if (table_stride < (batch > 1 ? max_pages : 0))
    return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: page_table rows overlap (stride %lld < %d)", fn,
                      static_cast<long long>(table_stride), max_pages);
  if (rows > 1 << 30) return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: more than 2^30 rows", fn);
  plan::Params p;
  p.fresh = new_rows;
  p.lens = seq_lens;
  p.free_pages = free_pages;
  p.free_count = free_count;
  p.table = page_table;
  p.lens_out = seq_lens_out;
  p.count_out = free_count_out;
  p.q_start = q_start;
  p.slots = reinterpret_cast<long long*>(slots);
  p.positions = reinterpret_cast<long long*>(positions);
  p.table_sb = table_stride;
  p.batch = batch;
  p.limit = page_size * max_pages;
  if (max_len >= 0 && max_len < p.limit) p.limit = max_len;
  p.page_shift = 0;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.num_pages = num_pages;
  p.free_size = free_size;
  p.rows = rows;
  const int smem = 3 * batch * static_cast<int>(sizeof(int));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (smem > 47 * 1024)
    e = cudaFuncSetAttribute(plan::paged_extend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             3 * plan::kMaxBatch * static_cast<int>(sizeof(int)));
  const int threads = batch <= 1024 && rows <= 1024 ? 256 : plan::kThreads;
  if (e == cudaSuccess) e = launch_dependent(dim3(1), threads, smem, st, plan::paged_extend_kernel, p);
  constexpr int kCtaRows = plan::kRowThreads * plan::kRowFlight;
  if (e == cudaSuccess && rows > plan::kOwnRows)
    e = launch_dependent(dim3((rows + kCtaRows - 1) / kCtaRows), plan::kRowThreads, 0, st, plan::paged_slots_kernel, p);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

}  // namespace paged
}  // namespace sabre

extern "C" {

int sabre_paged_extend(const int32_t* new_rows, int32_t* page_table, const int32_t* seq_lens, int32_t* seq_lens_out,
                       const int32_t* free_pages, const int32_t* free_count, int32_t* free_count_out,
                       int32_t* q_start, int64_t* slots, int64_t* positions, int rows, int batch, int num_pages,
                       int page_size, int max_pages, int free_size, int64_t table_stride, void* stream) {
  return sabre::paged::extend_call("sabre_paged_extend", new_rows, page_table, seq_lens, seq_lens_out, free_pages,
                                   free_count, free_count_out, q_start, slots, positions, rows, batch, num_pages,
                                   page_size, max_pages, free_size, -1, table_stride, stream);
}

int sabre_paged_extend_within(const int32_t* new_rows, int32_t* page_table, const int32_t* seq_lens,
                              int32_t* seq_lens_out, const int32_t* free_pages, const int32_t* free_count,
                              int32_t* free_count_out, int32_t* q_start, int64_t* slots, int64_t* positions, int rows,
                              int batch, int num_pages, int page_size, int max_pages, int free_size, int max_len,
                              int64_t table_stride, void* stream) {
  const char* fn = "sabre_paged_extend_within";
  if (max_len < 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: max_len must not be negative", fn);
  return sabre::paged::extend_call(fn, new_rows, page_table, seq_lens, seq_lens_out, free_pages, free_count,
                                   free_count_out, q_start, slots, positions, rows, batch, num_pages, page_size,
                                   max_pages, free_size, max_len, table_stride, stream);
}

}  // extern "C"
