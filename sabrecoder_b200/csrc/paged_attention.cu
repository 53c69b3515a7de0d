// Attention over a paged K/V cache, simplest form: one CTA per (row, query
// head), four warps that take every fourth key with an online softmax each and
// join through shared memory. Serves one new token per sequence
// (sabre_paged_decode) and ragged batches of rows (sabre_paged_prefill).
namespace sabre {
namespace paged {

struct AttnParams {
  Cache c;
  Window w;
  const void* q;
  const void* kp;
  const void* vp;
  void* o;
  const int32_t* starts;  // null: one row per sequence
  long long q_sr, q_sh, o_sr, o_sh;
  int rows, heads_q, heads_kv;
  float scale_log2;
};

template <typename T>
__global__ void __launch_bounds__(128) paged_rows_kernel(const AttnParams p) {
  const int row = blockIdx.x;
  const int h = blockIdx.y;
  const int hk = h / (p.heads_q / p.heads_kv);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int b = sequence_of(p.starts, p.c.batch, p.rows, row);
  if (b < 0) return;
  const int n = p.c.length(b);
  const int i = p.c.seq_lens[b] - (row_start(p.starts, b + 1, p.rows) - row);
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    q[e] = DT<T>::to_f(static_cast<const T*>(p.q)[row * p.q_sr + h * p.q_sh + lane * 4 + e]) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  const int lo = p.w.first(i);
  for (int j = warp; j <= i && j < n; j += 4) {
    if (j < lo && j >= p.w.prefix) continue;
    const int page = p.c.page_of(b, j);
    if (page < 0) continue;
    const int off = j & ((1 << p.c.page_shift) - 1);
    const T* kr = static_cast<const T*>(p.kp) + page * p.c.k_sp + hk * p.c.k_sh + off * p.c.k_st + lane * 4;
    const T* vr = static_cast<const T*>(p.vp) + page * p.c.v_sp + hk * p.c.v_sh + off * p.c.v_st + lane * 4;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(q[e], DT<T>::to_f(kr[e]), s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    if (mn == -INFINITY) continue;
    const float a = ex2(m - mn), w = ex2(s - mn);
    l = l * a + w;
    m = mn;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * a + w * DT<T>::to_f(vr[e]);
  }
  __shared__ float sm[4], sl[4], sa[4][kD];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sa[warp][lane * 4 + e] = acc[e];
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float L = 0.f, A = 0.f;
  if (M != -INFINITY)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float w = ex2(sm[r] - M);
      L += w * sl[r];
      A += w * sa[r][threadIdx.x];
    }
  static_cast<T*>(p.o)[row * p.o_sr + h * p.o_sh + threadIdx.x] = DT<T>::from_f(L > 0.f ? A / L : 0.f);
}

static int attend(const char* fn, const void* q, const void* k_pages, const void* v_pages, void* o,
                  const int32_t* page_table, const int32_t* seq_lens, const int32_t* q_start, int rows, int batch,
                  int heads_q, int heads_kv, int head_dim, int num_pages, int page_size, int max_pages, int window,
                  int prefix, const int64_t* q_strides, const int64_t* kp_strides, const int64_t* vp_strides,
                  const int64_t* o_strides, int64_t table_stride, float softmax_scale, int dtype, void* stream) {
  if (!q || !o || !q_strides || !o_strides) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  AttnParams p;
  const int st = make_cache(&p.c, fn, k_pages, v_pages, page_table, seq_lens, batch, heads_kv, head_dim, num_pages,
                            page_size, max_pages, kp_strides, vp_strides, table_stride, dtype);
  if (st != SABRE_OK) return st;
  if (rows <= 0 || heads_q <= 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: sizes must be positive", fn);
  if (heads_q % heads_kv != 0 || heads_q / heads_kv > 8)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: heads_q/heads_kv must be an integer <= 8", fn);
  if (prefix < 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: num_prefix_tokens %d < 0", fn, prefix);
  if (!aligned16(q) || !aligned16(o)) return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: q/o must be 16-byte aligned", fn);
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] % 8 != 0 || o_strides[i] % 8 != 0)
      return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: q/o strides must be multiples of 8 elements", fn);
  p.w = Window{window, window < 0 ? 0 : prefix};
  p.q = q;
  p.kp = k_pages;
  p.vp = v_pages;
  p.o = o;
  p.starts = q_start;
  p.q_sr = q_strides[0];
  p.q_sh = q_strides[1];
  p.o_sr = o_strides[0];
  p.o_sh = o_strides[1];
  p.rows = rows;
  p.heads_q = heads_q;
  p.heads_kv = heads_kv;
  const float scale = softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf(static_cast<float>(head_dim));
  p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid(rows, heads_q);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == SABRE_BF16)
    paged_rows_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else
    paged_rows_kernel<__half><<<grid, 128, 0, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

}  // namespace paged
}  // namespace sabre

extern "C" {

size_t sabre_paged_prefill_workspace_size(int rows, int batch, int heads_q, int heads_kv, int head_dim, int page_size,
                                          int max_pages, int window, int num_prefix_tokens) {
  (void)rows, (void)batch, (void)heads_q, (void)heads_kv, (void)head_dim, (void)page_size, (void)max_pages;
  (void)window, (void)num_prefix_tokens;
  return 0;
}

int sabre_paged_prefill(const void* q, const void* k_pages, const void* v_pages, void* o, const int32_t* page_table,
                        const int32_t* seq_lens, const int32_t* q_start, int rows, int batch, int heads_q,
                        int heads_kv, int head_dim, int num_pages, int page_size, int max_pages, int window,
                        int num_prefix_tokens, const int64_t* q_strides, const int64_t* kp_strides,
                        const int64_t* vp_strides, const int64_t* o_strides, int64_t table_stride,
                        float softmax_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace, (void)workspace_bytes;
  if (!q_start) return sabre_fail(SABRE_ERR_INVALID_ARG, "sabre_paged_prefill: null pointer argument");
  return sabre::paged::attend("sabre_paged_prefill", q, k_pages, v_pages, o, page_table, seq_lens, q_start, rows,
                              batch, heads_q, heads_kv, head_dim, num_pages, page_size, max_pages, window,
                              num_prefix_tokens, q_strides, kp_strides, vp_strides, o_strides, table_stride,
                              softmax_scale, dtype, stream);
}

}  // extern "C"
