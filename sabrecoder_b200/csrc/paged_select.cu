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
// The order is that of sums in 64 bits, a score rounded once to fp32: it depends on the
// order of a sum only for values that lie within 2^-30 or so of a border, where sums in
// 32 bits would make a list in a thousand depend on it. (The queries' sum is kept in two
// fp32 parts, which hold it exactly while the bits of its terms span no more than 48.)
namespace sabre {
namespace paged {

// ---------------------------------------------------------------------------
// mean keys: reads 256 bytes a row and head once. A warp takes one page of one
// head, half of it the even rows and half the odd ones, 16 bytes a lane and
// eight loads in flight; the sums are fp32 in row order. 16384 rows of 32 heads
// (138 MB) take 24.4 to 25.7 us, 5.4 to 5.7 TB/s; CTAs of eight warps 26.3.
// ---------------------------------------------------------------------------
namespace means {

constexpr int kMaxWarps = 4;

// volatile: eight of them go out before the first is used.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 x;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
               : "l"(p)
               : "memory");
  return x;
}

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
      for (int u = 0; u < 8; ++u) x[u] = load_once(src + (r + u) * 2 * p.c.k_st);
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

constexpr int kMaxPages = 32768;  // of a sequence: their keys are kept in shared memory
constexpr int kMaxCtas = 8;       // of a cluster: the portable size
constexpr int kSms = 148;         // a B200's
constexpr int kGroupBlocks = 4;   // query blocks that share the means they read
constexpr int kGroupPages = 2048; // columns up to which they do (32 KB of keys)

struct Params {
  Cache c;  // no pools
  const void* q;
  const float* means;
  const int32_t* starts;
  int32_t* lists;
  int32_t* counts;
  long long m_sp, m_sh;
  int q_sr, q_sh;       // one multiplication a row: sums of queries are bound by their instructions
  uint32_t per_group;   // ceil(2^32 / group), for rows / group (group > 1)
  int rows, heads_kv, group, tokens, topk, window, prefix, cap;
  int blocks, ctas, key_row;  // ctas: of a cluster; key_row: keys of a block in shared memory
};

// Scores as whole numbers in the same order: 0 is no candidate, 1 a NaN (taken
// last), numbers lie above, kAlways above them all.
constexpr uint32_t kAlways = 0xffffffffu;
__device__ __forceinline__ uint32_t order_key(float s) {
  if (s != s) return 1u;
  const uint32_t u = __float_as_uint(s + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_score(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Where the keys are cut: those above `limit` are taken, and of those equal to it
// the first `want`.
struct Cut {
  uint32_t limit;
  int want;
};

// The cut that takes the topk best of the candidates (more than topk > 0 of them,
// with keys from lo to hi), by one warp: the range is quartered until as many as
// wanted lie above a border. At first by scores, which are spread more evenly than
// their keys (six steps or so for two hundred), then by keys, which end anyway. The
// first 256 keys stay in registers. (A histogram in shared memory, whose bin is then
// ranked, takes twice as long for a warp: 3.9 K cycles against 2.3 for 190 pages.)
__device__ __forceinline__ Cut find_cut(const uint32_t* key, int pages, int topk, uint32_t lo, uint32_t hi) {
  constexpr int kHeld = 8;
  const int lane = threadIdx.x & 31;
  uint32_t held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held[i] = 32 * i + lane < pages ? key[32 * i + lane] : 0u;
    if (held[i] == kAlways) held[i] = 0u;
  }
  // More than topk keys in [lo, kAlways), fewer above hi.
  for (int round = 0;; ++round) {
    uint32_t at[3];
    const float a = key_score(lo), b = key_score(hi);
    if (round < 10 && fabsf(a) < 1e37f && fabsf(b) < 1e37f && hi - lo > 64u) {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        at[i] = min(max(order_key(fmaf(b - a, 0.25f * (i + 1), a)), lo + 1u + i), hi - 2u + i);
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        at[i] = lo + static_cast<uint32_t>((static_cast<unsigned long long>(hi - lo) * (i + 1) + 3) / 4);
    }
    int n[3] = {};
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
#pragma unroll
      for (int j = 0; j < 3; ++j) n[j] += held[i] >= at[j] ? 1 : 0;
    for (int i = 32 * kHeld + lane; i < pages; i += 32) {
      const uint32_t k = key[i];
#pragma unroll
      for (int j = 0; j < 3; ++j) n[j] += k >= at[j] && k != kAlways ? 1 : 0;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) n[j] = __reduce_add_sync(0xffffffffu, n[j]);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (n[j] == topk) return Cut{at[j] - 1u, 0};
    if (lo == hi) break;
    // Borders ascend, so the counts do not.
    if (n[2] > topk) {
      lo = at[2];
    } else if (n[1] > topk) {
      lo = at[1];
      hi = at[2] - 1u;
    } else if (n[0] > topk) {
      lo = at[0];
      hi = at[1] - 1u;
    } else {
      hi = at[0] - 1u;
    }
  }
  // More than topk keys from lo on, and fewer above it.
  int above = 0;
  for (int i = lane; i < pages; i += 32) above += key[i] > lo && key[i] != kAlways ? 1 : 0;
  return Cut{lo, topk - static_cast<int>(__reduce_add_sync(0xffffffffu, above))};
}

// A query block: `count` rows from `row` on, at positions i0, i0 + 1, ..
struct Block {
  long long row, i0;
  int count, pages, low;  // pages it may read, of which those from `low` on it always does
  __device__ __forceinline__ Block(const Params& p, const RowTile& t, int r) {
    count = max(0, min(p.tokens, t.len - r));
    row = static_cast<long long>(t.first) + r;
    i0 = static_cast<long long>(t.length) - t.len + r;  // lengths reach to the ends of int32
    const long long n = min(static_cast<long long>(min(max(t.length, 0), p.c.capacity())), i0 + count);
    pages = count > 0 && n > 0 ? static_cast<int>((n + (1 << p.c.page_shift) - 1) >> p.c.page_shift) : 0;
    low = static_cast<int>(min(max(i0 - p.window, 0ll) >> p.c.page_shift, static_cast<long long>(pages)));
  }
};

// hi + lo with what rounding takes from hi: hi + x is the new hi and the rounded-off
// part, exact, is added to lo (Knuth; two sums at a time).
__device__ __forceinline__ void add2(uint64_t& hi, uint64_t& lo, uint64_t x) {
  const uint64_t minus = f2_pack(-1.f, -1.f);
  const uint64_t s = f2_add(hi, x);
  const uint64_t b = f2_fma(hi, minus, s);
  const uint64_t a = f2_fma(b, minus, s);
  lo = f2_add(lo, f2_add(f2_fma(a, minus, hi), f2_fma(b, minus, x)));
  hi = s;
}

// hi the nearest to hi + lo, lo what is left. An infinity or NaN stays alone.
__device__ __forceinline__ void settle(float& hi, float& lo) {
  const float s = hi + lo;
  if (fabsf(s) < INFINITY) {
    lo += hi - s;
    hi = s;
  } else {
    hi = hi == hi ? hi : s;
    lo = 0.f;
  }
}

// Sums of this warp's share of the block's queries (rows first to first + 15 of every
// `step`) in two fp32 parts each, into hi[0, kD) and lo[0, kD): 16 threads a row, 16
// bytes each, eight loads in flight.
template <typename T>
__device__ __forceinline__ void sum_queries(const Params& p, const Block& blk, int hk, int first, int step, float* hi,
                                            float* lo) {
  const int lane = threadIdx.x & 31;
  const int many = blk.count * p.group;
  const T* const q = static_cast<const T*>(p.q) + blk.row * p.q_sr + static_cast<long long>(hk) * p.group * p.q_sh +
                     (lane & 15) * 8;
  uint64_t sum[4] = {}, rest[4] = {};
  auto load = [&](int r) -> uint4 {
    if (r >= many) return make_uint4(0u, 0u, 0u, 0u);
    const int tok = p.group == 1 ? r : __umulhi(r, p.per_group);  // exact for r < 2^32 / group
    return *reinterpret_cast<const uint4*>(q + (static_cast<long long>(tok) * p.q_sr +
                                                static_cast<long long>(r - tok * p.group) * p.q_sh));
  };
  uint4 x[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) x[u] = load(first + 2 * u + (lane >> 4));
  for (int r0 = first; r0 < many; r0 += step) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (r0 + 2 * u >= many) break;
      const T* e = reinterpret_cast<const T*>(&x[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) add2(sum[i], rest[i], f2_pack(DT<T>::to_f(e[2 * i]), DT<T>::to_f(e[2 * i + 1])));
      x[u] = load(r0 + step + 2 * u + (lane >> 4));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, rest[i], 16);
    add2(sum[i], rest[i], __shfl_xor_sync(0xffffffffu, sum[i], 16));
    rest[i] = f2_add(rest[i], other);
  }
  ulonglong2* const dst = reinterpret_cast<ulonglong2*>((lane < 16 ? hi : lo) + (lane & 15) * 8);
  dst[0] = lane < 16 ? make_ulonglong2(sum[0], sum[1]) : make_ulonglong2(rest[0], rest[1]);
  dst[1] = lane < 16 ? make_ulonglong2(sum[2], sum[3]) : make_ulonglong2(rest[2], rest[3]);
}

// The choice for one block, by one warp: from the keys of its pages, the sum of its
// queries (q_hi + q_lo) and `bound`, how far a score can be off. The candidates near
// the cut are scored again in 64 bits when some on both sides of it are.
__device__ __forceinline__ Cut choose(const Params& p, uint32_t* key, int pages, uint32_t lo, uint32_t hi,
                                      int candidates, float bound, const float* q_hi, const float* q_lo, int b, int hk,
                                      int* s_near) {
  const int lane = threadIdx.x & 31;
  if (p.topk == 0) return Cut{kAlways - 1u, 0};
  if (candidates <= p.topk) return Cut{0u, 0};
  const Cut cut = find_cut(key, pages, p.topk, lo, hi);
  // Everything from `border` on is taken, but for some of those equal to it (want > 0).
  const uint32_t border = cut.want > 0 ? cut.limit : cut.limit + 1u;
  const float at = key_score(border);
  const bool sure = bound < 1e37f && fabsf(at) < 1e37f;
  const uint32_t first = sure ? order_key(at - 2.002f * bound) : 1u;
  const uint32_t last = sure ? order_key(at + 2.002f * bound) : kAlways - 1u;
  bool in = false, out = false;
  int above = 0;
  for (int i = lane; i < pages; i += 32) {
    const uint32_t k = key[i];
    in = in || (k >= border && k <= last);
    out = out || (k >= first && k < border);
    above += k > last && k != kAlways ? 1 : 0;
  }
  const bool some_in = __any_sync(0xffffffffu, in), some_out = __any_sync(0xffffffffu, out);
  if (!some_in || !(some_out || cut.want > 0)) return cut;

  const int want = p.topk - static_cast<int>(__reduce_add_sync(0xffffffffu, above));
  // 32 near pages at a time: eight lanes a page, 16 columns each (four of every 32).
  const int sub = lane & 7;
  double q[16];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 32 * j + 4 * sub + e;
      q[4 * j + e] = static_cast<double>(q_hi[d]) + static_cast<double>(q_lo[d]);
    }
  uint32_t low = kAlways, high = 0u;
  int near = 0;
  for (int i0 = 0, held = 0; i0 < pages; i0 += 32) {
    const uint32_t k = i0 + lane < pages ? key[i0 + lane] : 0u;
    if (k > last) key[i0 + lane] = kAlways;
    if (k < first && k != 0u) key[i0 + lane] = 0u;
    const uint32_t these = __ballot_sync(0xffffffffu, k >= first && k <= last);
    const int place = held + __popc(these & ((1u << lane) - 1u));
    if (these >> lane & 1u) s_near[place] = i0 + lane;
    held += __popc(these);
    near += __popc(these);
    // Kept until there are 32, or no more.
    while (held >= 32 || (held > 0 && i0 + 32 >= pages)) {
      __syncwarp();
      const int n = min(held, 32);
      for (int g = 0; g < n; g += 4) {
        const int i = s_near[min(g + (lane >> 3), n - 1)];
        const float* m = p.means + p.c.page_of(b, i << p.c.page_shift) * p.m_sp + hk * p.m_sh + 4 * sub;
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(m + 32 * j);
          s = fma(q[4 * j], static_cast<double>(x.x), s);
          s = fma(q[4 * j + 1], static_cast<double>(x.y), s);
          s = fma(q[4 * j + 2], static_cast<double>(x.z), s);
          s = fma(q[4 * j + 3], static_cast<double>(x.w), s);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const uint32_t exact = order_key(static_cast<float>(s));
        if (sub == 0) key[i] = exact;
        low = min(low, exact);
        high = max(high, exact);
      }
      __syncwarp();
      const int moved = lane + 32 < held ? s_near[lane + 32] : 0;
      __syncwarp();
      if (lane + 32 < held) s_near[lane] = moved;
      held -= n;
    }
  }
  __syncwarp();
  if (near == want) return Cut{0u, 0};
  return find_cut(key, pages, want, __reduce_min_sync(0xffffffffu, low), __reduce_max_sync(0xffffffffu, high));
}

// Writes the list of a block, by one warp.
__device__ __forceinline__ void write_list(const Params& p, const Cut& cut, const uint32_t* key, int pages, int block,
                                           int hk) {
  const int lane = threadIdx.x & 31;
  int32_t* const out = p.lists + (static_cast<long long>(block) * p.heads_kv + hk) * p.cap;
  int total = 0, equal = 0;
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = 0; i0 < pages; i0 += 128) {  // four looks at a time
    uint32_t k[4], take[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = i0 + 32 * u + lane < pages ? key[i0 + 32 * u + lane] : 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u) take[u] = __ballot_sync(0xffffffffu, k[u] > cut.limit);
    if (cut.want > 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t same = __ballot_sync(0xffffffffu, k[u] == cut.limit);
        take[u] |= __ballot_sync(0xffffffffu, k[u] == cut.limit && equal + __popc(same & below) < cut.want);
        equal += __popc(same);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int place = total + __popc(take[u] & below);
      if ((take[u] >> lane & 1u) && place < p.cap) out[place] = i0 + 32 * u + lane;
      total += __popc(take[u]);
    }
  }
  total = min(total, p.cap);
  for (int i = total + lane; i < p.cap; i += 32) out[i] = -1;
  if (lane == 0) p.counts[static_cast<long long>(block) * p.heads_kv + hk] = total;
}

// kGroup = 1: a cluster of CTAs takes one query block and KV head; each scores a run
// of the pages and puts the keys into the shared memory of the first, one warp of
// which picks. kGroup > 1: a CTA takes that many consecutive blocks of a sequence,
// whose scores come from one read of the means, and each of its warps sums and picks
// for one.
//
// Scores are computed in 32 bits, from a sum of the queries in two parts whose first is
// within 2^-24 of it. A score is 16 products and sums a lane, three sums over the lanes
// and one rounding, so off by at most 24 * 2^-24 |q| |m| (lengths of vectors, the
// roundings of the bound in a factor 1.06). Two pages whose scores differ by more than
// two bounds are in their right order; where scores on both sides of the cut are
// nearer (one list in a thousand), those near it are computed in 64 bits. A bound that
// is not finite sends every page that way. 64 bits throughout cost 79 us for the
// 12288-row prompt at 16/16 heads; so it takes 25.5 (28.5 with inputs from HBM), of
// which half is the sum of the queries (128 registers, of which a few spill: 24 bytes of
// stack). Groups of two and of eight took 29 and 39 where four took 27. One row on 12288
// takes 5.8 us, 32 rows on up to 16383 (56/8 heads, 16-row pages) 25 to 32, 16
// continuations of up to 200 rows (32/32 heads, 16-row pages) 34 to 39, a chunk of 512 rows
// on 15872 (56/8 heads) 14 over 128-row pages and 35 over 16-row ones.
template <typename T, int kGroup, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kGroup == 1 ? 5 : 16 / kGroup) paged_select_kernel(const Params p) {
  constexpr int kThreads = kWarps * 32;
  constexpr int kInFlight = 2;  // a lane's pages on their way
  extern __shared__ __align__(16) uint32_t s_key[];  // [kGroup][key_row], of the first CTA
  __shared__ __align__(16) float s_hi[kWarps][kD], s_lo[kWarps][kD];  // sums of queries
  __shared__ int s_near[kGroup][64];
  // Of the first CTA, from every warp: its candidates' lowest and highest key and
  // their number, for each block, and the largest |m|^2.
  __shared__ uint4 s_told[kMaxCtas * kWarps];
  __shared__ int scratch[16];
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int warp = tid >> 5;
  const int hk = blockIdx.y;
  // Groups from the last, whose blocks see the most.
  const int slot = kGroup > 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x / p.ctas;
  const int rank = blockIdx.x % p.ctas;
  if (kGroup == 1 && tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (kGroup == 1 && p.ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  RowTile t{slot, 0, slot, 1, 0};
  int block = slot;
  if (!p.starts) {
    t.length = p.c.seq_lens[slot];
  } else {
    const int tile = p.tokens * kGroup;
    int before = 0, all = 0;  // blocks of the sequences before this one, and of all
    if (p.c.batch <= 32) {
      int len;
      if (!find_rows_warp(p.c, p.starts, p.rows, tile, slot, t, len)) t = RowTile{-1, 0, 0, 0, 0};
      const int n = (len + p.tokens - 1) / p.tokens;
      before = __reduce_add_sync(0xffffffffu, lane < t.b ? n : 0);
      all = __reduce_add_sync(0xffffffffu, n);
    } else if (!find_rows<kThreads>(p.c, p.starts, p.rows, tile, slot, scratch, t)) {
      t = RowTile{-1, 0, 0, 0, 0};
    }
    if constexpr (kGroup > 1) {
      if (p.c.batch > 32) {
        for (int b = tid; b < p.c.batch; b += kThreads) {
          const int len = max(row_start(p.starts, b + 1, p.rows) - row_start(p.starts, b, p.rows), 0);
          const int n = (len + p.tokens - 1) / p.tokens;
          all += n;
          before += b < t.b ? n : 0;
        }
        __syncthreads();  // scratch is read
        before = __reduce_add_sync(0xffffffffu, before);
        all = __reduce_add_sync(0xffffffffu, all);
        if (lane == 0) scratch[warp] = before, scratch[kWarps + warp] = all;
        __syncthreads();
        before = all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) before += scratch[w], all += scratch[kWarps + w];
      }
      block = before + t.r / p.tokens;
      // Blocks that the rows could make but do not hold have no pages. (A count past
      // int32, which only starts that do not ascend can make, is past them all.)
      for (long long i = (all < 0 ? p.blocks : all) + 0ll + slot * kWarps + warp; i < p.blocks; i += gridDim.x * kWarps)
        write_list(p, Cut{0u, 0}, s_key, 0, static_cast<int>(i), hk);
      if (t.b < 0) return;
    }
  }
  const Block mine(p, t, t.r + (kGroup > 1 ? warp * p.tokens : 0));
  // The last block sees the most; no block scores a page from its `low` on, and none
  // one that begins before the prefix's end.
  const int ahead = (min(kGroup * p.tokens, t.len - t.r) - 1) / p.tokens;
  const Block last = kGroup == 1 ? mine : Block(p, t, t.r + ahead * p.tokens);
  const int pages = last.pages;
  const int head = static_cast<int>((static_cast<long long>(p.prefix) + (1 << p.c.page_shift) - 1) >> p.c.page_shift);

  // This warp's pages, and the table's entries for the first 32 of them.
  const int slice = (pages + p.ctas - 1) / p.ctas;
  const int from = min(rank * slice, pages), to = min(from + slice, pages);
  const int chunk = (((to - from + kWarps - 1) / kWarps) + 3) & ~3;
  const int p0 = min(from + warp * chunk, to), p1 = min(p0 + chunk, to);
  int entry = p0 + lane < p1 ? p.c.entry(t.b, (p0 + lane) << p.c.page_shift) : -1;

  // kGroup = 1: each warp sums up to 16 rows for itself, which saves the barriers.
  const bool alone = kGroup > 1 || mine.count * p.group <= 16;
  const int of = alone ? warp : 0;  // whose sums this warp uses, if it scores one block
  sum_queries<T>(p, mine, hk, alone ? 0 : 16 * warp, alone ? 16 : 16 * kWarps, s_hi[warp], s_lo[warp]);
  if (kGroup > 1 || !alone) __syncthreads();
  if (kGroup == 1 && alone) {
    __syncwarp();
    for (int i = lane; i < kD; i += 32) settle(s_hi[warp][i], s_lo[warp][i]);
    __syncwarp();
  } else if constexpr (kGroup == 1) {
    for (int i = tid; i < kD; i += kThreads) {
      uint64_t hi = f2_pack(s_hi[0][i], 0.f), lo = f2_pack(s_lo[0][i], 0.f);
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        add2(hi, lo, f2_pack(s_hi[w][i], 0.f));
        lo = f2_add(lo, f2_pack(s_lo[w][i], 0.f));
      }
      float s, l, none;
      f2_unpack(hi, s, none);
      f2_unpack(lo, l, none);
      settle(s, l);
      s_hi[0][i] = s;
      s_lo[0][i] = l;
    }
    __syncthreads();
  } else {
    for (int i = tid; i < kGroup * kD; i += kThreads) settle(s_hi[0][i], s_lo[0][i]);
    __syncthreads();
  }

  // Scores: eight lanes share a page, 16 columns each (four of every 32).
  const int sub = lane & 7;
  ulonglong2 q1[kGroup == 1 ? 4 : 1];  // four columns as two pairs, as everything below
  if constexpr (kGroup == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) q1[j] = *reinterpret_cast<const ulonglong2*>(&s_hi[of][32 * j + 4 * sub]);
  }
  // The first CTA has started when its shared memory is written to.
  uint32_t keys = smem_u32(s_key), told = smem_u32(s_told);
  if (kGroup == 1 && p.ctas > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(keys) : "r"(keys), "r"(0));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(told) : "r"(told), "r"(0));
  }
  // kGroup > 1: the block whose scores end up in this lane.
  const int own_g = kGroup > 1 ? sub * kGroup / 8 : 0;
  const Block own(p, t, t.r + own_g * p.tokens);
  float size = 0.f;  // of |m|^2 this lane's 16 columns, the largest over the pages
  uint32_t lowest = kAlways, highest = 0u;
  int candidates = 0;
  for (int g0 = p0; g0 < p1; g0 += 32) {
    const int here = min(32, p1 - g0);
    const int id = g0 + lane < p1 ? p.c.checked(entry) : -1;
    const int next = g0 + 32 + lane;
    entry = next < p1 ? p.c.entry(t.b, next << p.c.page_shift) : -1;
    for (int u0 = 0; u0 < here; u0 += 4 * kInFlight) {
      ulonglong2 m[kInFlight][4];
      int page[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int i = u0 + 4 * u + (lane >> 3);
        page[u] = __shfl_sync(0xffffffffu, id, i & 31);
        if (i >= here) page[u] = -1;
        const bool scored = page[u] >= 0 && g0 + i >= head && g0 + i < last.low;
        const float* src = p.means + page[u] * p.m_sp + hk * p.m_sh + 4 * sub;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          m[u][j] = scored ? *reinterpret_cast<const ulonglong2*>(src + 32 * j) : make_ulonglong2(0ull, 0ull);
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        uint64_t n2 = 0ull;
#pragma unroll
        for (int j = 0; j < 4; ++j) n2 = f2_fma(m[u][j].x, m[u][j].x, f2_fma(m[u][j].y, m[u][j].y, n2));
        float a, b;
        f2_unpack(n2, a, b);
        size = a + b <= 1e37f ? fmaxf(size, a + b) : INFINITY;
      }
      float acc[kInFlight][kGroup];
#pragma unroll
      for (int g = 0; g < kGroup; ++g) {
        uint64_t two[kInFlight] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const ulonglong2 x = kGroup == 1 ? q1[j] : *reinterpret_cast<const ulonglong2*>(&s_hi[g][32 * j + 4 * sub]);
#pragma unroll
          for (int u = 0; u < kInFlight; ++u) two[u] = f2_fma(x.x, m[u][j].x, f2_fma(x.y, m[u][j].y, two[u]));
        }
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
          float a, b;
          f2_unpack(two[u], a, b);
          acc[u][g] = a + b;
        }
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        float s;
        if constexpr (kGroup == 1) {
          s = acc[u][0];
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        } else {
          // The eight lanes' parts of kGroup blocks: a step over lanes 4, 2 and 1 apart
          // leaves each half of the blocks while there are several.
          int have = kGroup;
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) {
            if (have > 1) {
              have /= 2;
#pragma unroll
              for (int g = 0; g < kGroup / 2; ++g) {
                if (g >= have) break;
                const float give = sub & o ? acc[u][g] : acc[u][g + have], keep = sub & o ? acc[u][g + have] : acc[u][g];
                acc[u][g] = keep + __shfl_xor_sync(0xffffffffu, give, o);
              }
            } else {
              acc[u][0] += __shfl_xor_sync(0xffffffffu, acc[u][0], o);
            }
          }
          s = acc[u][0];
        }
        const int i = u0 + 4 * u + (lane >> 3), pg = g0 + i;
        const bool scored = page[u] >= 0 && pg >= head && pg < own.low;
        const uint32_t key = page[u] < 0 ? 0u : scored ? order_key(s) : kAlways;
        if (scored) {
          lowest = min(lowest, key);
          highest = max(highest, key);
          ++candidates;
        }
        if (i < here && pg < own.pages) {
          if constexpr (kGroup > 1)
            s_key[own_g * p.key_row + pg] = key;
          else if (sub == 0)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(keys + 4u * pg), "r"(key) : "memory");
        }
      }
    }
  }
  // A grid whose CTAs run side by side leaves the places to the next one only now:
  // CTAs that came earlier would crowd where places are free.
  if (kGroup > 1 && tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // The eight lanes' largest parts add up to no less than the largest |m|^2.
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) size += __shfl_xor_sync(0xffffffffu, size, o);
  size = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(size)));  // >= 0: ordered as bits
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  highest = __reduce_max_sync(0xffffffffu, highest);
  if (kGroup == 1) candidates = __reduce_add_sync(0xffffffffu, sub == 0 ? candidates : 0);
  if (lane == 0)
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(told + 16u * (rank * kWarps + warp)),
                 "r"(lowest), "r"(highest), "r"(candidates), "r"(__float_as_uint(size))
                 : "memory");
  if (kGroup == 1 && p.ctas > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // A warp picks for its block; kGroup = 1: the first one. Starts that do not ascend
  // count more blocks than there is room for.
  const int pick = kGroup > 1 ? warp : 0;
  if (kGroup == 1 ? warp > 0 : mine.count == 0 || static_cast<uint32_t>(block + pick) >= p.blocks) return;
  uint32_t* const key = s_key + pick * p.key_row;
  uint4 sum = make_uint4(kAlways, 0u, 0u, 0u);
  for (int i = lane; i < p.ctas * kWarps; i += 32) {
    const uint4 w = s_told[i];
    sum = make_uint4(min(sum.x, w.x), max(sum.y, w.y), sum.z + w.z, max(sum.w, w.w));
  }
  const uint32_t lo = __reduce_min_sync(0xffffffffu, sum.x), hi = __reduce_max_sync(0xffffffffu, sum.y);
  size = __uint_as_float(__reduce_max_sync(0xffffffffu, sum.w));
  candidates = static_cast<int>(sum.z);
  if constexpr (kGroup > 1) {
    candidates = 0;
    for (int i = lane; i < mine.pages; i += 32) candidates += key[i] != 0u && key[i] != kAlways ? 1 : 0;
  }
  candidates = __reduce_add_sync(0xffffffffu, candidates);
  float q2 = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) q2 = fmaf(s_hi[of][32 * j + lane], s_hi[of][32 * j + lane], q2);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) q2 += __shfl_xor_sync(0xffffffffu, q2, o);
  // 2^-120 is more than what underflow takes from 128 squares, so that the lengths of
  // tiny vectors (below 2^-60) are bounded from above too; 1e-37 covers the products'.
  const float bound = 24.f * sqrtf(q2 + 0x1p-120f) * sqrtf(size + 0x1p-120f) * 0x1.1p-24f + 1e-37f;
  const Cut cut = choose(p, key, mine.pages, lo, hi, candidates, bound, s_hi[of], s_lo[of], t.b, hk, s_near[pick]);
  write_list(p, cut, key, mine.pages, block + pick, hk);
}

template <typename T, int kGroup, int kWarps>
static cudaError_t launch(const Params& p, long long slots, cudaStream_t s) {
  const auto kernel = paged_select_kernel<T, kGroup, kWarps>;
  const int most = kGroup > 1 ? kGroup * (kGroupPages + 1) : kMaxPages + 1;
  const int smem = kGroup * p.key_row * static_cast<int>(sizeof(uint32_t));
  if (smem > 32 * 1024) {  // with the kernel's own past what every launch may have
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               most * static_cast<int>(sizeof(uint32_t)));
    if (e != cudaSuccess) return e;
  }
  const dim3 grid(static_cast<unsigned>(slots * p.ctas), p.heads_kv);
  if (p.ctas == 1) return launch_dependent(grid, kWarps * 32, smem, s, kernel, p);
  return launch_cluster(grid, p.ctas, kWarps * 32, smem, s, kernel, p);
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
  if (heads_q % heads_kv != 0 || heads_q / heads_kv > 1024)  // rows of a block stay below 2^20
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: heads_q/heads_kv must be an integer <= 1024", fn);
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
  if (q_strides[0] < 0 || q_strides[1] < 0 || q_strides[0] > INT_MAX || q_strides[1] > INT_MAX)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: q strides must be from 0 to 2^31 - 1", fn);
  p.q_sr = static_cast<int>(q_strides[0]);
  p.q_sh = static_cast<int>(q_strides[1]);
  p.per_group = static_cast<uint32_t>(((1ull << 32) + heads_q / heads_kv - 1) / (heads_q / heads_kv));
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
  const long long blocks = row_slots(rows, batch, query_block);
  // Blocks that fill the card in groups run in groups; else clusters of as many CTAs
  // as leave each warp eight pages, while the card has places.
  // Device us in groups and without them, 16 heads, a table of 192 columns:
  //   groups * heads       128          160          192          256          320
  //   blocks of 128    17.0 / 14.5  18.2 / 15.4  17.8 / 15.7  20.8 / 20.4  23.4 / 25.1
  //   blocks of 16      6.9 / 12.1   7.9 / 9.3    8.3 / 11.7   9.7 / 14.0  10.8 / 16.9
  // (the 12288-row prompt in blocks of 128: 24.9 / 30.3), and by the table's width, whose
  // keys take 4 KB a 256 columns: 24.9 / 30.4 for 2049 columns, 25.4 / 30.7 for 4096, 43 /
  // 31 for 8192. Past 8192 columns a block's own keys leave few CTAs an SM: 38 us for
  // 16384 columns, 80 for 32768.
  const long long groups = q_start ? row_slots(rows, batch, query_block * sel::kGroupBlocks) : 0;
  const bool grouped = groups * heads_kv >= sel::kSms && max_pages <= sel::kGroupPages;
  p.ctas = 1;
  // Each CTA of a cluster sums the block's queries, so blocks of many rows run in
  // clusters over long tables only (32 blocks of 112 rows on 124 pages, 8 heads: 19 us
  // in pairs of CTAs, 13 alone; on 1000 pages 30 and 47).
  auto places = [&](int ctas) {
    return query_block * p.group <= 16 || max_pages > 256 * ctas ? 4 * sel::kSms : sel::kSms;
  };
  while (!grouped && p.ctas < sel::kMaxCtas && max_pages >= 32 * p.ctas && blocks * heads_kv * p.ctas <= places(p.ctas))
    p.ctas *= 2;
  if (blocks * p.ctas > INT_MAX) return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: too many query blocks", fn);
  p.blocks = static_cast<int>(blocks);
  p.key_row = max_pages | 1;  // the rows' banks differ
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (grouped)
    e = dtype == SABRE_BF16 ? sel::launch<__nv_bfloat16, sel::kGroupBlocks, sel::kGroupBlocks>(p, groups, s)
                            : sel::launch<__half, sel::kGroupBlocks, sel::kGroupBlocks>(p, groups, s);
  else
    e = dtype == SABRE_BF16 ? sel::launch<__nv_bfloat16, 1, 4>(p, blocks, s) : sel::launch<__half, 1, 4>(p, blocks, s);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

}  // extern "C"
