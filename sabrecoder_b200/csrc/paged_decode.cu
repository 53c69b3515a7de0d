// Attention of one new token per sequence over a paged K/V cache.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m), s_j = scale * log2(e) * q.k_j,
// over the visible keys, in one pass with a running maximum m. Bound by HBM:
// every visible K and V row is read once (512 bytes per KV head and key) for
// 512 flops per query head, so all heads of a KV head's group share the read.
//
// Work split. A (sequence, KV head) pair is a list of 64-key tiles (the tiles
// of the prefix tokens, then those of the window). The tiles of all pairs, in
// order, are dealt out in equal contiguous shares to at most two CTAs per SM,
// so a ragged batch, one long sequence and many short ones all fill the card,
// and lengths are only needed on the device (a captured call follows them). A
// CTA walks its share as segments (its part of one pair); a pair inside one
// share is finished there, the others leave (m, l, acc) per head and
// paged_join_kernel adds them in share order: results do not depend on timing.
//
// A CTA: warp 4 fetches K and V tiles by TMA into a three-stage ring (boxes of
// 16 rows; absent pages and boxes that nobody sees are not fetched) and runs
// ahead over segment ends; warps 0..3 each take 16 of a tile's 64 keys on the
// tensor cores with their own softmax state, so the tile loop has no barrier
// but the ring's:
//   S^T = K Q^T   (16 keys x 8 heads, K by ldmatrix, Q kept in registers)
//   O^T += V^T P^T (128 d x 8 heads, V by transposed ldmatrix; P^T is S^T's
//                   layout after one movmatrix per 8 keys)
// Eight heads fill the instruction's N: groups of up to eight cost the same.
// mma.sync is used rather than tcgen05: at the HBM rate the matrix work keeps
// the tensor pipe busy a tenth of the time (ncu), and there is no tensor memory
// to allocate, fill and read back per segment. 32 sequences of 1..16384 rows at
// 56/8 heads (917 MB) take 145 us, 6.3 TB/s.
// P is rounded to the type of V for the product (half a step of a weight,
// below the rounding of the output); scores, sums and acc are fp32.
namespace sabre {
namespace paged {

constexpr int kTile = 64;
constexpr int kStages = 3;
constexpr int kTileBytes = kTile * kD * 2;  // 16384
// A TMA box: 16 rows of one page, [d-half][16 rows][128 B] with the 128-byte
// swizzle. Boxes of up to 64 rows run long caches no faster and fetch rows that
// nobody sees at the ends of short ones: 64 sequences of 1..450 rows at 32/32
// heads 52.5 us against 58.4, the windowed batch of 64 178 against 185.
constexpr int kBoxRows = 16;
constexpr int kBoxes = kTile / kBoxRows;  // of a tile: one for each consumer warp
constexpr int kBoxBytes = kBoxRows * kD * 2;
constexpr int kConsumers = 4;
static_assert(kBoxes == kConsumers, "a consumer's 16 keys are one box");
constexpr int kDecThreads = (kConsumers + 1) * 32;
constexpr int kDecCtas = 2 * 148;
constexpr int kMaxParts = 128;  // parts of one pair, were all sequences alike
constexpr int kGroup = 8;       // query heads per KV head, at most
constexpr int kAccRow = 132;    // padded head row: the 32 lanes of a store hit 32 banks
constexpr int kRingOff = 0;
constexpr int kAccOff = kRingOff + kStages * 2 * kTileBytes;
constexpr int kMlOff = kAccOff + kConsumers * kGroup * kAccRow * 4;
constexpr int kBarOff = kMlOff + kConsumers * kGroup * 2 * 4;
constexpr int kMiscOff = kBarOff + 2 * kStages * 8;
constexpr int kDecSmem = kMiscOff + 48;
static_assert(2 * (kDecSmem + 1024) <= 228 * 1024, "two CTAs per SM");

struct DecodeParams {
  Cache c;
  Window w;
  const void* q;
  void* o;
  float* part_acc;  // [2 * kDecCtas][group][D]
  float* part_ml;   // [2 * kDecCtas][group][2]
  int4* joins;      // [kDecCtas]: {parts, b, hk, slot of the first part} of the pair whose first part ends share x
  long long q_sb, q_sh, o_sb, o_sh;
  int heads_kv, group, ctas;
  float scale_log2;
  Lists lists;  // of a call over listed pages
};

// The visible tiles of one sequence: `head` tiles from 0 (prefix tokens), then
// the tiles from `from` on.
struct Tiles {
  int n, lo, head, from, count;
  __device__ __forceinline__ Tiles(const DecodeParams& p, int b) {
    n = p.c.length(b);
    lo = n > 0 ? p.w.first(p.c.seq_lens[b] - 1) : 0;
    from = lo / kTile;
    // No tile past n: lengths and prefixes reach to the end of int32, tables do not.
    head = min((min(min(p.w.prefix, lo), n) + kTile - 1) / kTile, from);
    count = head + max(0, (n + kTile - 1) / kTile - from);
  }
  __device__ __forceinline__ int pos(int i) const { return (i < head ? i : from + i - head) * kTile; }
  __device__ __forceinline__ bool any(const Window& w, int t, int rows) const {  // a visible key in [t, t + rows)?
    return t < n && (t + rows > lo || t < w.prefix);
  }
};

// The same over the listed pages of one (sequence, KV head) pair: 64 list rows a
// tile, as many tiles as its list has entries for. Bound by HBM as the dense decode:
// 64 sequences at 56/8 heads over 22 pages of 128 rows (649 MB) take 106.5 us, 6.1
// TB/s; one sequence of 14 pages at 16/16 heads 6.8 (a cluster a pair, below).
struct ListedTiles {
  int n, entries, count;
  __device__ __forceinline__ ListedTiles(const DecodeParams& p, int b, int hk) {
    n = p.c.length(b);
    entries = n > 0 ? p.lists.count(b, hk) : 0;
    count = static_cast<int>(((static_cast<long long>(entries) << p.c.page_shift) + kTile - 1) / kTile);
  }
};

// What the shares are dealt out over, in order: without lists sequences, whose
// KV heads all have the same tiles; with lists pairs.
template <bool kListed>
struct Work {
  using Tiles_ = typename std::conditional<kListed, ListedTiles, Tiles>::type;
  static __device__ __forceinline__ int count(const DecodeParams& p) {
    return kListed ? p.c.batch * p.heads_kv : p.c.batch;
  }
  static __device__ __forceinline__ int heads(const DecodeParams& p) { return kListed ? 1 : p.heads_kv; }
  static __device__ __forceinline__ Tiles_ tiles(const DecodeParams& p, int x) {
    if constexpr (kListed)
      return ListedTiles(p, x / p.heads_kv, x % p.heads_kv);
    else
      return Tiles(p, x);
  }
};

// Shares: total tiles dealt to `ctas` CTAs; unit u belongs to CTA owner(u).
struct Shares {
  long long total;
  int ctas;
  __device__ __forceinline__ long long first(int x) const { return total * x / ctas; }
  __device__ __forceinline__ int owner(long long u) const { return static_cast<int>(((u + 1) * ctas - 1) / total); }
};

struct Place {
  int b, hk, tile;
};

// Finds the shares and the place of this CTA's first unit with the whole CTA
// (kDecThreads threads); scratch: 16 ints of shared memory. False for a CTA
// without a share. Calls on_empty(x) for the sequences (with lists: pairs)
// without a tile.
template <bool kListed, typename E>
__device__ __forceinline__ bool locate(const DecodeParams& p, int* scratch, Shares& sh, Place& at, E on_empty) {
  constexpr int kThreads = kDecThreads;
  using W = Work<kListed>;
  const int tid = threadIdx.x;
  const int per = (W::count(p) + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, W::count(p)), b1 = min(b0 + per, W::count(p));
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int nt = W::tiles(p, b).count;
    if (nt == 0) on_empty(b);
    mine += nt;
  }
  int incl = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, s);
    if ((tid & 31) >= s) incl += up;
  }
  if ((tid & 31) == 31) scratch[tid >> 5] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    before += w < (tid >> 5) ? scratch[w] : 0;
    all += scratch[w];
  }
  sh.total = static_cast<long long>(all) * W::heads(p);
  if (all == 0) return false;
  sh.ctas = static_cast<int>(min(static_cast<long long>(p.ctas), sh.total));
  if (static_cast<int>(blockIdx.x) >= sh.ctas) return false;
  long long left = sh.first(blockIdx.x) - static_cast<long long>(before + incl - mine) * W::heads(p);
  int* found = scratch + kThreads / 32;
  if (left >= 0 && left < static_cast<long long>(mine) * W::heads(p)) {
    for (int b = b0; b < b1; ++b) {
      const int nt = W::tiles(p, b).count;
      const long long here = static_cast<long long>(nt) * W::heads(p);
      if (left < here) {
        found[0] = b;
        found[1] = static_cast<int>(left / nt);
        found[2] = static_cast<int>(left % nt);
        break;
      }
      left -= here;
    }
  }
  __syncthreads();
  at.b = kListed ? found[0] / p.heads_kv : found[0];
  at.hk = kListed ? found[0] % p.heads_kv : found[1];
  at.tile = found[2];
  return true;
}

// Walks a share's segments: the same sequence for the producer and the consumers.
template <bool kListed>
struct Segments {
  const DecodeParams& p;
  int b, hk, t0, t1, seen;  // this segment: tiles [t0, t1) of pair (b, hk)
  long long left;
  typename Work<kListed>::Tiles_ tiles;
  __device__ __forceinline__ Segments(const DecodeParams& p_, const Place& at, long long units)
      : p(p_), b(at.b), hk(at.hk), t0(at.tile), t1(0), seen(-1), left(units),
        tiles(Work<kListed>::tiles(p_, kListed ? at.b * p_.heads_kv + at.hk : at.b)) {}
  __device__ __forceinline__ bool next() {
    if (left <= 0) return false;
    if (++seen > 0) {
      t0 = 0;
      if constexpr (kListed) {
        do {  // left > 0: another pair has tiles
          if (++hk == p.heads_kv) {
            hk = 0;
            ++b;
          }
          tiles = ListedTiles(p, b, hk);
        } while (tiles.count == 0 && b * p.heads_kv + hk < p.c.batch * p.heads_kv - 1);
      } else if (++hk == p.heads_kv) {
        hk = 0;
        do tiles = Tiles(p, ++b);  // left > 0: another sequence has tiles
        while (tiles.count == 0 && b < p.c.batch - 1);
      }
    }
    t1 = static_cast<int>(min(static_cast<long long>(tiles.count), t0 + left));
    left -= t1 - t0;
    return true;
  }
};

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* m, uint32_t bar, int row, int half,
                                              int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(0), "r"(row), "r"(half), "r"(head), "r"(page)
      : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8x8 matrix of 16-bit values over the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// c[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums.
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT<T>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
        " {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
        " {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// out[4 lane ..] = a / l, zeros where nothing was visible (l is exactly 0; a NaN
// sum is a NaN result).
template <typename T>
__device__ __forceinline__ void store_row(T* out, int lane, const float4& a, float l) {
  const float inv = 1.0f / l;
  *reinterpret_cast<uint2*>(out + lane * 4) =
      l == 0.f ? make_uint2(0u, 0u)
               : make_uint2(DT<T>::pack(a.x * inv, a.y * inv), DT<T>::pack(a.z * inv, a.w * inv));
}

// The running sum of a row's parts: maximum m, sum l and four columns a of the
// accumulator. Scores of NaN never raise m but make l NaN, also where m is still
// -inf: the l of such parts is added as it is (0 or NaN; a NaN l is enough for a
// NaN result). Scaling them like the others instead cost 0.3 us of the 23.4 of
// 12289 rows at 16/16 heads.
struct PartSum {
  float m = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void raise(float mn) {
    const float r = ex2(m - mn);
    m = mn;
    l *= r;
    a = make_float4(a.x * r, a.y * r, a.z * r, a.w * r);
  }
  __device__ __forceinline__ void add(float off, float pm, float pl, const float4& pa) {
    const float w = ex2(pm - off);
    l += w * pl;
    a.x += w * pa.x;
    a.y += w * pa.y;
    a.z += w * pa.z;
    a.w += w * pa.w;
  }
  // Parts first, first + step, .. below `parts`, eight in flight; slot(i): the
  // row of part i in ml and acc, this lane's columns from 4 lane on.
  template <typename S>
  __device__ __forceinline__ void add_parts(const float* part_ml, const float* part_acc, int first, int step, int parts,
                                            int lane, S slot) {
    constexpr int kBatch = 8;
    for (int i0 = first; i0 < parts; i0 += step * kBatch) {
      float2 ml[kBatch];
      float4 x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * step;
        ml[u] = i < parts ? *reinterpret_cast<const float2*>(part_ml + slot(i) * 2) : make_float2(-INFINITY, 0.f);
        x[u] = i < parts ? *reinterpret_cast<const float4*>(part_acc + slot(i) * kD + lane * 4)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) mn = fmaxf(mn, ml[u].x);
      if (mn == -INFINITY) {  // sums of 0 or NaN
#pragma unroll
        for (int u = 0; u < kBatch; ++u) l += ml[u].y;
        continue;
      }
      raise(mn);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) add(mn, ml[u].x, ml[u].y, x[u]);
    }
  }
};

// A barrier over all threads of the cluster.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Short lists of few pairs run in clusters: kCluster CTAs take a pair's tiles in equal
// runs and the first joins them over the cluster's shared memory, which spares the
// joining kernel (one sequence of 14 pages at 16/16 heads 8.0 -> 6.8 us). A CTA then has
// at most kClusterTiles tiles. Clusters find fewer places than CTAs alone do: 30 run at
// once here, and a 32nd waits for another's end, so kClusterPairs stays below that.
// Device us in clusters and in shares with the joining kernel, one head a group:
//   tiles a pair      2            8            16           32           33
//   1 pair        5.1 / 7.0    5.2 / 7.2    5.7 / 7.4    6.8 / 7.7    7.3 / 8.2
//   16 pairs      6.0 / 7.6    6.3 / 7.8    6.9 / 8.3    8.1 / 8.9    8.5 / 9.0
//   28 pairs      6.2 / 7.6    6.5 / 7.8    7.2 / 9.6    8.4 / 10.4
//   32 pairs      9.4 / 7.7    9.8 / 8.1   11.0 / 9.7   13.2 / 10.4
// (64 tiles: 8.9 / 8.7 for one pair; seven heads a group: 5.7 / 7.4 for one pair of two
// tiles, 9.4 / 12.0 for 28 of 32.)
constexpr int kCluster = 8;
constexpr int kClusterTiles = 4;
constexpr int kClusterPairs = 28;

// kMode: over all rows, or the window's; over the pages of p.lists; the same in clusters.
enum DecodeMode { kDense, kOverPages, kInClusters };
template <typename T, DecodeMode kMode>
__global__ void __launch_bounds__(kDecThreads, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const DecodeParams p) {
  constexpr bool kListed = kMode != kDense;
  constexpr bool kClustered = kMode == kInClusters;
  // paged_join_kernel (a programmatic dependent launch) may become resident
  // now; its griddepcontrol.wait still waits for this whole grid.
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const uint32_t sbase = smem_u32(smem);
  // [kStages]: fetched boxes of the tile; with lists also, from bit 4 on, how many
  // rows of each box the sequence has, in five bits each.
  uint32_t* valid = reinterpret_cast<uint32_t*>(smem + kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kMiscOff + 16);
  auto full_bar = [&](int s) -> uint32_t { return sbase + kBarOff + 8u * s; };
  auto empty_bar = [&](int s) -> uint32_t { return sbase + kBarOff + 8u * (kStages + s); };
  if (tid == 0) {
    const bool bad = (sbase & 1023u) != 0u;
    *abort_flag = bad ? 1 : 0;
    if (bad) record_status(SABRE_DEV_BAD_SMEM_ALIGN);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), kConsumers);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // Launched as a programmatic dependent of the previous kernel: nothing
  // below may read before its writes are visible.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned long long wlim = wait_limit_ns();
  Shares sh;
  Place at;
  T* const out = static_cast<T*>(p.o);
  long long units;
  if constexpr (kClustered) {
    const int pair = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
    at.b = pair / p.heads_kv;
    at.hk = pair % p.heads_kv;
    const int n = ListedTiles(p, at.b, at.hk).count;
    at.tile = n * rank / kCluster;
    units = n * (rank + 1) / kCluster - at.tile;
  } else {
    const bool some = locate<kListed>(p, reinterpret_cast<int*>(smem + kAccOff), sh, at, [&](int x) {
      // No visible tile: the sequence's (with lists: the pair's) rows are zero.
      if (x % p.ctas != static_cast<int>(blockIdx.x)) return;
      const int b = kListed ? x / p.heads_kv : x;
      const int h0 = kListed ? x % p.heads_kv * p.group : 0;
      for (int h = h0; h < h0 + (kListed ? 1 : p.heads_kv) * p.group; ++h)
        for (int d = 0; d < kD; d += 8)
          *reinterpret_cast<uint4*>(out + b * p.o_sb + h * p.o_sh + d) = make_uint4(0u, 0u, 0u, 0u);
    });
    // locate()'s barriers order the mbarrier set-up above before its use.
    if (!some) {
      if (tid == 0) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    units = sh.first(blockIdx.x + 1) - sh.first(blockIdx.x);
  }
  Segments<kListed> seg(p, at, units);
  __syncthreads();  // the scratch of locate() is free
  bool ok = *abort_flag == 0;

  if (warp == kConsumers) {
    // ---------------- producer ----------------
    int it = 0;
    int issued = 0;  // stages used, as a count of tiles
    while (ok && seg.next()) {
      const int nbox = (seg.t1 - seg.t0) * kBoxes;
      for (int i0 = 0; ok && i0 < nbox; i0 += 32) {
        // The pages of the next 32 boxes, one per lane.
        int page = -1, off = 0;
        uint32_t rows = 0;  // kListed: of this tile's boxes
        if constexpr (kListed) {
          const int at_row = seg.t0 * kTile + (i0 + lane) * kBoxRows;
          const int e = at_row >> p.c.page_shift;
          if (i0 + lane < nbox && e < seg.tiles.entries) {
            const int col = p.lists.column(seg.b, seg.hk, e, p.c);
            off = at_row & ((1 << p.c.page_shift) - 1);
            const int t = (col << p.c.page_shift) + off;
            if (col >= 0 && t < seg.tiles.n) {
              page = p.c.page_of(seg.b, t);
              rows = static_cast<uint32_t>(min(seg.tiles.n - t, kBoxRows)) << (4 + 5 * (lane % kBoxes));
            }
          }
          rows |= __shfl_xor_sync(0xffffffffu, rows, 1);
          rows |= __shfl_xor_sync(0xffffffffu, rows, 2);
        } else if (i0 + lane < nbox) {
          const int t = seg.tiles.pos(seg.t0 + (i0 + lane) / kBoxes) + (lane % kBoxes) * kBoxRows;
          if (seg.tiles.any(p.w, t, kBoxRows)) {
            page = p.c.page_of(seg.b, t);
            off = t & ((1 << p.c.page_shift) - 1);
          }
        }
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
        for (int i = 0; i < min(32, nbox - i0); i += kBoxes, ++it) {
          const int s = it % kStages;
          ok = mbar_wait_warp_lim(empty_bar(s), ((it / kStages) & 1) ^ 1, abort_flag, wlim);
          if (!ok) break;
          const uint32_t mask = (have >> i) & ((1u << kBoxes) - 1u);
          const uint32_t tile_rows = kListed ? __shfl_sync(0xffffffffu, rows, i) : 0u;
          if (lane == 0) {
            valid[s] = mask | tile_rows;
            mbar_arrive_expect_tx(full_bar(s), __popc(mask) * 2u * kBoxBytes);
          }
          __syncwarp();
          if (lane / kBoxes == i / kBoxes && page >= 0) {
            const uint32_t dst = sbase + kRingOff + s * 2 * kTileBytes + lane % kBoxes * kBoxBytes;
            tma_load_page(dst, &tmK, full_bar(s), off, 0, seg.hk, page);
            tma_load_page(dst + kTileBytes, &tmV, full_bar(s), off, 0, seg.hk, page);
          }
          issued = it + 1;
        }
      }
    }
    // Every issued copy must land before the CTA may exit.
    if (lane == 0)
      for (int i = max(0, issued - kStages); i < issued; ++i)
        mbar_wait_drain(full_bar(i % kStages), (i / kStages) & 1);
    if constexpr (kClustered) {  // the joining below
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  // ---------------- consumers: warp w owns keys [16w, 16w + 16) of a tile ----------------
  const int r4 = lane >> 2;       // S^T: keys r4 and r4 + 8; O^T: d r4 and r4 + 8 of 16
  const int c2 = (lane & 3) * 2;  // S^T and O^T: heads c2 and c2 + 1
  const uint32_t wrow = static_cast<uint32_t>(warp * kBoxBytes);  // this warp's box within a stage
  constexpr uint32_t half = kBoxBytes / 2;                        // from one d-half of it to the other
  // ldmatrix lane addresses: 16-byte chunk c of row r of a d-half lies at r * 128 + ((c ^ (r & 7)) << 4).
  const int mi = lane >> 3, ri = lane & 7;
  const uint32_t krow = wrow + static_cast<uint32_t>((mi & 1) * 8 + ri) * 128u;   // K: matrices by key, then d
  const uint32_t vrow = wrow + static_cast<uint32_t>((mi >> 1) * 8 + ri) * 128u;  // V: by d, then key
  float* acc_sm = reinterpret_cast<float*>(smem + kAccOff);
  float* ml_sm = reinterpret_cast<float*>(smem + kMlOff);
  int it = 0;
  // Q as the B operand: b0 = Q[head r4][16 kk + c2, +1], b1 the same 8 further.
  uint32_t qf[8][2];
  auto load_q = [&]() {
    const T* qp = static_cast<const T*>(p.q) + seg.b * p.q_sb + (seg.hk * p.group + r4) * p.q_sh + c2;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      qf[kk][0] = r4 < p.group ? *reinterpret_cast<const uint32_t*>(qp + kk * 16) : 0u;
      qf[kk][1] = r4 < p.group ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8) : 0u;
    }
  };
  // kClustered: what this CTA has of the two heads that a warp joins, four columns a lane.
  float4 mine_a[kGroup / kConsumers];
  float2 mine_ml[kGroup / kConsumers];
  if constexpr (kClustered) {
#pragma unroll
    for (int u = 0; u < kGroup / kConsumers; ++u) {
      mine_a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      mine_ml[u] = make_float2(-INFINITY, 0.f);
    }
  }
  bool more = seg.next();
  if (more) load_q();
  while (more) {
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      const int s = it % kStages;
      // After a timeout the segment walk goes on without waits or work, so
      // that every consumer still reaches the same barriers.
      if (ok) ok = mbar_wait_warp_lim(full_bar(s), (it / kStages) & 1, abort_flag, wlim);
      // The phase is complete; each lane's own probe gives it acquire order on the copied bytes.
      if (ok) (void)mbar_test_wait(full_bar(s), (it / kStages) & 1);
      if (ok && ((valid[s] >> warp) & 1u)) {
        int t = 0, rows = 0;  // the position of the 16 keys; kListed: how many of them there are
        if constexpr (kListed)
          rows = (valid[s] >> (4 + 5 * warp)) & 31u;
        else
          t = seg.tiles.pos(tile) + warp * 16;
        const uint32_t kb = sbase + kRingOff + s * 2 * kTileBytes + krow;
        const uint32_t vb = sbase + kRingOff + s * 2 * kTileBytes + kTileBytes + vrow;
        float sc[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const int ch = kk * 2 + (mi >> 1);
          uint32_t a[4];
          ldmatrix4(kb + (ch >> 3) * half + (((ch & 7) ^ ri) << 4), a);
          mma_16x8x16<T>(sc[kk & 1], a, qf[kk][0], qf[kk][1]);
        }
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (sc[0][e] + sc[1][e]) * p.scale_log2;
        // Some of the 16 keys may be hidden (ends of the sequence, the window
        // and the prefix): their scores become -inf and their V rows zero,
        // whatever the page holds there.
        bool whole;
        if constexpr (kListed)
          whole = rows == 16;
        else
          whole = t + 16 <= seg.tiles.n && (t >= seg.tiles.lo || t + 16 <= p.w.prefix);
        uint32_t vm0 = ~0u, vm1 = ~0u;
        if (!whole) {
          auto see = [&](int k) -> bool {
            if constexpr (kListed)
              return k < rows;
            else
              return t + k < seg.tiles.n && (t + k >= seg.tiles.lo || t + k < p.w.prefix);
          };
          if (!see(r4)) x[0] = x[1] = -INFINITY;
          if (!see(r4 + 8)) x[2] = x[3] = -INFINITY;
          vm0 = (see(c2) ? 0xffffu : 0u) | (see(c2 + 1) ? 0xffff0000u : 0u);
          vm1 = (see(c2 + 8) ? 0xffffu : 0u) | (see(c2 + 9) ? 0xffff0000u : 0u);
        }
        float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
        }
        float pr[4];
        const bool grow = mx[0] > m[0] || mx[1] > m[1];
        const float mn[2] = {fmaxf(m[0], mx[0]), fmaxf(m[1], mx[1])};
        const float off[2] = {mn[0] == -INFINITY ? 0.f : mn[0], mn[1] == -INFINITY ? 0.f : mn[1]};
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = ex2(x[e] - off[e & 1]);
        if (__any_sync(0xffffffffu, grow)) {
          const float a0 = ex2(m[0] - off[0]), a1 = ex2(m[1] - off[1]);
          l[0] *= a0;
          l[1] *= a1;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[i][0] *= a0;
            acc[i][1] *= a1;
            acc[i][2] *= a0;
            acc[i][3] *= a1;
          }
          m[0] = mn[0];
          m[1] = mn[1];
        }
        l[0] += pr[0] + pr[2];
        l[1] += pr[1] + pr[3];
        const uint32_t b0 = transpose8(DT<T>::pack(pr[0], pr[1]));
        const uint32_t b1 = transpose8(DT<T>::pack(pr[2], pr[3]));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int ch = i * 2 + (mi & 1);
          uint32_t a[4];
          ldmatrix4_trans(vb + (ch >> 3) * half + (((ch & 7) ^ ri) << 4), a);
          if (!whole) {
            a[0] &= vm0;
            a[1] &= vm0;
            a[2] &= vm1;
            a[3] &= vm1;
          }
          mma_16x8x16<T>(acc[i], a, b0, b1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(s));
    }

    const int b = seg.b, hk = seg.hk;
    const bool whole_pair = seg.t0 == 0 && seg.t1 == seg.tiles.count;
    // A part is kept as the share's first (0) or last (1) segment.
    const int place = 2 * static_cast<int>(blockIdx.x) + (seg.seen > 0 ? 1 : 0);
    if (!kClustered && tid == 0 && seg.left == 0) {
      // When the share ends inside a pair that began in it, the pair is joined for it.
      const int rest = seg.t0 == 0 ? seg.tiles.count - seg.t1 : 0;
      const int parts = rest > 0 ? sh.owner(sh.first(blockIdx.x + 1) + rest - 1) - static_cast<int>(blockIdx.x) + 1 : 0;
      p.joins[blockIdx.x] = make_int4(parts, b, hk, place);
    }
    // The next segment's Q is on its way while this one is joined.
    more = seg.next();
    if (more) load_q();

    // Join the four warps: (m, l, acc) through shared memory, then a warp sums
    // two heads, a lane four columns of each.
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
    if (r4 == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ml_sm[(warp * kGroup + c2 + e) * 2] = m[e];
        ml_sm[(warp * kGroup + c2 + e) * 2 + 1] = l[e];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc_sm[(warp * kGroup + c2 + (e & 1)) * kAccRow + i * 16 + r4 + (e >> 1) * 8] = acc[i][e];
    named_bar_sync(1, kConsumers * 32);
    const long long slot = static_cast<long long>(place) * p.group;
    // After a timeout anywhere in the CTA the segment is incomplete: store nothing.
    if (ok && *abort_flag == 0) {
#pragma unroll
      for (int u = 0; u < kGroup / kConsumers; ++u) {
        const int g = warp + u * kConsumers;
        if (g >= p.group) break;
        float mw[kConsumers], M = -INFINITY, L = 0.f;
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) {
          mw[w] = ml_sm[(w * kGroup + g) * 2];
          M = fmaxf(M, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) {
          const float a = M == -INFINITY ? 0.f : ex2(mw[w] - M);
          const float4 x = *reinterpret_cast<const float4*>(acc_sm + (w * kGroup + g) * kAccRow + lane * 4);
          L += a * ml_sm[(w * kGroup + g) * 2 + 1];
          A.x += a * x.x;
          A.y += a * x.y;
          A.z += a * x.z;
          A.w += a * x.w;
        }
        if constexpr (kClustered) {
          mine_a[u] = A;
          mine_ml[u] = make_float2(M, L);
          continue;
        }
        if (whole_pair)
          store_row<T>(out + b * p.o_sb + (hk * p.group + g) * p.o_sh, lane, A, L);
        else
          *reinterpret_cast<float4*>(p.part_acc + (slot + g) * kD + lane * 4) = A;
        if (!whole_pair && lane == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + g) * 2) = make_float2(M, L);
      }
    }
    named_bar_sync(1, kConsumers * 32);  // the joining buffers are free again
  }

  if constexpr (kClustered) {
    // Every CTA is done with its ring when the first barrier lets it through; the parts
    // then go into the first one's: [rank][head][kD], and (m, l, whether it is whole).
    ok = ok && *abort_flag == 0;
    const int rank = blockIdx.x % kCluster;
    const int pair = blockIdx.x / kCluster;
    constexpr int kMlAt = kCluster * kGroup * kD * 4;
    cluster_sync();
    uint32_t dst;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(sbase + kRingOff), "r"(0));
#pragma unroll
    for (int u = 0; u < kGroup / kConsumers; ++u) {
      const int slot = rank * kGroup + warp + u * kConsumers;
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + slot * kD * 4 + lane * 16),
                   "f"(mine_a[u].x), "f"(mine_a[u].y), "f"(mine_a[u].z), "f"(mine_a[u].w)
                   : "memory");
      if (lane == 0)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %3};" ::"r"(dst + kMlAt + slot * 16),
                     "f"(mine_ml[u].x), "f"(mine_ml[u].y), "f"(ok ? 1.f : 0.f)
                     : "memory");
    }
    cluster_sync();
    if (rank != 0) return;
#pragma unroll
    for (int u = 0; u < kGroup / kConsumers; ++u) {
      const int g = warp + u * kConsumers;
      if (g >= p.group) break;
      float4 ml[kCluster];
      float mn = -INFINITY;
      bool whole = true;
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        ml[r] = *reinterpret_cast<const float4*>(smem + kRingOff + kMlAt + (r * kGroup + g) * 16);
        mn = fmaxf(mn, ml[r].x);
        whole = whole && ml[r].z != 0.f;
      }
      PartSum sum;
      const float off = mn == -INFINITY ? 0.f : mn;
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        const float4 a = *reinterpret_cast<const float4*>(smem + kRingOff + (r * kGroup + g) * kD * 4 + lane * 16);
        // A part without a maximum has sums of 0 or NaN, which are added as they are.
        if (ml[r].x == -INFINITY)
          sum.l += ml[r].y;
        else
          sum.add(off, ml[r].x, ml[r].y, a);
      }
      // After a timeout in any CTA the result is incomplete: store nothing.
      if (whole)
        store_row<T>(out + (pair / p.heads_kv) * p.o_sb + (pair % p.heads_kv * p.group + g) * p.o_sh, lane, sum.a,
                     sum.l);
    }
  }
}

// One CTA per (share, head of the group): joins the parts of the pair whose
// first part ends the share, if there is one. Its warps (one for every eight
// parts, up to four) take the parts in turn, four columns a lane and eight
// parts in flight; the warps' sums are then added in order, so the result is
// the same every time. A CTA for each head rather than a warp of one CTA: 12289
// rows at 56/8 heads (37 parts a pair; 50 MB that stay in L2 from call to call)
// take 13.2 us a call instead of 16.5, 300 rows at 16/16 heads 6.6 instead of
// 7.0; the batches run alike.
constexpr int kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const DecodeParams p) {
  // The next call's kernel (a programmatic dependent too) may start its
  // set-up now; it waits for this grid before touching memory.
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float sm_m[kJoinWarps], sm_l[kJoinWarps];
  __shared__ float4 sm_a[kJoinWarps][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int x = blockIdx.x;
  const int g = blockIdx.y;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int4 job = p.joins[x];
  const int parts = job.x;
  if (parts == 0) return;
  const int warps = min(kJoinWarps, (parts + 7) / 8);
  // The first part is the last segment of its share, the others open theirs.
  PartSum sum;
  if (warp < warps)
    sum.add_parts(p.part_ml, p.part_acc, warp, warps, parts, lane,
                  [&](int i) -> long long { return (i == 0 ? job.w : 2ll * (x + i)) * p.group + g; });
  if (warps > 1) {
    if (lane == 0) {
      sm_m[warp] = sum.m;
      sm_l[warp] = sum.l;
    }
    sm_a[warp][lane] = sum.a;
    __syncthreads();
    float mn = -INFINITY;
    for (int w = 0; w < warps; ++w) mn = fmaxf(mn, sm_m[w]);
    sum = PartSum();
    const float off = mn == -INFINITY ? 0.f : mn;
    for (int w = 0; w < warps; ++w) sum.add(off, sm_m[w], sm_l[w], sm_a[w][lane]);
  }
  if (warp == 0)
    store_row<T>(static_cast<T*>(p.o) + job.y * p.o_sb + (job.z * p.group + g) * p.o_sh, lane, sum.a, sum.l);
}

// Tensor map of a pool [num_pages, H, page_size, D]: dims (64 d, page rows, 2
// d-halves, heads, pages), box = (64 d, box_rows, box_halves, 1, 1) with the
// 128-byte swizzle; pages outside the pool read as zero.
static int make_map_pages(CUtensorMap* m, const void* base, int dtype, int pages, int heads, int page_size,
                          long long sp, long long sh, long long st, int box_rows, int box_halves, const char* name) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return sabre_fail(SABRE_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  if (sp >= (1ll << 39) || sh >= (1ll << 39) || st >= (1ll << 39))
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: stride too large", name);
  const cuuint64_t gdim[5] = {64u, (cuuint64_t)page_size, 2u, (cuuint64_t)heads, (cuuint64_t)pages};
  const cuuint64_t gstr[4] = {(cuuint64_t)st * 2, 128u, (cuuint64_t)sh * 2, (cuuint64_t)sp * 2};
  const cuuint32_t box[5] = {64u, (cuuint32_t)box_rows, (cuuint32_t)box_halves, 1u, 1u};
  const cuuint32_t estr[5] = {1u, 1u, 1u, 1u, 1u};
  const CUresult r =
      fn(m, dtype == SABRE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
         const_cast<void*>(base), gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return sabre_fail(SABRE_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", name, (int)r);
  return SABRE_OK;
}

// Checks of the query side, shared by the attention entry points.
static int check_queries(const char* fn, const void* q, const void* o, int heads_q, int heads_kv, int prefix,
                         const int64_t* q_strides, const int64_t* o_strides) {
  if (!q || !o || !q_strides || !o_strides) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  if (heads_q <= 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: sizes must be positive", fn);
  if (heads_q % heads_kv != 0 || heads_q / heads_kv > kGroup)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: heads_q/heads_kv must be an integer <= %d", fn, kGroup);
  if (prefix < 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: num_prefix_tokens %d < 0", fn, prefix);
  if (!aligned16(q) || !aligned16(o)) return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: q/o must be 16-byte aligned", fn);
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] % 8 != 0 || o_strides[i] % 8 != 0)
      return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: q/o strides must be multiples of 8 elements", fn);
  return SABRE_OK;
}

static float scale_log2(float softmax_scale) {
  return (softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf(static_cast<float>(kD))) * 1.4426950408889634f;
}

// Parts of two segments of every share, and the shares' joins.
static size_t decode_workspace(int group) {
  return kDecCtas * sizeof(int4) + static_cast<size_t>(2) * kDecCtas * group * (kD + 2) * sizeof(float);
}

template <typename T, DecodeMode kMode>
static cudaError_t launch_paged_decode(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p,
                                       cudaStream_t s) {
  const auto kernel = paged_decode_kernel<T, kMode>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDecSmem);
  if (e != cudaSuccess) return e;
  if (kMode == kInClusters)
    return launch_cluster(dim3(p.c.batch * p.heads_kv * kCluster), kCluster, kDecThreads, kDecSmem, s, kernel, mk, mv,
                          p);
  e = launch_dependent(dim3(p.ctas), kDecThreads, kDecSmem, s, kernel, mk, mv, p);
  if (e != cudaSuccess || p.ctas == 1) return e;  // a single share is finished where it is
  return launch_dependent(dim3(p.ctas - 1, p.group), kJoinWarps * 32, 0, s, paged_join_kernel<T>, p);
}

// Both decode entries: over the pages of `lists`, or (null) over all rows or the window's.
static int decode_call(const char* fn, const void* q, const void* k_pages, const void* v_pages, void* o,
                  const int32_t* page_table, const int32_t* seq_lens, const Lists* lists, int batch, int heads_q,
                  int heads_kv, int head_dim, int num_pages, int page_size, int max_pages, int window,
                  int num_prefix_tokens, const int64_t* q_strides, const int64_t* kp_strides,
                  const int64_t* vp_strides, const int64_t* o_strides, int64_t table_stride, float softmax_scale,
                  int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  DecodeParams p;
  int st = make_cache(&p.c, fn, k_pages, v_pages, page_table, seq_lens, batch, heads_kv, head_dim, num_pages,
                      page_size, max_pages, kp_strides, vp_strides, table_stride, dtype);
  if (st == SABRE_OK) st = check_queries(fn, q, o, heads_q, heads_kv, num_prefix_tokens, q_strides, o_strides);
  if (st != SABRE_OK) return st;
  p.lists = lists ? *lists : Lists{};
  p.w = Window{window, window < 0 ? 0 : num_prefix_tokens};
  p.q = q;
  p.o = o;
  p.q_sb = q_strides[0];
  p.q_sh = q_strides[1];
  p.o_sb = o_strides[0];
  p.o_sh = o_strides[1];
  p.heads_kv = heads_kv;
  p.group = heads_q / heads_kv;
  p.scale_log2 = scale_log2(softmax_scale);
  if (!workspace || workspace_bytes < decode_workspace(p.group))
    return sabre_fail(SABRE_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn, workspace_bytes,
                      decode_workspace(p.group));
  if (!aligned16(workspace)) return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
  // No more CTAs than the table has tiles, nor parts of a pair than pay for
  // their joining (12000 rows of one KV head, 188 tiles: 11.2 us a call in 188
  // parts, 9.3 in 94; below that a tile a CTA is the fastest).
  if (lists && static_cast<long long>(page_size) * lists->cap > kMaxRows)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: page_size * list entries exceeds 2^30 rows", fn);
  const long long span = lists ? static_cast<long long>(page_size) * lists->cap
                               : static_cast<long long>(page_size) * max_pages;
  const long long per_head = static_cast<long long>(batch) * ((span + kTile - 1) / kTile);
  const long long tiles = per_head * heads_kv;
  // The kernel adds up a sequence's (with lists: a pair's) tiles in 32 bits.
  if ((lists ? tiles : per_head) > 0x7fffffffll)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, lists ? "%s: batch * heads_kv * page_size * list entries exceeds 2^37 rows"
                                                   : "%s: batch * page_size * max_pages exceeds 2^37 rows", fn);
  long long ctas = static_cast<long long>(batch) * heads_kv * kMaxParts;
  if (ctas > tiles) ctas = tiles;
  p.ctas = static_cast<int>(ctas < kDecCtas ? ctas : kDecCtas);
  p.joins = static_cast<int4*>(workspace);
  p.part_acc = reinterpret_cast<float*>(p.joins + kDecCtas);
  p.part_ml = p.part_acc + static_cast<size_t>(2) * kDecCtas * p.group * kD;
  CUtensorMap mk, mv;
  if ((st = make_map_pages(&mk, k_pages, dtype, num_pages, heads_kv, page_size, p.c.k_sp, p.c.k_sh, p.c.k_st,
                           kBoxRows, 2, "k_pages")) != SABRE_OK)
    return st;
  if ((st = make_map_pages(&mv, v_pages, dtype, num_pages, heads_kv, page_size, p.c.v_sp, p.c.v_sh, p.c.v_st,
                           kBoxRows, 2, "v_pages")) != SABRE_OK)
    return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  // tiles: of all pairs.
  const long long pairs = static_cast<long long>(batch) * heads_kv;
  if (lists && pairs <= kClusterPairs && tiles > pairs && tiles <= pairs * kCluster * kClusterTiles)
    e = dtype == SABRE_BF16 ? launch_paged_decode<__nv_bfloat16, kInClusters>(mk, mv, p, s)
                            : launch_paged_decode<__half, kInClusters>(mk, mv, p, s);
  else if (lists)
    e = dtype == SABRE_BF16 ? launch_paged_decode<__nv_bfloat16, kOverPages>(mk, mv, p, s)
                            : launch_paged_decode<__half, kOverPages>(mk, mv, p, s);
  else
    e = dtype == SABRE_BF16 ? launch_paged_decode<__nv_bfloat16, kDense>(mk, mv, p, s)
                            : launch_paged_decode<__half, kDense>(mk, mv, p, s);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

}  // namespace paged
}  // namespace sabre

extern "C" {

size_t sabre_paged_decode_workspace_size(int batch, int heads_q, int heads_kv, int head_dim) {
  using namespace sabre::paged;
  if (batch <= 0 || heads_q <= 0 || heads_kv <= 0 || head_dim != kD || heads_q % heads_kv != 0) return 0;
  return decode_workspace(heads_q / heads_kv);
}

int sabre_paged_decode(const void* q, const void* k_pages, const void* v_pages, void* o, const int32_t* page_table,
                       const int32_t* seq_lens, int batch, int heads_q, int heads_kv, int head_dim, int num_pages,
                       int page_size, int max_pages, int window, int num_prefix_tokens, const int64_t* q_strides,
                       const int64_t* kp_strides, const int64_t* vp_strides, const int64_t* o_strides,
                       int64_t table_stride, float softmax_scale, int dtype, void* workspace, size_t workspace_bytes,
                       void* stream) {
  return sabre::paged::decode_call("sabre_paged_decode", q, k_pages, v_pages, o, page_table, seq_lens, nullptr, batch,
                              heads_q, heads_kv, head_dim, num_pages, page_size, max_pages, window, num_prefix_tokens,
                              q_strides, kp_strides, vp_strides, o_strides, table_stride, softmax_scale, dtype,
                              workspace, workspace_bytes, stream);
}

int sabre_paged_decode_listed(const void* q, const void* k_pages, const void* v_pages, void* o,
                              const int32_t* page_table, const int32_t* seq_lens, const int32_t* lists,
                              const int32_t* counts, int list_entries, int batch, int heads_q, int heads_kv,
                              int head_dim, int num_pages, int page_size, int max_pages, const int64_t* q_strides,
                              const int64_t* kp_strides, const int64_t* vp_strides, const int64_t* o_strides,
                              const int64_t* list_strides, const int64_t* count_strides, int64_t table_stride,
                              float softmax_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sabre::paged;
  const char* fn = "sabre_paged_decode_listed";
  Lists l;
  const int st = make_lists(&l, fn, lists, counts, list_entries, list_strides, count_strides);
  if (st != SABRE_OK) return st;
  return decode_call(fn, q, k_pages, v_pages, o, page_table, seq_lens, &l, batch, heads_q, heads_kv, head_dim, num_pages,
                page_size, max_pages, -1, 0, q_strides, kp_strides, vp_strides, o_strides, table_stride,
                softmax_scale, dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
