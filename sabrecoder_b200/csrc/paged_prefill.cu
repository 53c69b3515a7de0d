// Causal attention of a ragged batch of new rows over a paged K/V cache, with
// an optional sliding window and prefix tokens that stay visible.
//
// o_i = sum_j p_ij v_j / sum_j p_ij over the visible keys j, in one pass over
// the keys with a running maximum per row (tensor-bound: 512 flops per query
// head and visible pair, while a tile of K and V is read once for 128 rows).
//
// Work split: a CTA owns 128 rows of one KV head and one sequence: 128 / g
// consecutive tokens times the g query heads of the group, token by token, so
// that a group's heads share each K/V tile, a short continuation fills its
// rows, and a window's span grows by fewer tokens. Its key tiles (64 keys) are
// the prefix tiles, then those of the window: nothing else is visited. Many
// (row tile, KV head) pairs run as one CTA each, in the batch's reverse order
// and so heaviest first within a sequence. When there are too few of them to
// fill the card evenly, and they are long, their key tiles are dealt out to two
// CTAs per SM instead (kShares, see RowShares): a CTA walks its share as
// segments, a pair inside one share is finished there, the others leave (m, l,
// O) per row and paged_combine_kernel adds them in share order. Sequences,
// lengths and pages are only read on the device, so a captured call follows
// them.
//
// Roles, tensor-memory layout and barrier protocol are those of
// prefill_bsa.cu (224 threads, two CTAs per SM: warps 0-3 softmax, 4 Q and K
// producer, 5 MMA issuer, 6 V producer; S = Q K^T of M=128 N=64 into two
// buffers, P over its S, O += P V with P from tensor memory); from one segment
// of a share to the next each role goes on by itself (model-checked:
// tests/test_paged_prefill_protocol.py, the V tiles below in
// tests/test_paged_prefill_zeroing_protocol.py). Different here: tiles come box
// by box from pages (a TMA box is min(page_size, 64) rows; absent pages and
// boxes that no row sees are read outside the pool and give zeros), and V rows
// that none of the CTA's rows sees (past the sequence's end, before the window)
// are zeroed in shared memory before their tile is handed to the MMA, since 0 *
// NaN would reach the result.
// P is rounded to the type of V for the product; scores, sums and O are fp32.
// A 12288-row prompt at 16/16 heads takes 555 us (1.11 PFLOP/s) in bursts of
// replays and 650 us (950 TFLOP/s) in a loop that holds the card at its power
// cap; the times in the comments below are of bursts. Neither the tensor pipe nor
// the exponential unit is busy more than about half the time: what bounds a CTA
// is its chain from S over the softmax to P.V.
namespace sabre {
namespace paged {
namespace pre {

using prefill::row_max64;

constexpr int kThreads = 224;
constexpr int kRows = 128;
constexpr int kShareBatch = 128;  // sequences of a call that runs in shares, at most
constexpr int kMinShare = 8;      // key tiles of a share, at least
constexpr int kMaxPairs = 2 * kDecCtas;
constexpr int kQBytes = kRows * kD * 2;  // [d-half][128 rows][128 B], 128-byte swizzle
constexpr int kQOff = 0;
constexpr int kKOff = kQOff + kQBytes;
constexpr int kVOff = kKOff + 2 * kTileBytes;
constexpr int kBarOff = kVOff + 2 * kTileBytes;
enum Bar {
  Q_FULL = 0,
  K_FULL = 1,  // [2]
  V_FULL = 3,  // [2]
  PRO = 5,     // [2] S(0), S(1) done
  DONE = 7,    // [2] commit C(j) on DONE[j%2]: P.V(j) and S(j+2) done
  P_FULL = 9,  // [2] P(j) stored over S buffer j%2 (one arrival per softmax warp)
  V_RAW = 11,  // the copies of a V tile some of whose rows are zeroed before V_FULL
  MMA_DONE = 12,
  NUM_BARS = 13
};
constexpr int kMiscOff = kBarOff + NUM_BARS * 8;
constexpr int kSmemBytes = kMiscOff + 72;
// kShares also keeps, per sequence: first row, rows, length, row tiles before it; and 64 counts.
constexpr int kSeqOff = kSmemBytes;
constexpr int kShareSmemBytes = kSeqOff + (4 * kShareBatch + 64) * 4;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kTmemS = 128;  // + 64 * buffer

struct Params {
  Cache c;
  Window w;
  const int32_t* starts;
  void* o;
  // kShares: the parts of two segments of every share, and for every pair (row
  // tile times KV heads plus head) {parts (0: finished), share and place of the
  // first, -}, {first row, tokens, -, -}.
  float* part_acc;  // [2 * kDecCtas][kRows][D]
  float* part_ml;   // [2 * kDecCtas][kRows][2]
  int4* joins;      // [kMaxPairs][2]
  long long o_sr, o_sh;
  int rows, heads_kv, group, tokens;  // tokens of a row tile: 128 / group
  int box_shift, slots;               // slots: row tiles of the grid
  int head_major, ctas;               // ctas: of a call in shares, else 0
  float scale_log2;
};

// P = 2^(x * sl2 - moff) for one row of 64 scores (-inf gives 0), rounded to the
// storage type and stored at column `col` of tensor memory, half a row at a time
// so that the first half's store runs under the exponentials of the second;
// returns the sum of the fp32 values.
template <typename T>
__device__ __forceinline__ float exp_store(const float (&x)[64], float sl2, float moff, uint32_t col) {
  const uint64_t sc = f2_pack(sl2, sl2);
  const uint64_t off = f2_pack(-moff, -moff);
  uint64_t acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f2_pack(0.f, 0.f);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y0, y1;
      f2_unpack(f2_fma(f2_pack(x[32 * half + 2 * i], x[32 * half + 2 * i + 1]), sc, off), y0, y1);
      const float p0 = ex2(y0);
      const float p1 = ex2(y1);
      acc[i & 3] = f2_add(acc[i & 3], f2_pack(p0, p1));
      pk[i] = DT<T>::pack(p0, p1);
    }
    tmem_st16(col + 16 * half, pk);
  }
  float s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(acc[i], s[2 * i], s[2 * i + 1]);
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// Bits [0, x) of a 64-bit mask, x clamped to [0, 64].
__device__ __forceinline__ unsigned long long low_bits(int x) {
  return x >= 64 ? ~0ull : (x <= 0 ? 0ull : (1ull << x) - 1ull);
}

// What a CTA works on: rows [row0, row0 + count) of sequence b, whose first is
// at position pos0, and the key tiles they see between them.
struct Job {
  int b, row0, count, pos0, n, lo, head, from, tiles;
  __device__ __forceinline__ int pos(int i) const { return (i < head ? i : from + i - head) * kTile; }
  __device__ __forceinline__ bool any(const Window& w, int t, int rows) const {
    return t < n && (t + rows > lo || t < w.prefix);
  }
};

// The row tile at row r of sequence b, whose `len` new rows begin at row
// `first` and end its `length` rows.
__device__ __forceinline__ Job make_job(const Params& p, int b, int r, int first, int len, int length) {
  Job job;
  job.b = b;
  job.row0 = first + r;
  job.count = min(p.tokens, len - r);
  job.pos0 = length - len + r;
  job.n = min(min(max(length, 0), p.c.capacity()), max(job.pos0 + job.count, 0));  // keys that some row may see
  job.lo = p.w.first(job.pos0);
  job.from = job.lo / kTile;
  const int whole = (job.n + kTile - 1) / kTile;
  job.head = min((min(min(p.w.prefix, job.lo), job.n) + kTile - 1) / kTile, job.from);
  job.tiles = job.head + max(0, whole - job.from);
  return job;
}

// Exclusive prefix sum over the CTA's threads; scratch: 8 ints. `all`: the total.
__device__ __forceinline__ int prefix_sum(int mine, int* scratch, int& all) {
  const int tid = threadIdx.x;
  int incl = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, s);
    if ((tid & 31) >= s) incl += up;
  }
  __syncthreads();  // scratch is free
  if ((tid & 31) == 31) scratch[tid >> 5] = incl;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    before += w < (tid >> 5) ? scratch[w] : 0;
    all += scratch[w];
  }
  return before + incl - mine;
}

// Row tile `slot` of the batch, found by the whole CTA; scratch: 16 ints.
__device__ __forceinline__ bool find_job(const Params& p, int slot, int* scratch, Job& job) {
  const int tid = threadIdx.x;
  const int per = (p.c.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.c.batch), b1 = min(b0 + per, p.c.batch);
  // The first length comes with the starts, not after them: one round trip
  // for as many sequences as threads.
  const int len0 = b0 < b1 ? p.c.seq_lens[b0] : 0;
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = row_start(p.starts, b + 1, p.rows) - row_start(p.starts, b, p.rows);
    mine += (max(len, 0) + p.tokens - 1) / p.tokens;
  }
  if (tid == 0) scratch[8] = -1;
  int all = 0;
  int left = slot - prefix_sum(mine, scratch, all);
  if (left >= 0 && left < mine) {
    for (int b = b0; b < b1; ++b) {
      const int first = row_start(p.starts, b, p.rows);
      const int len = row_start(p.starts, b + 1, p.rows) - first;
      const int nt = (max(len, 0) + p.tokens - 1) / p.tokens;
      if (left < nt) {
        scratch[8] = b;
        scratch[9] = left * p.tokens;
        scratch[10] = first;
        scratch[11] = len;
        scratch[12] = b == b0 ? len0 : p.c.seq_lens[b];
        break;
      }
      left -= nt;
    }
  }
  __syncthreads();
  if (scratch[8] < 0) return false;
  job = make_job(p, scratch[8], scratch[9], scratch[10], scratch[11], scratch[12]);
  return true;
}

// A place in a call's order of work: key tile `tile` of KV head hk and the row
// tile that begins at row r of sequence b.
struct RowPlace {
  int b, r, hk, tile;
};

// How a call in shares is dealt out. Whole parts: every pair is cut into equal
// parts of its own and a CTA has one of them, when that leaves none with more
// than kSlack key tiles above the mean. Else the tiles of all pairs, in order,
// are cut into equal shares: a CTA may then finish one pair and begin another,
// which costs it a second start and read-out, about kSlack tiles' time (300
// rows on 4000 at 16/16 heads, 48 pairs of 66 tiles: 30 us a call in parts, 35
// in shares; 256 rows on 1000 at 56/8 heads, 120 pairs of 18: 31 and 38; 8
// sequences of 32 rows on 2000 to 4000, ragged, in shares: 52).
constexpr int kSlack = 6;
struct RowShares : Shares {
  bool whole;
  int parts;        // whole: parts of the pair if this CTA has the first of several, else 0
  long long units;  // key tiles of this CTA
};

// kShares: lists the sequences in seq, then finds this CTA's share and the
// place of its first tile; scratch: 16 ints. Rows of row tiles that see no key
// are zeroed on the way. False without a share.
template <typename T>
__device__ __forceinline__ bool find_share(const Params& p, int* seq, int* scratch, RowShares& sh, RowPlace& at) {
  const int tid = threadIdx.x;
  int* const first_slot = seq + 3 * kShareBatch;
  int slots = 0;
  if (tid < p.c.batch) {
    const int first = row_start(p.starts, tid, p.rows);
    const int len = max(row_start(p.starts, tid + 1, p.rows) - first, 0);
    slots = (len + p.tokens - 1) / p.tokens;
    seq[tid] = first;
    seq[kShareBatch + tid] = len;
    seq[2 * kShareBatch + tid] = p.c.seq_lens[tid];
  }
  int nslots = 0;
  const int before = prefix_sum(slots, scratch, nslots);
  if (tid < p.c.batch) first_slot[tid] = before;
  __syncthreads();
  auto sequence = [&](int slot) -> int {  // the last b with first_slot[b] <= slot
    int lo = 0, hi = p.c.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (first_slot[mid] <= slot ? lo : hi) = mid;
    }
    return lo;
  };
  auto job_of = [&](int slot) -> Job {
    const int b = sequence(slot);
    return make_job(p, b, (slot - first_slot[b]) * p.tokens, seq[b], seq[kShareBatch + b], seq[2 * kShareBatch + b]);
  };
  const int per = (nslots + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, nslots), s1 = min(s0 + per, nslots);
  int mine = 0;
  for (int s = s0; s < s1; ++s) mine += job_of(s).tiles;
  int all = 0;
  const int ahead = prefix_sum(mine, scratch, all);
  const int units = p.heads_kv * p.group * (kD / 8);  // 16-byte stores of a row
  for (int s = blockIdx.x; s < p.slots; s += p.ctas) {
    const Job job = s < nslots ? job_of(s) : Job{};
    if (job.tiles > 0) continue;
    for (int h = tid; h < p.heads_kv; h += kThreads) p.joins[2 * (s * p.heads_kv + h)] = make_int4(0, 0, 0, 0);
    for (int i = tid; i < job.count * units; i += kThreads) {
      const int u = i % units;
      *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + static_cast<long long>(job.row0 + i / units) * p.o_sr +
                                u / (kD / 8) * p.o_sh + u % (kD / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (all == 0) return false;
  sh.total = static_cast<long long>(all) * p.heads_kv;
  // Parts of whole pairs of at most most + i tiles each, when so many CTAs do
  // for them all: the smallest i.
  const int most = static_cast<int>(max(static_cast<long long>(kMinShare), (sh.total + p.ctas - 1) / p.ctas));
  int count[kSlack + 1] = {};
  for (int s = s0; s < s1; ++s) {
    const int tiles = job_of(s).tiles;
#pragma unroll
    for (int i = 0; i <= kSlack; ++i) count[i] += (tiles + most + i - 1) / (most + i);
  }
  int* const counts = seq + 4 * kShareBatch;  // [kSlack + 1][8]
#pragma unroll
  for (int i = 0; i <= kSlack; ++i) {
    const int sum = __reduce_add_sync(0xffffffffu, count[i]);
    if ((tid & 31) == 0) counts[i * 8 + (tid >> 5)] = sum;
  }
  __syncthreads();
  int slack = kSlack + 1, mine_parts = 0;
#pragma unroll
  for (int i = kSlack; i >= 0; --i) {
    long long sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) sum += counts[i * 8 + w];
    if (sum * p.heads_kv <= p.ctas) slack = i, mine_parts = count[i];
  }
  sh.whole = slack <= kSlack;
  if (sh.whole) {
    int parts_all = 0;
    int left = static_cast<int>(blockIdx.x) - prefix_sum(mine_parts, scratch, parts_all) * p.heads_kv;
    sh.ctas = parts_all * p.heads_kv;
    if (static_cast<int>(blockIdx.x) >= sh.ctas) return false;
    if (left >= 0 && left < mine_parts * p.heads_kv) {
      for (int s = s0; s < s1; ++s) {
        const Job job = job_of(s);
        const int parts = (job.tiles + most + slack - 1) / (most + slack);
        if (left < parts * p.heads_kv) {
          const int k = left % parts;
          const long long from = static_cast<long long>(job.tiles) * k / parts;
          scratch[8] = job.b;
          scratch[9] = (s - first_slot[job.b]) * p.tokens;
          scratch[10] = left / parts;
          scratch[11] = static_cast<int>(from);
          scratch[12] = static_cast<int>(static_cast<long long>(job.tiles) * (k + 1) / parts - from);
          scratch[13] = k == 0 && parts > 1 ? parts : 0;
          break;
        }
        left -= parts * p.heads_kv;
      }
    }
  } else {
    sh.ctas = p.ctas;  // all busy: most > kMinShare, else parts would do
    long long left = sh.first(blockIdx.x) - static_cast<long long>(ahead) * p.heads_kv;
    if (left >= 0 && left < static_cast<long long>(mine) * p.heads_kv) {
      for (int s = s0; s < s1; ++s) {
        const Job job = job_of(s);
        const long long here = static_cast<long long>(job.tiles) * p.heads_kv;
        if (left < here) {
          scratch[8] = job.b;
          scratch[9] = (s - first_slot[job.b]) * p.tokens;
          scratch[10] = static_cast<int>(left / job.tiles);
          scratch[11] = static_cast<int>(left % job.tiles);
          break;
        }
        left -= here;
      }
    }
  }
  __syncthreads();
  at = RowPlace{scratch[8], scratch[9], scratch[10], scratch[11]};
  sh.units = sh.whole ? scratch[12] : sh.first(blockIdx.x + 1) - sh.first(blockIdx.x);
  sh.parts = scratch[13];
  return true;
}

// kShares: the CTA walks a share of all key tiles; else it owns a whole pair.
template <typename T, bool kShares>
__global__ void __launch_bounds__(kThreads, 2)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const uint32_t sbase = smem_u32(smem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kMiscOff + 4);
  auto bar = [&](int i) -> uint32_t { return sbase + kBarOff + 8u * i; };

  if (tid == 0) {
    const bool bad = (sbase & 1023u) != 0u;
    *abort_flag = bad ? 1 : 0;
    if (bad) record_status(SABRE_DEV_BAD_SMEM_ALIGN);
  }
  if (warp == 4 && lane == 0) {
    for (int i = 0; i < NUM_BARS; ++i) mbar_init(bar(i), i == P_FULL || i == P_FULL + 1 ? 4 : 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  // The set-up above overlaps the tail of the stream's previous kernel (this is
  // a programmatic dependent launch) and the loads below, whose barriers order
  // it before its use. Nothing before this line reads what that kernel wrote.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int* const scratch = reinterpret_cast<int*>(smem + kMiscOff + 8);
  int* const seq = reinterpret_cast<int*>(smem + kSeqOff);
  Job job;
  RowShares sh;
  RowPlace at;
  long long units = 0;  // key tiles of the share still to be done
  int hk = 0;
  bool some;
  if constexpr (kShares) {
    some = find_share<T>(p, seq, scratch, sh, at);
    if (some) units = sh.units;
  } else {
    // Later row tiles of a sequence see more keys: its heaviest first (sequences
    // come in the batch's reverse order, whatever their lengths). Row-major
    // (grid x = head) or head-major (grid x = row tile), as in prefill_bsa.cu.
    hk = p.head_major ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.x);
    some = find_job(p, p.slots - 1 - static_cast<int>(p.head_major ? blockIdx.x : blockIdx.y), scratch, job);
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int boxes = kTile >> p.box_shift;
  const int box_rows = 1 << p.box_shift;
  const bool start_ok = (*abort_flag == 0);

  // The barriers' phases run on over the segments: a wait's parity is that of a
  // first segment plus what the earlier ones completed: one phase a segment
  // (Q_FULL, PRO[0], MMA_DONE), one for each with a second tile (PRO[1]: twos),
  // one for each even (d0) or odd (d1) tile (K_FULL, V_FULL, P_FULL, DONE), one
  // for each tile that was zeroed (V_RAW: raws). No barrier can complete two
  // phases ahead of a waiter: the next segment's first loads wait for MMA_DONE,
  // which is committed after every other completion has been seen.
  int d0 = 0, d1 = 0, twos = 0, raws = 0;
  for (int segment = 0; some; ++segment) {
    const int seg_par = segment & 1, two_par = twos & 1;
    // After a timeout the walk goes on without work: every pair's record is written.
    const bool going = start_ok && (!kShares || __all_sync(0xffffffffu, *abort_flag == 0));
    // Parity of the completion for the k-th tile of stage s (0 or 1).
    auto par = [&](int s, int k) -> uint32_t { return static_cast<uint32_t>(k + (s ? d1 : d0)) & 1u; };
    // This segment: key tiles [j0, j0 + nt) of the pair.
    int j0 = 0, nt = job.tiles, place = 0;
    bool part = false;
    if constexpr (kShares) {
      if (segment > 0) {
        at.tile = 0;
        if (++at.hk == p.heads_kv) {
          at.hk = 0;
          at.r += p.tokens;
        }
      }
      for (;;) {  // the next row tile that sees a key; units > 0: there is one
        while (at.b < p.c.batch - 1 && at.r >= seq[kShareBatch + at.b]) {
          ++at.b;
          at.r = 0;
        }
        job = make_job(p, at.b, at.r, seq[at.b], seq[kShareBatch + at.b], seq[2 * kShareBatch + at.b]);
        if (job.tiles > 0 || job.count <= 0) break;
        at.r += p.tokens;
      }
      hk = at.hk;
      j0 = at.tile;
      nt = static_cast<int>(min(static_cast<long long>(job.tiles - j0), units));
      units -= nt;
      part = nt < job.tiles;
      // A part is kept as the share's first (0) or last (1) segment.
      place = 2 * static_cast<int>(blockIdx.x) + (segment > 0 ? 1 : 0);
      if (j0 == 0 && tid == 0) {
        // The pair begins here: does it end here too?
        const int rest = job.tiles - nt;
        int parts = sh.parts;
        if (!sh.whole)
          parts = rest > 0 ? sh.owner(sh.first(blockIdx.x + 1) + rest - 1) - static_cast<int>(blockIdx.x) + 1 : 0;
        const int pair = (seq[3 * kShareBatch + at.b] + at.r / p.tokens) * p.heads_kv + hk;
        p.joins[2 * pair] = make_int4(parts, static_cast<int>(blockIdx.x), place, 0);
        p.joins[2 * pair + 1] = make_int4(job.row0, job.count, 0, 0);
      }
    }

    constexpr uint32_t kIdescQK = idesc_f16(128, 64, DT<T>::kBf16, false);
    constexpr uint32_t kIdescPV = idesc_f16(128, 128, DT<T>::kBf16, true);

    if (warp == 4 || warp == 6) {
      // ---------------- TMA producers (warp 4: K, warp 6: V) ----------------
      const bool is_k = (warp == 4);
      const int full0 = is_k ? K_FULL : V_FULL;
      const uint32_t ring = sbase + (is_k ? kKOff : kVOff);
      const CUtensorMap* map = is_k ? &tmK : &tmV;
      // The segment before is done with the Q tile and both stages (while its O is
      // still read out).
      bool ok = going;
      if (kShares && segment > 0 && ok) ok = mbar_wait_warp(bar(MMA_DONE), seg_par ^ 1, abort_flag);
      if (is_k && lane == 0 && ok) {
        mbar_arrive_expect_tx(bar(Q_FULL), static_cast<uint32_t>(p.group * p.tokens) * 256u);
        const uint64_t pol = l2_policy_evict_first();
        tma_load_4d_hint(sbase + kQOff, &tmQ, bar(Q_FULL), 0, 0, job.row0, hk, pol);
        tma_load_4d_hint(sbase + kQOff + kQBytes / 2, &tmQ, bar(Q_FULL), 64, 0, job.row0, hk, pol);
      }
      int issued = 0;    // tiles
      bool raw = false;  // the last tile went through V_RAW
      const bool began = ok;
      for (int i0 = 0; ok && i0 < nt * boxes; i0 += 32) {
        // The pages of the next 32 boxes, one per lane; num_pages reads zeros.
        int page = p.c.num_pages, off = 0;
        if (i0 + lane < nt * boxes) {
          const int t = job.pos(j0 + (i0 + lane) / boxes) + (((i0 + lane) % boxes) << p.box_shift);
          off = t & ((1 << p.c.page_shift) - 1);
          if (job.any(p.w, t, box_rows)) {
            const int pg = p.c.page_of(job.b, t);
            if (pg >= 0) page = pg;
          }
        }
        for (int i = i0; i < min(i0 + 32, nt * boxes); i += boxes) {
          const int j = i / boxes;
          const int s = j & 1;
          if (j >= 2) {
            // As in prefill_bsa.cu: K(j) may overwrite its stage after S(j-2)
            // (PRO[j-2] for j < 4, else in C(j-4)), V(j) after P.V(j-2) (C(j-2)).
            if (is_k && j < 4)
              ok = mbar_wait_warp(bar(PRO + (j - 2)), j == 2 ? seg_par : two_par, abort_flag);
            else
              ok = mbar_wait_warp(bar(DONE + s), par(s, (j >> 1) - (is_k ? 2 : 1)), abort_flag);
            if (!ok) break;
          }
          // Rows of V that none of this CTA's rows sees (past the end, before the
          // window) but that share a box with some that one does are zeroed.
          unsigned long long hidden = 0;
          if (!is_k) {
            const int t = job.pos(j0 + j);
            hidden = ~low_bits(job.n - t) | (low_bits(job.lo - t) & ~low_bits(p.w.prefix - t));
            for (int x = 0; x < boxes && hidden != 0ull; ++x) {  // a box that is hidden as a whole is zero already
              const unsigned long long box = low_bits(box_rows) << (x << p.box_shift);
              if ((hidden & box) == box) hidden &= ~box;
            }
          }
          const bool clean = hidden != 0ull;
          const uint32_t full = bar(clean ? V_RAW : full0 + s);
          if (lane == 0) mbar_arrive_expect_tx(full, kTileBytes);
          __syncwarp();
          const int x = lane - (i - i0);
          const uint32_t dst = ring + s * kTileBytes;
          if (x >= 0 && x < boxes) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              tma_load_page(dst + h * (kTileBytes / 2) + x * box_rows * 128, map, full, off, h, hk, page);
          }
          issued = j + 1;
          raw = clean;
          if (clean) {
            const int raw_par = raws++ & 1;
            ok = mbar_wait_warp(bar(V_RAW), raw_par, abort_flag);
            if (!ok) break;
            (void)mbar_test_wait(bar(V_RAW), raw_par);  // each lane's own acquire of the copied bytes
            // Half a warp zeroes the even rows, half the odd ones, 16 bytes a lane.
            uint8_t* const at16 = smem + kVOff + s * kTileBytes + ((lane >> 3) & 1) * (kTileBytes / 2) + (lane & 7) * 16;
            for (unsigned long long m = hidden & (0x5555555555555555ull << (lane >> 4)); m != 0ull; m &= m - 1ull)
              *reinterpret_cast<uint4*>(at16 + (__ffsll(m) - 1) * 128) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(full0 + s));
          }
        }
      }
      // Every issued copy must land before the CTA may exit.
      if (lane == 0 && began) {
        if (is_k) mbar_wait_drain(bar(Q_FULL), seg_par);
        for (int j = max(0, issued - 2); j < issued; ++j) {
          if (raw && j == issued - 1)
            mbar_wait_drain(bar(V_RAW), (raws - 1) & 1);
          else
            mbar_wait_drain(bar(full0 + (j & 1)), par(j & 1, j >> 1));
        }
      }
    } else if (warp == 5) {
      // ---------------- MMA issuer ----------------
      if (lane == 0 && going) {
        const uint64_t qd = smem_desc_sw128(sbase + kQOff, 16, 1024);
        const uint64_t kd0 = smem_desc_sw128(sbase + kKOff, 16, 1024);
        const uint64_t vd0 = smem_desc_sw128(sbase + kVOff, kTileBytes / 2, 1024);
        const uint32_t s_tmem = tmem + kTmemS;
        const unsigned long long lim = wait_limit_ns();
        auto wait = [&](int i, uint32_t parity) -> bool { return mbar_wait_lim<8>(bar(i), parity, abort_flag, lim); };
        bool ok = wait(Q_FULL, seg_par);
        auto issue_s = [&](int j) -> bool {
          const int ks = j & 1;
          if (!wait(K_FULL + ks, par(ks, j >> 1))) return false;
          tc_fence_after();
          const uint64_t kd = kd0 + static_cast<uint64_t>(ks * (kTileBytes >> 4));
          const uint32_t dst = s_tmem + 64 * ks;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint64_t qo = ((kk >> 2) * (kQBytes / 2) + (kk & 3) * 32) >> 4;
            const uint64_t ko = ((kk >> 2) * (kTileBytes / 2) + (kk & 3) * 32) >> 4;
            mma_f16_ss(dst, qd + qo, kd + ko, kIdescQK, kk > 0 ? 1u : 0u);
          }
          return true;
        };
        auto issue_pv = [&](int i) -> bool {
          const int pb = i & 1;
          if (!wait(V_FULL + pb, par(pb, i >> 1))) return false;
          if (!wait(P_FULL + pb, par(pb, i >> 1))) return false;
          tc_fence_after();
          const uint64_t vd = vd0 + static_cast<uint64_t>(pb * (kTileBytes >> 4));
          const uint32_t pa = s_tmem + 64 * pb;
          mma_f16_ts(tmem, pa, vd, kIdescPV, i > 0 ? 1u : 0u);
#pragma unroll
          for (int kk = 1; kk < 4; ++kk) mma_f16_ts(tmem, pa + 8 * kk, vd + kk * (2048 >> 4), kIdescPV, 1u);
          return true;
        };
        for (int j = 0; ok && j < 2 && j < nt; ++j) {
          ok = issue_s(j);
          if (ok) mma_commit(bar(PRO + j));
        }
        for (int j = 0; ok && j < nt; ++j) {
          if (!issue_pv(j)) { ok = false; break; }
          if (j + 2 < nt && !issue_s(j + 2)) { ok = false; break; }
          mma_commit(bar(DONE + (j & 1)));
        }
        if constexpr (kShares) {
          // The next segment's waiters start from known phases: C(nt-2), which
          // nobody else may wait for, has arrived too.
          for (int x = 0; ok && x < 2; ++x)
            if (nt > x) mbar_wait_drain(bar(DONE + x), par(x, (nt - x - 1) >> 1));
        }
        // Whatever was issued must finish before tensor memory is released.
        mma_commit(bar(MMA_DONE));
        mbar_wait_drain(bar(MMA_DONE), seg_par);
      }
    } else {
      // ---------------- softmax + epilogue (warps 0-3) ----------------
      const int tok = tid / p.group;
      const int head = hk * p.group + tid - tok * p.group;
      const bool real = tok < job.count;
      const int pos = job.pos0 + tok;
      const int seen = real ? min(pos + 1, job.n) : 0;  // keys [0, seen), less the window's gap
      const int wlo = p.w.first(pos);
      // Every row of the warp, if it has any, sees the keys [all_wlo, all_seen).
      const int all_seen = __any_sync(0xffffffffu, real) ? __reduce_min_sync(0xffffffffu, real ? seen : INT_MAX) : 0;
      const int all_wlo = __reduce_max_sync(0xffffffffu, wlo);
      const uint32_t tl = tmem + (static_cast<uint32_t>(warp * 32) << 16);
      const float sl2 = p.scale_log2;
      float m_run = -INFINITY;
      float l_run = 0.f;
      bool ok = going;
      // Absent pages are not visible: the boxes of the next 32 / boxes tiles are
      // looked up by the lanes, a batch ahead.
      auto lookup = [&](int i) -> int {
        const int t = job.pos(j0 + i / boxes) + ((i % boxes) << p.box_shift);
        return i < nt * boxes && job.any(p.w, t, box_rows) ? p.c.entry(job.b, t) : 0;
      };
      int entry_ahead = lookup(lane);
      uint32_t absent = 0;
      for (int j = 0; ok && j < nt; ++j) {
        const int t = job.pos(j0 + j);
        const int i = j * boxes;
        if ((i & 31) == 0) {
          absent = __ballot_sync(0xffffffffu, p.c.checked(entry_ahead) < 0);
          entry_ahead = lookup(i + 32 + lane);
        }
        const uint32_t missing = (absent >> (i & 31)) & ((1u << boxes) - 1u);
        // Which keys the row sees; most tiles are seen whole by the whole warp (the
        // masks left out there: 592 -> 574 us for the prompt below).
        unsigned long long see = ~0ull;
        bool dead = false;
        if (t + kTile > all_seen || (t < all_wlo && t + kTile > p.w.prefix) || missing != 0u) {
          see = low_bits(seen - t) & (~low_bits(wlo - t) | low_bits(p.w.prefix - t));
          if (missing != 0u) {
#pragma unroll 1
            for (int x = 0; x < boxes; ++x)
              if ((missing >> x) & 1u) see &= ~(low_bits(box_rows) << (x << p.box_shift));
          }
          // A warp whose rows see no key of this tile stores P = 0 and leaves the
          // exponential unit to the others.
          dead = __all_sync(0xffffffffu, see == 0ull);
        }
        const int sb = j & 1;
        const uint32_t ts = tl + kTmemS + 64 * sb;
        // S(j): PRO[j] for j < 2, else in C(j-2)
        const uint32_t s_bar = bar(j < 2 ? PRO + j : DONE + sb);
        const uint32_t s_par = j < 2 ? (j == 0 ? seg_par : two_par) : par(sb, (j >> 1) - 1);
        // Mostly there already: every lane looks, which spares the hand-over from
        // lane 0 (a 12288-row prompt at 16/16 heads: 574 -> 560 us; looking on
        // instead of waiting takes issue slots from the other warps, 567).
        if (!__all_sync(0xffffffffu, mbar_test_wait(s_bar, s_par))) ok = mbar_wait_warp(s_bar, s_par, abort_flag);
        if (!ok) break;
        tc_fence_after();
        bool rescale = false;
        float alpha = 1.0f;
        if (dead) {
          uint32_t zero[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) zero[c] = 0u;
          tmem_st32(ts, zero);
        } else {
          uint32_t sr0[32], sr1[32];
          tmem_ld32(ts, sr0);
          tmem_ld32(ts + 32, sr1);
          tmem_wait_ld();
          float x[64];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            x[c] = __uint_as_float(sr0[c]);
            x[c + 32] = __uint_as_float(sr1[c]);
          }
          if (see != ~0ull) {
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (!((see >> c) & 1ull)) x[c] = -INFINITY;
          }
          const float m_tile = row_max64(x) * sl2;
          // The maximum used to scale P is only raised when it grows by more
          // than 2^8 (exact: O and l share it).
          rescale = m_tile > m_run + 8.0f;
          const float m_use = rescale ? m_tile : m_run;
          alpha = rescale ? ex2(m_run - m_use) : 1.0f;
          const float moff = (m_use == -INFINITY) ? 0.0f : m_use;
          l_run = l_run * alpha + exp_store<T>(x, sl2, moff, ts);
          m_run = m_use;
        }
        // O must not change under a running P.V: rescale only after P.V(j-1).
        if (j >= 1 && __any_sync(0xffffffffu, rescale)) {
          ok = mbar_wait_warp(bar(DONE + ((j - 1) & 1)), par((j - 1) & 1, (j - 1) >> 1), abort_flag);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t ov[32];
            tmem_ld32(tl + ch * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
            tmem_st32(tl + ch * 32, ov);
          }
          tmem_wait_st();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL + sb));
      }
      if (ok && nt >= 1) {
        ok = mbar_wait(bar(DONE + ((nt - 1) & 1)), par((nt - 1) & 1, (nt - 1) >> 1), abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      // After a timeout anywhere in the CTA the tile is incomplete: store nothing.
      ok = __all_sync(0xffffffffu, ok && *abort_flag == 0);
      if (ok) {
        T* orow = static_cast<T*>(p.o) + static_cast<long long>(job.row0 + tok) * p.o_sr + head * p.o_sh;
        const long long prow = static_cast<long long>(place) * kRows + tid;
        const float inv = 1.0f / l_run;  // unused where the row saw nothing (l_run is exactly 0): it is zero
        const uint64_t opol = l2_policy_evict_first();
        auto quad = [&](const uint32_t (&ov)[32], int q4) -> uint4 {  // 8 columns of the result
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = l_run == 0.f ? 0u
                                : DT<T>::pack(__uint_as_float(ov[8 * q4 + 2 * e]) * inv,
                                              __uint_as_float(ov[8 * q4 + 2 * e + 1]) * inv);
          return make_uint4(w[0], w[1], w[2], w[3]);
        };
        if (!kShares && nt >= 1) {
          // Every S is done, so the Q tile is free: the warp turns its rows in
          // their place and writes two whole rows at a time (windowed prompts 767
          // -> 752 us). In shares the next Q may be on its way there already.
          uint8_t* const turn = smem + kQOff + warp * (32 * kD * 2);
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t ov[32];
            tmem_ld32(tl + ch * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
              *reinterpret_cast<uint4*>(turn + lane * 256 + (((ch * 4 + q4) ^ (lane & 7)) << 4)) = quad(ov, q4);
          }
          __syncwarp();
          const uint32_t rows = __ballot_sync(0xffffffffu, real);
          const unsigned long long mine = reinterpret_cast<unsigned long long>(orow);
#pragma unroll 4
          for (int i = 0; i < 32; i += 2) {
            const int r = i + (lane >> 4);
            uint4* const dst = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, mine, r)) + (lane & 15);
            const uint4 v = *reinterpret_cast<const uint4*>(turn + r * 256 + (((lane & 15) ^ (r & 7)) << 4));
            if ((rows >> r) & 1u) st_global_v4_hint(dst, v, opol);
          }
          break;
        }
#pragma unroll 1
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t ov[32];
          if (nt >= 1) {
            tmem_ld32(tl + ch * 32, ov);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) ov[c] = 0u;
          }
          if (!real) continue;
          if (part) {
            uint4* dst = reinterpret_cast<uint4*>(p.part_acc + prow * kD + ch * 32);
#pragma unroll
            for (int q4 = 0; q4 < 8; ++q4)
              dst[q4] = make_uint4(ov[4 * q4], ov[4 * q4 + 1], ov[4 * q4 + 2], ov[4 * q4 + 3]);
          } else {
            uint4* dst = reinterpret_cast<uint4*>(orow + ch * 32);
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) st_global_v4_hint(dst + q4, quad(ov, q4), opol);
          }
        }
        if (real && part) *reinterpret_cast<float2*>(p.part_ml + prow * 2) = make_float2(m_run, l_run);
      }
    }

    // Each role goes on to the next segment by itself: the producers wait for
    // MMA_DONE, S(0) and S(1) are made while this segment's O is read out, and
    // P.V(0) waits for P(0), which the softmax stores after that.
    if (!kShares || units == 0) break;
    d0 += (nt + 1) >> 1;
    d1 += nt >> 1;
    twos += nt >= 2 ? 1 : 0;
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, kTmemCols);
}

// Joins the parts of pair blockIdx.x, if it has several, in share order: a warp
// per row, four columns a lane, eight parts in flight.
template <typename T>
__global__ void __launch_bounds__(256) paged_combine_kernel(const Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int4 pair = p.joins[2 * blockIdx.x];
  const int parts = pair.x;
  if (parts == 0) return;
  const int4 rows = p.joins[2 * blockIdx.x + 1];
  const int tok = row / p.group;
  if (tok >= rows.y) return;
  // The first part is the last segment of its share, the others open theirs.
  PartSum sum;
  sum.add_parts(p.part_ml, p.part_acc, 0, 1, parts, lane, [&](int i) -> long long {
    return static_cast<long long>(i == 0 ? pair.z : 2 * (pair.y + i)) * kRows + row;
  });
  store_row<T>(static_cast<T*>(p.o) + static_cast<long long>(rows.x + tok) * p.o_sr +
                   (static_cast<int>(blockIdx.x) % p.heads_kv * p.group + row - tok * p.group) * p.o_sh,
               lane, sum.a, sum.l);
}

// Row tiles that `rows` rows of `batch` sequences need at most: a sequence of
// l > 0 rows takes (l - 1) / tokens + 1.
static inline long long row_slots(int rows, int batch, int tokens) {
  const int k = rows < batch ? rows : batch;
  return static_cast<long long>(rows - k) / tokens + k;
}

// Whether a call runs in shares, as far as the host can tell: by the pairs (row
// tile, KV head) there may be and the key tiles of one, counted for a row tile
// in the middle of its sequence's new rows. The table's width stands for the
// sequences' length, so callers pass the columns in use: with the table of a
// 16384-row cache 1280 fresh rows at 32/32 heads take 66 us instead of 24, 256 on
// 1000 at 56/8 31.5 instead of 19.6. Where a pair can be cut in k >= 2
// parts, when that saves it 13 tiles or more: less does not pay for the larger
// start and the joining. Else equal shares fill the places that the last pairs
// leave empty (counted for the pairs there are when row tiles end anywhere),
// which pays when those are many and the pairs long: a CTA alone on its SM is
// faster than one of two. Measured, us a call, a CTA each against shares (pairs
// x tiles):
//   64 rows on 1000, 16/16 heads (16 x 16)          18.6 / 16.1
//   64 rows on 16000, 16/16 heads (16 x 250)         240 / 36
//   256 rows on 1000, 56/8 heads (120 x 18)         22.3 / 31.4
//   1000 rows on 1000, 16/16 heads (128 x 23)       31.0 / 35.5
//   400 rows on 4000, 56/8 heads (184 x 66)         72.1 / 78.5
//   400 rows on 8000, 56/8 heads (184 x 129)         133 / 118
//   512 rows on 12000, 56/8 heads (232 x 192)        195 / 203
//   512 rows on 15872, 56/8 heads (232 x 252)        257 / 251
//   2300 rows on 8000, 16/16 heads (288 x 143)       174 / 220
//   1280 rows on 6000, 32/32 heads (320 x 104)       198 / 190
//   1500 rows on 12000, 32/32 heads (384 x 199)      370 / 410
//   16 sequences of 1..200 rows on 100..8000, 16/16  152 / 141
static bool in_shares(int rows, int batch, int heads_q, int heads_kv, int page_size, int max_pages, int window,
                      int prefix) {
  const int tokens = kRows / (heads_q / heads_kv);
  long long span = static_cast<long long>(page_size) * max_pages;
  span -= (rows / batch < span ? rows / batch : span) / 2;
  if (window >= 0) {
    const long long seen = static_cast<long long>(window) + tokens + prefix;
    if (seen < span) span = seen;
  }
  const long long slots = row_slots(rows, batch, tokens), pairs = slots * heads_kv, tiles = span / kTile;
  if (batch > kShareBatch || pairs > kMaxPairs) return false;
  // find_share() counts the tiles of all row tiles in 32 bits.
  if (slots * ((static_cast<long long>(page_size) * max_pages + kTile - 1) / kTile) > INT_MAX) return false;
  const long long k = kDecCtas / pairs;
  if (k >= 2) return tiles - tiles / k >= 13;
  const long long likely = (2ll * rows + static_cast<long long>(batch) * tokens) * heads_kv / (2 * tokens);
  if (likely <= kDecCtas) return tiles * (kDecCtas - likely) >= 48 * kDecCtas;
  return tiles >= 96 && 2 * kDecCtas - likely >= 250;
}

// Joins, then the parts of two segments of every share.
static constexpr size_t kShareWorkspace =
    kMaxPairs * 2 * sizeof(int4) + static_cast<size_t>(2) * kDecCtas * kRows * (kD + 2) * sizeof(float);

// Tensor map of q [rows, Hq, D]: dims (128 d, g heads of a group, rows, KV
// heads); box = (64 d, g, tokens, 1): one d-half of a row tile, token by token.
static int make_map_q(CUtensorMap* m, const void* q, int dtype, int rows, int heads_kv, int group, int tokens,
                      long long sr, long long sh) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return sabre_fail(SABRE_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  if (heads_kv * group == 1) sh = kD;  // dimensions of size one may carry any stride
  if (rows == 1) sr = sh * heads_kv * group;
  if (sr <= 0 || sh <= 0 || sr >= (1ll << 39) || sh * group >= (1ll << 39))
    return sabre_fail(SABRE_ERR_ALIGNMENT, "sabre_paged_prefill: q strides must be positive");
  const cuuint64_t gdim[4] = {(cuuint64_t)kD, (cuuint64_t)group, (cuuint64_t)rows, (cuuint64_t)heads_kv};
  const cuuint64_t gstr[3] = {(cuuint64_t)sh * 2, (cuuint64_t)sr * 2, (cuuint64_t)sh * group * 2};
  const cuuint32_t box[4] = {64u, (cuuint32_t)group, (cuuint32_t)tokens, 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUresult r =
      fn(m, dtype == SABRE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
         const_cast<void*>(q), gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return sabre_fail(SABRE_ERR_CUDA, "q: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return SABRE_OK;
}

template <typename T>
static cudaError_t launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Params& p,
                          cudaStream_t s) {
  const int smem = p.ctas > 0 ? kShareSmemBytes : kSmemBytes;
  auto kernel = p.ctas > 0 ? paged_prefill_kernel<T, true> : paged_prefill_kernel<T, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid = p.ctas > 0 ? dim3(p.ctas) : p.head_major ? dim3(p.slots, p.heads_kv) : dim3(p.heads_kv, p.slots);
  e = launch_dependent(grid, kThreads, smem, s, kernel, mq, mk, mv, p);
  if (e != cudaSuccess || p.ctas == 0) return e;
  const int tile_rows = (p.rows < p.tokens ? p.rows : p.tokens) * p.group;
  return launch_dependent(dim3(p.slots * p.heads_kv, (tile_rows + 7) / 8), 256, 0, s, paged_combine_kernel<T>, p);
}

}  // namespace pre
}  // namespace paged
}  // namespace sabre

extern "C" {

size_t sabre_paged_prefill_workspace_size(int rows, int batch, int heads_q, int heads_kv, int head_dim, int page_size,
                                          int max_pages, int window, int num_prefix_tokens) {
  using namespace sabre::paged;
  if (rows <= 0 || batch <= 0 || heads_q <= 0 || heads_kv <= 0 || head_dim != kD || heads_q % heads_kv != 0 ||
      heads_q / heads_kv > kGroup || page_size <= 0 || max_pages <= 0)
    return 0;
  return pre::in_shares(rows, batch, heads_q, heads_kv, page_size, max_pages, window, num_prefix_tokens)
             ? pre::kShareWorkspace
             : 0;
}

int sabre_paged_prefill(const void* q, const void* k_pages, const void* v_pages, void* o, const int32_t* page_table,
                        const int32_t* seq_lens, const int32_t* q_start, int rows, int batch, int heads_q,
                        int heads_kv, int head_dim, int num_pages, int page_size, int max_pages, int window,
                        int num_prefix_tokens, const int64_t* q_strides, const int64_t* kp_strides,
                        const int64_t* vp_strides, const int64_t* o_strides, int64_t table_stride,
                        float softmax_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sabre::paged;
  const char* fn = "sabre_paged_prefill";
  if (!q_start) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  pre::Params p;
  int st = make_cache(&p.c, fn, k_pages, v_pages, page_table, seq_lens, batch, heads_kv, head_dim, num_pages,
                      page_size, max_pages, kp_strides, vp_strides, table_stride, dtype);
  if (st == SABRE_OK) st = check_queries(fn, q, o, heads_q, heads_kv, num_prefix_tokens, q_strides, o_strides);
  if (st != SABRE_OK) return st;
  if (rows <= 0) return sabre_fail(SABRE_ERR_INVALID_ARG, "%s: rows must be positive", fn);
  p.w = Window{window, window < 0 ? 0 : num_prefix_tokens};
  p.starts = q_start;
  p.o = o;
  p.o_sr = o_strides[0];
  p.o_sh = o_strides[1];
  p.rows = rows;
  p.heads_kv = heads_kv;
  p.group = heads_q / heads_kv;
  p.tokens = pre::kRows / p.group;
  p.box_shift = p.c.page_shift < 6 ? p.c.page_shift : 6;
  p.scale_log2 = scale_log2(softmax_scale);
  const bool shares =
      pre::in_shares(rows, batch, heads_q, heads_kv, page_size, max_pages, window, num_prefix_tokens);
  p.ctas = shares ? kDecCtas : 0;
  if (shares && (!workspace || workspace_bytes < pre::kShareWorkspace))
    return sabre_fail(SABRE_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn, workspace_bytes, pre::kShareWorkspace);
  if (shares && !aligned16(workspace))
    return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
  p.joins = static_cast<int4*>(workspace);
  p.part_acc = shares ? reinterpret_cast<float*>(p.joins + 2 * pre::kMaxPairs) : nullptr;
  p.part_ml = shares ? p.part_acc + static_cast<size_t>(2) * kDecCtas * pre::kRows * kD : nullptr;
  const long long slots = pre::row_slots(rows, batch, p.tokens);
  // The rule of prefill_bsa.cu: K/V larger than this -> head-major order.
  const long long kv_bytes = 4ll * heads_kv * kD * batch * page_size * max_pages;
  p.head_major = kv_bytes > (112ll << 20) || slots > 65535 ? 1 : 0;
  p.slots = static_cast<int>(slots);
  CUtensorMap mq, mk, mv;
  if ((st = pre::make_map_q(&mq, q, dtype, rows, heads_kv, p.group, p.tokens, q_strides[0], q_strides[1])) != SABRE_OK)
    return st;
  if ((st = make_map_pages(&mk, k_pages, dtype, num_pages, heads_kv, page_size, p.c.k_sp, p.c.k_sh, p.c.k_st,
                           1 << p.box_shift, 1, "k_pages")) != SABRE_OK)
    return st;
  if ((st = make_map_pages(&mv, v_pages, dtype, num_pages, heads_kv, page_size, p.c.v_sp, p.c.v_sh, p.c.v_st,
                           1 << p.box_shift, 1, "v_pages")) != SABRE_OK)
    return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == SABRE_BF16 ? pre::launch<__nv_bfloat16>(mq, mk, mv, p, s)
                                            : pre::launch<__half>(mq, mk, mv, p, s);
  return e == cudaSuccess ? SABRE_OK : sabre_cuda_fail(e, fn);
}

}  // extern "C"
