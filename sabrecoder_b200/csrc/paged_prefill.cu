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
// the prefix tiles, then those of the window: nothing else is visited. When
// the tiles of rows alone would leave SMs idle, the key tiles of a row tile
// are dealt out to `splits` CTAs whose parts paged_combine_kernel joins.
// Sequences, lengths and pages are only read on the device, so a captured
// call follows them; the grid is the most row tiles that the rows could need.
//
// Roles, tensor-memory layout and barrier protocol are those of
// prefill_bsa.cu (224 threads, two CTAs per SM: warps 0-3 softmax, 4 Q and K
// producer, 5 MMA issuer, 6 V producer; S = Q K^T of M=128 N=64 into two
// buffers, P over its S, O += P V with P from tensor memory), whose model
// check covers them. Different here: tiles come box by box from pages (a TMA
// box is min(page_size, 64) rows; absent pages and boxes that no row sees are
// read outside the pool and give zeros), and rows past the sequence's end
// inside a page are zeroed in V before its tile is handed to the MMA, since
// 0 * NaN would reach the result.
// P is rounded to the type of V for the product; scores, sums and O are fp32.
namespace sabre {
namespace paged {
namespace pre {

using prefill::exp_tile;
using prefill::row_max64;

constexpr int kThreads = 224;
constexpr int kRows = 128;
constexpr int kMaxSplits = 32;
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
  V_RAW = 11,  // the copies of the tile that ends inside a page, before its rows are zeroed
  MMA_DONE = 12,
  NUM_BARS = 13
};
constexpr int kMiscOff = kBarOff + NUM_BARS * 8;
constexpr int kSmemBytes = kMiscOff + 72;
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kTmemS = 128;  // + 64 * buffer

struct Params {
  Cache c;
  Window w;
  const int32_t* starts;
  void* o;
  float* part_acc;  // [splits][rows][Hq][D]
  float* part_ml;   // [splits][rows][Hq][2]
  long long o_sr, o_sh;
  int rows, heads_kv, group, tokens;  // tokens of a row tile: 128 / group
  int box_shift, splits, slots;       // slots: row tiles of the grid
  int head_major;
  float scale_log2;
};

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
  int incl = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, s);
    if ((tid & 31) >= s) incl += up;
  }
  if ((tid & 31) == 31) scratch[tid >> 5] = incl;
  if (tid == 0) scratch[8] = -1;
  __syncthreads();
  int left = slot - (incl - mine);
  for (int w = 0; w < (tid >> 5); ++w) left -= scratch[w];
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
  job.b = scratch[8];
  if (job.b < 0) return false;
  const int r = scratch[9], len = scratch[11], length = scratch[12];
  job.row0 = scratch[10] + r;
  job.count = min(p.tokens, len - r);
  job.pos0 = length - len + r;
  job.n = min(min(max(length, 0), p.c.capacity()), max(job.pos0 + job.count, 0));  // keys that some row may see
  job.lo = p.w.first(job.pos0);
  job.from = job.lo / kTile;
  job.head = min((min(p.w.prefix, job.lo) + kTile - 1) / kTile, job.from);
  const int whole = (job.n + kTile - 1) / kTile;
  job.head = min(job.head, whole);
  job.tiles = job.head + max(0, whole - job.from);
  return true;
}

template <typename T>
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

  // Later row tiles of a sequence see more keys: heaviest first. Row-major
  // (grid x = head) or head-major (grid x = row tile), as in prefill_bsa.cu.
  const int hs = p.head_major ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.x);
  const int hk = hs / p.splits;
  const int split = hs - hk * p.splits;
  const int slot = p.slots - 1 - static_cast<int>(p.head_major ? blockIdx.x : blockIdx.y);
  if (tid == 0) {
    const bool bad = (sbase & 1023u) != 0u;
    *abort_flag = bad ? 1 : 0;
    if (bad) record_status(SABRE_DEV_BAD_SMEM_ALIGN);
  }
  if (warp == 4 && lane == 0) {
    mbar_init(bar(Q_FULL), 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(K_FULL + s), 1);
      mbar_init(bar(V_FULL + s), 1);
      mbar_init(bar(PRO + s), 1);
      mbar_init(bar(DONE + s), 1);
      mbar_init(bar(P_FULL + s), 4);
    }
    mbar_init(bar(V_RAW), 1);
    mbar_init(bar(MMA_DONE), 1);
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
  // a programmatic dependent launch) and the loads of find_job, whose barriers
  // order it before its use. Nothing before this line reads what that kernel wrote.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Job job;
  const bool any_job = find_job(p, slot, reinterpret_cast<int*>(smem + kMiscOff + 8), job);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (!any_job) {
    if (warp == 5) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  // This part's key tiles.
  const int j0 = static_cast<int>(static_cast<long long>(job.tiles) * split / p.splits);
  const int nt = static_cast<int>(static_cast<long long>(job.tiles) * (split + 1) / p.splits) - j0;
  const bool start_ok = (*abort_flag == 0);
  const int boxes = kTile >> p.box_shift;
  const int box_rows = 1 << p.box_shift;

  constexpr uint32_t kIdescQK = idesc_f16(128, 64, DT<T>::kBf16, false);
  constexpr uint32_t kIdescPV = idesc_f16(128, 128, DT<T>::kBf16, true);

  if (warp == 4 || warp == 6) {
    // ---------------- TMA producers (warp 4: K, warp 6: V) ----------------
    const bool is_k = (warp == 4);
    const int full0 = is_k ? K_FULL : V_FULL;
    const uint32_t ring = sbase + (is_k ? kKOff : kVOff);
    const CUtensorMap* map = is_k ? &tmK : &tmV;
    if (is_k && lane == 0 && start_ok) {
      mbar_arrive_expect_tx(bar(Q_FULL), static_cast<uint32_t>(p.group * p.tokens) * 256u);
      const uint64_t pol = l2_policy_evict_first();
      tma_load_4d_hint(sbase + kQOff, &tmQ, bar(Q_FULL), 0, 0, job.row0, hk, pol);
      tma_load_4d_hint(sbase + kQOff + kQBytes / 2, &tmQ, bar(Q_FULL), 64, 0, job.row0, hk, pol);
    }
    int issued = 0;    // tiles
    bool raw = false;  // the last one went through V_RAW
    bool ok = start_ok;
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
          const int wb = is_k && j < 4 ? PRO + (j - 2) : DONE + s;
          const int par = is_k ? (j < 4 ? 0 : (j >> 1) & 1) : ((j >> 1) - 1) & 1;
          ok = mbar_wait_warp(bar(wb), par, abort_flag);
          if (!ok) break;
        }
        // Rows of V at and past the sequence's end inside a box are zeroed.
        const int over = job.n - job.pos(j0 + j);
        const bool clean = !is_k && over < kTile && (over & (box_rows - 1)) != 0;
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
        if (clean) {
          raw = true;
          ok = mbar_wait_warp(bar(V_RAW), 0, abort_flag);
          if (!ok) break;
          (void)mbar_test_wait(bar(V_RAW), 0);  // each lane's own acquire of the copied bytes
          const int end = (over + box_rows) & ~(box_rows - 1);
          for (int c = lane; c < (end - over) * 16; c += 32) {
            const int row = over + (c >> 4);
            *reinterpret_cast<uint4*>(smem + kVOff + s * kTileBytes + ((c >> 3) & 1) * (kTileBytes / 2) + row * 128 +
                                      (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(full0 + s));
        }
      }
    }
    // Every issued copy must land before the CTA may exit. (The tile that ends
    // the sequence is the last one: only it can have gone through V_RAW.)
    if (lane == 0 && start_ok) {
      if (is_k) mbar_wait_drain(bar(Q_FULL), 0);
      for (int j = max(0, issued - 2); j < issued; ++j) {
        if (raw && j == issued - 1)
          mbar_wait_drain(bar(V_RAW), 0);
        else
          mbar_wait_drain(bar(full0 + (j & 1)), (j >> 1) & 1);
      }
    }
  } else if (warp == 5) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && start_ok) {
      const uint64_t qd = smem_desc_sw128(sbase + kQOff, 16, 1024);
      const uint64_t kd0 = smem_desc_sw128(sbase + kKOff, 16, 1024);
      const uint64_t vd0 = smem_desc_sw128(sbase + kVOff, kTileBytes / 2, 1024);
      const uint32_t s_tmem = tmem + kTmemS;
      bool ok = mbar_wait(bar(Q_FULL), 0, abort_flag);
      auto issue_s = [&](int j) -> bool {
        const int ks = j & 1;
        if (!mbar_wait(bar(K_FULL + ks), (j >> 1) & 1, abort_flag)) return false;
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
        if (!mbar_wait(bar(P_FULL + pb), (i >> 1) & 1, abort_flag)) return false;
        if (!mbar_wait(bar(V_FULL + pb), (i >> 1) & 1, abort_flag)) return false;
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
      // Whatever was issued must finish before tensor memory is released.
      mma_commit(bar(MMA_DONE));
      mbar_wait_drain(bar(MMA_DONE), 0);
    }
  } else {
    // ---------------- softmax + epilogue (warps 0-3) ----------------
    const int tok = tid / p.group;
    const int head = hk * p.group + tid - tok * p.group;
    const bool real = tok < job.count;
    const int pos = job.pos0 + tok;
    const int seen = real ? min(pos + 1, job.n) : 0;  // keys [0, seen), less the window's gap
    const int wlo = p.w.first(pos);
    const uint32_t tl = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const float sl2 = p.scale_log2;
    float m_run = -INFINITY;
    float l_run = 0.f;
    bool ok = start_ok;
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
      unsigned long long see = low_bits(seen - t) & (~low_bits(wlo - t) | low_bits(p.w.prefix - t));
      const uint32_t missing = (absent >> (i & 31)) & ((1u << boxes) - 1u);
      if (missing != 0u) {
#pragma unroll 1
        for (int x = 0; x < boxes; ++x)
          if ((missing >> x) & 1u) see &= ~(low_bits(box_rows) << (x << p.box_shift));
      }
      // A warp whose rows see no key of this tile stores P = 0 and leaves the
      // exponential unit to the others.
      const bool dead = __all_sync(0xffffffffu, see == 0ull);
      const int sb = j & 1;
      const uint32_t ts = tl + kTmemS + 64 * sb;
      // S(j): PRO[j] for j < 2, else in C(j-2)
      ok = j < 2 ? mbar_wait_warp(bar(PRO + j), 0, abort_flag)
                 : mbar_wait_warp(bar(DONE + sb), ((j >> 1) - 1) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t pk[32];
      bool rescale = false;
      float alpha = 1.0f;
      if (dead) {
#pragma unroll
        for (int c = 0; c < 32; ++c) pk[c] = 0u;
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
        const float rs = exp_tile<T>(x, sl2, moff, pk);
        l_run = l_run * alpha + rs;
        m_run = m_use;
      }
      // O must not change under a running P.V: rescale only after P.V(j-1).
      if (j >= 1 && __any_sync(0xffffffffu, rescale)) {
        ok = mbar_wait_warp(bar(DONE + ((j - 1) & 1)), ((j - 1) >> 1) & 1, abort_flag);
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
      tmem_st32(ts, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(P_FULL + sb));
    }
    if (ok && nt >= 1) {
      ok = mbar_wait(bar(DONE + ((nt - 1) & 1)), ((nt - 1) >> 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    ok = __all_sync(0xffffffffu, ok);
    // After a timeout anywhere in the CTA the tile is incomplete: store nothing.
    if (ok && *abort_flag == 0) {
      const long long row = job.row0 + tok;
      const long long part = (split * static_cast<long long>(p.rows) + row) * (p.heads_kv * p.group) + head;
      T* orow = static_cast<T*>(p.o) + row * p.o_sr + head * p.o_sh;
      const float inv = 1.0f / l_run;  // unused where the row saw nothing: it is zero
      const uint64_t opol = l2_policy_evict_first();
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
        if (p.splits > 1) {
          uint4* dst = reinterpret_cast<uint4*>(p.part_acc + part * kD + ch * 32);
#pragma unroll
          for (int q4 = 0; q4 < 8; ++q4)
            dst[q4] = make_uint4(ov[4 * q4], ov[4 * q4 + 1], ov[4 * q4 + 2], ov[4 * q4 + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(orow + ch * 32);
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = l_run > 0.f ? DT<T>::pack(__uint_as_float(ov[8 * q4 + 2 * e]) * inv,
                                               __uint_as_float(ov[8 * q4 + 2 * e + 1]) * inv)
                                 : 0u;
            st_global_v4_hint(dst + q4, make_uint4(w[0], w[1], w[2], w[3]), opol);
          }
        }
      }
      if (real && p.splits > 1) {
        p.part_ml[part * 2] = m_run;
        p.part_ml[part * 2 + 1] = l_run;
      }
    }
  }

  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// One warp per (row, head): joins the parts of a split call in order.
template <typename T>
__global__ void __launch_bounds__(256) paged_combine_kernel(const Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int heads = p.heads_kv * p.group;
  const long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const long long row = i / heads;
  const int head = static_cast<int>(i - row * heads);
  // No sequence's row: padding behind the last one.
  if (row < row_start(p.starts, 0, p.rows) || row >= row_start(p.starts, p.c.batch, p.rows)) return;
  const long long step = static_cast<long long>(p.rows) * heads;
  float m = -INFINITY, l = 0.f;
  if (lane < p.splits) {
    m = p.part_ml[(i + lane * step) * 2];
    l = p.part_ml[(i + lane * step) * 2 + 1];
  }
  float M = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float w = M == -INFINITY ? 0.f : ex2(m - M);
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < p.splits; ++s) {
    const float ws = __shfl_sync(0xffffffffu, w, s);
    L += ws * __shfl_sync(0xffffffffu, l, s);
    if (ws == 0.f) continue;  // a part that saw nothing
    const float4 a = *reinterpret_cast<const float4*>(p.part_acc + (i + s * step) * kD + lane * 4);
    acc.x += ws * a.x;
    acc.y += ws * a.y;
    acc.z += ws * a.z;
    acc.w += ws * a.w;
  }
  const float inv = L > 0.f ? 1.0f / L : 0.f;
  *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + row * p.o_sr + head * p.o_sh + lane * 4) =
      make_uint2(DT<T>::pack(acc.x * inv, acc.y * inv), DT<T>::pack(acc.z * inv, acc.w * inv));
}

// Row tiles that `rows` rows of `batch` sequences need at most: a sequence of
// l > 0 rows takes (l - 1) / tokens + 1.
static inline long long row_slots(int rows, int batch, int tokens) {
  const int k = rows < batch ? rows : batch;
  return static_cast<long long>(rows - k) / tokens + k;
}

// CTAs per row tile, as far as the host can tell: enough that the card's 296
// places are filled, with at least eight key tiles each, counted for a row
// tile in the middle of its sequence's new rows. A part costs a CTA's start
// and read-out and 516 bytes per row and head through the workspace: 512 rows
// of a single sequence at 56/8 heads on 15872 rows run 297 us whole and 307 in
// two parts (232 row tiles), 64 rows at 16 heads on 16000 rows 234 us whole
// and 37 in 16 parts; 1000 rows on none run 22 us whole and 25 in two.
static int plan_splits(int rows, int batch, int heads_q, int heads_kv, int page_size, int max_pages, int window,
                       int prefix) {
  const int tokens = kRows / (heads_q / heads_kv);
  long long span = static_cast<long long>(page_size) * max_pages;
  span -= (rows / batch < span ? rows / batch : span) / 2;
  if (window >= 0) {
    const long long seen = static_cast<long long>(window) + tokens + prefix;
    if (seen < span) span = seen;
  }
  const long long tiles = span / kTile;
  if (tiles < 32) return 1;
  long long s = kDecCtas / (row_slots(rows, batch, tokens) * heads_kv);
  if (s > tiles / 8) s = tiles / 8;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : static_cast<int>(s);
}

static size_t workspace_bytes(int rows, int heads_q, int splits) {
  return splits == 1 ? 0 : static_cast<size_t>(splits) * rows * heads_q * (kD + 2) * sizeof(float);
}

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
  cudaError_t e = cudaFuncSetAttribute(paged_prefill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return e;
  const unsigned hs = static_cast<unsigned>(p.heads_kv * p.splits);
  const dim3 grid = p.head_major ? dim3(p.slots, hs) : dim3(hs, p.slots);
  e = launch_dependent(grid, kThreads, kSmemBytes, s, paged_prefill_kernel<T>, mq, mk, mv, p);
  if (e != cudaSuccess || p.splits == 1) return e;
  const long long warps = static_cast<long long>(p.rows) * p.heads_kv * p.group;
  return launch_dependent(dim3(static_cast<unsigned>((warps + 7) / 8)), 256, 0, s, paged_combine_kernel<T>, p);
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
  return pre::workspace_bytes(rows, heads_q, pre::plan_splits(rows, batch, heads_q, heads_kv, page_size, max_pages,
                                                              window, num_prefix_tokens));
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
  p.splits = pre::plan_splits(rows, batch, heads_q, heads_kv, page_size, max_pages, window, num_prefix_tokens);
  p.scale_log2 = scale_log2(softmax_scale);
  const size_t need = pre::workspace_bytes(rows, heads_q, p.splits);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return sabre_fail(SABRE_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn, workspace_bytes, need);
  if (need > 0 && !aligned16(workspace))
    return sabre_fail(SABRE_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
  p.part_acc = static_cast<float*>(workspace);
  p.part_ml = need > 0 ? p.part_acc + static_cast<size_t>(p.splits) * rows * heads_q * kD : nullptr;
  const long long slots = pre::row_slots(rows, batch, p.tokens);
  // The rule of prefill_bsa.cu: K/V larger than this -> head-major order.
  const long long kv_bytes = 4ll * heads_kv * kD * batch * page_size * max_pages;
  p.head_major = kv_bytes > (112ll << 20) ? 1 : 0;
  const long long hs = static_cast<long long>(heads_kv) * p.splits;
  if ((p.head_major ? hs : slots) > 65535) p.head_major ^= 1;
  if ((p.head_major ? hs : slots) > 65535)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: %lld row tiles of %lld head parts exceed the grid", fn, slots, hs);
  if ((static_cast<long long>(rows) * heads_q + 7) / 8 > 0x7fffffffll)
    return sabre_fail(SABRE_ERR_UNSUPPORTED, "%s: rows * heads_q too large", fn);
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
