// Attention of many requests over one NVFP4 pool, many query rows a request
// (verify windows, prompt chunks), sm_100a, tcgen05 with the accumulators in
// tensor memory.  The formula is that of batch_few.cu.
//
// An item is one request, one KV head and 128 / group query positions: their
// (position, head) rows are the M = 128 rows of every MMA.  It visits the
// 128-token KV tiles up to its last row's causal limit.  One persistent CTA per
// SM takes an equal share of all items' tiles (batch_common.cuh); 17 warps:
//   warps 0-7   softmax, thread = row (TMEM lane), in two groups of four that
//               take the even and the odd tiles; Q staging and epilogue (half of
//               the head dims a group)
//   warps 8-11  dequantise K(j), warps 12-15 V(j): codes straight from the pool
//               into registers one tile ahead, FP16 into shared memory as
//               [128 tok][D] (64-wide head-dim atoms, 128-byte swizzle): the same
//               bytes are the K-major B operand of QK and the MN-major B
//               operand of PV
//   warp 16     tensor-memory owner and MMA issuer (one thread)
// Per tile: S(j) [128 x 128] = Q K(j)^T into the group's S buffer, softmax
// writes P(j) (FP16, 11 significant bits as the output has) over S(j), and
// O [128 x D] += P(j) V(j) with P from tensor memory.  A row's reference
// seldom moves (batch_common.cuh); it is handed from one group's warp to the other's
// before the exponentials, so the two groups' exponentials overlap.  The MMA
// thread queues QK(j + 1) ahead of PV(j).  K and V have two buffers each below D
// 256 and one at D 256 (192 KB of operands): there K(j + 1) is dequantised while
// PV(j - 1) runs and V(j) while QK(j + 1) does.
//
// What bounds it: a tile's MMAs take 8 D cycles, its 128 x 128 exponentials 1,024
// (16 a cycle and SM).  At D 256 shared memory carries 320 KB a tile (128 of QK
// operands, 64 of V, 128 of dequantised stores: 2,560 cycles) and the four warps
// that dequantise K are busy for about 5,400 cycles a tile whose codes come from
// HBM (3,000 converting and storing, 2,400 issuing loads); a second K buffer does
// not fit.  At D 128 the period is about 2,500 cycles, the softmax's chain from
// S(j) to P(j).  The rest is changes of item: the first QK waits for the old item's
// last PV, and the softmax warps stage Q and write O before the next P.  A chunk
// of 4,096 rows onto 61,440 tokens, with few of them, takes 2.5 us a tile (6,685 us,
// 58 % of the measured bf16 rate); of the 299,000 cycles that the windows below
// take, 46 tiles of 5,400 are 248,000, and of the 775,000 of the prompts 106 are
// 572,000.
//
// batch_few.cu, which converts for every eight columns, has an item's first eight
// (sixteen where a group has 9 to 16 heads).  On 16 requests of 4,096 to 32,768
// tokens, 24/4/256, it takes 63 us with 6 columns where this kernel takes 172; with
// 12 columns this one takes 176, and two groups of eight there would take 109, but
// their launch takes 108 with 6 columns (capi_batch.cu).
//
// Measured, 24/4/256: 16 requests of 4,096 to 32,768 tokens, 7 rows each, 174 us
// (22 % of the HBM rate, 13 % of the measured bf16 rate in useful rows, two thirds
// of the tile's rows being empty); a step of prompt chunks, windows and decode
// rows, 467 us (32 % of the measured bf16 rate).  16 x 7 rows at 32,768 tokens of
// 32/8/128: 376 us.
#include "attn_common.cuh"
#include "batch_common.cuh"
#include "tc_common.cuh"

namespace qwz {

using namespace detail;

namespace {

constexpr int kRwTok = 128;                 // tokens of a tile
constexpr int kRwRows = 128;                // MMA M
constexpr int kRwSoft = 8;                  // softmax warps, two groups
constexpr int kRwDq = 4;                    // dequant warps of K, and of V
constexpr int kRwMma = kRwSoft + 2 * kRwDq;  // MMA warp
constexpr int kRwWarps = kRwMma + 1;
constexpr int kRwThreads = kRwWarps * 32;
constexpr int kRwScan = 256;                // threads that scan the requests

// Every barrier whose phases are not all waited for by everyone is per tile
// parity or per warp pair, so that a waiter is never two phases off.
enum RwBar : int {
  kRwKReady = 0,            // [2] K buffer written
  kRwKFree = 2,             // [2] QK has read it
  kRwVReady = 4,            // [2]
  kRwVFree = 6,             // [2]
  kRwSFull = 8,             // [2] S(j) is there (j's parity)
  kRwPReady = 10,           // [2] P(j) is written
  kRwPvDone = 12,           // [2] PV(j) is done
  kRwRef = 14,              // [4 warps][2] the reference maxima after tile j
  kRwSum = 22,              // [4 warps] both groups' row sums of the item
  kRwQReady = 26,           // the item's Q is staged
  kRwEpi = 27,              // the item's O has been read
  kRwFin = 28,
  kRwNumBars = 29
};

template <int D>
struct Rows {
  static constexpr int kBufs = D == 256 ? 1 : 2;         // K and V buffers
  static constexpr int kTile = kRwTok * D * 2;           // FP16 K or V tile
  static constexpr int kQ = 0;                           // D / 64 atoms of [128 rows x 128 B]
  static constexpr int kK = kQ + kRwRows * D * 2;
  static constexpr int kV = kK + kBufs * kTile;
  static constexpr int kBars = kV + kBufs * kTile;
  static constexpr int kMeta = kBars + 8 * ((kRwNumBars + 1) / 2 * 2);  // TMEM base, abort flag
  static constexpr int kRowfac = kMeta + 16;             // [2][128] by item parity
  static constexpr int kRef = kRowfac + 8 * kRwRows;     // [2][128] by tile parity
  static constexpr int kSum = kRef + 8 * kRwRows;        // [2][2][128] by item parity and group
  static constexpr int kStarts = kSum + 16 * kRwRows;     // [kRwScan] units before each scanning thread
  static constexpr int kSums = kStarts + 8 * kRwScan;    // [kRwWarps]
  static constexpr int kSmem = kSums + 8 * 32 + 1024;
  static_assert(kSmem <= 227 * 1024 && kStarts % 8 == 0, "shared memory");
  // tensor memory: S of even and odd tiles, O; P has columns of its own where
  // they fit, so that S is free for QK(j + 2) as soon as the softmax has read it
  static constexpr bool kOwnP = D <= 128;
  static constexpr uint32_t kTmS = 0, kTmO = 256, kTmP = kOwnP ? 384 : 0, kTmPStep = kOwnP ? 64 : 128, kTmCols = 512;
  static constexpr size_t kRec = (size_t)kRwRows * (D + 2);  // floats of a record
};

// Walks the units (request, head, group of positions, tile) of the launch.
struct RowsWalk {
  int b, h, i, tile;
  int tiles, groups;
  int per;                 // positions of an item
  batch::Req r;

  QWZ_DEVINL static int tiles_of(const batch::Req& r, int per, int i) {
    const int lim = r.kv - r.n + min((i + 1) * per, r.n);
    return max(1, (lim + kRwTok - 1) / kRwTok);
  }
  QWZ_DEVINL static long long head_cost(const batch::Req& r, int per) {
    long long c = 0;
    for (int i = 0; i * per < r.n; ++i) c += tiles_of(r, per, i);
    return c;
  }
  QWZ_DEVINL static bool many(const BatchAttnParams& p, const batch::Req& r) { return r.n * p.group > p.few_cols; }
  QWZ_DEVINL static long long cost(const BatchAttnParams& p, int b, int per) {
    const batch::Req r = batch::load_req(p, b);
    return many(p, r) ? p.kv_heads * head_cost(r, per) : 0;
  }
  QWZ_DEVINL void enter(const BatchAttnParams& p, int bb) {
    b = bb;
    r = batch::load_req(p, b);
    groups = (r.n + per - 1) / per;
  }
  QWZ_DEVINL void seek(const BatchAttnParams& p, int b0, long long u) {
    for (b = b0; b < p.requests - 1; ++b) {
      const long long c = cost(p, b, per);
      if (u < c) break;
      u -= c;
    }
    enter(p, b);
    const long long c = max(1LL, head_cost(r, per));
    h = (int)(u / c);
    u %= c;
    for (i = 0; i < groups - 1; ++i) {
      const int t = tiles_of(r, per, i);
      if (u < t) break;
      u -= t;
    }
    tiles = tiles_of(r, per, i);
    tile = (int)u;
  }
  QWZ_DEVINL void next(const BatchAttnParams& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++i >= groups) {
      i = 0;
      if (++h >= p.kv_heads) {
        h = 0;
        int bb = b + 1;
        for (; bb < p.requests; ++bb) {
          enter(p, bb);
          if (many(p, r)) break;
        }
      }
    }
    tiles = tiles_of(r, per, i);
  }
  QWZ_DEVINL int entry(const BatchAttnParams& p) const {
    return __ldg(p.block_table + (size_t)b * p.table_width + tile / (kPage / kRwTok));
  }
  QWZ_DEVINL bool present(const BatchAttnParams& p, int pp) const {
    if (r.kv <= 0) return false;
    if (pp >= 0 && pp < p.num_pages) return true;
    flag_error(kErrPageRange);
    return false;
  }
};

QWZ_DEVINL void rw_ld32(uint32_t taddr, float (&x)[32]) {
  uint32_t a[16], b[16];
  tc::ld_32x32b_x16(taddr, a);
  tc::ld_32x32b_x16(taddr + 16, b);
  tc::wait_ld();
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    asm volatile("" : "+r"(a[e]), "+r"(b[e])::"memory");
    x[e] = __uint_as_float(a[e]);
    x[16 + e] = __uint_as_float(b[e]);
  }
}

// Columns at or past `room` do not count.
QWZ_DEVINL void rw_mask(float (&x)[32], int room) {
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = e < room ? x[e] : -CUDART_INF_F;
}

// Codes and scales of one thread's share of a tile: D / 32 chunks of 32 head dims.
template <int D>
struct RwChunks {
  uint4 w[D / 32];
  uint32_t s[D / 32];
};

// Thread t of the dequant warps, load 0: token row and 32-dim chunk; load k is
// kRwStep<D> rows further.  Eight neighbouring lanes hold eight token rows of one
// chunk, so the swizzled 16-byte stores of a quarter warp touch every bank once.
template <int D>
constexpr int kRwStep = kRwDq * 32 / (D / 32);
template <int D>
QWZ_DEVINL void rw_place(int t, int& row, int& chunk) {
  constexpr int CPR = D / 32;
  row = (t & 7) + 8 * (t / (8 * CPR));
  chunk = (t >> 3) % CPR;
}

// codes and scales point at the thread's row 0 of the pool; token0: first token.
template <int D>
QWZ_DEVINL void rw_load(const uint8_t* codes, const uint8_t* scales, size_t token0, int kv_heads, int row, int valid,
                        RwChunks<D>& out) {
  const uint8_t* c = codes + token0 * (size_t)(kv_heads * (D / 2));
  const uint8_t* s = scales + token0 * (size_t)(kv_heads * (D / 16));
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    out.w[k] = make_uint4(0u, 0u, 0u, 0u);
    out.s[k] = 0u;
    if (row + k * kRwStep<D> < valid) {
      out.w[k] = __ldg(reinterpret_cast<const uint4*>(c + k * kRwStep<D> * kv_heads * (D / 2)));
      out.s[k] = __ldg(reinterpret_cast<const unsigned short*>(s + k * kRwStep<D> * kv_heads * (D / 16)));
    }
  }
}

template <int D>
QWZ_DEVINL void rw_store(uint32_t tile, int row, int c, const RwChunks<D>& in) {
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    uint32_t s01, unused;
    e4m3x4_to_f16x2x2(in.s[k], s01, unused);
    const uint32_t s0 = __byte_perm(s01, 0, 0x1010), s1 = __byte_perm(s01, 0, 0x3232);
    const uint32_t base = tile + (c >> 1) * (kRwTok * 128) + (row + k * kRwStep<D>) * 128;
    const uint32_t w[4] = {in.w[k].x, in.w[k].y, in.w[k].z, in.w[k].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t h[4];
      e2m1x8_to_f16x2x4(w[j], h);
      const uint32_t s = j < 2 ? s0 : s1;
      sts128(base + (((4 * (c & 1) + j) ^ (row & 7)) << 4), hmul2_u32(h[0], s), hmul2_u32(h[1], s),
             hmul2_u32(h[2], s), hmul2_u32(h[3], s));
    }
  }
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kRwThreads, 1) batch_rows_kernel(const __grid_constant__ BatchAttnParams p) {
  using R = Rows<D>;
  constexpr int NB = R::kBufs;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sraw = smem_u32(smem);
  const uint32_t sb = (sraw + 1023u) & ~1023u;
  uint8_t* sg = smem + (sb - sraw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) -> uint32_t { return sb + R::kBars + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sg + R::kMeta + 4);
  float* rowfac = reinterpret_cast<float*>(sg + R::kRowfac);
  float* ref_s = reinterpret_cast<float*>(sg + R::kRef);
  float* sum_s = reinterpret_cast<float*>(sg + R::kSum);
  long long* starts = reinterpret_cast<long long*>(sg + R::kStarts);
  long long* sums = reinterpret_cast<long long*>(sg + R::kSums);

  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kRwKReady + i), kRwDq);
      mbar_init(bar(kRwKFree + i), 1);
      mbar_init(bar(kRwVReady + i), kRwDq);
      mbar_init(bar(kRwVFree + i), 1);
      mbar_init(bar(kRwSFull + i), 1);
      mbar_init(bar(kRwPReady + i), kRwSoft / 2);
      mbar_init(bar(kRwPvDone + i), 1);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) mbar_init(bar(kRwRef + i), 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) mbar_init(bar(kRwSum + i), 2);
    mbar_init(bar(kRwQReady), kRwSoft);
    mbar_init(bar(kRwEpi), kRwSoft);
    mbar_init(bar(kRwFin), 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kRwMma) {
    tc::tmem_alloc(sb + R::kMeta, R::kTmCols);
    tc::tmem_relinquish();
  }
  griddep_wait();

  // ---------------------------------------------------- this CTA's share
  const int per_pos = kRwRows / p.group;
  const int per = (p.requests + kRwScan - 1) / kRwScan;
  long long mine = 0, total;
  if (tid < kRwScan)
    for (int b = tid * per; b < min(p.requests, (tid + 1) * per); ++b) mine += RowsWalk::cost(p, b, per_pos);
  const long long before = batch::block_scan(mine, sums, total);
  if (tid < kRwScan) starts[tid] = before;
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tbase = *reinterpret_cast<volatile uint32_t*>(sg + R::kMeta);
  const long long n_cta = gridDim.x;
  const long long lo = (long long)blockIdx.x * total / n_cta, hi = ((long long)blockIdx.x + 1) * total / n_cta;
  const int units = (int)(hi - lo);
  int32_t* meta = p.meta + (kBatchMaxCtas + blockIdx.x) * kBatchMeta;
  RowsWalk cur;
  cur.per = per_pos;
  if (units > 0) {
    int at = 0;
    for (int step = kRwScan / 2; step > 0; step >>= 1)
      if (starts[at + step] <= lo) at += step;
    cur.seek(p, at * per, lo - starts[at]);
  }
  if (tid == 0) meta[0] = 0;

  if (units == 0) {
    // nothing to do
  } else if (warp == kRwMma) {
    // ------------------------------------------------------------------ MMA
    if (lane == 0) {
      constexpr uint32_t idesc_qk = tc::idesc_f16_f32(kRwRows, kRwTok);
      constexpr uint32_t idesc_pv = tc::idesc_f16_f32(kRwRows, D, /*b_mn_major=*/true);
      const uint64_t dq = tc::smem_desc_k128(sb + R::kQ);
      const uint64_t dk = tc::smem_desc_k128(sb + R::kK);
      const uint64_t dv = tc::smem_desc_mn128(sb + R::kV, kRwTok * 128, 1024);
      int item = -1, item_cur = -1;  // items of this CTA: of the last QK, of the current tile
      unsigned firsts = 0;           // bit j % 4: tile j is its item's first here
      bool fresh = true;  // the next QK begins an item of this CTA
      // first tile of its item in this CTA? (PV then overwrites O), for tiles j and j + 1
      bool first_next = false, first_cur = false;
      auto qk = [&](int j) -> bool {
        if (fresh) {
          ++item;
          if (!mbar_wait(bar(kRwQReady), item & 1)) return false;
        }
        first_next = fresh;
        fresh = cur.tile + 1 == cur.tiles;
        cur.next(p);
        const int kb = j % NB;
        if (!mbar_wait(bar(kRwKReady + kb), (j / NB) & 1)) return false;
        // S(j) goes where P(j - 2) was read from (with a P of its own: where S(j - 2)
        // was read, and PV(j - 2) has waited for that)
        if (!R::kOwnP && j >= 2 && !mbar_wait(bar(kRwPvDone + (j & 1)), ((j - 2) >> 1) & 1)) return false;
        tc::fence_after();
        const uint32_t d = tbase + R::kTmS + 128u * (j & 1);
        const uint64_t dkj = dk + (uint64_t)((kb * R::kTile) >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          tc::mma_ss(d, dq + (uint64_t)(((ks >> 2) * (kRwRows * 128) + (ks & 3) * 32) >> 4),
                     dkj + (uint64_t)(((ks >> 2) * (kRwTok * 128) + (ks & 3) * 32) >> 4), idesc_qk, ks > 0);
        tc::commit(bar(kRwSFull + (j & 1)));
        tc::commit(bar(kRwKFree + kb));
        return true;
      };
      auto pv = [&](int j) -> bool {
        const int vb = j % NB;
        if (!mbar_wait(bar(kRwVReady + vb), (j / NB) & 1)) return false;
        // a new item's first PV overwrites O: all of the old one has been read
        if (first_cur && item_cur > 0 && !mbar_wait(bar(kRwEpi), (item_cur - 1) & 1)) return false;
        tc::fence_after();
        const uint64_t dvj = dv + (uint64_t)((vb * R::kTile) >> 4);
#pragma unroll
        for (int kk = 0; kk < kRwTok / 16; ++kk)
          tc::mma_ts(tbase + R::kTmO, tbase + R::kTmP + R::kTmPStep * (j & 1) + 8u * kk, dvj + (uint64_t)((kk * 2048) >> 4),
                     idesc_pv, (!first_cur || kk > 0) ? 1u : 0u);
        tc::commit(bar(kRwPvDone + (j & 1)));
        tc::commit(bar(kRwVFree + vb));
        return true;
      };
      // QK runs one tile ahead of PV, two once P(j) is there where P has columns
      // of its own; a new item's first QK comes after the old one's last PV (its Q
      // is staged after the last softmax)
      int next = 0;  // tile of the next QK
      bool fine = true;
      for (int j = 0; fine && j < units; ++j) {
        if (*abort_flag) break;
        while (fine && next < units && next <= j + 1 && (!fresh || next == j)) {
          fine = qk(next);
          firsts = (firsts & ~(1u << (next & 3))) | ((first_next ? 1u : 0u) << (next & 3));
          ++next;
        }
        if (!fine || !(fine = mbar_wait(bar(kRwPReady + (j & 1)), (j >> 1) & 1))) break;
        if (R::kOwnP && next == j + 2 && next < units && !fresh) {
          if (!(fine = qk(next))) break;
          firsts = (firsts & ~(1u << (next & 3))) | ((first_next ? 1u : 0u) << (next & 3));
          ++next;
        }
        first_cur = ((firsts >> (j & 3)) & 1u) != 0u;
        item_cur += first_cur ? 1 : 0;
        fine = pv(j);
      }
      if (!fine) {
        flag_error(kErrTimeout);
        *abort_flag = 1;
      }
      tc::commit(bar(kRwFin));  // never leave with MMAs in flight
      if (!mbar_wait(bar(kRwFin), 0)) flag_error(kErrTimeout);
    }
  } else if (warp >= kRwSoft) {
    // ------------------------------------------------------------- dequant
    const bool is_k = warp < kRwSoft + kRwDq;
    int row, chunk;
    rw_place<D>(tid - (is_k ? kRwSoft : kRwSoft + kRwDq) * 32, row, chunk);
    const uint8_t* c0 = (is_k ? p.k_codes : p.v_codes) + (size_t)row * p.kv_heads * (D / 2) + chunk * 16;
    const uint8_t* s0 = (is_k ? p.k_scales : p.v_scales) + (size_t)row * p.kv_heads * (D / 16) + chunk * 2;
    const uint32_t tiles = sb + (is_k ? R::kK : R::kV);
    const int ready = is_k ? kRwKReady : kRwVReady, free = is_k ? kRwKFree : kRwVFree;
    RwChunks<D> regs;
    int entry = cur.entry(p);
    auto load = [&]() {
      const int at = cur.tile * kRwTok;
      const int valid = cur.present(p, entry) ? min(kRwTok, cur.r.kv - at) : 0;
      const size_t token0 = valid > 0 ? (size_t)entry * kPage + (at & (kPage - 1)) : 0;
      rw_load<D>(c0 + cur.h * (D / 2), s0 + cur.h * (D / 16), token0, p.kv_heads, row, valid, regs);
    };
    load();
    if (units > 1) {
      cur.next(p);
      entry = cur.entry(p);
    }
    bool ok = true;
    for (int j = 0; j < units; ++j) {
      const int b = j % NB;
      if (j >= NB) ok &= mbar_wait(bar(free + b), (j / NB - 1) & 1);
      if (__any_sync(kFull, !ok || *abort_flag)) break;
      rw_store<D>(tiles + b * R::kTile, row, chunk, regs);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(ready + b));
      if (j + 1 < units) {
        load();
        if (j + 2 < units) {
          cur.next(p);
          entry = cur.entry(p);
        }
      }
    }
    if (__any_sync(kFull, !ok) && lane == 0) {
      flag_error(kErrTimeout);
      *abort_flag = 1;
    }
  } else {
    // ------------------------------------------------- softmax (thread = row)
    // tcgen05.ld / st / wait are warp-collective: every branch around them is
    // decided by a warp vote.
    const int grp = warp >> 2, wq = warp & 3;  // tiles of parity grp; TMEM lane quadrant
    const int r = 32 * wq + lane;
    const int rpos = r / p.group, rhead = r % p.group;
    const uint32_t lane_base = (uint32_t)(32 * wq) << 16;
    const uint32_t ts = tbase + lane_base + R::kTmS + 128u * grp, to = tbase + lane_base + R::kTmO;
    const uint32_t tp = tbase + lane_base + R::kTmP + R::kTmPStep * grp;
    bool ok = true;
    // 16 of the quadrant's Q rows of the walker's item -> K-major FP16 operand,
    // each row scaled by a power of two (exact for BF16 and FP16)
    auto stage_q = [&](const RowsWalk& w, int item) {
      constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes a row, rows a load
      const int sub = lane / LPR, ln = lane % LPR;
      const int pos0 = w.i * per_pos, npos = min(per_pos, w.r.n - pos0);
      const T* q = reinterpret_cast<const T*>(p.q);
#pragma unroll 1
      for (int base = 32 * wq + 16 * grp; base < 32 * wq + 16 * grp + 16; base += 4) {
        constexpr int U = RPI < 4 ? 4 / RPI : 1;
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int row = base + u * RPI + sub;
          const int pos = row / p.group;
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if (pos < npos)
            v[u] = __ldg(reinterpret_cast<const uint4*>(q + (long long)(w.r.row0 + pos0 + pos) * p.q_stride +
                                                        (w.h * p.group + row % p.group) * D) + ln);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int row = base + u * RPI + sub;
          const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
          float amax = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = InTraits<T>::to_float2(x[e]);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, shfl_xor(amax, o));
          const float sc = pow2_row_scale(amax);
          uint32_t hh[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = InTraits<T>::to_float2(x[e]);
            hh[e] = pack_half2(f.x * sc, f.y * sc);
          }
          sts128(sb + R::kQ + (ln >> 3) * (kRwRows * 128) + row * 128 + (((ln & 7) ^ (row & 7)) << 4), hh[0], hh[1],
                 hh[2], hh[3]);
          if (ln == 0) rowfac[(item & 1) * kRwRows + row] = p.sm_scale_log2 / sc;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kRwQReady));
    };

    stage_q(cur, 0);
    int entry = cur.entry(p);
    int j = 0;  // tile of the CTA
    for (int item = 0; j < units; ++item) {
      // ------------------------------------------------------------ an item
      const int pos0 = cur.i * per_pos, npos = min(per_pos, cur.r.n - pos0);
      const int tile0 = cur.tile, n_tiles = min(cur.tiles - tile0, units - j), head = cur.h;
      const int row0 = cur.r.row0 + pos0;
      const bool starts_here = tile0 == 0, ends_here = tile0 + n_tiles == cur.tiles, valid = rpos < npos;
      const int all_tiles = cur.tiles;
      // keys below lim are visible; rows that do not exist are all zeros in Q
      const int lim = valid ? cur.r.kv - cur.r.n + pos0 + rpos + 1 : 0x7fffffff;
      const int last = j + n_tiles - 1;
      ok &= mbar_wait(bar(kRwQReady), item & 1);  // the other warps' row factors
      if (__any_sync(kFull, !ok || *abort_flag)) break;
      const float fac = rowfac[(item & 1) * kRwRows + r];
      float m_own = -CUDART_INF_F, la = 0.f, lb = 0.f;  // the row sum relative to m_own
      bool fine = true;
      for (int k = 0; k < n_tiles; ++k, ++j) {
        const int t0 = cur.tile * kRwTok;
        const bool here = cur.present(p, entry);
        if (j + 1 < units) {
          cur.next(p);
          entry = cur.entry(p);
        }
        if ((j & 1) != grp) continue;
        ok &= mbar_wait(bar(kRwSFull + grp), (j >> 1) & 1);
        if (__any_sync(kFull, !ok || *abort_flag)) {
          fine = false;
          break;
        }
        tc::fence_after();
        const int room = here ? lim - t0 : 0;  // columns below it count
        const bool masked = !__all_sync(kFull, room >= kRwTok);
        // (loops, not unrolled over the columns: with three roles in one kernel
        // the instruction cache is short)
        float mr = -CUDART_INF_F;
#pragma unroll 1
        for (int c = 0; c < kRwTok; c += 32) {
          float x[32];
          rw_ld32(ts + c, x);
          if (masked) rw_mask(x, room - c);
#pragma unroll
          for (int e = 0; e < 32; e += 2) mr = pf_fmax3(mr, x[e], x[e + 1]);
        }
        const float mt = mr * fac;
        float m_ref = -CUDART_INF_F;
        if (k > 0) {  // the reference after tile j - 1, from the other group's warp
          ok &= mbar_wait(bar(kRwRef + 2 * wq + (grp ^ 1)), ((j - 1) >> 1) & 1);
          if (__any_sync(kFull, !ok)) {
            fine = false;
            break;
          }
          m_ref = ref_s[(grp ^ 1) * kRwRows + r];
        }
        const bool need = mt > m_ref + batch::kRoom;
        const float m_new = need ? mt - batch::kLift : m_ref;
        ref_s[grp * kRwRows + r] = m_new;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kRwRef + 2 * wq + grp));
        const float alpha = (need && m_ref != -CUDART_INF_F) ? exp2_approx(m_ref - m_new) : 1.f;
        const float own = m_own != -CUDART_INF_F ? exp2_approx(m_own - m_new) : 1.f;
        const float mu = m_new == -CUDART_INF_F ? 0.f : m_new;
        la *= own;
        lb *= own;
        m_own = m_new;
        if (R::kOwnP && j >= 2) {  // PV(j - 2) has read this P
          ok &= mbar_wait(bar(kRwPvDone + grp), ((j - 2) >> 1) & 1);
          if (__any_sync(kFull, !ok)) {
            fine = false;
            break;
          }
          tc::fence_after();
        }
#pragma unroll 1
        for (int c = 0; c < kRwTok; c += 32) {
          float x[32];
          rw_ld32(ts + c, x);
          if (masked) rw_mask(x, room - c);
          uint32_t pw[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float p0, p1;
            pf_ffma2(p0, p1, x[2 * e], x[2 * e + 1], fac, -mu);
            pw[e] = pack_half2(exp2_approx(p0), exp2_approx(p1));
            const float2 f = InTraits<__half>::to_float2(pw[e]);  // the sum is of the rounded weights
            pf_fadd2(la, lb, f.x, f.y);
          }
          tc::st_32x32b_x16(tp + c / 2, pw);  // (on top of S: over columns that have been read)
        }
        if (k > 0 && __any_sync(kFull, alpha != 1.f)) {
          ok &= mbar_wait(bar(kRwPvDone + (grp ^ 1)), ((j - 1) >> 1) & 1);
          if (__any_sync(kFull, !ok)) {
            fine = false;
            break;
          }
          tc::fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tc::ld_32x32b_x16(to + c, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              asm volatile("" : "+r"(o[e])::"memory");
              o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            }
            tc::st_32x32b_x16(to + c, o);
          }
        }
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kRwPReady + grp));
      }
      if (!fine) break;
      // the next item's Q while the last PV runs, once the last QK has read this one
      ok &= mbar_wait(bar(kRwSFull + (last & 1)), (last >> 1) & 1);
      if (__any_sync(kFull, !ok)) break;
      if (j < units) stage_q(cur, item + 1);
      // the row's reference and sum over both groups
      ok &= mbar_wait(bar(kRwRef + 2 * wq + (last & 1)), (last >> 1) & 1);
      if (__any_sync(kFull, !ok)) break;
      const float m_fin = ref_s[(last & 1) * kRwRows + r];
      float* sums_of = sum_s + (item & 1) * 2 * kRwRows;
      // (without a reference of its own the group's sum is 0, or NaN from NaN scores)
      sums_of[grp * kRwRows + r] = m_own != -CUDART_INF_F ? (la + lb) * exp2_approx(m_own - m_fin) : la + lb;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kRwSum + wq));
      ok &= mbar_wait(bar(kRwSum + wq), item & 1);
      // ---------------------------------------------------------- epilogue
      ok &= mbar_wait(bar(kRwPvDone + (last & 1)), (last >> 1) & 1);
      if (__any_sync(kFull, !ok)) break;
      tc::fence_after();
      const float l = sums_of[r] + sums_of[kRwRows + r];
      if (starts_here && ends_here) {
        T* out = reinterpret_cast<T*>(p.out) + (long long)(row0 + (valid ? rpos : 0)) * p.out_stride +
                 (head * p.group + rhead) * D;
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
        for (int c = grp * (D / 2); c < (grp + 1) * (D / 2); c += 32) {
          float x[32];
          rw_ld32(to + c, x);
          if (!valid) continue;
          uint4* dst = reinterpret_cast<uint4*>(out + c);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const T a = InTraits<T>::from_float(x[e + 2 * i] * inv), b = InTraits<T>::from_float(x[e + 2 * i + 1] * inv);
              w[i] = (uint32_t)(*reinterpret_cast<const uint16_t*>(&a)) |
                     ((uint32_t)(*reinterpret_cast<const uint16_t*>(&b)) << 16);
            }
            dst[e / 8] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      } else {
        // record [D / 4][128 rows] of float4, then (m, l) a row
        float* rec = p.row_records + (size_t)(blockIdx.x * 2 + (starts_here ? 1 : 0)) * R::kRec;
        float4* ro = reinterpret_cast<float4*>(rec) + r;
#pragma unroll 1
        for (int c = grp * (D / 2); c < (grp + 1) * (D / 2); c += 32) {
          float x[32];
          rw_ld32(to + c, x);
          if (!valid) continue;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            ro[(size_t)((c + e) / 4) * kRwRows] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        }
        if (valid && grp == 0) *reinterpret_cast<float2*>(rec + kRwRows * D + 2 * r) = make_float2(m_fin, l);
        if (starts_here && tid == 0) {
          const long long last_unit = lo + (j - n_tiles) + all_tiles - 1;
          meta[0] = npos * p.group;
          meta[1] = row0;
          meta[3] = head;
          meta[4] = (int)(((last_unit + 1) * n_cta - 1) / total);
          meta[5] = (int)min(total, n_cta);
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kRwEpi));
    }
    if (__any_sync(kFull, !ok) && lane == 0) {
      flag_error(kErrTimeout);
      *abort_flag = 1;
    }
  }

  griddep_launch_dependents();
  tc::fence_before();
  __syncthreads();
  if (warp == kRwMma) {
    tc::fence_after();
    tc::tmem_dealloc(tbase, R::kTmCols);
  }
}

// Merges the records of items that more than one CTA worked on, in CTA order:
// block (i, y) takes rows 8y .. 8y + 7 of the item that CTA i began.
template <typename T, int D>
__global__ void __launch_bounds__(256) batch_rows_combine_kernel(const __grid_constant__ BatchAttnParams p) {
  using R = Rows<D>;
  __shared__ float w[8][kBatchMaxCtas];
  __shared__ float inv_l[8];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, i0 = blockIdx.x, n_cta = gridDim.x, y0 = blockIdx.y * 8;
  const int32_t* meta = p.meta + (kBatchMaxCtas + i0) * kBatchMeta;
  const int rows = __ldcg(meta);
  if (y0 >= rows) return;
  const int base = __ldcg(meta + 1), hd = __ldcg(meta + 3), parts = __ldcg(meta + 4) - i0 + 1, busy = __ldcg(meta + 5);
  auto record = [&](int j) { return p.row_records + (size_t)((i0 + j) * 2 + (j == 0 ? 1 : 0)) * R::kRec; };
  auto empty = [&](int j) {
    const long long i = i0 + j;
    return i * busy / n_cta == (i + 1) * busy / n_cta;
  };
  {  // one warp a row: weights of the parts
    const int row = y0 + (tid >> 5), lane = tid & 31;
    float M = -CUDART_INF_F;
    for (int j = lane; j < parts; j += 32)
      if (row < rows && !empty(j)) M = fmaxf(M, __ldcg(record(j) + kRwRows * D + 2 * row));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, shfl_xor(M, o));
    float L = 0.f;
    for (int j = lane; j < parts; j += 32) {
      float wt = 0.f;
      if (row < rows && !empty(j)) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(record(j) + kRwRows * D + 2 * row));
        wt = batch::part_weight(v.x, v.y, M);
        L += wt * v.y;
      }
      w[tid >> 5][j] = wt;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += shfl_xor(L, o);
    if (lane == 0) inv_l[tid >> 5] = L > 0.f ? 1.f / L : 0.f;
  }
  __syncthreads();
  const int row = y0 + (tid & 7);
  if (row >= rows) return;
  T* out = reinterpret_cast<T*>(p.out) + (long long)(base + row / p.group) * p.out_stride + (hd * p.group + row % p.group) * D;
  for (int d4 = tid >> 3; d4 < D / 4; d4 += 32) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < parts; ++j) {
      const float wj = w[tid & 7][j];
      if (wj == 0.f) continue;
      const float4 v = __ldcg(reinterpret_cast<const float4*>(record(j)) + (size_t)d4 * kRwRows + row);
      a.x += wj * v.x;
      a.y += wj * v.y;
      a.z += wj * v.z;
      a.w += wj * v.w;
    }
    const float s = inv_l[tid & 7];
    T* dst = out + d4 * 4;
    dst[0] = InTraits<T>::from_float(a.x * s);
    dst[1] = InTraits<T>::from_float(a.y * s);
    dst[2] = InTraits<T>::from_float(a.z * s);
    dst[3] = InTraits<T>::from_float(a.w * s);
  }
}

template <typename T, int D>
cudaError_t launch_rows(const BatchAttnParams& p, int ctas, cudaStream_t stream) {
  auto kernel = batch_rows_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Rows<D>::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(ctas), dim3(kRwThreads), Rows<D>::kSmem, stream, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(batch_rows_combine_kernel<T, D>, dim3(ctas, kRwRows / 8), dim3(256), 0, stream, p);
}

}  // namespace qwz
