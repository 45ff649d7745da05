// Attention behind shared prefixes, the parts of many query rows (sm_100a, tcgen05):
// the rows of all requests that read a prefix over the prefix's tokens, and the rows
// of windows and prompt chunks over their own.  The formula is that of batch_few.cu;
// each part (m, l, o) goes to batch_join.cu.
//
// An item is one KV head and 128 (row, head) pairs of a prefix's readers or of a
// request, 256 at D 256; the pairs are the M rows of every MMA, and it visits the
// 128-token tiles of the prefix, or those up to its last row's causal limit.  The
// prefixes' items come first, then the requests'; persistent CTAs, one an SM, take
// equal shares of all tiles (batch_common.cuh).
//
// At D 256 two CTAs of a cluster are one unit (cta_group::2, M = 256): each has 128 of
// the rows, and converts half of K's tokens and half of V's dims into its own shared
// memory for both, which halves the conversions and the shared-memory traffic a row (a
// CTA by itself: 320 KB a tile and 64 K conversions).  The first CTA issues the MMAs.
//
// 20 warps a CTA, the last one idle:
//   warps 0-7    softmax, thread = row (TMEM lane), two groups of four that take the
//                even and the odd tiles; Q staging and the epilogue
//   warps 8-11   dequantise K, warps 12-15 V: codes from the pool into shared memory by
//                cp.async, a ring of the thread's own two slots ahead, FP16 into the
//                operands' layout
//   warp 16      tensor memory; one thread issues QK
//   warp 17      walks the CTA's share and hands its items to the others in a ring,
//                so that no other role reads lengths or plans
//   warp 18      one thread issues PV (with QK from one thread, its waits and commits left
//                the tensor pipe idle for a third of the time)
// K and V pass through rings of 16 KB slots, which are written, read by the MMAs and
// freed one by one: a slot of K is 64 head dims of a tile's 128 tokens (of a CTA's 64:
// 128 dims), one of V 128 / (slots of a tile) tokens of the CTA's dims.
//
// The roles' loops stay rolled: together they have to fit the instruction cache.
// (Codes held four slots ahead in registers, which unrolls the conversion by four, made
// every conversion of a slot take 450 to 1,250 cycles instead of 300.)
//
// What bounds it.  At D 256 S and O fill the tensor memory, so P lies on its own S and
// QK(j + 2) waits for PV(j): a tile's chain QK (1,300 cycles), softmax (3,100), PV (1,300)
// and the waits between take 8,200 cycles, two tiles at a time, 4,100 a tile of 256 rows
// where its MMAs need 2,048.  At D 128 a tile of 128 rows takes 3,200 (1,024): the MMAs of a
// single CTA, whose operands take all of the shared memory's bandwidth, run at half rate
// (two CTAs a unit there: 119 us against 90, since the items are not 256 rows wide).  An item
// costs another 10 us (Q staged 4, the end 5, the first waits), which its weight in the
// shares stands for, at every head dim.  With a weight of two, three, five and eight tiles: 12
// requests with questions behind two prompts of 8,192 tokens, 24/4/256, 461, 402, 348 and
// 359 us, 32/8/128 445, 385, 352 and 361, 14/2/64 165, 151, 142 and 144; 24 windows of 7
// rows behind two of 16,384, 168, 157, 159 and 166, 166, 148, 146 and 154, 74, 66, 66 and
// 67; decode rows differ by less than 3 %.
// Measured, whole calls on the GPU, against the same rows in batch_rows.cu's form: 64 rows
// behind 32,768 tokens, 24/4/256, 130 us (141); 256 of 32/8/128 167 (251); 24 x 7-row
// windows 203 (278); questions of 12 requests 205 (306).
// Not kept, while the windows took 215 us: Q staged by the V warps (219), the softmax's next
// chunk loaded ahead (230), QK(1) of an item held back until P(0) so that the groups
// alternate (228).
#include "attn_common.cuh"
#include "batch_common.cuh"
#include "tc_common.cuh"

namespace qwz {

using namespace detail;

namespace {

constexpr int kTlTok = 128;                  // tokens of a tile
constexpr int kTlRows = 128;                 // MMA rows of a CTA
constexpr int kTlSoft = 8;                   // softmax warps, two groups
constexpr int kTlDq = 4;                     // dequant warps of K, and of V
constexpr int kTlQk = kTlSoft + 2 * kTlDq;
constexpr int kTlSched = kTlQk + 1, kTlPv = kTlQk + 2;
constexpr int kTlWarps = 20;                 // whole warpgroups
constexpr int kTlThreads = kTlWarps * 32;
constexpr int kTlScan = 256;                 // threads that scan the requests
constexpr int kTlSlot = 16384;
constexpr int kTlAhead = 2;                  // slots whose codes are on their way
constexpr int kTlItems = 4;                  // items in flight
constexpr int kTlOver = 5;                   // what an item costs beside its tiles, in tiles (Q, the first waits, the end)
// registers a thread: 640 x 96 at launch; 256 x 112 + 256 x 80 + 128 x 64 after the
// split.  (Spills in these loops cost an L2 access each: there is no L1 left.)
constexpr int kTlSoftRegs = 112, kTlDqRegs = 80, kTlRestRegs = 64;
static_assert(256 * kTlSoftRegs + 256 * kTlDqRegs + 128 * kTlRestRegs <= kTlThreads * 96, "register split");

// Every barrier whose phases are not all waited for by everyone is per slot, tile
// parity or warp pair, so that a waiter is never two phases off.
enum TlBar : int {
  kTlKReady = 0,       // [4] K slot written (by both CTAs, at the first one)
  kTlKFree = 4,        // [4] QK has read it
  kTlVReady = 8,       // [4]
  kTlVFree = 12,       // [4]
  kTlSFull = 16,       // [2] S(j) is there (j's parity)
  kTlPReady = 18,      // [2] P(j) is written (both CTAs, at the first one)
  kTlPvDone = 20,      // [2] PV(j) is done
  kTlRef = 22,         // [4 warps][2] the reference maxima after tile j
  kTlSum = 30,         // [4 warps] both groups' row sums of the item
  kTlQReady = 34,      // the item's Q is staged (both CTAs, at the first one)
  kTlEpi = 35,         // the item's O has been read (both CTAs, at the first one)
  kTlFin = 36,         // [2] the last QK, the last PV
  kTlItemFull = 38,    // [4]
  kTlItemFree = 42,    // [4]
  kTlQHere = 46,       // the item's row factors of this CTA are written
  kTlNumBars = 48      // (one unused)
};

// One item of a share (n_tiles 0: the share's end).
struct TlItem {
  int n_tiles, tile0;         // of this share
  int parts;                  // where it begins here: CTAs (clusters) that share it
  int head, table;            // KV head, row of the block table
  int kv, lim;                // tokens; tokens that the request's first row sees
  int pair0, pairs;           // the item's first (row, head) pair and their number
  int row0;                   // of q, of a prefix: place in shared_rows
  int pre, joins;             // a prefix; whether the rows have parts
};

template <int D>
struct Tiles {
  static constexpr int kCtas = D == 256 ? 2 : 1;         // of a cluster
  static constexpr int kRows = kTlRows * kCtas;          // pairs of an item
  static constexpr int kSub = D / 64 / kCtas;            // slots of a tile
  static constexpr int kSlots = kCtas == 2 ? 3 : 4;      // of a ring
  static constexpr int kQ = 0;                           // D / 64 atoms of [128 rows x 128 B]
  static constexpr int kK = kQ + kTlRows * D * 2;
  static constexpr int kV = kK + kSlots * kTlSlot;
  static constexpr int kCode = kV + kSlots * kTlSlot;    // [K, V][kTlAhead + 1][256 chunks of 32 dims] x 16 B
  static constexpr int kScale = kCode + 2 * (kTlAhead + 1) * 4096;  // and the 4 B that hold their scales
  static constexpr int kBars = kScale + 2 * (kTlAhead + 1) * 1024;
  static constexpr int kMeta = kBars + 8 * kTlNumBars;   // TMEM base, abort flag
  static constexpr int kRowfac = kMeta + 16;             // [2][128] by item parity
  static constexpr int kRef = kRowfac + 8 * kTlRows;     // [2][128] by tile parity
  static constexpr int kSum = kRef + 8 * kTlRows;        // [2][2][128] by item parity and group
  static constexpr int kItem = kSum + 16 * kTlRows;      // [kTlItems]
  static constexpr int kStarts = kItem + kTlItems * (int)sizeof(TlItem);  // [kTlScan] units before each scanning thread
  static constexpr int kSums = kStarts + 8 * kTlScan;    // [32]
  static constexpr int kStage = kSums + 8 * 32;          // [kTlSoft][32 rows][kPitch] of the epilogue
  static constexpr int kPitch = 80;                      // 64 B of a row, and 16 that spread the rows over the banks
  static constexpr int kSmem = kStage + kTlSoft * 32 * kPitch + 1024;
  static_assert(kSmem <= 227 * 1024 && kBars % 16 == 0 && kMeta % 16 == 0 && kStarts % 8 == 0 && kStage % 16 == 0,
                "shared memory");
  // tensor memory: S of even and odd tiles, O; P has columns of its own where they
  // fit, so that S is free for QK(j + 2) as soon as the softmax has read it
  static constexpr bool kOwnP = D <= 128;
  static constexpr uint32_t kTmS = 0, kTmO = 256, kTmP = kOwnP ? 384 : 0, kTmPStep = kOwnP ? 64 : 128, kTmCols = 512;
  static constexpr size_t kRec = (size_t)kRows * (D + 2);  // floats of a record
};

// The units (request, head, group of pairs, tile) of the launch.  `b` below p.requests
// is the prefix b, whose rows are those that read it; b - p.requests a request.
template <int PER>
struct TilesWalk {
  int b, h, i, at, tiles, groups, pairs;  // at: weighed unit of the item
  bool pre, small;
  batch::Req r;

  // Whether those that read prefix b do so in batch_few.cu, in front of their own
  // tokens: a request alone behind it with few columns (no records, and no tile of
  // 128 rows for eight), or all of them where that is little work.
  QWZ_DEVINL static bool direct(const BatchAttnParams& p, int b, const batch::Req& r, bool small) {
    return small || (r.n * p.group <= p.few_cols && __ldg(p.alone + b) >= 0);
  }
  QWZ_DEVINL static batch::Req load(const BatchAttnParams& p, int b, bool small) {
    batch::Req r;
    if (b >= p.requests) {
      r = batch::load_req(p, b - p.requests);
      if (r.n * p.group <= p.few_cols) r.n = 0;  // batch_few.cu's
    } else {
      r = batch::load_prefix(p, b);
      if (direct(p, b, r, small)) r.n = 0;
    }
    return r;
  }
  QWZ_DEVINL static int tiles_of(const BatchAttnParams& p, const batch::Req& r, int i, bool pre) {
    const int last = min((i + 1) * PER, r.n * p.group) - 1;  // pair
    const int lim = pre ? r.kv : r.kv - r.n + last / p.group + 1;
    return max(1, (lim + kTlTok - 1) / kTlTok);
  }
  // Weighed units of a KV head: an item has kTlOver of them in front of its tiles.
  QWZ_DEVINL static long long head_cost(const BatchAttnParams& p, const batch::Req& r, bool pre) {
    const int groups = (r.n * p.group + PER - 1) / PER;
    if (pre) return groups > 0 ? (long long)groups * (kTlOver + tiles_of(p, r, 0, true)) : 0;
    long long c = 0;
    for (int i = 0; i < groups; ++i) c += kTlOver + tiles_of(p, r, i, false);
    return c;
  }
  QWZ_DEVINL static long long cost(const BatchAttnParams& p, int b, bool small) {
    return p.kv_heads * head_cost(p, load(p, b, small), b < p.requests);
  }
  QWZ_DEVINL void enter(const BatchAttnParams& p, int bb) {
    b = bb;
    pre = b < p.requests;
    r = load(p, b, small);
    pairs = r.n * p.group;
    groups = (pairs + PER - 1) / PER;
  }
  QWZ_DEVINL void seek(const BatchAttnParams& p, int b0, long long u) {
    for (b = b0; b < 2 * p.requests - 1; ++b) {
      const long long c = cost(p, b, small);
      if (u < c) break;
      u -= c;
    }
    enter(p, b);
    const long long c = max(1LL, head_cost(p, r, pre));
    h = (int)(u / c);
    u %= c;
    for (i = 0; i < groups - 1; ++i) {
      const int t = kTlOver + tiles_of(p, r, i, pre);
      if (u < t) break;
      u -= t;
    }
    tiles = tiles_of(p, r, i, pre);
    at = (int)u;
  }
  QWZ_DEVINL void next_item(const BatchAttnParams& p) {
    at = 0;
    if (++i >= groups) {
      i = 0;
      if (++h >= p.kv_heads) {
        h = 0;
        for (int bb = b + 1; bb < 2 * p.requests; ++bb) {
          enter(p, bb);
          if (r.n > 0) break;
        }
      }
    }
    tiles = tiles_of(p, r, i, pre);
  }
  QWZ_DEVINL void item(const BatchAttnParams& p, TlItem& t) const {
    t.head = h;
    t.table = pre ? b : b - p.requests;
    t.kv = r.kv;
    t.lim = r.kv - r.n + 1;
    t.pair0 = i * PER;
    t.pairs = min(PER, pairs - i * PER);
    t.row0 = r.row0;
    t.pre = pre;
    t.joins = pre || batch::prefix_of(p, b - p.requests) >= 0;
  }
};

// The row of q and out at a place of shared_rows (-1, and the error bit, for an
// entry that is none).
QWZ_DEVINL int tl_shared_row(const BatchAttnParams& p, int at) {
  const int row = __ldg(p.shared_rows + at);
  if (row >= 0 && row < p.rows) return row;
  flag_error(kErrTableRange);
  return -1;
}

// Whether every row behind a prefix is one of few and what they would read of
// prefixes by themselves (tokens x KV heads) costs less than the records, the 128-row
// tiles and the first wait of this kernel.  Calls with decode rows of own lengths to 500,
// read by themselves and in tiles: 24/4/256, 4 behind 4,096 (65,536) 27 and 48 us, 16
// behind 4,096 (262,144) 39 and 50, 64 behind 2,048 (524,288) 64 and 66, 16 behind 10,240
// (655,360) 60 and 57, 16 behind 16,384 81 and 63; 32/8/128, 64 behind 1,024 (524,288) 52
// and 58, 64 behind 1,536 (786,432) 60 and 59; 14/2/64, 64 behind 4,096 (524,288) 35 and
// 39, 64 behind 6,144 (786,432) 40 and 41, 64 behind 8,192 45 and 42.
constexpr long long kTlSmall = 600 * 1024;
// Also: `any`, whether a request has more rows than batch_few.cu takes.
QWZ_DEVINL bool tl_small(const BatchAttnParams& p, long long* sums, bool& any) {
  const int per = (p.requests + kTlScan - 1) / kTlScan;
  long long mine = 0, total;
  int wide = 0;  // 1: a request with many rows, 2: one that reads a prefix
  if (threadIdx.x < kTlScan)
    for (int b = threadIdx.x * per; b < min(p.requests, (int)(threadIdx.x + 1) * per); ++b) {
      const int g = batch::prefix_of(p, b), n = batch::load_req(p, b).n;
      if (g >= 0 && n > 0) mine += batch::tokens_of(p, g);
      if (n * p.group > p.few_cols) wide |= g >= 0 ? 3 : 1;
    }
  any = __syncthreads_or(wide) != 0;
  const bool behind = __syncthreads_or(wide & 2) != 0;
  batch::block_scan(mine, sums, total);
  return !behind && total * p.kv_heads <= kTlSmall;
}

// BYTES (4 or 16) to shared memory; zeros without a read where there is nothing.
template <int BYTES>
QWZ_DEVINL void tl_copy(uint32_t dst, const uint8_t* src, bool some) {
  if constexpr (BYTES == 16)
    cp_async16(dst, src, some ? 16u : 0u);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(some ? 4u : 0u));
}

// What two CTAs of a cluster do together; with C 1 all of it stays in the CTA.
template <int C>
struct Pair {
  QWZ_DEVINL static int rank() {
    if constexpr (C == 1) return 0;
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return (int)r;
  }
  QWZ_DEVINL static void sync() {
    if constexpr (C == 1) {
      __syncthreads();
    } else {
      asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    }
  }
  // Arrives at the barrier of the first CTA.  What it stands for is in the arriving
  // CTA's own shared or tensor memory, behind a proxy fence or a tcgen05 wait: no
  // release to the cluster, which takes a thousand cycles here.
  QWZ_DEVINL static void arrive(uint32_t bar) {
    if constexpr (C == 1) {
      mbar_arrive(bar);
    } else {
      asm volatile(
          "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n"
          " mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(bar)
          : "memory");
    }
  }
  QWZ_DEVINL static void alloc(uint32_t dst, uint32_t cols) {
    if constexpr (C == 1) {
      tc::tmem_alloc(dst, cols);
      tc::tmem_relinquish();
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(dst), "r"(cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
  }
  QWZ_DEVINL static void dealloc(uint32_t at, uint32_t cols) {
    if constexpr (C == 1)
      tc::tmem_dealloc(at, cols);
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(at), "r"(cols) : "memory");
  }
  QWZ_DEVINL static void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (C == 1) {
      tc::mma_ss(d, a, b, idesc, accumulate);
    } else {
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
          " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n}\n" ::"r"(d),
          "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
          : "memory");
    }
  }
  QWZ_DEVINL static void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (C == 1) {
      tc::mma_ts(d, a, b, idesc, accumulate);
    } else {
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
          " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n}\n" ::"r"(d),
          "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
          : "memory");
    }
  }
  // Arrives once at the barrier of every CTA when the MMAs issued so far are done.
  QWZ_DEVINL static void commit(uint32_t bar) {
    if constexpr (C == 1)
      tc::commit(bar);
    else
      asm volatile(
          "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
          "h"((uint16_t)3)
          : "memory");
  }
};

// The weighed units of batch_few.cu before each request, by one CTA: each of its CTAs
// would else scan all requests, five dependent loads each, before its first copy.
template <int D>
QWZ_DEVINL void tl_few_starts(const BatchAttnParams& p, bool small, long long* sums) {
  using Walk = FewWalk<Few<D>::kUnit, kBatchShared>;
  const int per = (p.requests + kTlThreads - 1) / kTlThreads, b0 = threadIdx.x * per, b1 = min(p.requests, b0 + per);
  for (int c = 0; c < p.col_groups; ++c) {
    long long* out = p.few_starts + (size_t)c * (p.requests + 1);
    long long mine = 0, total;
    for (int b = b0; b < b1; ++b) {
      const batch::Req r = batch::load_req(p, b);
      int g = batch::prefix_of(p, b);
      if (g >= 0 && !TilesWalk<Tiles<D>::kRows>::direct(p, g, batch::load_prefix(p, g), small)) g = -1;
      const long long cost = Walk::few(p, r, c * kFewCols) ? Walk::units_of(p, r, g) + Walk::kOver : 0;
      out[b] = cost;  // (its own cost for now)
      mine += cost;
    }
    long long at = batch::block_scan(mine, sums, total);
    for (int b = b0; b < b1; ++b) {
      const long long cost = out[b];
      out[b] = at;
      at += cost;
    }
    if (threadIdx.x == 0) out[p.requests] = total;
  }
}

// a and b plus the two weights of w.  The sums take the rounded weights, as in
// batch_few.cu: a row's weights add up to one, and the rounding of a dominant weight
// cancels (the error is then at most 2^-11 of the sum of p |v - out|).  (FP16 and FP32 in one addition; a conversion and an addition in pairs behind the
// chunk's vote: 24 windows of 7 rows 233 us, 216 so; of the unrounded weights 212.)
QWZ_DEVINL void tl_add_pair(float& a, float& b, uint32_t w) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n add.f32.f16 %0, l, %0;\n add.f32.f16 %1, h, %1;\n}\n"
      : "+f"(a), "+f"(b)
      : "r"(w));
}

template <int REGS>
QWZ_DEVINL void tl_more_regs() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS));
}
template <int REGS>
QWZ_DEVINL void tl_fewer_regs() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS));
}

// Columns [first, first + D / 2) of the warp's 32 tensor-memory rows to the places of
// the lanes' rows (null: not stored), through shared memory so that four lanes write
// 64 bytes of a row: as FP32, or as T times the row's factor.  (A lane writing its own
// row 16 bytes at a time took 7 us an item instead of 5.)
template <typename T, int D, bool FINAL>
QWZ_DEVINL void tl_store_rows(uint32_t stage, uint32_t taddr, int first, void* dst, float factor) {
  constexpr int kPitch = Tiles<D>::kPitch, kCols = FINAL ? 32 : 16;
  const int lane = threadIdx.x & 31, quarter = lane & 3;
  uint8_t* rows[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    rows[i] = reinterpret_cast<uint8_t*>(__shfl_sync(kFull, reinterpret_cast<unsigned long long>(dst), 8 * i + (lane >> 2)));
#pragma unroll 1
  for (int c = first; c < first + D / 2; c += kCols) {
    uint32_t x[16];
    if constexpr (FINAL) {
      float f[32];
      rw_ld32(taddr + c, f);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const T a = InTraits<T>::from_float(f[2 * e] * factor), b = InTraits<T>::from_float(f[2 * e + 1] * factor);
        x[e] = (uint32_t)(*reinterpret_cast<const uint16_t*>(&a)) | ((uint32_t)(*reinterpret_cast<const uint16_t*>(&b)) << 16);
      }
    } else {
      tc::ld_32x32b_x16(taddr + c, x);
      tc::wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) asm volatile("" : "+r"(x[e])::"memory");
    }
#pragma unroll
    for (int e = 0; e < 16; e += 4) sts128(stage + lane * kPitch + 4 * e, x[e], x[e + 1], x[e + 2], x[e + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = lds128(stage + (8 * i + (lane >> 2)) * kPitch + 16 * quarter);
      if (rows[i] != nullptr) *reinterpret_cast<uint4*>(rows[i] + c * (FINAL ? 2 : 4) + 16 * quarter) = v;
    }
    __syncwarp();
  }
}

// The warp's first n chunks (of 32 columns) of P times the row's factor, a power of two
// (references are whole numbers), in two steps, since FP16 has no powers below 2^-24.  Weights
// that stay above 2^-14 keep their bits; below it they lose up to 2^-25, of a largest weight
// of 2^6 at least (the row's sum keeps them: 2^-31 of it a weight).
__noinline__ __device__ void tl_scale_p(uint32_t tp, int n, float factor) {
  tc::wait_st();
  const float first = fmaxf(factor, 6.103515625e-5f), second = factor / first;  // 2^-14 at least, the rest
  const uint32_t f = pack_half2(first, first), f2 = pack_half2(second, second);
#pragma unroll 1
  for (int c = 0; c < n; ++c) {
    uint32_t x[16];
    tc::ld_32x32b_x16(tp + 16 * c, x);
    tc::wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      asm volatile("" : "+r"(x[e])::"memory");
      x[e] = hmul2_u32(hmul2_u32(x[e], f), f2);
    }
    tc::st_32x32b_x16(tp + 16 * c, x);
  }
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kTlThreads, 1) batch_tiles_kernel(const __grid_constant__ BatchAttnParams p) {
  using R = Tiles<D>;
  constexpr int S = R::kSub, C = R::kCtas;
  using G = Pair<C>;
  using Walk = TilesWalk<R::kRows>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sraw = smem_u32(smem);
  const uint32_t sb = (sraw + 1023u) & ~1023u;
  uint8_t* sg = smem + (sb - sraw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = G::rank();
  auto bar = [&](int i) -> uint32_t { return sb + R::kBars + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sg + R::kMeta + 4);
  const volatile TlItem* items = reinterpret_cast<const volatile TlItem*>(sg + R::kItem);
  long long* starts = reinterpret_cast<long long*>(sg + R::kStarts);
  long long* sums = reinterpret_cast<long long*>(sg + R::kSums);

  if (tid == 0) {
#pragma unroll 1
    for (int i = 0; i < kTlNumBars; ++i) {
      const int count = i < kTlKFree || (i >= kTlVReady && i < kTlVFree) ? kTlDq * C
                        : i == kTlPReady || i == kTlPReady + 1           ? kTlSoft / 2 * C
                        : i >= kTlSum && i < kTlQReady                   ? 2
                        : i == kTlQReady || i == kTlEpi                  ? kTlSoft * C
                        : i == kTlQHere                                  ? kTlSoft
                        : i >= kTlItemFree && i < kTlQHere               ? kTlQk + (rank == 0 ? 2 : 0)
                                                                         : 1;
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kTlQk) G::alloc(sb + R::kMeta, R::kTmCols);
  griddep_wait();

  // ---------------------------------------------------- this CTA's (cluster's) share
  bool any;
  const bool small = tl_small(p, sums, any);
  if (blockIdx.x == 0)
    for (int g = tid; g < p.requests; g += kTlThreads) p.direct[g] = Walk::direct(p, g, batch::load_prefix(p, g), small);
  const int per = (2 * p.requests + kTlScan - 1) / kTlScan;
  long long mine = 0, total = 0;
  if (any || !small) {
    if (tid < kTlScan)
      for (int b = tid * per; b < min(2 * p.requests, (tid + 1) * per); ++b) mine += Walk::cost(p, b, small);
    const long long before = batch::block_scan(mine, sums, total);
    if (tid < kTlScan) starts[tid] = before;
  }
  if (blockIdx.x + 1 == gridDim.x) tl_few_starts<D>(p, small, sums);  // batch_few.cu's shares, for all of its CTAs
  const int cluster = blockIdx.x / C, clusters = gridDim.x / C;
  const long long lo = (long long)cluster * total / clusters, hi = ((long long)cluster + 1) * total / clusters;
  if (tid == 0 && blockIdx.x == 0) p.busy[0] = (int)min(total, (long long)clusters);
  tc::fence_before();
  __syncthreads();
  if (C > 1) G::sync();  // the barriers of both CTAs
  tc::fence_after();
  const uint32_t tbase = *reinterpret_cast<volatile uint32_t*>(sg + R::kMeta);

  // Item k of the share, for the calling warp (whole warps only).
  auto take = [&](int k, TlItem& t) -> bool {
    const bool ok = mbar_wait(bar(kTlItemFull + k % kTlItems), (k / kTlItems) & 1);
    const volatile TlItem& src = items[k % kTlItems];
    t.n_tiles = ok ? src.n_tiles : 0;
    t.tile0 = src.tile0;
    t.parts = src.parts;
    t.head = src.head;
    t.table = src.table;
    t.kv = src.kv;
    t.lim = src.lim;
    t.pair0 = src.pair0;
    t.pairs = src.pairs;
    t.row0 = src.row0;
    t.pre = src.pre;
    t.joins = src.joins;
    return ok;
  };
  auto taken = [&](int k) { mbar_arrive(bar(kTlItemFree + k % kTlItems)); };

  if (lo == hi) {
    // nothing to do
  } else if (warp >= kTlQk) {
    tl_fewer_regs<kTlRestRegs>();
    if (warp == kTlSched && lane == 0) {
      // ------------------------------------------------------------ items
      Walk w;
      w.small = small;
      int at = 0;
      for (int step = kTlScan / 2; step > 0; step >>= 1)
        if (starts[at + step] <= lo) at += step;
      w.seek(p, at * per, lo - starts[at]);
      bool ok = true;
      long long pos = lo;  // weighed unit of the launch
      for (int k = 0;; ++k) {
        int tile0 = 0, n = 0, rest = 0;  // (rest: units of the item from pos on)
        while (pos < hi) {
          rest = w.tiles + kTlOver - w.at;
          const int take_units = (int)min((long long)rest, hi - pos);
          tile0 = max(w.at - kTlOver, 0);
          n = max(w.at + take_units - kTlOver, 0) - tile0;
          if (n > 0) break;
          pos += take_units;  // the item's tiles are the next CTA's
        }
        if (k >= kTlItems) ok = mbar_wait(bar(kTlItemFree + k % kTlItems), (k / kTlItems - 1) & 1);
        if (!ok || *abort_flag) break;
        TlItem& t = reinterpret_cast<TlItem*>(sg + R::kItem)[k % kTlItems];
        t.n_tiles = n;
        t.tile0 = tile0;
        t.parts = 1;
        if (n > 0) {
          w.item(p, t);
          if (rest > hi - pos) t.parts = (int)(((pos + rest) * clusters - 1) / total) - cluster + 1;
        }
        mbar_arrive(bar(kTlItemFull + k % kTlItems));
        if (n == 0) break;
        pos += rest;
        if (pos < hi) w.next_item(p);
      }
      if (!ok) {
        flag_error(kErrTimeout);
        *abort_flag = 1;
      }
    } else if (warp == kTlQk && lane == 0 && rank == 0) {
      // --------------------------------------------------------------- QK
      constexpr uint32_t idesc = tc::idesc_f16_f32(kTlRows * C, kTlTok);
      constexpr int kAtom = kTlTok / C * 128;  // bytes of 64 dims in a slot
      const uint64_t dq = tc::smem_desc_k128(sb + R::kQ), dk = tc::smem_desc_k128(sb + R::kK);
      int slot = 0, phase = 0, j = 0;
      bool fine = true;
#pragma unroll 1
      for (int item = 0; fine; ++item) {
        fine = mbar_wait(bar(kTlItemFull + item % kTlItems), (item / kTlItems) & 1);
        const int end = j + (fine ? items[item % kTlItems].n_tiles : 0);
        if (end == j) break;
        taken(item);
        if (fine) fine = mbar_wait(bar(kTlQReady), item & 1);
#pragma unroll 1
        for (; fine && j < end; ++j) {
          // S(j) goes where P(j - 2) was read from; with a P of its own, where the softmax has read S(j - 2)
          if (j >= 2) fine = mbar_wait(bar((R::kOwnP ? kTlPReady : kTlPvDone) + (j & 1)), ((j - 2) >> 1) & 1);
          const uint32_t d = tbase + R::kTmS + 128u * (j & 1);
#pragma unroll 1
          for (int a = 0; fine && a < S; ++a) {
            fine = mbar_wait(bar(kTlKReady + slot), phase) && !*abort_flag;
            if (!fine) break;
            tc::fence_after();
            const uint64_t dka = dk + (uint64_t)((slot * kTlSlot) >> 4), dqa = dq + (uint64_t)((a * C * (kTlRows * 128)) >> 4);
#pragma unroll
            for (int i = 0; i < 4 * C; ++i)
              G::mma_ss(d, dqa + (uint64_t)(((i >> 2) * (kTlRows * 128) + (i & 3) * 32) >> 4),
                        dka + (uint64_t)(((i >> 2) * kAtom + (i & 3) * 32) >> 4), idesc, a + i > 0);
            G::commit(bar(kTlKFree + slot));
            if (++slot == R::kSlots) {
              slot = 0;
              phase ^= 1;
            }
          }
          if (fine) G::commit(bar(kTlSFull + (j & 1)));
        }
      }
      if (!fine) {
        flag_error(kErrTimeout);
        *abort_flag = 1;
      }
      G::commit(bar(kTlFin));  // never leave with MMAs in flight
      if (!mbar_wait(bar(kTlFin), 0)) flag_error(kErrTimeout);
    } else if (warp == kTlPv && lane == 0 && rank == 0) {
      // --------------------------------------------------------------- PV
      constexpr uint32_t idesc = tc::idesc_f16_f32(kTlRows * C, D, /*b_mn_major=*/true);
      const uint64_t dv = tc::smem_desc_mn128(sb + R::kV, kTlTok / S * 128, 1024);
      int slot = 0, phase = 0, j = 0;
      bool fine = true;
#pragma unroll 1
      for (int item = 0; fine; ++item) {
        fine = mbar_wait(bar(kTlItemFull + item % kTlItems), (item / kTlItems) & 1);
        const int begin = j, end = j + (fine ? items[item % kTlItems].n_tiles : 0);
        if (end == j) break;
        taken(item);
        // the item's first PV overwrites O: all of the old one has been read
        if (fine && item > 0) fine = mbar_wait(bar(kTlEpi), (item - 1) & 1);
#pragma unroll 1
        for (; fine && j < end; ++j) {
          fine = mbar_wait(bar(kTlPReady + (j & 1)), (j >> 1) & 1);
#pragma unroll 1
          for (int s = 0; fine && s < S; ++s) {
            fine = mbar_wait(bar(kTlVReady + slot), phase) && !*abort_flag;
            if (!fine) break;
            tc::fence_after();
            const uint64_t dva = dv + (uint64_t)((slot * kTlSlot) >> 4);
            const uint32_t ap = tbase + R::kTmP + R::kTmPStep * (j & 1) + 8u * (8 / S) * s;
#pragma unroll
            for (int kk = 0; kk < 8 / S; ++kk)
              G::mma_ts(tbase + R::kTmO, ap + 8u * kk, dva + (uint64_t)((kk * 2048) >> 4), idesc,
                        (j > begin || s + kk > 0) ? 1u : 0u);
            G::commit(bar(kTlVFree + slot));
            if (++slot == R::kSlots) {
              slot = 0;
              phase ^= 1;
            }
          }
          if (fine) G::commit(bar(kTlPvDone + (j & 1)));
        }
      }
      if (!fine) {
        flag_error(kErrTimeout);
        *abort_flag = 1;
      }
      G::commit(bar(kTlFin + 1));
      if (!mbar_wait(bar(kTlFin + 1), 0)) flag_error(kErrTimeout);
    }
  } else if (warp >= kTlSoft) {
    tl_fewer_regs<kTlDqRegs>();
    // ------------------------------------------------------------- dequant
    // A thread has 32 head dims of two tokens in a slot.  Eight neighbouring lanes hold
    // eight tokens of one chunk, so the swizzled 16-byte stores of a quarter warp touch
    // every bank once.
    const bool is_k = warp < kTlSoft + kTlDq;
    const int t = tid - (is_k ? kTlSoft : kTlSoft + kTlDq) * 32;
    constexpr int CK = 2 * C, CV = D / (32 * C);  // chunks of a token in a slot
    const int row = (t & 7) + 8 * (t / (8 * (is_k ? CK : CV)));
    const int chunk = (t >> 3) % (is_k ? CK : CV);
    const int half = is_k ? 128 / CK : 128 / CV;  // tokens from the thread's first one to its second
    const int tstep = is_k ? 0 : kTlTok / S;      // tokens from a slot of a tile to the next one
    // in the pool: the thread's first token of a tile, its chunk, and the chunk's step from slot to slot
    const int tok0 = row + (is_k ? rank * (kTlTok / C) : 0), chunk0 = chunk + (is_k ? 0 : rank * CV), cstep = is_k ? CK : 0;
    const int ready = is_k ? kTlKReady : kTlVReady, free = is_k ? kTlKFree : kTlVFree;
    const uint32_t codes = sb + R::kCode + (is_k ? 0 : (kTlAhead + 1) * 4096) + t * 16;
    const uint32_t scales = sb + R::kScale + (is_k ? 0 : (kTlAhead + 1) * 1024) + t * 4;
    // where the thread's two halves of a slot go, but for the slot and the swizzle
    const uint32_t to = sb + (is_k ? R::kK : R::kV) + (chunk >> 1) * (is_k ? kTlTok / C : kTlTok / S) * 128 + row * 128;
    const uint32_t swz = (uint32_t)(row & 7) << 4, inner = (uint32_t)(chunk & 1) << 6;
    bool ok = true, more = true;
    int made = 0;  // slots whose copies are on their way
    // place of the next copy: item, tile, slot of the tile, the thread's codes and scales there
    int k = 0, left = 0, tile = 0, head = 0, kv = 0, entry = 0, room = 0, table = 0, sub = 0, buf = 0;
    const uint8_t *cp = nullptr, *sp = nullptr;
    auto copy = [&]() {
      if (sub == 0) {  // a new tile
        if (left == 0) {
          TlItem it;
          if (more) ok &= take(k, it);
          more = more && __all_sync(kFull, ok) && it.n_tiles > 0;
          if (!more) return;
          __syncwarp();
          if (lane == 0) taken(k);
          ++k;
          left = it.n_tiles;
          tile = it.tile0;
          head = it.head;
          kv = it.kv;
          table = it.table;
          entry = __ldg(p.block_table + (size_t)table * p.table_width + tile / (kPage / kTlTok));
        }
        const int at = tile * kTlTok;
        const bool in_pool = kv > 0 && entry >= 0 && entry < p.num_pages;
        if (kv > 0 && !in_pool) flag_error(kErrPageRange);  // its tokens count as absent
        room = in_pool ? kv - at - tok0 : 0;  // tokens of the tile from the thread's first one on
        const size_t unit = ((size_t)(in_pool ? entry * (long long)kPage + (at & (kPage - 1)) : 0) + tok0) * p.kv_heads + head;
        cp = (is_k ? p.k_codes : p.v_codes) + unit * (D / 2) + chunk0 * 16;
        sp = (is_k ? p.k_scales : p.v_scales) + unit * (D / 16) + (chunk0 & ~1) * 2;  // (4 bytes: two chunks' scales)
        ++tile;
        if (--left > 0) entry = __ldg(p.block_table + (size_t)table * p.table_width + tile / (kPage / kTlTok));
      }
      const int pitch = p.kv_heads * (D / 32);  // chunks of a token
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool some = room > sub * tstep + e * half;
        const int step = some ? sub * cstep + (sub * tstep + e * half) * pitch : 0;
        tl_copy<16>(codes + buf * 4096 + e * 2048, some ? cp + step * 16 : p.k_codes, some);
        tl_copy<4>(scales + buf * 1024 + e * 512, some ? sp + step * 2 : p.k_scales, some);
      }
      if (++sub == S) sub = 0;
      if (++buf == kTlAhead + 1) buf = 0;
      ++made;
    };
    int slot = 0, phase = 1, from = 0;  // ring slot; parity of its last freeing; code buffer
#pragma unroll 1
    for (int n = -kTlAhead;; ++n) {
      copy();
      cp_async_commit();
      if (n < 0) continue;
      if (n >= made) break;
      if (n >= R::kSlots) ok &= mbar_wait(bar(free + slot), phase);
      if (__any_sync(kFull, !ok || *abort_flag)) break;
      cp_async_wait<kTlAhead>();  // the thread's own copies of this slot
      uint32_t sc = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        sc |= ((lds32(scales + from * 1024 + e * 512) >> (16 * (chunk0 & 1))) & 0xffffu) << (16 * e);
      uint32_t sp01[2];
      e4m3x4_to_f16x2x2(sc, sp01[0], sp01[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 words = lds128(codes + from * 4096 + e * 2048);
        const uint32_t sl = __byte_perm(sp01[e], 0, 0x1010), sh = __byte_perm(sp01[e], 0, 0x3232);
        const uint32_t x[4] = {words.x, words.y, words.z, words.w};
        const uint32_t base = to + slot * kTlSlot + e * half * 128;  // (half is a multiple of 8)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t h[4];
          e2m1x8_to_f16x2x4(x[j], h);
          const uint32_t s = j < 2 ? sl : sh;
          sts128(base + ((inner + 16 * j) ^ swz), hmul2_u32(h[0], s), hmul2_u32(h[1], s), hmul2_u32(h[2], s),
                 hmul2_u32(h[3], s));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) G::arrive(bar(ready + slot));
      if (++slot == R::kSlots) {
        slot = 0;
        phase ^= 1;
      }
      if (++from == kTlAhead + 1) from = 0;
    }
    cp_async_wait<0>();
    if (__any_sync(kFull, !ok) && lane == 0) {
      flag_error(kErrTimeout);
      *abort_flag = 1;
    }
  } else {
    tl_more_regs<kTlSoftRegs>();
    // ------------------------------------------------- softmax (thread = row)
    // tcgen05.ld / st / wait are warp-collective: every branch around them is
    // decided by a warp vote.
    const int grp = warp >> 2, wq = warp & 3;  // tiles of parity grp; TMEM lane quadrant
    const int r = 32 * wq + lane, rr = rank * kTlRows + r;  // row of the CTA, pair of the item
    const uint32_t lane_base = (uint32_t)(32 * wq) << 16;
    const uint32_t ts = tbase + lane_base + R::kTmS + 128u * grp, to = tbase + lane_base + R::kTmO;
    const uint32_t tp = tbase + lane_base + R::kTmP + R::kTmPStep * grp;
    bool ok = true;
    // 16 of the quadrant's Q rows of an item -> K-major FP16 operand, two lanes a row:
    // copied to its place as it is; BF16 rows are then scaled there by a power of two that
    // makes them exact in FP16.  (Rolled, and without sums over lanes in the loops: code
    // that runs once an item comes from L2, and a chain of shuffles a row took 7 us.)
    auto stage_q = [&](const TlItem& it, int item) {
      constexpr int N = D / 16;  // 16-byte chunks of a lane
      const int row = 32 * wq + 16 * grp + (lane >> 1), at = rank * kTlRows + row, c = it.pair0 + at;
      int q_row = -1;
      if (at < it.pairs) q_row = it.pre ? tl_shared_row(p, it.row0 + c / p.group) : it.row0 + c / p.group;
      const int first = (lane & 1) * N;
      const T* from = reinterpret_cast<const T*>(p.q);
      if (q_row >= 0) from += q_row * p.q_stride + (it.head * p.group + c % p.group) * D + first * 8;
      auto place = [&](int n) {  // of the lane's chunk n
        return sb + R::kQ + ((first + n) >> 3) * (kTlRows * 128) + row * 128 + ((((first + n) & 7) ^ (row & 7)) << 4);
      };
#pragma unroll 4
      for (int n = 0; n < N; ++n) cp_async16(place(n), from + (q_row >= 0 ? n * 8 : 0), q_row >= 0 ? 16u : 0u);
      cp_async_commit();
      cp_async_wait<0>();
      float s = 1.f;
      if constexpr (!std::is_same<T, __half>::value) {
        float amax = 0.f;
#pragma unroll 2
        for (int n = 0; n < N; ++n) {
          const uint4 v = lds128(place(n));
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = InTraits<T>::to_float2(x[e]);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        amax = fmaxf(amax, shfl_xor(amax, 1));
        s = pow2_row_scale(amax);
#pragma unroll 2
        for (int n = 0; n < N; ++n) {
          const uint4 v = lds128(place(n));
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
          uint32_t hh[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = InTraits<T>::to_float2(x[e]);
            hh[e] = pack_half2(f.x * s, f.y * s);
          }
          sts128(place(n), hh[0], hh[1], hh[2], hh[3]);
        }
      }
      if ((lane & 1) == 0) sts32(sb + R::kRowfac + 4 * ((item & 1) * kTlRows + row), __float_as_uint(p.sm_scale_log2 / s));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (C > 1) mbar_arrive(bar(kTlQHere));
        G::arrive(bar(kTlQReady));
      }
    };

    auto lds_f = [&](int at, int i) { return __uint_as_float(lds32(sb + at + 4 * i)); };
    auto sts_f = [&](int at, int i, float x) { sts32(sb + at + 4 * i, __float_as_uint(x)); };
    {
      TlItem it;
      ok &= take(0, it);
      if (__all_sync(kFull, ok && it.n_tiles > 0)) stage_q(it, 0);
    }
    int j = 0;  // tile of the CTA
#pragma unroll 1
    for (int item = 0;; ++item) {
      // ------------------------------------------------------------ an item
      int lim, last, t0, table;
      {
        TlItem it;
        ok &= take(item, it);
        if (__any_sync(kFull, it.n_tiles == 0)) break;
        // keys below lim are visible; rows that do not exist are all zeros in Q
        lim = rr >= it.pairs ? 0x7fffffff : it.pre ? it.kv : it.lim + (it.pair0 + rr) / p.group;
        last = j + it.n_tiles - 1;
        t0 = it.tile0 * kTlTok;
        table = it.table;
      }
      ok &= mbar_wait(bar(C > 1 ? kTlQHere : kTlQReady), item & 1);  // the other warps' row factors
      if (__any_sync(kFull, !ok || *abort_flag)) break;
      const float fac = lds_f(R::kRowfac, (item & 1) * kTlRows + r);
      float m_own = -CUDART_INF_F, la = 0.f, lb = 0.f;  // the group's reference; the row sum relative to it
      bool fine = true, later = false;  // later: the item has tiles in front of this one
      if ((j & 1) != grp) {
        ++j;
        t0 += kTlTok;
        later = true;
      }
#pragma unroll 1
      for (; j <= last; j += 2, t0 += 2 * kTlTok, later = true) {
        const int entry = __ldg(p.block_table + (size_t)table * p.table_width + t0 / kPage);
        ok &= mbar_wait(bar(kTlSFull + grp), (j >> 1) & 1);
        if (R::kOwnP && j >= 2) ok &= mbar_wait(bar(kTlPvDone + grp), ((j - 2) >> 1) & 1);  // PV(j - 2) has read this P
        if (__any_sync(kFull, !ok || *abort_flag)) {
          fine = false;
          break;
        }
        tc::fence_after();
        const bool here = entry >= 0 && entry < p.num_pages;
        const int room = here ? lim - t0 : 0;  // columns below it count
        const bool masked = !__all_sync(kFull, room >= kTlTok);
        // One pass over the scores: weights relative to the group's reference, which
        // seldom moves, and the largest of them.  Only where one is above 2^kRoom (or
        // the row has no reference yet) is the chunk's maximum taken, the row's chunks
        // so far rescaled and the chunk done again.  (Loops, not unrolled over the
        // columns: with three roles in one kernel the instruction cache is short.)
#pragma unroll 1
        for (int c = 0; c < kTlTok; c += 32) {
          float x[32];
          rw_ld32(ts + c, x);
          if (masked) rw_mask(x, room - c);
          uint32_t pw[16];
          float sa, sb2;
          bool again = false;
          while (true) {
            const float mu = m_own == -CUDART_INF_F ? 0.f : m_own;
            uint32_t top = 0;
            sa = sb2 = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float p0, p1;
              pf_ffma2(p0, p1, x[2 * e], x[2 * e + 1], fac, -mu);
              p0 = exp2_approx(p0);
              p1 = exp2_approx(p1);
              pw[e] = pack_half2(p0, p1);
              tl_add_pair(sa, sb2, pw[e]);
              asm("max.u16x2 %0, %0, %1;\n" : "+r"(top) : "r"(pw[e]));
            }
            // FP16 2^15; infinities and NaN are above it
            const bool over = (top & 0xffffu) > 0x7800u || (top >> 16) > 0x7800u;
            if (again || !__any_sync(kFull, over || m_own == -CUDART_INF_F)) break;
            again = true;
            float mr = -CUDART_INF_F;
#pragma unroll
            for (int e = 0; e < 32; e += 2) mr = pf_fmax3(mr, x[e], x[e + 1]);
            const float mt = mr * fac;
            const float m_new = mt > m_own + batch::kRoom ? ceilf(mt) - batch::kLift : m_own;
            const float a = m_own != -CUDART_INF_F ? exp2_approx(m_own - m_new) : 1.f;
            la *= a;
            lb *= a;
            if (c > 0 && __any_sync(kFull, a != 1.f)) tl_scale_p(tp, c / 32, a);
            m_own = m_new;
          }
          la += sa;
          lb += sb2;
          tc::st_32x32b_x16(tp + c / 2, pw);  // (on top of S: over columns that have been read)
        }
        if (later) {  // the reference after tile j - 1, from the other group's warp
          ok &= mbar_wait(bar(kTlRef + 2 * wq + (grp ^ 1)), ((j - 1) >> 1) & 1);
          if (__any_sync(kFull, !ok)) {
            fine = false;
            break;
          }
          const float m_ref = lds_f(R::kRef, (grp ^ 1) * kTlRows + r);
          const float m_new = fmaxf(m_own, m_ref);
          const float a = m_own != -CUDART_INF_F ? exp2_approx(m_own - m_new) : 1.f;
          const float alpha = m_ref != -CUDART_INF_F ? exp2_approx(m_ref - m_new) : 1.f;
          m_own = m_new;
          if (__any_sync(kFull, a != 1.f)) {
            la *= a;
            lb *= a;
            tl_scale_p(tp, 4, a);
          }
          if (__any_sync(kFull, alpha != 1.f)) {
            ok &= mbar_wait(bar(kTlPvDone + (grp ^ 1)), ((j - 1) >> 1) & 1);
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
        }
        sts_f(R::kRef, grp * kTlRows + r, m_own);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kTlRef + 2 * wq + grp));
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) G::arrive(bar(kTlPReady + grp));
      }
      if (!fine) break;
      j = last + 1;
      // the next item's Q while the last PV runs, once the last QK has read this one
      ok &= mbar_wait(bar(kTlSFull + (last & 1)), (last >> 1) & 1);
      if (__any_sync(kFull, !ok)) break;
      {
        TlItem it;
        ok &= take(item + 1, it);
        if (__any_sync(kFull, !ok)) break;
        if (__all_sync(kFull, it.n_tiles > 0)) stage_q(it, item + 1);
      }
      // the row's reference and sum over both groups
      ok &= mbar_wait(bar(kTlRef + 2 * wq + (last & 1)), (last >> 1) & 1);
      if (__any_sync(kFull, !ok)) break;
      const float m_fin = lds_f(R::kRef, (last & 1) * kTlRows + r);
      const int sums_of = (item & 1) * 2 * kTlRows + r;
      // (without a reference of its own the group's sum is 0, or NaN from NaN scores)
      sts_f(R::kSum, sums_of + grp * kTlRows, m_own != -CUDART_INF_F ? (la + lb) * exp2_approx(m_own - m_fin) : la + lb);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kTlSum + wq));
      ok &= mbar_wait(bar(kTlSum + wq), item & 1);
      // ---------------------------------------------------------- epilogue
      ok &= mbar_wait(bar(kTlPvDone + (last & 1)), (last >> 1) & 1);
      if (__any_sync(kFull, !ok)) break;
      tc::fence_after();
      const float l = lds_f(R::kSum, sums_of) + lds_f(R::kSum, sums_of + kTlRows);
      TlItem it;
      take(item, it);  // (it is there)
      const int head = it.head, rhead = (it.pair0 + rr) % p.group, at_row = it.row0 + (it.pair0 + rr) / p.group;
      const bool pre = it.pre != 0, joins = it.joins != 0;
      const bool starts_here = it.tile0 == 0;
      // (-1: no such pair, or, of a prefix, for a bad entry, which has no output)
      const int row = rr >= it.pairs ? -1 : pre ? tl_shared_row(p, at_row) : at_row;
      const bool whole = starts_here && it.parts == 1;
      const uint32_t stage = sb + R::kStage + warp * 32 * R::kPitch;
      // (kind, row, head) of the row's part
      const size_t part = ((size_t)(pre ? 0 : p.rows) + max(row, 0)) * (p.kv_heads * p.group) + head * p.group + rhead;
      if (starts_here && grp == 0 && row >= 0) {
        // (of a prefix with the row's place in shared_rows, by which batch_join.cu knows this call's parts)
        const uint32_t place = pre ? (uint32_t)at_row : 0u;
        p.where[part] = !whole ? batch::where_word(kWhereRows, cluster, it.parts, rr)
                        : joins ? (uint32_t)kWhereWhole | place << 2
                                : (uint32_t)kWhereDone;
        if (pre && !whole) p.part_ml[2 * part] = __uint_as_float(place);
      }
      if (whole && !joins) {
        T* out = reinterpret_cast<T*>(p.out) + (long long)max(row, 0) * p.out_stride + (head * p.group + rhead) * D;
        tl_store_rows<T, D, true>(stage, to, grp * (D / 2), row >= 0 ? out : nullptr, l > 0.f ? 1.f / l : 0.f);
      } else {
        // a whole part to its row's place, others to a record [pairs][D], then (m, l) a pair
        float* rec = p.row_records + (size_t)(cluster * 2 + (starts_here ? 1 : 0)) * R::kRec;
        float* dst = whole ? p.part_o + part * D : rec + rr * D;
        float2* ml = whole ? reinterpret_cast<float2*>(p.part_ml) + part : reinterpret_cast<float2*>(rec + R::kRows * D) + rr;
        tl_store_rows<T, D, false>(stage, to, grp * (D / 2), row >= 0 ? dst : nullptr, 1.f);
        if (row >= 0 && grp == 0) *ml = make_float2(m_fin, l);
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        G::arrive(bar(kTlEpi));
        taken(item);
      }
    }
    if (__any_sync(kFull, !ok) && lane == 0) {
      flag_error(kErrTimeout);
      *abort_flag = 1;
    }
  }

  griddep_launch_dependents();
  tc::fence_before();
  G::sync();  // (neither CTA leaves before the other's MMAs and arrivals)
  if (warp == kTlQk) {
    tc::fence_after();
    G::dealloc(tbase, R::kTmCols);
  }
}

template <typename T, int D>
cudaError_t launch_tiles(const BatchAttnParams& p, int ctas, cudaStream_t stream) {  // ctas: whole clusters
  auto kernel = batch_tiles_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tiles<D>::kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kTlThreads);
  cfg.dynamicSmemBytes = Tiles<D>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = Tiles<D>::kCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = Tiles<D>::kCtas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace qwz
