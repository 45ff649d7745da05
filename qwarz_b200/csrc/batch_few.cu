// Attention of many requests over one NVFP4 pool, few query rows a request
// (decode, short windows), sm_100a.
//
//   out[r, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(sm_scale q_r.k_j - max),
//   j < kv - n + s + 1 for row s of the n rows of a request with kv tokens.
//
// A token costs D/2 + D/16 bytes of K and as many of V a head, and 4 D
// multiply-adds a query column, far below the tensor rate.  What bounds it is
// the work between: each pair of codes is converted and each pair of halves
// scaled on the way to a fragment, and with those instructions taken out the
// loads alone run at 92 % of the measured copy bandwidth.  They do not fill a
// unit, though (ALU 51 %, issue slots 54 %, DRAM 57 %): eight warps an SM, at 236
// registers, wait on their own chains.
//
// The (row, head of the group) pairs of one request and KV head are the columns
// of an item, eight at most (9 to 16 heads of a group make two items that run
// side by side, the second reading the tokens from L2).  A CTA has one KV head and
// a share of all requests' units of 128 or 256 tokens (batch_common.cuh); the CTAs
// of the other heads work on the same tokens at the same time, so that the slices
// of a token's row leave HBM together.  A warp owns 32 or 64 tokens of a unit and
// streams them through a ring of its own: the codes by TMA (one box of its rows
// of K and one of V, on the warp's own mbarrier), the scales, whose rows can be
// narrower than a TMA box, by cp.async.  No warp waits for another inside an
// item, and the ring runs on across items, so a CTA's loads never drain.  Tokens
// are on the M side of mma.sync.m16n8k16 and columns on N, where eight columns
// fill the tile (tcgen05 would take the operands from shared memory, four bytes of
// FP16 written and read there for each byte of codes): K codes become A
// fragments of S^T in registers, V codes A fragments of O^T, P^T comes from the
// S^T fragment by movmatrix.  Base-2 online softmax with a reference that seldom
// moves; P is rounded to FP16 for its product (11 significant bits, as the output
// has), all sums are FP32.  At an item's end the warps' (m, l, O) are merged in
// shared memory in warp order.
//
// Measured: 524,288 tokens in one request, 24/4/256, 122 us (4.9 TB/s, 76 % of
// the measured copy bandwidth); 64 requests of 256 to 32,768 tokens, 24/4/256,
// 112 us (72 %); 256 of 32/8/128, 100 us (47 %: short items, whose ends cost
// two units each); one of 4,000 tokens 14 us, the latency of two launches.
#include "attn_common.cuh"
#include "batch_common.cuh"

namespace qwz {

using namespace detail;

namespace {

constexpr int kFewCols = kBatchFewCols;  // query columns of an item
constexpr int kFewScan = 128;  // threads that scan the requests

template <int D>
struct Few {
  // measured at 524,288 tokens of 24/4/256 and 262,144 of 32/8/128 (us):
  //   D 256: 4 warps x 32 tokens, 3 stages, 2 CTAs 125; 8 x 32, 3, 1 CTA 126
  //     (short items: 187 against 248 at 1,024 x 512 tokens); 4 x 32, 2, 3 CTAs 148
  //   D 128: 4 x 64, 2, 3 CTAs 78; 4 x 32, 3, 4 CTAs 81; 8 x 32, 3, 2 CTAs 80
  //   D 64:  4 x 64, 2, 4 CTAs 37; 4 x 64, 3, 4 CTAs 39; 4 x 32, 3, 5 CTAs 45
  static constexpr int kWarps = 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTok = D == 256 ? 32 : 64;    // tokens of a unit a warp owns
  static constexpr int kUnit = kWarps * kTok;        // tokens of a unit of work (divides a page)
  static constexpr int kStages = D == 256 ? 3 : 2;
  static constexpr int kCtas = D == 256 ? 2 : D == 128 ? 3 : 4;  // per SM
  static constexpr int kMT = D / 16;                 // MMA row tiles of O^T
  static constexpr int kRow = D / 2;                 // code bytes of a row
  static constexpr int kSRow = D / 16;               // scale bytes of a row
  static constexpr int kCodes = kTok * kRow;
  static constexpr int kScales = kTok * kSRow;
  // per CTA: code slots [warp][stage] {K, V}, scale slots, barriers
  static constexpr int kRing = kWarps * kStages * 2 * kCodes;
  static constexpr int kScaleRing = kWarps * kStages * 2 * kScales;
  static constexpr int kSmem = kRing + kScaleRing + 8 * kWarps * kStages + 1024;
  // for the merge a warp's O takes the code slot its last unit left, (m, l) the scale slot
  static_assert(kMT * 512 <= 2 * kCodes && kFewCols * 8 <= 2 * kScales, "merge area");
  static_assert(kMT % kWarps == 0 && kTok % 32 == 0, "merge share, tile pairs");
};

// Byte offset of 16-byte chunk c of code row r as the TMA box lays it out: rows
// of 128, 64 or 32 bytes with the swizzle of that width.
template <int D>
QWZ_DEVINL uint32_t few_swz(int r, int c) {
  const uint32_t at = (uint32_t)(r * Few<D>::kRow + c * 16);
  return at ^ ((at >> 3) & (D == 256 ? 0x70u : D == 128 ? 0x30u : 0x10u));
}

QWZ_DEVINL uint2 few_lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// N words (1, 2 or 4) from shared memory.
template <int N>
QWZ_DEVINL void lds_words(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = lds32(addr);
  } else if constexpr (N == 2) {
    const uint2 v = few_lds64(addr);
    w[0] = v.x; w[1] = v.y;
  } else {
    const uint4 v = lds128(addr);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
}

template <int BYTES>
QWZ_DEVINL void cp_async_small(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(BYTES));
}

// Walks the units (request, U tokens) of one KV head in order.  A request
// weighs its units and kOver more for what its item costs beside them (its Q,
// the merge and the store), so that CTAs with many short items get fewer.
template <int U>
struct FewWalk {
  static constexpr int kOver = 256 / U;
  int b, unit;             // request (p.requests: past the end), unit
  int units;               // of request b
  long long base;          // weighed units before the request
  batch::Req r;

  // whether request r has columns of the group that begins at c0 (those with more
  // than few_cols are batch_rows.cu's)
  static QWZ_DEVINL bool few(const BatchAttnParams& p, const batch::Req& r, int c0) {
    const int cols = r.n * p.group;
    return cols > c0 && cols <= p.few_cols;
  }
  // a request without tokens still has rows to write
  static QWZ_DEVINL int units_of(const batch::Req& r) { return max(1, (r.kv + U - 1) / U); }
  static QWZ_DEVINL long long cost(const BatchAttnParams& p, int b, int c0) {
    const batch::Req r = batch::load_req(p, b);
    return few(p, r, c0) ? units_of(r) + kOver : 0;
  }
  QWZ_DEVINL void enter(const BatchAttnParams& p, int bb) {
    b = bb;
    r = batch::load_req(p, b);
    units = units_of(r);
  }
  // Weighed unit u, `before` of which precede request b0.
  QWZ_DEVINL void seek(const BatchAttnParams& p, int c0, int b0, long long before, long long u) {
    base = before;
    u -= before;
    for (b = b0; b < p.requests; ++b) {
      const long long c = cost(p, b, c0);
      if (u < c) break;
      u -= c;
      base += c;
    }
    unit = 0;
    if (b == p.requests) return;
    enter(p, b);
    unit = max((int)u - kOver, 0);
  }
  // To the next request that has work here.
  QWZ_DEVINL void next_request(const BatchAttnParams& p, int c0) {
    unit = 0;
    base += units + kOver;
    for (int bb = b + 1; bb < p.requests; ++bb) {
      enter(p, bb);
      if (few(p, r, c0)) return;
    }
    b = p.requests;
  }
  QWZ_DEVINL bool at(const FewWalk& o) const { return b == o.b && unit == o.unit; }
  // Units from here on, of this request, before the walk's end.
  QWZ_DEVINL int left(int end_b, int end_unit) const { return (b == end_b ? end_unit : units) - unit; }
  // Table entry of the unit's page, unchecked (the load is in flight until it is used).
  QWZ_DEVINL int entry(const BatchAttnParams& p) const {
    return __ldg(p.block_table + (size_t)b * p.table_width + unit / (kPage / U));
  }
  // Whether the unit has tokens and lies in the pool.
  QWZ_DEVINL bool present(const BatchAttnParams& p, int pp) const {
    if (r.kv <= 0) return false;
    if (pp >= 0 && pp < p.num_pages) return true;
    flag_error(kErrPageRange);  // a bad entry: its tokens count as absent
    return false;
  }
};

template <int D>
struct FewV {  // V codes of tokens ra, ra+1, ra+8, ra+9: head dims [D/8 g, D/8 (g+1))
  static constexpr int W = D / 64;
  uint32_t a[W], b[W], c[W], d[W];
  uint32_t sab[2], scd[2];
};

// Scales of rows at or past `end` are zeroed, so stale bytes add nothing.
template <int D>
QWZ_DEVINL void few_v_load(uint32_t codes, uint32_t scales, int ra, int g, bool tail, int end, FewV<D>& v) {
  constexpr int SB = Few<D>::kRow / 8;  // slice bytes of a lane: 16, 8, 4
  const int c = g * SB / 16, in = g * SB % 16;
  lds_words(codes + few_swz<D>(ra, c) + in, v.a);
  lds_words(codes + few_swz<D>(ra + 1, c) + in, v.b);
  lds_words(codes + few_swz<D>(ra + 8, c) + in, v.c);
  lds_words(codes + few_swz<D>(ra + 9, c) + in, v.d);
  uint32_t s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = ra + (i & 1) + (i >> 1) * 8;
    if constexpr (D == 256) s[i] = lds16(scales + row * 16 + 2 * g);
    else if constexpr (D == 128) s[i] = lds8(scales + row * 8 + g);
    else s[i] = lds8(scales + row * 4 + (g >> 1));
    if (tail && row >= end) s[i] = 0;
  }
  e4m3x4_to_f16x2x2(__byte_perm(s[0], s[1], 0x5140), v.sab[0], v.sab[1]);
  e4m3x4_to_f16x2x2(__byte_perm(s[2], s[3], 0x5140), v.scd[0], v.scd[1]);
}

// O^T += V^T P^T of one 16-token tile.
template <int D>
QWZ_DEVINL void few_pv(const FewV<D>& v, const PFrag& pf, float (&o)[D / 16][4]) {
#pragma unroll
  for (int w = 0; w < FewV<D>::W; ++w) {
    const uint32_t xab = (v.a[w] & 0x0F0F0F0Fu) | ((v.b[w] << 4) & 0xF0F0F0F0u);
    const uint32_t yab = ((v.a[w] >> 4) & 0x0F0F0F0Fu) | (v.b[w] & 0xF0F0F0F0u);
    const uint32_t xcd = (v.c[w] & 0x0F0F0F0Fu) | ((v.d[w] << 4) & 0xF0F0F0F0u);
    const uint32_t ycd = ((v.c[w] >> 4) & 0x0F0F0F0Fu) | (v.d[w] & 0xF0F0F0F0u);
    uint32_t hxab[4], hyab[4], hxcd[4], hycd[4];
    e2m1x8_to_f16x2x4(xab, hxab);
    e2m1x8_to_f16x2x4(yab, hyab);
    e2m1x8_to_f16x2x4(xcd, hxcd);
    e2m1x8_to_f16x2x4(ycd, hycd);
    const uint32_t sab = v.sab[D == 256 ? w >> 1 : 0], scd = v.scd[D == 256 ? w >> 1 : 0];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      mma_16816(o[4 * w + kk], hmul2_u32(hxab[kk], sab), hmul2_u32(hyab[kk], sab), hmul2_u32(hxcd[kk], scd),
                hmul2_u32(hycd[kk], scd), pf.hi0, pf.hi1);
  }
}

// Raw S^T of the 16-token tile at row r0 - g of the slot.
template <int D>
QWZ_DEVINL void few_qk(uint32_t codes, uint32_t scales, int r0, int qd, const uint32_t (&qf)[D / 8], float (&s)[4]) {
  constexpr int KW = D / 32;  // code words of a lane: 8, 4, 2
  const int r1 = r0 + 8;
  uint32_t kw0[KW], kw1[KW], sc0[4], sc1[4];
  if constexpr (D == 256) {
    uint32_t a[4], b[4], c[4], d[4];
    lds_words(codes + few_swz<D>(r0, 2 * qd), a);
    lds_words(codes + few_swz<D>(r0, 2 * qd + 1), b);
    lds_words(codes + few_swz<D>(r1, 2 * qd), c);
    lds_words(codes + few_swz<D>(r1, 2 * qd + 1), d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kw0[i] = a[i];
      kw0[4 + i] = b[i];
      kw1[i] = c[i];
      kw1[4 + i] = d[i];
    }
    scales_bcast4(lds32(scales + r0 * 16 + 4 * qd), sc0);
    scales_bcast4(lds32(scales + r1 * 16 + 4 * qd), sc1);
  } else if constexpr (D == 128) {
    lds_words(codes + few_swz<D>(r0, qd), kw0);
    lds_words(codes + few_swz<D>(r1, qd), kw1);
    scales_bcast4(lds16(scales + r0 * 8 + 2 * qd), sc0);
    scales_bcast4(lds16(scales + r1 * 8 + 2 * qd), sc1);
  } else {
    lds_words(codes + few_swz<D>(r0, qd >> 1) + (qd & 1) * 8, kw0);
    lds_words(codes + few_swz<D>(r1, qd >> 1) + (qd & 1) * 8, kw1);
    scales_bcast4(lds8(scales + r0 * 4 + qd), sc0);
    scales_bcast4(lds8(scales + r1 * 4 + qd), sc1);
  }
  float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w8 = 0; w8 < KW; ++w8) {
    uint32_t h0[4], h1[4];
    e2m1x8_to_f16x2x4(kw0[w8], h0);
    e2m1x8_to_f16x2x4(kw1[w8], h1);
    const uint32_t s0 = sc0[w8 >> 1], s1 = sc1[w8 >> 1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h0[j] = hmul2_u32(h0[j], s0);
      h1[j] = hmul2_u32(h1[j], s1);
    }
    mma_16816(sa, h0[0], h1[0], h0[1], h1[1], qf[4 * w8 + 0], qf[4 * w8 + 1]);
    mma_16816(sb, h0[2], h1[2], h0[3], h1[3], qf[4 * w8 + 2], qf[4 * w8 + 3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = sa[i] + sb[i];
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(Few<D>::kThreads, Few<D>::kCtas)
    batch_few_kernel(const __grid_constant__ BatchAttnParams p, const __grid_constant__ BatchPoolMaps maps) {
  using F = Few<D>;
  using Walk = FewWalk<F::kUnit>;
  constexpr int MT = F::kMT, QW = D / 8, TILES = F::kTok / 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sraw = smem_u32(smem);
  const uint32_t sbase = (sraw + 1023u) & ~1023u;
  uint8_t* sgen = smem + (sbase - sraw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, qd = lane & 3;
  const uint32_t codes = sbase + warp * F::kStages * 2 * F::kCodes;
  const uint32_t scales = sbase + F::kRing + warp * F::kStages * 2 * F::kScales;
  const uint32_t bars = sbase + F::kRing + F::kScaleRing + warp * F::kStages * 8;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < F::kStages; ++s) mbar_init(bars + 8 * s, 1);
    mbar_fence_init();
    if (warp == 0) {
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
    }
  }
  griddep_wait();

  // x: KV head and group of columns, y: share
  const int hd = blockIdx.x / p.col_groups, c0 = blockIdx.x % p.col_groups * kFewCols;
  const int split = blockIdx.y, cta = split * gridDim.x + blockIdx.x;
  const long long splits = gridDim.y;
  // ---------------------------------------------------- this CTA's share
  // (the ring's memory holds the scan until the first copy)
  long long* starts = reinterpret_cast<long long*>(sgen);  // weighed units before each scanning thread's requests
  long long* warp_sums = starts + kFewScan;
  const int per = (p.requests + kFewScan - 1) / kFewScan;
  long long mine = 0;
  if (tid < kFewScan)
    for (int b = tid * per; b < min(p.requests, (tid + 1) * per); ++b) mine += Walk::cost(p, b, c0);
  long long total;
  const long long before = batch::block_scan(mine, warp_sums, total);
  if (tid < kFewScan) starts[tid] = before;
  __syncthreads();
  auto seek = [&](long long u) {
    int at = 0;
    for (int step = kFewScan / 2; step > 0; step >>= 1)
      if (starts[at + step] <= u) at += step;
    Walk w;
    w.seek(p, c0, min(at * per, p.requests), starts[at], u);
    return w;
  };
  Walk cur = seek(split * total / splits);
  int end_b, end_unit;
  bool none;
  {
    const Walk end = seek((split + 1) * total / splits);
    end_b = end.b;
    end_unit = end.unit;
    none = cur.at(end);
  }
  __syncthreads();
  int32_t* meta = p.meta + cta * kBatchMeta;
  if (tid == 0) meta[0] = 0;
  if (none) {
    griddep_launch_dependents();
    return;
  }

  // The loads run kStages - 1 units ahead of the math, with their own place.
  int pre_b = cur.b, pre_unit = cur.unit, pre_left = cur.left(end_b, end_unit), pre_kv = cur.r.kv;
  const int32_t* pre_row = p.block_table + (size_t)pre_b * p.table_width;
  constexpr int kPerPage = kPage / F::kUnit;
  int pre_page = __ldg(pre_row + pre_unit / kPerPage);
  unsigned filled = 0;  // bit s: ring slot s holds (or will hold) tokens of the pool
  // False once a wait gave up: nothing more is copied, what is on its way is still
  // waited for, and the result is marked by the error.
  bool ok = true;
  unsigned late = 0, phases = 0;  // bits of slots: whose wait gave up; their barriers' parity
  const int step = p.kv_heads * F::kSRow;  // scale bytes of a token row
  const uint8_t* ks_lane = p.k_scales + hd * F::kSRow + (size_t)lane * step;
  const uint8_t* vs_lane = p.v_scales + hd * F::kSRow + (size_t)lane * step;

  // Copies this warp's tokens of the next unit into ring slot `slot`.
  auto advance = [&](int slot) {
    if (pre_left > 0) {
      bool in_pool = pre_page >= 0 && pre_page < p.num_pages;
      if (!in_pool && pre_kv > 0) flag_error(kErrPageRange);  // a bad entry: its tokens count as absent
      in_pool = in_pool && pre_kv > 0 && ok;
      filled = in_pool ? filled | (1u << slot) : filled & ~(1u << slot);
      const int t0 = pre_unit * F::kUnit + warp * F::kTok;
      if (in_pool && t0 < pre_kv) {
        const int row0 = pre_page * kPage + (t0 & (kPage - 1));
        if (lane == 0) {
          const uint32_t bar = bars + 8 * slot, dst = codes + slot * 2 * F::kCodes;
          fence_proxy_async_smem();  // the slot's last reads and merge writes before the copies
          mbar_arrive_expect_tx(bar, 2 * F::kCodes);
          tma_load_2d(dst, &maps.k, hd * F::kRow, row0, bar);
          tma_load_2d(dst + F::kCodes, &maps.v, hd * F::kRow, row0, bar);
        }
        const uint8_t* kp = ks_lane + (size_t)(unsigned)row0 * (unsigned)step;
        const uint8_t* vp = vs_lane + (size_t)(unsigned)row0 * (unsigned)step;
        const uint32_t dst = scales + slot * 2 * F::kScales + lane * F::kSRow;
#pragma unroll
        for (int r = 0; r < F::kTok; r += 32) {
          cp_async_small<F::kSRow>(dst + r * F::kSRow, kp + r * step);
          cp_async_small<F::kSRow>(dst + F::kScales + r * F::kSRow, vp + r * step);
        }
      }
      ++pre_unit;
      if (--pre_left == 0 && pre_b != end_b) {  // on to the next request
        batch::Req r = {0, 0, 0};
        while (++pre_b < p.requests) {
          r = batch::load_req(p, pre_b);
          if (Walk::few(p, r, c0)) break;
        }
        if (pre_b < p.requests) {
          pre_unit = 0;
          pre_left = pre_b == end_b ? end_unit : Walk::units_of(r);
          pre_kv = r.kv;
          pre_row = p.block_table + (size_t)pre_b * p.table_width;
          if (pre_left > 0 && warp == 0) {  // the item's Q on its way into L1
            constexpr int kLines = D * 2 / 128;
            const int c = c0 + lane / kLines;
            if (c < r.n * p.group && c < c0 + kFewCols)
              asm volatile("prefetch.global.L1 [%0];\n" ::"l"(reinterpret_cast<const T*>(p.q) +
                                                             (r.row0 + c / p.group) * p.q_stride +
                                                             (hd * p.group + c % p.group) * D + (lane % kLines) * 64));
          }
        }
      }
      if (pre_left > 0) pre_page = __ldg(pre_row + pre_unit / kPerPage);
    }
    cp_async_commit();  // one group a unit, empty past the share's end
  };
#pragma unroll
  for (int s = 0; s < F::kStages - 1; ++s) advance(s);

  float o[MT][4];
  uint32_t qf[QW];
  int slot = 0, fill = F::kStages - 1;

  while (true) {  // ------------------------------------------------ an item
    const int first_unit = cur.unit, cols = min(kFewCols, cur.r.n * p.group - c0);
    float cf0, cf1;
    {
      float amax = 0.f;
      if (g < cols) {
        const uint4* src = reinterpret_cast<const uint4*>(
            reinterpret_cast<const T*>(p.q) + (cur.r.row0 + (c0 + g) / p.group) * p.q_stride +
            (hd * p.group + (c0 + g) % p.group) * D + qd * (D / 4));
#pragma unroll
        for (int i = 0; i < QW / 4; ++i) {
          const uint4 v = __ldg(src + i);
          qf[4 * i + 0] = v.x;
          qf[4 * i + 1] = v.y;
          qf[4 * i + 2] = v.z;
          qf[4 * i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < QW; ++i) qf[i] = 0u;
      }
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        const float2 f = InTraits<T>::to_float2(qf[i]);
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      amax = fmaxf(amax, shfl_xor(amax, 1));
      amax = fmaxf(amax, shfl_xor(amax, 2));
      const float sc = pow2_row_scale(amax);
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        const float2 f = InTraits<T>::to_float2(qf[i]);
        qf[i] = pack_half2(f.x * sc, f.y * sc);
      }
      const float rowfac = p.sm_scale_log2 / sc;
      cf0 = __shfl_sync(kFull, rowfac, 8 * qd);
      cf1 = __shfl_sync(kFull, rowfac, 8 * qd + 4);
    }
    const int lim_base = cur.r.kv - cur.r.n + 1, min_lim = lim_base + c0 / p.group;
    const int lim0 = 2 * qd < cols ? lim_base + (c0 + 2 * qd) / p.group : 0;
    const int lim1 = 2 * qd + 1 < cols ? lim_base + (c0 + 2 * qd + 1) / p.group : 0;
    // reference maxima in base-2 units, and the raw scores that move them
    float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, top0 = -CUDART_INF_F, top1 = -CUDART_INF_F;
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    int tw = cur.unit * F::kUnit + warp * F::kTok;
    for (int n = cur.left(end_b, end_unit); n > 0; --n, tw += F::kUnit) {
      cp_async_wait<F::kStages - 2>();
      const bool here = ((filled >> slot) & 1u) != 0u && tw < cur.r.kv;
      if (here) {  // this warp's copy was issued
        if (!__all_sync(kFull, mbar_wait(bars + 8 * slot, (phases >> slot) & 1u))) {
          flag_error(kErrTimeout);
          ok = false;
          late |= 1u << slot;
        }
        phases ^= 1u << slot;
      }
      __syncwarp();
      const uint32_t kc = codes + slot * 2 * F::kCodes, vc = kc + F::kCodes;
      const uint32_t ks = scales + slot * 2 * F::kScales, vs = ks + F::kScales;
      advance(fill);
      fill = fill + 1 == F::kStages ? 0 : fill + 1;
      slot = slot + 1 == F::kStages ? 0 : slot + 1;
      if (!here) continue;

      const bool tail = tw + F::kTok > min_lim;
      const int end_row = cur.r.kv - tw;
      float t[TILES][4];
#pragma unroll
      for (int i = 0; i < TILES; ++i) few_qk<D>(kc, ks, 16 * i + g, qd, qf, t[i]);
      if (tail) {
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const int at = tw + 16 * i + g;
          if (at >= lim0) t[i][0] = -CUDART_INF_F;
          if (at >= lim1) t[i][1] = -CUDART_INF_F;
          if (at + 8 >= lim0) t[i][2] = -CUDART_INF_F;
          if (at + 8 >= lim1) t[i][3] = -CUDART_INF_F;
        }
      }
      // V codes first: their shared-memory latency hides behind the softmax
      FewV<D> va, vb;
      few_v_load<D>(vc, vs, 2 * qd, g, tail, end_row, va);
      few_v_load<D>(vc, vs, 2 * qd + 16, g, tail, end_row, vb);

      // The references move only when some score exceeds one by 2^15: one
      // vote a unit, and the reduction over the lanes only then.
      float mx0 = fmaxf(t[0][0], t[0][2]), mx1 = fmaxf(t[0][1], t[0][3]);
#pragma unroll
      for (int i = 1; i < TILES; ++i) {
        mx0 = fmaxf(mx0, fmaxf(t[i][0], t[i][2]));
        mx1 = fmaxf(mx1, fmaxf(t[i][1], t[i][3]));
      }
      if (__any_sync(kFull, mx0 > top0 || mx1 > top1)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, shfl_xor(mx0, off));
          mx1 = fmaxf(mx1, shfl_xor(mx1, off));
        }
        const float n0 = fmaxf(m0, mx0 * cf0 - batch::kLift), n1 = fmaxf(m1, mx1 * cf1 - batch::kLift);
        const float a0 = (n0 == -CUDART_INF_F) ? 1.f : exp2_approx(m0 - n0);
        const float a1 = (n1 == -CUDART_INF_F) ? 1.f : exp2_approx(m1 - n1);
        m0 = n0;
        m1 = n1;
        top0 = (m0 + batch::kRoom) / cf0;
        top1 = (m1 + batch::kRoom) / cf1;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          o[j][0] *= a0;
          o[j][1] *= a1;
          o[j][2] *= a0;
          o[j][3] *= a1;
        }
      }
      const float mu0 = (m0 == -CUDART_INF_F) ? 0.f : m0;
      const float mu1 = (m1 == -CUDART_INF_F) ? 0.f : m1;
      PFrag pf[TILES];
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        t[i][0] = exp2_approx(fmaf(t[i][0], cf0, -mu0));
        t[i][1] = exp2_approx(fmaf(t[i][1], cf1, -mu1));
        t[i][2] = exp2_approx(fmaf(t[i][2], cf0, -mu0));
        t[i][3] = exp2_approx(fmaf(t[i][3], cf1, -mu1));
        // P rounded to FP16 once; the sums take the rounded weights, so a row's
        // weights add up to one and a rounding of a dominant weight cancels
        const uint32_t a = pack_half2(t[i][0], t[i][1]), b = pack_half2(t[i][2], t[i][3]);
        const float2 fa = InTraits<__half>::to_float2(a), fb = InTraits<__half>::to_float2(b);
        l0 += fa.x + fb.x;
        l1 += fa.y + fb.y;
        pf[i].hi0 = movmatrix_trans(a);
        pf[i].hi1 = movmatrix_trans(b);
      }
#pragma unroll
      for (int i = 0; i < TILES; i += 2) {
        few_pv<D>(va, pf[i], o);
        if (i + 2 < TILES) few_v_load<D>(vc, vs, 2 * qd + 16 * (i + 2), g, tail, end_row, va);
        few_pv<D>(vb, pf[i + 1], o);
        if (i + 3 < TILES) few_v_load<D>(vc, vs, 2 * qd + 16 * (i + 3), g, tail, end_row, vb);
      }
    }

    {  // ---------------------------------------------------- the item's end
      constexpr int kPitch = F::kStages * 2 * F::kCodes;
      const int used = fill;  // the slot that the last unit left (the next copy's)
      uint8_t* area = sgen + used * 2 * F::kCodes;  // of warp 0
      auto ml_of = [&](int w) {
        return reinterpret_cast<float2*>(sgen + F::kRing + (w * F::kStages + used) * 2 * F::kScales);
      };
      float4* red = reinterpret_cast<float4*>(area + warp * kPitch);
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += shfl_xor(l0, off);
        l1 += shfl_xor(l1, off);
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < MT; ++j) red[j * 32 + lane] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
      if (g == 0) {
        ml_of(warp)[2 * qd] = make_float2(m0, l0);
        ml_of(warp)[2 * qd + 1] = make_float2(m1, l1);
      }
      const bool starts_here = first_unit == 0, ends_here = cur.b != end_b;
      const bool whole = starts_here && ends_here;
      float* rec = p.records + (size_t)(cta * 2 + (starts_here ? 1 : 0)) * (kFewCols * (D + 2));
      __syncthreads();
      // the lane's two columns: weights of the warps
      float w0[F::kWarps], w1[F::kWarps], M0 = -CUDART_INF_F, M1 = -CUDART_INF_F, L0 = 0.f, L1 = 0.f;
#pragma unroll
      for (int w = 0; w < F::kWarps; ++w) {
        w0[w] = ml_of(w)[2 * qd].x;
        w1[w] = ml_of(w)[2 * qd + 1].x;
        M0 = fmaxf(M0, w0[w]);
        M1 = fmaxf(M1, w1[w]);
      }
#pragma unroll
      for (int w = 0; w < F::kWarps; ++w) {
        w0[w] = w0[w] == -CUDART_INF_F ? 0.f : exp2_approx(w0[w] - M0);
        w1[w] = w1[w] == -CUDART_INF_F ? 0.f : exp2_approx(w1[w] - M1);
        L0 += w0[w] * ml_of(w)[2 * qd].y;
        L1 += w1[w] * ml_of(w)[2 * qd + 1].y;
      }
      const float i0 = L0 > 0.f ? 1.f / L0 : 0.f, i1 = L1 > 0.f ? 1.f / L1 : 0.f;
      if (!whole && warp == 0 && g == 0) {
        float2* ml = reinterpret_cast<float2*>(rec + kFewCols * D);
        ml[2 * qd] = make_float2(M0, L0);
        ml[2 * qd + 1] = make_float2(M1, L1);
      }
#pragma unroll
      for (int jj = 0; jj < MT / F::kWarps; ++jj) {
        const int j = jj * F::kWarps + warp;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < F::kWarps; ++w) {
          const float4 v = reinterpret_cast<const float4*>(area + w * kPitch)[j * 32 + lane];
          a.x += w0[w] * v.x;
          a.y += w1[w] * v.y;
          a.z += w0[w] * v.z;
          a.w += w1[w] * v.w;
        }
        // (x, z): d = D/8 g + 2j and d + 1 of column 2qd; (y, w): of column 2qd + 1
        const int d = D / 8 * g + 2 * j;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 2 * qd + e;
          if (c >= cols) continue;
          const float x = e ? a.y : a.x, y = e ? a.w : a.z, inv = e ? i1 : i0;
          if (whole) {
            T* dst = reinterpret_cast<T*>(p.out) + (cur.r.row0 + (c0 + c) / p.group) * p.out_stride +
                     (hd * p.group + (c0 + c) % p.group) * D + d;
            const T h[2] = {InTraits<T>::from_float(x * inv), InTraits<T>::from_float(y * inv)};
            *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(h);
          } else {
            *reinterpret_cast<float2*>(rec + c * D + d) = make_float2(x, y);
          }
        }
      }
      if (starts_here && !ends_here && tid == 0) {  // the rest of the item is the next CTAs'
        const long long last_unit = cur.base + Walk::kOver + cur.units - 1;
        meta[0] = cols;
        meta[1] = cur.r.row0;
        meta[4] = (int)(((last_unit + 1) * splits - 1) / total);
        meta[5] = (int)min(total, splits);  // fewer units than splits leave some without a record
      }
      __syncthreads();
    }
    if (cur.b == end_b) break;
    cur.next_request(p, c0);
    if (cur.b == p.requests || (cur.b == end_b && end_unit == 0)) break;
  }
  if (!ok) {  // never leave with copies in flight
    cp_async_wait<0>();
    for (int s = 0; s < F::kStages; ++s)
      if ((late >> s) & 1u) mbar_wait(bars + 8 * s, ((phases >> s) & 1u) ^ 1u);
  }
  griddep_launch_dependents();
}

// Merges the records of the items that more than one CTA worked on, in the
// order of the splits: block (head, split, y) takes columns y, y + gridDim.z,
// ... of the item that this split began and did not finish.
template <typename T, int D>
__global__ void __launch_bounds__(256) batch_combine_kernel(const __grid_constant__ BatchAttnParams p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float w[kBatchMaxCtas], sums[kBatchMaxCtas];
  __shared__ float red[8];
  __shared__ float4 acc_s[kGroups][kLanes];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, hd = blockIdx.x, heads = gridDim.x, i0 = blockIdx.y;
  const long long splits = gridDim.y;
  const int32_t* meta = p.meta + (i0 * heads + hd) * kBatchMeta;
  const int cols = __ldcg(meta);
  if (cols == 0) return;
  const int row0 = __ldcg(meta + 1), parts = __ldcg(meta + 4) - i0 + 1, busy = __ldcg(meta + 5);
  constexpr size_t kRec = (size_t)kFewCols * (D + 2);
  // split i0 left its part in record 1, the later ones in record 0
  auto record = [&](int j) { return p.records + (size_t)(((i0 + j) * heads + hd) * 2 + (j == 0 ? 1 : 0)) * kRec; };
  auto empty = [&](int j) {
    const long long i = i0 + j;
    return i * busy / splits == (i + 1) * busy / splits;
  };
  for (int c = blockIdx.z; c < cols; c += gridDim.z) {
    auto stat = [&](int j) { return __ldcg(reinterpret_cast<const float2*>(record(j) + kFewCols * D + 2 * c)); };
    float M = -CUDART_INF_F;
    for (int j = tid; j < parts; j += 256) {
      const float2 v = stat(j);
      const bool skip = empty(j);  // its record is another call's
      w[j] = skip ? -CUDART_INF_F : v.x;
      sums[j] = skip ? 0.f : v.y;
      M = fmaxf(M, w[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if ((tid & 31) == 0) red[tid >> 5] = M;
    __syncthreads();
    M = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) M = fmaxf(M, red[i]);
    __syncthreads();
    float L = 0.f;
    for (int j = tid; j < parts; j += 256) {
      const float wt = batch::part_weight(w[j], sums[j], M);
      L += wt * sums[j];
      w[j] = wt;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if ((tid & 31) == 0) red[tid >> 5] = L;
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) L += red[i];
    const int grp = tid / kLanes, ln = tid % kLanes;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int j = grp; j < parts; j += kGroups) {
      const float wj = w[j];
      const float4 v = __ldcg(reinterpret_cast<const float4*>(record(j) + c * D) + ln);
      a.x += wj == 0.f ? 0.f : wj * v.x;  // (v can be anything where wj is 0)
      a.y += wj == 0.f ? 0.f : wj * v.y;
      a.z += wj == 0.f ? 0.f : wj * v.z;
      a.w += wj == 0.f ? 0.f : wj * v.w;
    }
    acc_s[grp][ln] = a;
    __syncthreads();
    if (tid < kLanes) {
      a = acc_s[0][tid];
#pragma unroll
      for (int i = 1; i < kGroups; ++i) {
        const float4 v = acc_s[i][tid];
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
      }
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const int cc = hd % p.col_groups * kFewCols + c;  // column of the KV head
      const int s = cc / p.group, h = hd / p.col_groups * p.group + cc % p.group;
      T* dst = reinterpret_cast<T*>(p.out) + (row0 + s) * p.out_stride + h * D + tid * 4;
      dst[0] = InTraits<T>::from_float(a.x * inv);
      dst[1] = InTraits<T>::from_float(a.y * inv);
      dst[2] = InTraits<T>::from_float(a.z * inv);
      dst[3] = InTraits<T>::from_float(a.w * inv);
    }
    __syncthreads();
  }
}

// The same with a warp a column and a block an item: for many requests, whose
// items have a few parts each.
constexpr int kCombineThreads = kFewCols * 32;

template <typename T, int D>
__global__ void __launch_bounds__(kCombineThreads)
    batch_combine_short_kernel(const __grid_constant__ BatchAttnParams p, int splits) {
  constexpr int kVecs = (D + 127) / 128;  // float4s of a lane (D 64: half the lanes)
  extern __shared__ float weights[];      // [warps][splits]
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = warp;
  const int hd = blockIdx.x, heads = gridDim.x;
  const int i0 = blockIdx.y;
  const int32_t* meta = p.meta + (i0 * heads + hd) * kBatchMeta;
  const int cols = __ldcg(meta);
  if (cols == 0) return;
  const int row0 = __ldcg(meta + 1), parts = __ldcg(meta + 4) - i0 + 1, busy = __ldcg(meta + 5);
  constexpr size_t kRec = (size_t)kFewCols * (D + 2);
  // split i0 left its part in record 1, the later ones in record 0
  auto record = [&](int j) { return p.records + (size_t)(((i0 + j) * heads + hd) * 2 + (j == 0 ? 1 : 0)) * kRec; };
  float* w = weights + warp * splits;
  float4 a[kVecs];
#pragma unroll
  for (int v = 0; v < kVecs; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
  const bool mine = lane * 4 < D;
  if (c < cols) {
    auto stat = [&](int j) {
      const long long i = i0 + j;
      if (i * busy / splits == (i + 1) * busy / splits) return make_float2(-CUDART_INF_F, 0.f);  // a split without units
      return __ldcg(reinterpret_cast<const float2*>(record(j) + kFewCols * D + 2 * c));
    };
    float M = -CUDART_INF_F;
    for (int j = lane; j < parts; j += 32) M = fmaxf(M, stat(j).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    for (int j = lane; j < parts; j += 32) {
      const float2 v = stat(j);
      const float wt = batch::part_weight(v.x, v.y, M);
      L += wt * v.y;
      w[j] = wt;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    __syncwarp();
    if (mine) {
#pragma unroll 4
      for (int j = 0; j < parts; ++j) {
        const float wj = w[j];
        if (wj == 0.f) continue;  // (a split without units has no record)
        const float4* src = reinterpret_cast<const float4*>(record(j) + c * D) + lane;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const float4 x = __ldcg(src + 32 * v);
          a[v].x += wj * x.x;
          a[v].y += wj * x.y;
          a[v].z += wj * x.z;
          a[v].w += wj * x.w;
        }
      }
    }
  }
  if (c >= cols || !mine) return;
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const int cc = hd % p.col_groups * kFewCols + c;  // column of the KV head
  T* dst = reinterpret_cast<T*>(p.out) + (row0 + cc / p.group) * p.out_stride +
           (hd / p.col_groups * p.group + cc % p.group) * D;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    T h[4] = {InTraits<T>::from_float(a[v].x * inv), InTraits<T>::from_float(a[v].y * inv),
              InTraits<T>::from_float(a[v].z * inv), InTraits<T>::from_float(a[v].w * inv)};
    *reinterpret_cast<uint2*>(dst + (lane + 32 * v) * 4) = *reinterpret_cast<const uint2*>(h);
  }
}

namespace {

template <typename T, int D>
cudaError_t launch_few(const BatchAttnParams& p, const BatchPoolMaps& maps, int sms, cudaStream_t stream) {
  using F = Few<D>;
  // the heads of a token range run side by side: their slices of a token row
  // share DRAM pages and sectors
  const int heads = p.kv_heads * p.col_groups;
  const dim3 grid(heads, max(1, sms * F::kCtas / heads));
  auto kernel = batch_few_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, grid, dim3(F::kThreads), F::kSmem, stream, p, maps);
  if (e != cudaSuccess) return e;
  // Few requests have items of many parts: a block a column (one request of 4,000
  // tokens: 14 us a call against 17 with a warp a column); otherwise a warp a
  // column (256 requests: 100 us a call against 106 with a block a column).
  const int splits = (int)grid.y;
  e = p.requests * 4 <= splits
          ? launch_pdl(batch_combine_kernel<T, D>, dim3(grid.x, grid.y, kFewCols), dim3(256), 0, stream, p)
          : launch_pdl(batch_combine_short_kernel<T, D>, grid, dim3(kCombineThreads), kFewCols * splits * sizeof(float),
                       stream, p, splits);
  if (e != cudaSuccess || (long long)p.max_rows * p.group <= p.few_cols) return e;
  return launch_rows<T, D>(p, sms, stream);
}

template <typename T>
cudaError_t launch_attend(const BatchAttnParams& p, const BatchPoolMaps& maps, int dim, int sms, cudaStream_t stream) {
  switch (dim) {
    case 64: return launch_few<T, 64>(p, maps, sms, stream);
    case 128: return launch_few<T, 128>(p, maps, sms, stream);
    case 256: return launch_few<T, 256>(p, maps, sms, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

size_t batch_few_record_bytes(int dim) { return (size_t)kBatchMaxCtas * 2 * kFewCols * (dim + 2) * sizeof(float); }
size_t batch_workspace_bytes(int dim) {
  return kBatchMetaBytes + batch_few_record_bytes(dim) + (size_t)kBatchMaxSms * 2 * kRwRows * (dim + 2) * sizeof(float);
}
int batch_few_box_rows(int dim) { return dim == 256 ? Few<256>::kTok : dim == 128 ? Few<128>::kTok : Few<64>::kTok; }

cudaError_t launch_batch_attend(const BatchAttnParams& p, const BatchPoolMaps& maps, int dim, int dtype, int sms,
                                cudaStream_t stream) {
  return dtype == kDtypeBF16 ? launch_attend<__nv_bfloat16>(p, maps, dim, sms, stream)
                             : launch_attend<__half>(p, maps, dim, sms, stream);
}

}  // namespace qwz
