// Attention of many requests over one NVFP4 pool, few query rows a request
// (decode, short windows), sm_100a.
//
//   out[r, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(sm_scale q_r.k_j - max),
//   j < kv - n + s + 1 for row s of the n rows of a request with kv tokens.
//
// Bound by HBM: a token costs D/2 + D/16 bytes of K and as many of V a head,
// and 4 D multiply-adds a query column, far below the tensor rate.
//
// The (row, head of the group) pairs of one request and KV head are the
// columns of an item: kCols of them (2048 / D, so that O^T [D x kCols] is 64
// registers a thread at every head size).  CTA = 8 warps, one CTA per SM, and
// a share of all items' 256-token pages (batch_common.cuh).  A warp owns 32
// tokens of each page and streams them through a ring of its own with
// cp.async (16-byte copies straight from the pool's rows, so any head layout,
// page order and ragged end needs no descriptor); no warp waits for another
// inside an item, and the ring runs on across items, so a CTA's loads never
// drain.  A warp's 32 tokens are two 16-token MMA tiles, tokens on M and
// columns on N: K codes become A fragments of S^T in registers, V codes A
// fragments of O^T, P^T comes from the S^T fragment by movmatrix.  Base-2
// online softmax, the reference maximum moves only by more than 2^8; P is
// rounded to FP16 for its product (11 significant bits, the output's own), all
// sums are FP32.  At an item's end the eight warps' (m, l, O) are merged in
// shared memory in warp order.
#include "attn_common.cuh"
#include "batch_common.cuh"

namespace qwz {

using namespace detail;

namespace {

constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewTok = 32;  // tokens of a page a warp owns

template <int D>
struct Few {
  static constexpr int kCols = 2048 / D;             // query columns of an item
  static constexpr int kNT = kCols / 8;              // MMA column tiles
  static constexpr int kMT = D / 16;                 // MMA row tiles of O^T
  static constexpr int kRow = D / 2;                 // code bytes of a row
  static constexpr int kSRow = D / 16;               // scale bytes of a row
  static constexpr int kCodes = kFewTok * kRow;
  static constexpr int kStage = 2 * (kCodes + kFewTok * kSRow);
  static constexpr int kStages = D == 256 ? 3 : D == 128 ? 4 : 6;
  static constexpr int kMergeWarp = 16 * kEpiRowF4 * 16 + kCols * 8;  // O and (m, l) of a warp
  // D 256: the merge uses the slot that the item's last page left
  static constexpr bool kMergeInRing = kMergeWarp <= kStage;
  static constexpr int kRing = kFewWarps * kStages * kStage;
  static constexpr int kMerge = kMergeInRing ? 0 : kFewWarps * kMergeWarp;
  static constexpr int kSmem = kRing + kMerge;
};

// Byte offset of 16-byte chunk c of code row r: 128-byte lines of 128 / kRow
// rows, chunks XOR-swizzled by the line so that the K reads (8 rows x 4 lanes)
// and the V reads (rows 0, 2, 4, 6 x 8 lanes) both touch every bank once.
template <int D>
QWZ_DEVINL uint32_t few_swz(int r, int c) {
  constexpr int rpl = 128 / Few<D>::kRow, cpr = Few<D>::kRow / 16;
  const int line = r / rpl, ch = (r % rpl) * cpr + c;
  const int x = D == 256 ? (line & 7) : D == 128 ? (line & 3) * 2 : (line & 1) * 2;
  return (uint32_t)(line * 128 + ((ch ^ x) << 4));
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

// Walks the units (request, item, page) of the launch in order.
template <int D>
struct FewWalk {
  int b, head, page;       // request, KV head, page
  int pages;               // of request b
  batch::Req r;

  static QWZ_DEVINL bool few(const BatchAttnParams& p, const batch::Req& r) {
    return r.n > 0 && r.n * p.group <= p.few_cols;  // the others are batch_rows.cu's
  }
  // a request without tokens still has rows to write
  static QWZ_DEVINL int pages_of(const batch::Req& r) { return max(1, (r.kv + kPage - 1) / kPage); }
  static QWZ_DEVINL long long cost(const BatchAttnParams& p, int b) {
    const batch::Req r = batch::load_req(p, b);
    return few(p, r) ? (long long)p.kv_heads * pages_of(r) : 0;
  }
  QWZ_DEVINL void enter(const BatchAttnParams& p, int bb) {
    b = bb;
    r = batch::load_req(p, b);
    pages = pages_of(r);
  }
  // Unit `u` counted from the start of request b0.
  QWZ_DEVINL void seek(const BatchAttnParams& p, int b0, long long u) {
    for (b = b0; b < p.requests; ++b) {
      const long long c = cost(p, b);
      if (u < c) break;
      u -= c;
    }
    enter(p, min(b, p.requests - 1));
    head = (int)(u / pages);
    page = (int)(u % pages);
  }
  QWZ_DEVINL void next(const BatchAttnParams& p) {
    if (++page < pages) return;
    page = 0;
    if (++head < p.kv_heads) return;
    head = 0;
    for (int bb = b + 1; bb < p.requests; ++bb) {
      enter(p, bb);
      if (few(p, r)) return;
    }
  }
  // Table entry of the unit, unchecked (the load is in flight until it is used).
  QWZ_DEVINL int entry(const BatchAttnParams& p) const {
    return __ldg(p.block_table + (size_t)b * p.table_width + page);
  }
  // Whether the unit has tokens in a page of the pool.
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

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kFewThreads, 1) batch_few_kernel(const __grid_constant__ BatchAttnParams p) {
  using F = Few<D>;
  constexpr int NT = F::kNT, MT = F::kMT, QW = D / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ long long starts[kFewThreads + 1];  // units before each thread's requests
  __shared__ long long warp_sums[kFewWarps];
  __shared__ float weights[F::kCols * kFewWarps];
  __shared__ float col_l[F::kCols];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, qd = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * F::kStages * F::kStage;

  griddep_wait();

  // ---------------------------------------------------- this CTA's share
  const int per = (p.requests + kFewThreads - 1) / kFewThreads;
  long long mine = 0;
  for (int b = tid * per; b < min(p.requests, (tid + 1) * per); ++b) mine += FewWalk<D>::cost(p, b);
  long long total;
  starts[tid] = batch::block_scan(mine, warp_sums, total);
  __syncthreads();
  const long long n_cta = gridDim.x;
  const long long lo = (long long)blockIdx.x * total / n_cta, hi = ((long long)blockIdx.x + 1) * total / n_cta;
  const int units = (int)(hi - lo);
  int32_t* meta = p.meta + blockIdx.x * kBatchMeta;
  if (units == 0) {
    if (tid == 0) meta[0] = 0;
    griddep_launch_dependents();
    return;
  }
  int at = 0;
  for (int step = kFewThreads / 2; step > 0; step >>= 1)
    if (starts[at + step] <= lo) at += step;
  FewWalk<D> cur;
  cur.seek(p, at * per, lo - starts[at]);
  FewWalk<D> pre = cur;
  int pre_page = pre.entry(p);

  // Copies this warp's 32 tokens of the walker's unit into ring slot `slot`.
  auto issue = [&](int slot) {
    const int t0 = pre.page * kPage + warp * kFewTok;
    const int valid = pre.present(p, pre_page) ? min(kFewTok, pre.r.kv - t0) : 0;
    if (valid > 0) {
      const size_t row0 = (size_t)pre_page * kPage + warp * kFewTok;
      const size_t hd = pre.head;
      const uint32_t dst = ring + slot * F::kStage;
      constexpr int CPR = F::kRow / 16;
#pragma unroll
      for (int i = 0; i < CPR; ++i) {
        const int idx = i * 32 + lane, row = idx / CPR, c = idx % CPR;
        if (row < valid) {
          const size_t src = ((row0 + row) * p.kv_heads + hd) * F::kRow + c * 16;
          const uint32_t off = few_swz<D>(row, c);
          cp_async_small<16>(dst + off, p.k_codes + src);
          cp_async_small<16>(dst + F::kCodes + off, p.v_codes + src);
        }
      }
      if (lane < valid) {
        const size_t src = ((row0 + lane) * p.kv_heads + hd) * F::kSRow;
        const uint32_t off = dst + 2 * F::kCodes + lane * F::kSRow;
        cp_async_small<F::kSRow>(off, p.k_scales + src);
        cp_async_small<F::kSRow>(off + kFewTok * F::kSRow, p.v_scales + src);
      }
    }
  };

  int issued = 0;
  auto advance = [&](int slot) {  // one group a unit, empty past the share's end
    if (issued < units) {
      issue(slot);
      if (++issued < units) {
        pre.next(p);
        pre_page = pre.entry(p);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < F::kStages - 1; ++s) advance(s);

  float o[NT][MT][4];
  float m[NT][2], l[NT][2], cf[NT][2];
  int lim[NT][2];
  uint32_t qf[NT][QW];
  int first_page = 0, min_lim = 0, max_lim = 0, cols = 0;
  bool fresh = true;
  if (tid == 0) meta[0] = 0;
  int slot = 0, fill = F::kStages - 1;

  for (int k = 0; k < units; ++k) {
    if (fresh) {  // ------------------------------------------- a new item
      fresh = false;
      first_page = cur.page;
      const int hd = cur.head;
      cols = cur.r.n * p.group;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int c = nt * 8 + g;
        float amax = 0.f;
        if (c < cols) {
          const int s = c / p.group, h = hd * p.group + c % p.group;
          const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) +
                                                            (cur.r.row0 + s) * p.q_stride + h * D + qd * (D / 4));
#pragma unroll
          for (int i = 0; i < QW / 4; ++i) {
            const uint4 v = __ldg(src + i);
            qf[nt][4 * i + 0] = v.x;
            qf[nt][4 * i + 1] = v.y;
            qf[nt][4 * i + 2] = v.z;
            qf[nt][4 * i + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < QW; ++i) qf[nt][i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          const float2 f = InTraits<T>::to_float2(qf[nt][i]);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        amax = fmaxf(amax, shfl_xor(amax, 1));
        amax = fmaxf(amax, shfl_xor(amax, 2));
        const float sc = pow2_row_scale(amax);
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          const float2 f = InTraits<T>::to_float2(qf[nt][i]);
          qf[nt][i] = pack_half2(f.x * sc, f.y * sc);
        }
        const float rowfac = p.sm_scale_log2 / sc;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          cf[nt][i] = __shfl_sync(kFull, rowfac, 4 * (2 * qd + i));
          const int cc = nt * 8 + 2 * qd + i;
          lim[nt][i] = cc < cols ? cur.r.kv - cur.r.n + cc / p.group + 1 : 0;
          m[nt][i] = -CUDART_INF_F;
          l[nt][i] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      }
      min_lim = cur.r.kv - cur.r.n + 1;
      max_lim = cur.r.kv - cur.r.n + (cols - 1) / p.group + 1;
    }

    cp_async_wait<F::kStages - 2>();
    __syncwarp();
    const bool here = cur.present(p, cur.entry(p));
    advance(fill);
    fill = fill + 1 == F::kStages ? 0 : fill + 1;

    const uint32_t st = ring + slot * F::kStage;
    const uint32_t k_codes = st, v_codes = st + F::kCodes;
    const uint32_t k_scales = st + 2 * F::kCodes, v_scales = k_scales + kFewTok * F::kSRow;
    const int tw = cur.page * kPage + warp * kFewTok;
    if (tw < max_lim && here) {
      const bool tail = tw + kFewTok > min_lim;
      // ------------------------------------------------ S^T of both tiles
      float t[NT][8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float sa[NT][4], sb[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sa[nt][i] = sb[nt][i] = 0.f;
        const int r0 = 16 * half + g, r1 = r0 + 8;
        constexpr int KW = D / 32;  // code words of a lane: 8, 4, 2
        uint32_t kw0[KW], kw1[KW], sc0[4], sc1[4];
        if constexpr (D == 256) {
          uint32_t(&a)[4] = reinterpret_cast<uint32_t(&)[4]>(kw0[0]);
          uint32_t(&b)[4] = reinterpret_cast<uint32_t(&)[4]>(kw0[4]);
          uint32_t(&c)[4] = reinterpret_cast<uint32_t(&)[4]>(kw1[0]);
          uint32_t(&d)[4] = reinterpret_cast<uint32_t(&)[4]>(kw1[4]);
          lds_words(k_codes + few_swz<D>(r0, 2 * qd), a);
          lds_words(k_codes + few_swz<D>(r0, 2 * qd + 1), b);
          lds_words(k_codes + few_swz<D>(r1, 2 * qd), c);
          lds_words(k_codes + few_swz<D>(r1, 2 * qd + 1), d);
          scales_bcast4(lds32(k_scales + r0 * 16 + 4 * qd), sc0);
          scales_bcast4(lds32(k_scales + r1 * 16 + 4 * qd), sc1);
        } else if constexpr (D == 128) {
          lds_words(k_codes + few_swz<D>(r0, qd), kw0);
          lds_words(k_codes + few_swz<D>(r1, qd), kw1);
          scales_bcast4(lds16(k_scales + r0 * 8 + 2 * qd), sc0);
          scales_bcast4(lds16(k_scales + r1 * 8 + 2 * qd), sc1);
        } else {
          lds_words(k_codes + few_swz<D>(r0, qd >> 1) + (qd & 1) * 8, kw0);
          lds_words(k_codes + few_swz<D>(r1, qd >> 1) + (qd & 1) * 8, kw1);
          scales_bcast4(lds8(k_scales + r0 * 4 + qd), sc0);
          scales_bcast4(lds8(k_scales + r1 * 4 + qd), sc1);
        }
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
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816(sa[nt], h0[0], h1[0], h0[1], h1[1], qf[nt][4 * w8 + 0], qf[nt][4 * w8 + 1]);
            mma_16816(sb[nt], h0[2], h1[2], h0[3], h1[3], qf[nt][4 * w8 + 2], qf[nt][4 * w8 + 3]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = (sa[nt][i] + sb[nt][i]) * cf[nt][i & 1];
            if (tail && tw + 16 * half + g + 8 * (i >> 1) >= lim[nt][i & 1]) x = -CUDART_INF_F;
            t[nt][4 * half + i] = x;
          }
      }

      // V codes first: their shared-memory latency hides behind the softmax
      const int end = cur.r.kv - tw;
      FewV<D> va, vb;
      few_v_load<D>(v_codes, v_scales, 2 * qd, g, tail, end, va);
      few_v_load<D>(v_codes, v_scales, 2 * qd + 16, g, tail, end, vb);

      // ------------------------------------------------ online softmax
      PFrag pa[NT], pb[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx0 = fmaxf(fmaxf(t[nt][0], t[nt][2]), fmaxf(t[nt][4], t[nt][6]));
        float mx1 = fmaxf(fmaxf(t[nt][1], t[nt][3]), fmaxf(t[nt][5], t[nt][7]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, shfl_xor(mx0, off));
          mx1 = fmaxf(mx1, shfl_xor(mx1, off));
        }
        if (__any_sync(kFull, (mx0 > m[nt][0] + kLazy) || (mx1 > m[nt][1] + kLazy))) {
          const float n0 = fmaxf(m[nt][0], mx0), n1 = fmaxf(m[nt][1], mx1);
          const float a0 = (n0 == -CUDART_INF_F) ? 1.f : exp2_approx(m[nt][0] - n0);
          const float a1 = (n1 == -CUDART_INF_F) ? 1.f : exp2_approx(m[nt][1] - n1);
          m[nt][0] = n0;
          m[nt][1] = n1;
          l[nt][0] *= a0;
          l[nt][1] *= a1;
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[nt][j][0] *= a0;
            o[nt][j][1] *= a1;
            o[nt][j][2] *= a0;
            o[nt][j][3] *= a1;
          }
        }
        const float mu0 = (m[nt][0] == -CUDART_INF_F) ? 0.f : m[nt][0];
        const float mu1 = (m[nt][1] == -CUDART_INF_F) ? 0.f : m[nt][1];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          t[nt][i] = exp2_approx(t[nt][i] - mu0);
          t[nt][i + 1] = exp2_approx(t[nt][i + 1] - mu1);
        }
        l[nt][0] += (t[nt][0] + t[nt][2]) + (t[nt][4] + t[nt][6]);
        l[nt][1] += (t[nt][1] + t[nt][3]) + (t[nt][5] + t[nt][7]);
        pa[nt] = p_fragments(t[nt][0], t[nt][1], t[nt][2], t[nt][3]);
        pb[nt] = p_fragments(t[nt][4], t[nt][5], t[nt][6], t[nt][7]);
      }

      // ------------------------------------------------ O^T += V^T P^T
#pragma unroll
      for (int w = 0; w < FewV<D>::W; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const FewV<D>& v = half ? vb : va;
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
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t a0 = hmul2_u32(hxab[kk], sab), a1 = hmul2_u32(hyab[kk], sab);
            const uint32_t a2 = hmul2_u32(hxcd[kk], scd), a3 = hmul2_u32(hycd[kk], scd);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_16816(o[nt][4 * w + kk], a0, a1, a2, a3, half ? pb[nt].hi0 : pa[nt].hi0,
                        half ? pb[nt].hi1 : pa[nt].hi1);
          }
        }
      }
    }

    if (cur.page + 1 == cur.pages || k + 1 == units) {  // --------- item's end
      uint8_t* area = F::kMergeInRing ? smem + slot * F::kStage : smem + F::kRing;
      constexpr int kPitch = F::kMergeInRing ? F::kStages * F::kStage : F::kMergeWarp;
      float4* red = reinterpret_cast<float4*>(area + warp * kPitch);
      float* ml = reinterpret_cast<float*>(red + 16 * kEpiRowF4);
      __syncwarp();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[nt][i] += shfl_xor(l[nt][i], off);
#pragma unroll
        for (int j = 0; j < MT; ++j)
          red[(nt * MT + j) * kEpiRowF4 + lane] =
              make_float4(o[nt][j][0], o[nt][j][1], o[nt][j][2], o[nt][j][3]);
        if (g == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ml[(nt * 8 + 2 * qd + i) * 2 + 0] = m[nt][i];
            ml[(nt * 8 + 2 * qd + i) * 2 + 1] = l[nt][i];
          }
        }
      }
      const bool starts_here = first_page == 0, ends_here = cur.page + 1 == cur.pages;
      const bool whole = starts_here && ends_here;
      float* rec = p.records + (size_t)(blockIdx.x * 2 + (starts_here ? 1 : 0)) * (F::kCols * (D + 2));
      __syncthreads();
      if (tid < F::kCols) {
        float mm[kFewWarps], M = -CUDART_INF_F, ls = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
          const float* s = reinterpret_cast<const float*>(area + w * kPitch + 16 * kEpiRowF4 * 16) + tid * 2;
          mm[w] = s[0];
          M = fmaxf(M, mm[w]);
        }
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
          const float* s = reinterpret_cast<const float*>(area + w * kPitch + 16 * kEpiRowF4 * 16) + tid * 2;
          const float wt = mm[w] == -CUDART_INF_F ? 0.f : exp2_approx(mm[w] - M);
          weights[tid * kFewWarps + w] = wt;
          ls += wt * s[1];
        }
        col_l[tid] = ls > 0.f ? 1.f / ls : 0.f;
        if (!whole) {
          rec[F::kCols * D + 2 * tid] = M;
          rec[F::kCols * D + 2 * tid + 1] = ls;
        }
      }
      __syncthreads();
      const int hd = cur.head;
      for (int idx = tid; idx < cols * (D / 2); idx += kFewThreads) {
        const int c = idx / (D / 2), d = idx % (D / 2) * 2;
        // d = D/8 gg + 2j sits in m-tile j, lane row gg: (d, col) in c0/c1, (d + 1, col) in c2/c3
        const int gg = d / (D / 8), j = d % (D / 8) / 2;
        const int src = ((((c >> 3) * MT + j) * kEpiRowF4) + 4 * gg + ((c & 7) >> 1)) * 4 + (c & 1);
        float a0 = 0.f, a1 = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
          const float* s = reinterpret_cast<const float*>(area + w * kPitch);
          a0 += weights[c * kFewWarps + w] * s[src];
          a1 += weights[c * kFewWarps + w] * s[src + 2];
        }
        if (whole) {
          const int s = c / p.group, h = hd * p.group + c % p.group;
          T* dst = reinterpret_cast<T*>(p.out) + (cur.r.row0 + s) * p.out_stride + h * D + d;
          dst[0] = InTraits<T>::from_float(a0 * col_l[c]);
          dst[1] = InTraits<T>::from_float(a1 * col_l[c]);
        } else {
          *reinterpret_cast<float2*>(rec + c * D + d) = make_float2(a0, a1);
        }
      }
      if (starts_here && !ends_here && tid == 0) {  // the rest of the item is the next CTAs'
        const long long last_unit = hi - 1 - cur.page + cur.pages - 1;
        meta[0] = cols;
        meta[1] = cur.r.row0;
        meta[3] = hd;
        meta[4] = (int)(((last_unit + 1) * n_cta - 1) / total);
        meta[5] = (int)min(total, n_cta);  // fewer units than CTAs leave some CTAs without a record
      }
      __syncthreads();
      fresh = true;
    }
    cur.next(p);
    slot = slot + 1 == F::kStages ? 0 : slot + 1;
  }
  griddep_launch_dependents();
}

// Merges the records of the items that more than one CTA worked on, CTA by
// CTA in order: block (i, y) takes columns y, y + gridDim.y, ... of the item
// that CTA i began and did not finish.  
template <typename T, int D, int COLS>
__global__ void __launch_bounds__(256) batch_combine_kernel(const __grid_constant__ BatchAttnParams p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float w[256];
  __shared__ float red[8];
  __shared__ float4 acc_s[kGroups][kLanes];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, i0 = blockIdx.x, n_cta = gridDim.x;
  const int32_t* meta = p.meta + i0 * kBatchMeta;
  const int cols = __ldcg(meta);
  if (cols == 0) return;
  const int row0 = __ldcg(meta + 1), hd = __ldcg(meta + 3), last = __ldcg(meta + 4);
  const int busy = __ldcg(meta + 5);
  const int parts = last - i0 + 1;
  constexpr size_t kRec = (size_t)COLS * (D + 2);
  // CTA i0 left its part in record 1, the later ones in record 0
  auto record = [&](int j) { return p.records + (size_t)((i0 + j) * 2 + (j == 0 ? 1 : 0)) * kRec; };
  auto empty = [&](int j) {
    const long long i = i0 + j;
    return i * busy / n_cta == (i + 1) * busy / n_cta;
  };
  for (int c = blockIdx.y; c < cols; c += gridDim.y) {
    float m = -CUDART_INF_F, l = 0.f;
    if (tid < parts && !empty(tid)) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(record(tid) + COLS * D + 2 * c));
      m = v.x;
      l = v.y;
    }
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if ((tid & 31) == 0) red[tid >> 5] = M;
    __syncthreads();
    M = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) M = fmaxf(M, red[i]);
    __syncthreads();
    const float wt = m == -CUDART_INF_F ? 0.f : exp2_approx(m - M);
    w[tid] = wt;
    float L = wt * l;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if ((tid & 31) == 0) red[tid >> 5] = L;
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) L += red[i];
    const int grp = tid / kLanes, ln = tid % kLanes;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = grp; j < parts; j += kGroups) {
      const float wj = w[j];
      if (wj == 0.f) continue;
      const float4 v = __ldcg(reinterpret_cast<const float4*>(record(j) + c * D) + ln);
      a.x += wj * v.x;
      a.y += wj * v.y;
      a.z += wj * v.z;
      a.w += wj * v.w;
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
      const int s = c / p.group, h = hd * p.group + c % p.group;
      T* dst = reinterpret_cast<T*>(p.out) + (row0 + s) * p.out_stride + h * D + tid * 4;
      dst[0] = InTraits<T>::from_float(a.x * inv);
      dst[1] = InTraits<T>::from_float(a.y * inv);
      dst[2] = InTraits<T>::from_float(a.z * inv);
      dst[3] = InTraits<T>::from_float(a.w * inv);
    }
    __syncthreads();
  }
}

namespace {

template <typename T, int D>
cudaError_t launch_few(const BatchAttnParams& p, int ctas, cudaStream_t stream) {
  auto kernel = batch_few_kernel<T, D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<D>::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(ctas), dim3(kFewThreads), Few<D>::kSmem, stream, p);
  if (e != cudaSuccess) return e;
  e = launch_pdl(batch_combine_kernel<T, D, Few<D>::kCols>, dim3(ctas, 8), dim3(256), 0, stream, p);
  if (e != cudaSuccess || (long long)p.max_rows * p.group <= p.few_cols) return e;
  return launch_rows<T, D>(p, ctas, stream);
}

template <typename T>
cudaError_t launch_attend(const BatchAttnParams& p, int dim, int ctas, cudaStream_t stream) {
  switch (dim) {
    case 64: return launch_few<T, 64>(p, ctas, stream);
    case 128: return launch_few<T, 128>(p, ctas, stream);
    case 256: return launch_few<T, 256>(p, ctas, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

size_t batch_few_record_bytes(int dim) {
  return (size_t)kBatchMaxCtas * 2 * (2048 / dim) * (dim + 2) * sizeof(float);
}
size_t batch_workspace_bytes(int dim) {
  return kBatchMetaBytes + batch_few_record_bytes(dim) +
         (size_t)kBatchMaxCtas * 2 * kRwRows * (dim + 2) * sizeof(float);
}

cudaError_t launch_batch_attend(const BatchAttnParams& p, int dim, int dtype, int ctas, cudaStream_t stream) {
  if (p.requests <= 0 || p.rows <= 0) return cudaSuccess;
  return dtype == kDtypeBF16 ? launch_attend<__nv_bfloat16>(p, dim, ctas, stream)
                             : launch_attend<__half>(p, dim, ctas, stream);
}

}  // namespace qwz
