// The parts of every row behind shared prefixes, merged (sm_100a): the prefix's part
// (batch_tiles.cu) and that of the request's own tokens (batch_few.cu or
// batch_tiles.cu), each whole or in records of the CTAs that shared it.
//
//   out = sum_i w_i o_i / sum_i w_i l_i,  w_i = 2^(m_i - max m)
//
// over the parts (m_i, l_i, o_i) in a fixed order: the prefix's by CTA, then the own
// tokens' by CTA.  A row that the plan does not list behind its prefix has no part there in
// this call, and what the workspace holds is an earlier call's: the part counts only where
// the place it was made for lies in the prefix's range and names the row.
// A warp has one (row, head), or G warps take every G-th part of
// it (up to eight (row, head) pairs an SM, which leave warps idle and have many parts each).  It reads D + 2 floats a
// part, mostly from L2; the chain of loads from the row's request over `where` and the
// statistics to the outputs bounds it.
// Measured, from the end of the launch before it: 96 pairs 7 us, 1,536 of about 14 parts 14 us,
// 4,032 11 us, 8,192 of three 18 us.
#include "batch_common.cuh"

namespace qwz {

namespace {

constexpr int kJoinWarps = 8;

// The records of one item: part 0 in the second one of the CTA that began it, the
// others in the first one of the CTAs after it.
struct JoinSide {
  const float* o = nullptr;   // of the row in part 0
  const float* ml = nullptr;
  size_t step = 0, rec = 0;   // floats from a CTA's records to the next one's, of a record
  int parts = 0, first = 0, ctas = 1, busy = 0;

  QWZ_DEVINL size_t at(int j) const { return j == 0 ? 0 : j * step - rec; }
  // Reference and sum of part j; a CTA without units left no record.
  QWZ_DEVINL float2 stat(int j) const {
    if (j >= parts) return make_float2(-CUDART_INF_F, 0.f);
    const long long i = first + j;
    if (parts > 1 && i * busy / ctas == (i + 1) * busy / ctas) return make_float2(-CUDART_INF_F, 0.f);
    return __ldcg(reinterpret_cast<const float2*>(ml + at(j)));
  }
};

// The request that a row belongs to, by the warp (the last one that begins at or
// before it; -1: none).
QWZ_DEVINL int join_request(const BatchAttnParams& p, int row) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = p.requests;
  while (true) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const int count = __popc(__ballot_sync(0xffffffffu, lane * step < n && __ldg(p.cu_rows + at) <= row));
    if (count == 0) return -1;
    lo += (count - 1) * step;
    n = min(step, n - (count - 1) * step);
    if (n <= 1) return lo;
  }
}

}  // namespace

template <typename T, int D, int G>
__global__ void __launch_bounds__(kJoinWarps * 32)
    batch_join_kernel(const __grid_constant__ BatchAttnParams p, int few_splits, int row_ctas) {
  constexpr int kVecs = (D + 127) / 128, kPairs = kJoinWarps / G;
  __shared__ float4 acc_s[G > 1 ? kJoinWarps : 1][kVecs * 32];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pg = warp % G;
  const int q_heads = p.kv_heads * p.group, few_heads = p.kv_heads * p.col_groups;
  const long long pairs = (long long)p.rows * q_heads;
  const bool mine = lane * 4 < D;
  constexpr size_t kRows = Tiles<D>::kRows;  // of a record of batch_tiles.cu
  constexpr size_t kFewRec = (size_t)kBatchFewCols * (D + 2), kRowRec = Tiles<D>::kRec;
  // (the loop's bounds are the same for all warps of the CTA)
  for (long long at = (long long)blockIdx.x * kPairs; at < pairs; at += (long long)gridDim.x * kPairs) {
    const long long rh = min(at + warp / G, pairs - 1);
    const int out_row = (int)(rh / q_heads), head = (int)(rh % q_heads);
    const int b = join_request(p, out_row);
    batch::Req r = {0, 0, 0};
    if (b >= 0) r = batch::load_req(p, b);
    const int s = out_row - r.row0;
    bool work = at + warp / G < pairs && b >= 0 && s < r.n;
    bool joins = false;
    batch::Req of_prefix = {0, 0, 0};
    if (work) {
      const int g = batch::prefix_of(p, b);
      if (g >= 0) {
        joins = __ldcg(p.direct + g) == 0;
        if (joins) of_prefix = batch::load_prefix(p, g);
        // many rows whose prefix was left to their request: the plan lists fewer
        if (!joins && r.n * p.group > p.few_cols) flag_error(kErrTableRange);
      }
    }
    JoinSide side[2];  // 0: the prefix, 1: own tokens
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!work || (k == 0 && !joins)) continue;
      JoinSide& x = side[k];
      const size_t part = (size_t)k * p.rows * q_heads + rh;
      const uint32_t w = __ldcg(p.where + part), what = w & 3u;
      const int first = (w >> 2) & 1023, parts = (int)((w >> 12) & 1023) + 1, row = (w >> 22) & 255;
      if (k == 0) {
        const long long place = what == kWhereWhole ? w >> 2 : __float_as_uint(__ldcg(p.part_ml + 2 * part));
        const bool there = what != kWhereDone && what != kWhereFew && place >= of_prefix.row0 &&
                           place < (long long)of_prefix.row0 + of_prefix.n && __ldg(p.shared_rows + place) == out_row;
        if (!there) {
          flag_error(kErrTableRange);
          continue;
        }
      }
      if (what == kWhereDone) {  // out has it
        work = work && k == 0;
      } else if (what == kWhereWhole) {
        x.parts = 1;
        x.o = p.part_o + part * D;
        x.ml = p.part_ml + part * 2;
      } else if (what == kWhereRows) {
        x.first = min(first, row_ctas - 1);
        x.ctas = row_ctas;
        x.busy = __ldcg(p.busy);
        x.rec = kRowRec;
        x.step = 2 * kRowRec;
        const float* rec = p.row_records + (size_t)x.first * x.step + kRowRec;
        x.o = rec + (row % kRows) * D;
        x.ml = rec + kRows * D + 2 * (row % kRows);
        x.parts = min(parts, row_ctas - x.first);
      } else {
        const int column = s * p.group + head % p.group;
        const int hd = head / p.group * p.col_groups + column / kBatchFewCols % p.col_groups;
        x.first = min(first, few_splits - 1);
        x.ctas = few_splits;
        x.busy = __ldcg(p.busy + 1 + hd);
        x.rec = kFewRec;
        x.step = 2 * few_heads * kFewRec;
        const float* rec = p.records + (size_t)x.first * x.step + (size_t)(2 * hd + 1) * kFewRec;
        x.o = rec + (size_t)(row % kBatchFewCols) * D;
        x.ml = rec + (size_t)kBatchFewCols * D + 2 * (row % kBatchFewCols);
        x.parts = min(parts, few_splits - x.first);
      }
    }
    float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      for (int j = lane; j < side[k].parts; j += 32) M = fmaxf(M, side[k].stat(j).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float4 a[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const JoinSide& x = side[k];
      for (int j0 = 0; j0 < x.parts; j0 += 32) {
        const float2 st = x.stat(j0 + lane);
        const float wt = batch::part_weight(st.x, st.y, M);
        L += wt * st.y;
        const int n = min(32, x.parts - j0);
#pragma unroll 4
        for (int i = pg; i < n; i += G) {
          const float wi = __shfl_sync(0xffffffffu, wt, i);
          if (wi == 0.f || !mine) continue;  // (a CTA without units has no record)
          const float4* src = reinterpret_cast<const float4*>(x.o + x.at(j0 + i)) + lane;
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            const float4 y = __ldcg(src + 32 * v);
            a[v].x += wi * y.x;
            a[v].y += wi * y.y;
            a[v].z += wi * y.z;
            a[v].w += wi * y.w;
          }
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if constexpr (G > 1) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) acc_s[warp][32 * v + lane] = a[v];
      __syncthreads();
      if (pg == 0) {
#pragma unroll
        for (int i = 1; i < G; ++i)
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            const float4 y = acc_s[warp + i][32 * v + lane];
            a[v].x += y.x;
            a[v].y += y.y;
            a[v].z += y.z;
            a[v].w += y.w;
          }
      }
      __syncthreads();
    }
    if (!work || !mine || pg != 0) continue;
    const float inv = L > 0.f ? 1.f / L : 0.f;
    T* dst = reinterpret_cast<T*>(p.out) + (long long)out_row * p.out_stride + (long long)head * D;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      T h[4] = {InTraits<T>::from_float(a[v].x * inv), InTraits<T>::from_float(a[v].y * inv),
                InTraits<T>::from_float(a[v].z * inv), InTraits<T>::from_float(a[v].w * inv)};
      *reinterpret_cast<uint2*>(dst + (lane + 32 * v) * 4) = *reinterpret_cast<const uint2*>(h);
    }
  }
}

namespace {

template <typename T, int D>
cudaError_t launch_shared(const BatchAttnParams& p, const BatchPoolMaps& maps, int sms, cudaStream_t stream) {
  const int clusters = sms / Tiles<D>::kCtas;
  cudaError_t e = launch_tiles<T, D>(p, clusters * Tiles<D>::kCtas, stream);
  if (e == cudaSuccess) e = launch_few<T, D, kBatchShared>(p, maps, sms, stream);
  if (e != cudaSuccess) return e;
  // Four warps a (row, head) where there are few of them (the parts are many then).  Calls with
  // four and with one, decode rows behind 8,192 tokens: 24/4/256, 16 rows (384 pairs) 54.9 and
  // 59.1 us, 43 (1,032) 64.1 and 65.4, 53 (1,272) 70.3 and 67.2, 64 (1,536) 76.8 and 73.1;
  // 32/8/128, 32 rows (1,024) 51.9 and 53.6, 40 (1,280) 61.3 and 57.1; 14/2/64, 72 rows
  // (1,008) 43.0 and 45.8, 96 (1,344) 51.4 and 47.7.
  const long long pairs = (long long)p.rows * p.kv_heads * p.group;
  const int splits = few_splits<D>(p, sms);
  auto launch = [&](auto kernel, int per_cta) {
    const dim3 grid((unsigned)min((pairs + per_cta - 1) / per_cta, 8LL * sms));
    return launch_pdl(kernel, grid, dim3(kJoinWarps * 32), 0, stream, p, splits, clusters);
  };
  return pairs <= 8LL * sms ? launch(batch_join_kernel<T, D, 4>, 2) : launch(batch_join_kernel<T, D, 1>, 8);
}

template <typename T>
cudaError_t launch_shared_of(const BatchAttnParams& p, const BatchPoolMaps& maps, int dim, int sms, cudaStream_t stream) {
  switch (dim) {
    case 64: return launch_shared<T, 64>(p, maps, sms, stream);
    case 128: return launch_shared<T, 128>(p, maps, sms, stream);
    case 256: return launch_shared<T, 256>(p, maps, sms, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_batch_attend_shared(const BatchAttnParams& p, const BatchPoolMaps& maps, int dim, int dtype, int sms,
                                       cudaStream_t stream) {
  return dtype == kDtypeBF16 ? launch_shared_of<__nv_bfloat16>(p, maps, dim, sms, stream)
                             : launch_shared_of<__half>(p, maps, dim, sms, stream);
}

}  // namespace qwz
