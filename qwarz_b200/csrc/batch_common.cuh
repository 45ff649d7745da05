// Device helpers shared by the kernels that serve many requests from one
// NVFP4 pool: the split of all requests' work over the CTAs of a launch, and
// the records through which CTAs that share an item hand over their partials.
//
// The work of a launch is the concatenation, over requests, heads and groups
// of query rows, of the KV tiles each of them has to visit.  CTA i of N takes
// units [i * total / N, (i + 1) * total / N), so the CTAs' shares differ by at
// most one tile whatever the lengths are, and only the first and the last item
// of a CTA can be shared with other CTAs: two records a CTA hold every partial,
// independent of the number of requests.  Every CTA finds its share from the
// lengths alone (one scan), so a call needs no schedule made beforehand.
#pragma once

#include "qwz_common.cuh"
#include "batch_kernels.h"
#include "qwz_kernels.h"

#include <math_constants.h>

namespace qwz {
namespace batch {

// A row's weights are 2^(score - m).  The reference m is set kLift below the
// maximum and moves when a score exceeds it by more than kRoom, so that weights
// lie below 2^15 and, rounded to FP16, keep their 11 bits down to 2^-21 of the
// largest (with m at the maximum itself they would lose them at 2^-14).
constexpr float kLift = 7.f, kRoom = 15.f;

// Rows and tokens of request b, clipped to what the buffers hold.
struct Req {
  int row0;  // first row in q / out
  int n;     // rows
  int kv;    // tokens after the step
};

QWZ_DEVINL Req load_req(const BatchAttnParams& p, int b) {
  Req r;
  const int lo = __ldg(p.cu_rows + b), hi = __ldg(p.cu_rows + b + 1);
  r.row0 = lo;
  r.n = hi - lo;
  r.kv = __ldg(p.kv_lens + b);
  if (lo < 0 || hi < lo || hi > p.rows || r.n > p.max_rows) {  // never address rows that do not exist
    flag_error(kErrTableRange);
    r.row0 = 0;
    r.n = 0;
  }
  if (r.kv > p.table_width * kPage) {
    flag_error(kErrTableRange);
    r.kv = p.table_width * kPage;
  }
  if (r.kv < 0) r.kv = 0;
  return r;
}

// Weight of a part (m, l) of a row whose parts have the maximum M.  A part
// without tokens (m -inf, l 0) has none; one that saw nothing but NaN scores (m
// -inf, l NaN) makes the row NaN, as it would be in one piece.
QWZ_DEVINL float part_weight(float m, float l, float M) {
  return m == -CUDART_INF_F ? 0.f * l : exp2_approx(m - M);
}

// Exclusive scan of one value a thread over the CTA (blockDim.x <= 1024, a
// multiple of 32); returns the thread's prefix, the CTA's total in `total`.
QWZ_DEVINL long long block_scan(long long v, long long* warp_sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int w = 0; w < warps; ++w) {
    const long long s = warp_sums[w];
    if (w < warp) before += s;
    total += s;
  }
  __syncthreads();
  return before + x - v;
}

}  // namespace batch
}  // namespace qwz
