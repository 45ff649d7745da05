// Paging of many requests on the device: page allocation, block tables, slot
// map and row offsets of one step from the requests' lengths; and the writer
// that quantises the step's K/V rows into their slots (sm_100a).
//
// Tables.  Request b holds held[b] pages and lengths[b] tokens and adds
// new[b] rows, or ends (new[b] < 0).  With
//   grow[b] = max(0, ceil((lengths[b] + new[b]) / 256) - held[b])  (new[b] > 0)
// pages are taken from a ring of free ids in request order (exclusive scan of
// grow), those of requests that end go behind the free ones as far as the ring
// has places there.  Row r of request b, position p = lengths[b] + r, gets slot
// table[b][p / 256] * 256 + p % 256.
// All of it is a few bytes a request and 12 bytes a row: the launch and the
// latency of one scan bound it, so every CTA scans all requests by itself (one
// scan of three counts) instead of waiting for another CTA, and then fills its
// part of the rows and of the tables.  Requests that are denied count with all
// they ask for, which need not fit 32 bits together: sums stop at 2^31 - 1, beyond
// every row of the slot map and every free page.  Measured: 4.8 us for 8 requests,
// 7.1 us for 2,048 with prompts (a thread copying a request's pages: 22 us; two
// scans, of pages asked for and of pages granted: 6.5 and 9.0 us).
#include "batch_common.cuh"
#include "nvfp4_quant.cuh"

namespace qwz {

namespace {

constexpr int kTabThreads = 1024;

struct TabReq {
  int len, n, held, grow;  // n: rows; grow before the pool's limit
  bool ends, wide;         // wide: does not fit the table
};

QWZ_DEVINL TabReq tab_req(const BatchTablesParams& p, int b) {
  TabReq t;
  t.len = max(__ldg(p.lengths + b), 0);
  t.n = __ldg(p.new_rows + b);
  t.held = min(max(__ldg(p.held + b), 0), p.table_width);
  t.ends = t.n < 0;
  t.n = max(t.n, 0);
  const long long end = (long long)t.len + t.n;
  t.wide = t.n > 0 && end > (long long)p.table_width * kPage;
  t.grow = (t.n > 0 && !t.wide) ? max((int)((end + kPage - 1) / kPage) - t.held, 0) : 0;
  return t;
}

// Sum of two counts, at most 2^31 - 1 (associative for counts).
QWZ_DEVINL int add_sat(int a, int b) { return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu); }
// Rows, pages asked for and pages of requests that end.
struct TabSum {
  int rows, grow, freed;
};
QWZ_DEVINL TabSum add_sat(TabSum a, TabSum b) {
  return {add_sat(a.rows, b.rows), add_sat(a.grow, b.grow), add_sat(a.freed, b.freed)};
}
QWZ_DEVINL TabSum tab_sum(const TabReq& t) { return {t.n, t.grow, t.ends ? t.held : 0}; }
QWZ_DEVINL TabSum tab_shfl_up(TabSum v, int o) {
  return {__shfl_up_sync(0xffffffffu, v.rows, o), __shfl_up_sync(0xffffffffu, v.grow, o),
          __shfl_up_sync(0xffffffffu, v.freed, o)};
}

// Exclusive scan over the CTA; all threads' rows in `rows`.
QWZ_DEVINL TabSum tab_scan(TabSum v, TabSum* warp_sums, int& rows) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const TabSum y = tab_shfl_up(v, o);
    if (lane >= o) v = add_sat(v, y);
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  TabSum before = {0, 0, 0};
  rows = 0;
#pragma unroll
  for (int w = 0; w < kTabThreads / 32; ++w) {
    const TabSum s = warp_sums[w];
    if (w < warp) before = add_sat(before, s);
    rows = add_sat(rows, s.rows);
  }
  const TabSum y = tab_shfl_up(v, 1);
  return lane > 0 ? add_sat(before, y) : before;
}

}  // namespace

__global__ void __launch_bounds__(kTabThreads) batch_tables_kernel(const __grid_constant__ BatchTablesParams p) {
  __shared__ int2 starts[kTabThreads];  // (rows, grown pages) before each thread's requests
  __shared__ TabSum sums[kTabThreads / 32];
  __shared__ int granted_s, put_back_s;
  const int tid = threadIdx.x;
  griddep_wait();
  const int F = p.ring_size, head = __ldg(p.ring_state), count = __ldg(p.ring_state + 1);
  const bool state_ok = head >= 0 && head < F && count >= 0 && count <= F;  // else no page moves and no row has a slot
  const int per = (p.requests + kTabThreads - 1) / kTabThreads;
  const int b_lo = min(tid * per, p.requests), b_hi = min(b_lo + per, p.requests);

  if (tid == 0) granted_s = put_back_s = 0;
  TabSum v = {0, 0, 0};
  for (int b = b_lo; b < b_hi; ++b) v = add_sat(v, tab_sum(tab_req(p, b)));
  int rows;
  v = tab_scan(v, sums, rows);  // before this thread's requests
  starts[tid] = make_int2(v.rows, v.grow);
  // granted and freed pages: a request is granted while the pool lasts, one that
  // ends puts its pages back while the ring has room (places that this step takes
  // from do not count: another CTA may not have read them yet)
  auto denied = [&](const TabReq& t, int first) {
    return t.n > 0 && (!state_ok || t.wide || (t.grow > 0 && t.grow > count - first));
  };
  auto kept = [&](const TabReq& t, int freed) {
    return t.ends && t.held > 0 && (!state_ok || t.held > F - count - freed);
  };

  // the requests: CTA 0 writes the per-request words; the table entries and the
  // ring are shared out by request, a warp copies one request's pages at a time
  auto ring_at = [&](long long i) { return (int)((head + i) % F); };
  int granted = 0, put_back = 0;  // pages, up to the thread's last request that has any
  for (int k = 0; k < per; ++k) {
    const int b = b_lo + k;
    const bool mine = b < b_hi;
    TabReq t = {0, 0, 0, 0, false, false};
    if (mine) t = tab_req(p, b);
    const bool no = denied(t, v.grow), stays = kept(t, v.freed);
    if (t.grow > 0 && !no) granted = v.grow + t.grow;
    if (t.ends && t.held > 0 && !stays) put_back = v.freed + t.held;
    if (mine && blockIdx.x == 0) {
      p.cu_rows[b] = v.rows;
      p.kv_lens[b] = (t.ends || no) ? 0 : t.len + t.n;
      p.held_out[b] = t.ends ? (stays ? t.held : 0) : t.held + (no ? 0 : t.grow);
      if (no && t.wide) flag_error(kErrTableRange);
      else if ((no || stays) && state_ok) flag_error(kErrPoolEmpty);
    }
    const int pages_moved = t.ends ? (stays ? 0 : t.held) : no ? 0 : t.grow;
    unsigned work = __ballot_sync(0xffffffffu, mine && pages_moved > 0 && (unsigned)b % gridDim.x == blockIdx.x);
    while (work) {
      const int src = __ffs(work) - 1;
      work &= work - 1;
      const int n = __shfl_sync(0xffffffffu, pages_moved, src), ends = __shfl_sync(0xffffffffu, (int)t.ends, src);
      const int have = __shfl_sync(0xffffffffu, t.held, src);
      const int from = __shfl_sync(0xffffffffu, t.ends ? v.freed : v.grow, src);
      int32_t* table = p.block_table + (size_t)__shfl_sync(0xffffffffu, b, src) * p.table_width;
      for (int j = tid & 31; j < n; j += 32) {
        if (ends) {
          p.ring[ring_at((long long)count + from + j)] = table[j];
        } else {
          table[have + j] = __ldg(p.ring + ring_at((long long)from + j));
        }
      }
    }
    v = add_sat(v, tab_sum(t));
  }
  if (blockIdx.x == 0) {  // no request is served after one that was not: the furthest is the sum
    granted = __reduce_max_sync(0xffffffffu, granted);
    put_back = __reduce_max_sync(0xffffffffu, put_back);
    if ((tid & 31) == 0) {
      atomicMax(&granted_s, granted);
      atomicMax(&put_back_s, put_back);
    }
  }
  __syncthreads();  // (and `starts` is whole)
  if (blockIdx.x == 0 && tid == 0) {
    p.cu_rows[p.requests] = rows;
    p.ring_out[0] = state_ok ? ring_at(granted_s) : head;
    p.ring_out[1] = state_ok ? count - granted_s + put_back_s : count;
    if (!state_ok) flag_error(kErrPageRange);
    if (rows > p.rows) flag_error(kErrSlotRange);  // rows past the slot map's end get no slot
  }

  // the rows: find the thread whose requests hold the row, walk to the request
  for (long long r = (long long)blockIdx.x * kTabThreads + tid; r < p.rows; r += (long long)gridDim.x * kTabThreads) {
    int slot = -1, pos = 0, req = -1;
    if (r < rows) {
      int at = 0;
      for (int step = kTabThreads / 2; step > 0; step >>= 1)
        if (starts[at + step].x <= r) at += step;
      int off = (int)r - starts[at].x, first = starts[at].y;
      int b = at * per;
      TabReq t = tab_req(p, b);
      while (off >= t.n && b + 1 < p.requests) {
        off -= t.n;
        first = add_sat(first, t.grow);
        t = tab_req(p, ++b);
      }
      req = b;
      pos = add_sat(t.len, off);
      if (!denied(t, first)) {
        const int j = pos / kPage;
        int page;
        if (j < t.held) page = p.block_table[(size_t)b * p.table_width + j];
        else page = __ldg(p.ring + ring_at((long long)first + j - t.held));
        if (page >= 0 && page <= 0x7fffffff / kPage - 1) slot = page * kPage + pos % kPage;
        else flag_error(kErrPageRange);
      }
    }
    p.slots[r] = slot;
    p.positions[r] = pos;
    p.request_of[r] = req;
  }
  griddep_launch_dependents();
}

// One thread quantises one 16-element block of K or V: 32 bytes in, 8 code
// bytes, one scale byte and (optionally) the 32 bytes the cache now stands for
// out; bound by HBM.  The rounding is that of nvfp4_quant.cuh: s = E4M3(amax /
// 6), code = E2M1 of the correctly rounded x / s.  The quotient is made from
// the correctly rounded reciprocal by one residual step (Markstein: correctly
// rounded when the reciprocal is), 3 operations instead of a division, and
// converted two at a time; |x| is first cut at 8 s (E2M1 ends at 6), which also
// keeps infinities out of the residual and sends NaN to +6, as there.  Measured:
// 16,384 rows of 4 x 256, 26 us (90 % of the measured copy bandwidth); 224 rows
// 1.9 us, below what a launch costs the host.
template <typename T>
__global__ void __launch_bounds__(256) batch_append_kernel(const __grid_constant__ BatchAppendParams p) {
  griddep_wait();
  const int blocks = p.dim / 16;
  const long long per_row = (long long)p.kv_heads * blocks;
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  const bool is_v = blockIdx.y != 0;
  if (idx >= p.rows * per_row) return;
  const long long row = idx / per_row;
  const int in = (int)(idx % per_row);  // head * blocks + block
  const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + row * (is_v ? p.v_stride : p.k_stride) + in * 16;
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
  const uint4 b = __ldg(reinterpret_cast<const uint4*>(src) + 1);
  const int slot = __ldg(p.slots + row);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  float x[16], amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = InTraits<T>::to_float2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
  }
  const uint32_t sbits = quant::e4m3_encode_nonneg(__fdiv_rn(amax, 6.0f));
  const float s = quant::e4m3_decode(sbits);
  uint32_t code[2] = {0u, 0u};
  if (s > 0.f) {
    const float r = __frcp_rn(s), cut = 8.f * s;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float c = fmaxf(fminf(x[i + e], cut), -cut);
        const float q = __fmul_rn(c, r);
        y[e] = __fmaf_rn(__fmaf_rn(-q, s, c), r, q);
      }
      uint32_t pair;
      asm("{\n .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n cvt.u32.u8 %0, t;\n}\n"
          : "=r"(pair)
          : "f"(y[0]), "f"(y[1]));
      code[i >> 3] |= pair << (4 * (i & 7));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // a zero magnitude carries no sign
      const uint32_t m = code[i] & 0x77777777u;
      const uint32_t some = (m | (m >> 1) | (m >> 2)) & 0x11111111u;
      code[i] = m | (code[i] & (some << 3));
    }
  }
  if (slot >= 0 && (slot >> 8) < p.num_pages) {
    const size_t at = (size_t)slot * per_row + in;
    *reinterpret_cast<uint2*>((is_v ? p.v_cache : p.k_cache) + at * 8) = make_uint2(code[0], code[1]);
    (is_v ? p.v_scales : p.k_scales)[at] = (uint8_t)sbits;
  } else if (slot >= 0) {
    flag_error(kErrSlotRange);
  }
  void* held = is_v ? p.v_held : p.k_held;
  if (held != nullptr) {  // code x scale: at most 6 significant bits, exact in FP16 and BF16
    uint32_t h[8], s0, s1;
    {
      uint32_t t[4];
      e2m1x8_to_f16x2x4(code[0], t);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = t[i];
      e2m1x8_to_f16x2x4(code[1], t);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[4 + i] = t[i];
    }
    e4m3x4_to_f16x2x2(sbits * 0x0101u, s0, s1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] = hmul2_u32(h[i], s0);
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
        const float2 f = InTraits<__half>::to_float2(h[i]);
        const __nv_bfloat162 v = __floats2bfloat162_rn(f.x, f.y);
        h[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(held) + (row * per_row + in) * 16);
    dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
    dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
  }
}

cudaError_t launch_batch_tables(const BatchTablesParams& p, int sms, cudaStream_t stream) {
  const long long want = (p.rows + kTabThreads - 1) / kTabThreads;
  const int grid = (int)max(1LL, min(want, (long long)sms));
  return launch_pdl(batch_tables_kernel, dim3(grid), dim3(kTabThreads), 0, stream, p);
}

cudaError_t launch_batch_append(const BatchAppendParams& p, int dtype, cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  const long long n = p.rows * (long long)p.kv_heads * (p.dim / 16);
  const dim3 grid((unsigned)((n + 255) / 256), 2);
  if (dtype == kDtypeBF16) return launch_pdl(batch_append_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, p);
  return launch_pdl(batch_append_kernel<__half>, grid, dim3(256), 0, stream, p);
}

}  // namespace qwz
