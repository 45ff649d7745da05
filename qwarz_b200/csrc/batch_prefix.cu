// Requests behind shared prefixes, sm_100a: the step's rows sorted by the prefix
// they read, and the writer that norms and rotates Q and K on the way (the
// attention is that of batch_rows.cu and batch_few.cu).
//
// A prefix is a request that has none itself; e(b) is the one that request b
// reads, n(b) the request's rows.  Rows are listed by prefix, then by row, so
// the place of request b's first row is the sum of n(b') over the requests with
// (e(b'), b') < (e(b), b).  With R requests a CTA compares its 32 with all of
// them (R / 8 comparisons a thread); for 2^14 requests, the most a call takes,
// that is still less than what a sort's passes would wait for one another.
#include "batch_common.cuh"
#include "nvfp4_quant.cuh"

namespace qwz {

namespace {

constexpr int kShReq = 32;              // requests of a CTA
constexpr int kShSub = 8;               // threads a request
constexpr int kShThreads = kShReq * kShSub;
constexpr int kShTile = 1024;           // requests in shared memory at a time

// The prefix that request b reads: one that exists, is another and has none itself.
QWZ_DEVINL int share_prefix(const BatchShareParams& p, int b) {
  const int g = __ldg(p.prefix_of + b);
  if (g < 0) return -1;
  if (g < p.requests && g != b && __ldg(p.prefix_of + g) < 0) return g;
  flag_error(kErrTableRange);
  return -1;
}
// Rows of request b: [lo, lo + n).
QWZ_DEVINL int share_rows(const BatchShareParams& p, int b, int& lo) {
  lo = __ldg(p.cu_rows + b);
  const int hi = __ldg(p.cu_rows + b + 1);
  if (lo >= 0 && hi >= lo && hi <= p.rows) return hi - lo;
  flag_error(kErrTableRange);
  return 0;
}

}  // namespace

__global__ void __launch_bounds__(kShThreads) batch_share_kernel(const __grid_constant__ BatchShareParams p) {
  __shared__ int2 tile[kShTile];        // (prefix, rows)
  griddep_wait();
  const int tid = threadIdx.x, sub = tid % kShSub;
  const int b = blockIdx.x * kShReq + tid / kShSub;
  const int key = b < p.requests ? share_prefix(p, b) : -1;
  int before = 0, of_lower = 0, readers = 0, reader = -1, total = 0;
  for (int t0 = 0; t0 < p.requests; t0 += kShTile) {
    const int n = min(kShTile, p.requests - t0);
    __syncthreads();
    for (int i = tid; i < n; i += kShThreads) {
      int lo;
      tile[i] = make_int2(share_prefix(p, t0 + i), share_rows(p, t0 + i, lo));
    }
    __syncthreads();
    for (int i = sub; i < n; i += kShSub) {
      const int2 o = tile[i];
      if (o.x < 0 || o.y == 0) continue;
      total += o.y;
      if (o.x < key || (o.x == key && t0 + i < b)) before += o.y;
      if (o.x < b) of_lower += o.y;
      if (o.x == b) {
        ++readers;
        reader = t0 + i;
      }
    }
  }
#pragma unroll
  for (int o = 1; o < kShSub; o <<= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    of_lower += __shfl_xor_sync(0xffffffffu, of_lower, o);
    readers += __shfl_xor_sync(0xffffffffu, readers, o);
    reader = max(reader, __shfl_xor_sync(0xffffffffu, reader, o));
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  int lo = 0, n = 0;
  if (b < p.requests) n = share_rows(p, b, lo);
  if (sub == 0 && b < p.requests) {
    p.reads[b] = key;
    p.alone[b] = readers == 1 ? reader : -1;
    p.cu_shared[b] = of_lower;
    if (b == 0) p.cu_shared[p.requests] = total;
  }
  // the rows of the CTA's requests, by eight threads each
  const int place = key >= 0 ? before : -1;
  if (place >= 0)
    for (int i = sub; i < n && place + i < p.rows; i += kShSub) p.shared_rows[place + i] = lo + i;
  // positions from the prefix's start, and the places behind the last row
  const int step = gridDim.x * kShThreads;
  for (int t = blockIdx.x * kShThreads + tid; t < p.rows; t += step) {
    const int r = __ldg(p.request_of + t);
    int pos = p.positions[t];
    if (r >= 0 && r < p.requests) {
      const int g = share_prefix(p, r);
      if (g >= 0) pos += max(__ldg(p.kv_lens + g), 0);
    }
    p.positions_out[t] = pos;
    if (t >= total) p.shared_rows[t] = -1;
  }
  griddep_launch_dependents();
}

cudaError_t launch_batch_share(const BatchShareParams& p, int sms, cudaStream_t stream) {
  const int by_request = (p.requests + kShReq - 1) / kShReq;
  const int by_row = min((p.rows + kShThreads - 1) / kShThreads, sms);
  return launch_pdl(batch_share_kernel, dim3(max(max(by_request, by_row), 1)), dim3(kShThreads), 0, stream, p);
}

// ---------------------------------------------------------------------------
// Norm, rotation and quantisation of a step's rows.
//
//   x' = x w / sqrt(mean(x^2) + eps)                      (with a weight)
//   (y_i, y_j) = (x'_i cos a - x'_j sin a, x'_j cos a + x'_i sin a),  a = position * inv_freq_i
// with j = i + freqs, or the pairs (2i, 2i + 1); dims from 2 freqs on keep x'.
// q_out is y rounded once.  K's y goes to the quantiser without a rounding in
// between: E4M3 scales and E2M1 codes are those of the exact y, up to the
// error of 64 bits, so they do not depend on how 32 bits round next to a border.
// 64-bit arithmetic is half as fast as 32-bit here and only K's rotated dims need
// it; angles of far positions need it anyway (a position of 10^6 leaves 32 bits
// 0.06 radians).
namespace {

// Nearest float with an odd last bit unless y is a float itself: later roundings
// to fewer bits, and comparisons with numbers of fewer bits, come out as those of y.
QWZ_DEVINL float float_odd(double y) {
  const float f = __double2float_rz(y);
  return __uint_as_float(__float_as_uint(f) | ((__double2loint(y) & 0x1fffffff) != 0 ? 1u : 0u));
}
// The same of an IEEE quotient q whose remainder has the sign of `rem`.
QWZ_DEVINL float odd_of(float q, float rem) {
  const uint32_t u = __float_as_uint(q);
  const int up = ((rem > 0.f) == (q > 0.f)) ? 1 : -1;
  return (rem > 0.f || rem < 0.f) && q != 0.f && (u & 1u) == 0u ? __uint_as_float(u + up) : q;
}

// Eight elements of one 16-element block, whose other half the lane next to this
// one has: code word and scale byte, with the rounding of nvfp4_quant.cuh for the
// numbers that x stands for (exact, or rounded to odd).
QWZ_DEVINL void quantise8(const float (&x)[8], uint32_t& code, uint32_t& sbits) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  const float q6 = __fdiv_rn(amax, 6.f);
  sbits = quant::e4m3_encode_nonneg(odd_of(q6, __fmaf_rn(-q6, 6.f, amax)));
  const float s = quant::e4m3_decode(sbits);
  code = 0u;
  if (s > 0.f) {
    const float r = __frcp_rn(s), cut = 8.f * s;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float c = fmaxf(fminf(x[i + e], cut), -cut);
        const float q = __fmul_rn(c, r);
        const float d = __fmaf_rn(__fmaf_rn(-q, s, c), r, q);  // c / s, correctly rounded
        y[e] = odd_of(d, __fmaf_rn(-d, s, c));
      }
      uint32_t pair;
      asm("{\n .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n cvt.u32.u8 %0, t;\n}\n"
          : "=r"(pair)
          : "f"(y[0]), "f"(y[1]));
      code |= pair << (4 * i);
    }
    const uint32_t m = code & 0x77777777u;  // a zero magnitude carries no sign
    const uint32_t some = (m | (m >> 1) | (m >> 2)) & 0x11111111u;
    code = m | (code & (some << 3));
  }
}

// The eight values that a code word and its scale stand for, as T.
template <typename T>
QWZ_DEVINL uint4 held8(uint32_t code, uint32_t sbits) {
  uint32_t h[4], s0, s1;
  e2m1x8_to_f16x2x4(code, h);
  e4m3x4_to_f16x2x2(sbits * 0x0101u, s0, s1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = hmul2_u32(h[i], s0);
    if constexpr (!std::is_same<T, __half>::value) {
      const float2 f = InTraits<__half>::to_float2(h[i]);
      const __nv_bfloat162 v = __floats2bfloat162_rn(f.x, f.y);
      h[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}

template <typename T, typename F>
QWZ_DEVINL void to_floats(const uint4& v, F (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = InTraits<T>::to_float2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename F>
QWZ_DEVINL void scale8(F (&x)[8], const float* weight, F r) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(weight)), b = __ldg(reinterpret_cast<const float4*>(weight) + 1);
  const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
}

QWZ_DEVINL float rsqrt_of(float x) { return rsqrtf(x); }
QWZ_DEVINL double rsqrt_of(double x) { return rsqrt(x); }
QWZ_DEVINL float shfl_xor_any(float x, int o) { return __shfl_xor_sync(0xffffffffu, x, o); }
QWZ_DEVINL double shfl_xor_any(double x, int o) { return __shfl_xor_sync(0xffffffffu, x, o); }

// Norm and rotation of one head, eight dims a lane (chunk c of D / 8), in F's
// precision.  cos_sin: the row's table.
template <typename T, int D, typename F, typename F2>
QWZ_DEVINL void turn8(const uint4& raw, int c, const float* weight, float eps, int freqs, bool neighbours,
                      const F2* cos_sin, F (&x)[8]) {
  constexpr int kLanes = D / 8;
  to_floats<T>(raw, x);
  F r = 1;
  if (weight != nullptr) {
    F sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += shfl_xor_any(sum, o);
    r = rsqrt_of(sum / D + (F)eps);
    scale8(x, weight + 8 * c, r);
  }
  if (neighbours) {
    if (c < freqs / 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 t = cos_sin[4 * c + i];
        const F a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = a * t.x - b * t.y;
        x[2 * i + 1] = b * t.x + a * t.y;
      }
    }
  } else {
    // the chunk `half` chunks away has the pairs' other halves
    const int half = freqs / 8, lane = threadIdx.x & 31;
    const bool turns = c < 2 * half, low = c < half;
    const int other = turns ? (low ? c + half : c - half) : c;
    const int from = lane - c + other;
    uint4 w;
    w.x = __shfl_sync(0xffffffffu, raw.x, from);
    w.y = __shfl_sync(0xffffffffu, raw.y, from);
    w.z = __shfl_sync(0xffffffffu, raw.z, from);
    w.w = __shfl_sync(0xffffffffu, raw.w, from);
    if (turns) {
      F y[8];
      to_floats<T>(w, y);
      if (weight != nullptr) scale8(y, weight + 8 * other, r);
      const int f0 = 8 * (low ? c : c - half);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const F2 t = cos_sin[f0 + i];
        x[i] = low ? x[i] * t.x - y[i] * t.y : x[i] * t.x + y[i] * t.y;
      }
    }
  }
}

constexpr int kRotThreads = 256;

template <int ROWS>
struct RotTable {
  double2 wide[ROWS][128];  // (cos, sin) of a row's angles
  float2 narrow[ROWS][128];
};

}  // namespace

// A CTA has ROWS rows: their angles' cosines and sines first, then heads, D / 8
// lanes each, the row's Q heads, K heads and V heads in turn.  grid.y CTAs share
// the heads of the same rows.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kRotThreads) batch_rotate_kernel(const __grid_constant__ BatchRotateParams p) {
  constexpr int kLanes = D / 8, kHeads = 32 / kLanes;  // lanes a head, heads a warp
  __shared__ RotTable<ROWS> table;
  griddep_wait();
  const BatchAppendParams& a = p.kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = lane % kLanes;
  const long long row0 = (long long)blockIdx.x * ROWS;
  const int rows = (int)min((long long)ROWS, a.rows - row0);
  for (int i = tid; i < rows * p.freqs; i += kRotThreads) {
    const int r = i / p.freqs, f = i % p.freqs;
    // the angle in turns, its whole part taken off: position * inv_freq / 2 pi with 1 / 2 pi in two parts
    constexpr double kTurn = 0.15915494309189535, kTurnLow = -9.839338337591243e-18;
    const double pos = __ldg(p.positions + row0 + r), freq = __ldg(p.inv_freq + f);
    const double angle = pos * freq, rest = __fma_rn(pos, freq, -angle);
    const double turns = angle * kTurn;
    const double low = __fma_rn(angle, kTurn, -turns) + angle * kTurnLow + rest * kTurn;
    double s, co;
    sincospi(2.0 * ((turns - rint(turns)) + low), &s, &co);
    table.wide[r][f] = make_double2(co, s);
    table.narrow[r][f] = make_float2((float)co, (float)s);
  }
  __syncthreads();
  const int qu = (p.q_heads + kHeads - 1) / kHeads, ku = (a.kv_heads + kHeads - 1) / kHeads;
  const int per_row = qu + 2 * ku, step = gridDim.y * (kRotThreads / 32);
  for (int u = blockIdx.y * (kRotThreads / 32) + warp; u < rows * per_row; u += step) {
    const int r = u / per_row, v = u % per_row;
    const long long row = row0 + r;
    const int kind = v < qu ? 0 : v < qu + ku ? 1 : 2;  // Q, K, V
    const int head = (kind == 0 ? v : kind == 1 ? v - qu : v - qu - ku) * kHeads + lane / kLanes;
    const bool mine = head < (kind == 0 ? p.q_heads : a.kv_heads);
    const T* src = reinterpret_cast<const T*>(kind == 0 ? p.q : kind == 1 ? a.k : a.v) +
                   row * (kind == 0 ? p.q_stride : kind == 1 ? a.k_stride : a.v_stride) + head * D + 8 * c;
    const uint4 raw = mine ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
    if (kind == 0) {
      float x[8];
      turn8<T, D, float, float2>(raw, c, p.q_weight, p.eps, p.freqs, p.neighbours != 0, table.narrow[r], x);
      if (mine) {
        T h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = InTraits<T>::from_float(x[i]);
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out) + row * p.q_out_stride + head * D + 8 * c) =
            *reinterpret_cast<const uint4*>(h);
      }
      continue;
    }
    float x[8];
    if (kind == 1) {
      double y[8];
      turn8<T, D, double, double2>(raw, c, p.k_weight, p.eps, p.freqs, p.neighbours != 0, table.wide[r], y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = float_odd(y[i]);
    } else {
      to_floats<T>(raw, x);
    }
    uint32_t code, sbits;
    quantise8(x, code, sbits);
    if (!mine) continue;
    const int slot = __ldg(a.slots + row);
    if (slot >= 0 && (slot >> 8) < a.num_pages) {
      const size_t at = (size_t)slot * a.kv_heads + head;
      reinterpret_cast<uint32_t*>(kind == 1 ? a.k_cache : a.v_cache)[at * kLanes + c] = code;
      if ((c & 1) == 0) (kind == 1 ? a.k_scales : a.v_scales)[at * (D / 16) + c / 2] = (uint8_t)sbits;
    } else if (slot >= 0) {
      flag_error(kErrSlotRange);
    }
    void* held = kind == 1 ? a.k_held : a.v_held;
    if (held != nullptr)
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(held) + (row * a.kv_heads + head) * D + 8 * c) =
          held8<T>(code, sbits);
  }
  griddep_launch_dependents();
}

namespace {

template <typename T, int D>
cudaError_t launch_rotate(const BatchRotateParams& p, cudaStream_t stream) {
  constexpr int kHeads = 256 / D;
  const int per_row = (p.q_heads + kHeads - 1) / kHeads + 2 * ((p.kv.kv_heads + kHeads - 1) / kHeads);
  // few rows: a row's heads over several CTAs, each with the row's angles
  if (p.kv.rows <= 256)
    return launch_pdl(batch_rotate_kernel<T, D, 1>, dim3((unsigned)p.kv.rows, (per_row + 7) / 8), dim3(kRotThreads), 0,
                      stream, p);
  constexpr int kRows = 4;
  return launch_pdl(batch_rotate_kernel<T, D, kRows>, dim3((unsigned)((p.kv.rows + kRows - 1) / kRows)),
                    dim3(kRotThreads), 0, stream, p);
}

template <typename T>
cudaError_t launch_rotate_of(const BatchRotateParams& p, cudaStream_t stream) {
  switch (p.kv.dim) {
    case 64: return launch_rotate<T, 64>(p, stream);
    case 128: return launch_rotate<T, 128>(p, stream);
    case 256: return launch_rotate<T, 256>(p, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_batch_rotate(const BatchRotateParams& p, int dtype, cudaStream_t stream) {
  return dtype == kDtypeBF16 ? launch_rotate_of<__nv_bfloat16>(p, stream) : launch_rotate_of<__half>(p, stream);
}

}  // namespace qwz
