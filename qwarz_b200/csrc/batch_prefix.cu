// Requests behind shared prefixes, sm_100a: the step's rows sorted by the prefix
// they read, and the writer that norms and rotates Q and K on the way (the
// attention is that of batch_tiles.cu, batch_few.cu and batch_join.cu).
//
// A prefix is a request that has none itself; e(b) is the one that request b
// reads, n(b) the request's rows.  Rows are listed by prefix, then by row, so
// the place of request b's first row is the sum of n(b') over the requests with
// (e(b'), b') < (e(b), b).  A warp has one request and compares it with all R (no
// request waits for another's sums); a step's bytes are nothing beside the launch.
// Measured: 3.6 us for 66 requests of 64 rows, 12.3 us for 2,072 of 21,130: the latency of
// the loads that depend on one another.  (Eight threads a request: 28 us for the latter.)
#include "batch_common.cuh"
#include "nvfp4_quant.cuh"

namespace qwz {

namespace {

constexpr int kShReq = 32;              // requests of a CTA, a warp each
constexpr int kShThreads = kShReq * 32;
constexpr int kShTile = 4096;           // requests in shared memory at a time

// The prefix that request b reads: one that exists, is another and has none itself, and
// whose rows, if it has any in this step, were not denied (they would be its tokens).
QWZ_DEVINL int share_prefix(const BatchShareParams& p, int b) {
  const int g = __ldg(p.prefix_of + b);
  if (g < 0) return -1;
  if (g < p.requests && g != b && __ldg(p.prefix_of + g) < 0 &&
      (__ldg(p.kv_lens + g) > 0 || __ldg(p.cu_rows + g + 1) <= __ldg(p.cu_rows + g)))
    return g;
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
  __shared__ int2 tile[kShTile];        // (prefix, rows; -1, 0: the request reads none or has no rows)
  griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int b = blockIdx.x * kShReq + (tid >> 5);
  // positions from the prefix's start (their loads are on their way during the rest)
  // (64 bits: a step more than the last row may pass 32)
  for (long long t = blockIdx.x * kShThreads + tid; t < p.rows; t += gridDim.x * kShThreads) {
    const int r = __ldg(p.request_of + t);
    int pos = p.positions[t];
    if (r >= 0 && r < p.requests) {
      const int g = share_prefix(p, r);
      if (g >= 0) pos += max(__ldg(p.kv_lens + g), 0);
    }
    p.positions_out[t] = pos;
  }
  if (blockIdx.x * kShReq >= p.requests && blockIdx.x > 0) return;
  const int key = b < p.requests ? share_prefix(p, b) : -1;
  int before = 0, of_lower = 0, readers = 0, reader = -1, total = 0;
  for (int t0 = 0; t0 < p.requests; t0 += kShTile) {
    const int n = min(kShTile, p.requests - t0);
    __syncthreads();
    for (int i = tid; i < n; i += kShThreads) {
      int lo;
      const int rows = share_rows(p, t0 + i, lo), g = share_prefix(p, t0 + i);
      tile[i] = g >= 0 && rows > 0 ? make_int2(g, rows) : make_int2(0x7fffffff, 0);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = lane; i < n; i += 32) {
      const int2 o = tile[i];
      total += o.y;
      before += o.x < key || (o.x == key && t0 + i < b) ? o.y : 0;
      of_lower += o.x < b ? o.y : 0;
      readers += o.x == b ? 1 : 0;
      reader = o.x == b ? t0 + i : reader;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    of_lower += __shfl_xor_sync(0xffffffffu, of_lower, o);
    readers += __shfl_xor_sync(0xffffffffu, readers, o);
    reader = max(reader, __shfl_xor_sync(0xffffffffu, reader, o));
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (b < p.requests) {
    if (lane == 0) {
      p.reads[b] = key;
      p.alone[b] = readers == 1 ? reader : -1;
      p.cu_shared[b] = of_lower;
      if (b == 0) p.cu_shared[p.requests] = total;
    }
    if (key >= 0) {
      int lo;
      const int n = share_rows(p, b, lo);
      for (long long i = lane; i < n && before + i >= 0 && before + i < p.rows; i += 32) p.shared_rows[before + i] = (int)(lo + i);
    }
  }
  // the places behind the last row
  const int ctas = (p.requests + kShReq - 1) / kShReq;
  for (long long t = max(total, 0) + blockIdx.x * kShThreads + tid; t < p.rows; t += ctas * kShThreads) p.shared_rows[t] = -1;
  griddep_launch_dependents();
}

cudaError_t launch_batch_share(const BatchShareParams& p, int sms, cudaStream_t stream) {
  const int by_request = (p.requests + kShReq - 1) / kShReq;
  const int by_row = (int)min((p.rows + kShThreads - 1LL) / kShThreads, (long long)sms);
  return launch_pdl(batch_share_kernel, dim3(max(max(by_request, by_row), 1)), dim3(kShThreads), 0, stream, p);
}

// ---------------------------------------------------------------------------
// Norm, rotation and quantisation of a step's rows.
//
//   x' = x w / sqrt(mean(x^2) + eps)                      (with a weight)
//   (y_i, y_j) = (x'_i cos a - x'_j sin a, x'_j cos a + x'_i sin a),  a = position * inv_freq_i
// with j = i + freqs, or the pairs (2i, 2i + 1); dims from 2 freqs on keep x'.
// q_out is y rounded once.  K's y goes to the quantiser without a rounding in
// between: E4M3 scales and E2M1 codes are those of the exact y, up to the error of
// 64 bits, so they do not depend on how 32 bits round next to a border.  They are made
// from 32 bits and an error bound, and again from 64 where a border is inside it (a few
// groups of heads in a hundred).  Angles are taken in 64 bits: 32 leave 0.06 radians of a position
// of 10^6.
//
// Q's y is made in 32 bits; BF16 heads whose squares 32 bits do not hold are left for 64.
//
// Instructions bound it for long steps (issue slots 57 %, DRAM 41 %).  Measured, GPU times:
// 16,384 rows of 24/4/256 in BF16, a quarter of the dims turned, with norm and held values,
// 148 us (57 % of the measured copy bandwidth); 5,001 rows of 14/2/64 12.0 us; 448 rows of
// 32/8/128 8.1 us; 16 rows of 24/4/256 4.5 us, less than the call costs the host.  Forms that
// were slower on the first, while it took 145 us: all of K in 64 bits with 8 dims a lane for
// Q, whose pairs' other dims came by shuffles, 214 us; the same with factors made once a row,
// 187 us; CTAs of 256 threads, two an SM 160 us, three 151 us.
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
// numbers that x stands for: 16-bit ones, or (ODD) what was rounded to odd.  16-bit
// numbers need no care: of 11 bits, they and their quotients are borders or keep 2^-12
// away from them.
template <bool ODD>
QWZ_DEVINL void quantise8(const float (&x)[8], uint32_t& code, uint32_t& sbits) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  float q6 = __fdiv_rn(amax, 6.f);
  if constexpr (ODD) q6 = odd_of(q6, __fmaf_rn(-q6, 6.f, amax));
  uint32_t pair, s2, unused;
  asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n cvt.u32.u16 %0, t;\n}\n" : "=r"(pair) : "f"(q6), "f"(0.f));
  sbits = pair;  // (the high one is 0)
  e4m3x4_to_f16x2x2(pair, s2, unused);
  const float s = InTraits<__half>::to_float2(s2).x;
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
        y[e] = __fmaf_rn(__fmaf_rn(-q, s, c), r, q);  // c / s, correctly rounded (Markstein, as in batch_tables.cu)
        if constexpr (ODD) y[e] = odd_of(y[e], __fmaf_rn(-y[e], s, c));
      }
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

// (x0, x1) * (a0, a1) + (c0, c1) in one instruction.
QWZ_DEVINL void fma_pair(float& d0, float& d1, float x0, float x1, float a0, float a1, float c0, float c1) {
  asm("{\n .reg .b64 x, a, c;\n mov.b64 x, {%2, %3};\n mov.b64 a, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 x, x, a, c;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d0), "=f"(d1)
      : "f"(x0), "f"(x1), "f"(a0), "f"(a1), "f"(c0), "f"(c1));
}
// Whether squares of T's numbers need more than 32 bits' range.
template <typename T>
constexpr bool kWide = !std::is_same<T, __half>::value;
QWZ_DEVINL float rsqrt_of(float x) { return rsqrtf(x); }
QWZ_DEVINL double rsqrt_of(double x) { return rsqrt(x); }
QWZ_DEVINL float shfl_xor_any(float x, int o) { return __shfl_xor_sync(0xffffffffu, x, o); }
QWZ_DEVINL double shfl_xor_any(double x, int o) { return __shfl_xor_sync(0xffffffffu, x, o); }

// A lane's two chunks of eight dims of a Q head, D / 16 lanes a head.  Where the pairs
// are (i, i + freqs) a turning lane has both of a pair, so no lane needs another's dims.
// y0 = x0 a0 + p0 b0, y1 = x1 a1 + p1 b1 with the pairs' other dims p, the cosines, sines
// and weights in a and b, made once for all heads of a row.
struct TurnQ {
  float a[2][8], b[2][8];
  int chunk[2];
  bool turns;  // (both chunks or neither: freqs is a multiple of 8)

  QWZ_DEVINL void set(int l, const float* weight, int freqs, bool neighbours, const float2* cos_sin) {
    const int half = freqs / 8;
    const bool both = !neighbours && l < half;
    chunk[0] = both ? l : 2 * l;
    chunk[1] = both ? l + half : 2 * l + 1;
    turns = neighbours ? l < freqs / 8 : both;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[k][i] = weight != nullptr ? __ldg(weight + 8 * chunk[k] + i) : 1.f;
        b[k][i] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w0 = a[0][i], w1 = a[1][i];
      if (both) {
        const float2 t = cos_sin[8 * l + i];
        a[0][i] = t.x * w0;
        a[1][i] = t.x * w1;
        b[0][i] = -t.y * w1;
        b[1][i] = t.y * w0;
      }
    }
    if (neighbours && turns) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 t = cos_sin[4 * chunk[k] + i / 2];
          const float w0 = a[k][i], w1 = a[k][i + 1];
          a[k][i] = t.x * w0;
          a[k][i + 1] = t.x * w1;
          b[k][i] = -t.y * w1;
          b[k][i + 1] = t.y * w0;
        }
    }
  }

  // False where 32 bits do not hold the head's squares (q_from_64; never in FP16).
  template <typename T, int LANES, bool NEIGHBOURS>
  QWZ_DEVINL bool apply(uint4 (&raw)[2], bool norm, float eps) const {
    float x[2][8], y[2][8];
    to_floats<T>(raw[0], x[0]);
    to_floats<T>(raw[1], x[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if (turns) {
          const float p0 = NEIGHBOURS ? x[k][i + 1] : x[1 - k][i], p1 = NEIGHBOURS ? x[k][i] : x[1 - k][i + 1];
          fma_pair(y[k][i], y[k][i + 1], p0, p1, b[k][i], b[k][i + 1], 0.f, 0.f);
          fma_pair(y[k][i], y[k][i + 1], x[k][i], x[k][i + 1], a[k][i], a[k][i + 1], y[k][i], y[k][i + 1]);
        } else {  // (0 times an infinity is no 0)
          y[k][i] = x[k][i] * a[k][i];
          y[k][i + 1] = x[k][i + 1] * a[k][i + 1];
        }
      }
    float r = 1.f;
    if (norm) {
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 8; i += 2) fma_pair(s0, s1, x[k][i], x[k][i + 1], x[k][i], x[k][i + 1], s0, s1);
      float sum = s0 + s1;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      r = rsqrtf(sum / (16 * LANES) + eps);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      T h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = InTraits<T>::from_float(y[k][i] * r);
      raw[k] = *reinterpret_cast<const uint4*>(h);
    }
    return !kWide<T> || (r > 1e-15f && r < 1e15f);
  }
};

// One Q head (where `mine`) of a row from 64 bits, rounded once.
template <typename T, int D>
__device__ __noinline__ void q_from_64(const BatchRotateParams& p, long long row, int head, bool mine, const double2* cos_sin) {
  constexpr int kLanes = D / 16;
  const int l = threadIdx.x % kLanes, half = p.freqs / 8;
  const bool neighbours = p.neighbours != 0, both = !neighbours && l < half;
  const int c[2] = {both ? l : 2 * l, both ? l + half : 2 * l + 1};
  double x[2][8], sum = 0.0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (mine) raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + row * p.q_stride + head * D + 8 * c[k]);
    to_floats<T>(raw, x[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[k][i] * x[k][i];
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) sum += shfl_xor_any(sum, o);
  const double r = rsqrt_of(sum / D + (double)p.eps);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[k][i] = x[k][i] * r * __ldg(p.q_weight + 8 * c[k] + i);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    T h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double y = x[k][i];
      if (both) {
        const double2 t = cos_sin[8 * l + i];
        y = y * t.x + x[1 - k][i] * (k == 0 ? -t.y : t.y);
      } else if (neighbours && c[k] < p.freqs / 4) {
        const double2 t = cos_sin[4 * c[k] + i / 2];
        y = y * t.x + x[k][i ^ 1] * (i % 2 == 0 ? -t.y : t.y);
      }
      h[i] = InTraits<T>::from_float(float_odd(y));
    }
    if (mine)
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out) + row * p.q_out_stride + head * D + 8 * c[k]) =
          *reinterpret_cast<const uint4*>(h);
  }
}

// The eight dims `c` of a K head in F's precision, D / 8 lanes a head (all lanes of the
// warp take part).
template <typename T, int LANES, typename F, typename F2>
QWZ_DEVINL void turn_k(const uint4& raw, int c, const float* weight, float eps, int freqs, bool neighbours,
                       const F2* cos_sin, F (&y)[8]) {
  const int half = freqs / 8, lane = threadIdx.x & 31;
  const bool turns = c < 2 * half, low = c < half;
  const int other = turns && !neighbours ? (low ? c + half : c - half) : c, from = lane - c + other;
  uint4 w;
  w.x = __shfl_sync(0xffffffffu, raw.x, from);
  w.y = __shfl_sync(0xffffffffu, raw.y, from);
  w.z = __shfl_sync(0xffffffffu, raw.z, from);
  w.w = __shfl_sync(0xffffffffu, raw.w, from);
  F x[8];
  to_floats<T>(raw, x);
  F r = 1;
  if (weight != nullptr) {
    F sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
    for (int k = LANES / 2; k > 0; k >>= 1) sum += shfl_xor_any(sum, k);
    r = rsqrt_of(sum / (8 * LANES) + (F)eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * __ldg(weight + 8 * c + i);
  }
  if (!turns) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  } else if (neighbours) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const F2 t = cos_sin[4 * c + i / 2];
      y[i] = x[i] * t.x - x[i + 1] * t.y;
      y[i + 1] = x[i + 1] * t.x + x[i] * t.y;
    }
  } else {
    F o[8];
    to_floats<T>(w, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const F2 t = cos_sin[8 * (low ? c : c - half) + i];
      if (weight != nullptr) o[i] = o[i] * r * __ldg(weight + 8 * other + i);
      y[i] = low ? x[i] * t.x - o[i] * t.y : x[i] * t.x + o[i] * t.y;
    }
  }
}

// Code word and scale byte of a K head's eight dims from 64 bits.
template <typename T, int LANES>
__device__ __noinline__ void k_from_64(const uint4 raw, int c, const float* weight, float eps, int freqs, bool neighbours,
                                       const double2* cos_sin, uint32_t& code, uint32_t& sbits) {
  double y[8];
  turn_k<T, LANES, double, double2>(raw, c, weight, eps, freqs, neighbours, cos_sin, y);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = float_odd(y[i]);
  quantise8<true>(x, code, sbits);
}

// The same from 32 bits; false where a border lies inside the error bound.
//
// Errors in parts of 2^-24 of |a| + |b|, the two terms of a dim, which is at most twice the
// head's largest |x'|: cosine or sine, product and sum 3; with a norm also half of the sum of
// squares' 14 and of eps' 1, the root's 4 (two places), two products: 16.5.  So 6 x 2^-24 =
// 3.6e-7 of max |x'|, and 33 x 2^-24 = 2.0e-6.  A head without norm has its other dims
// exactly.  The quotient adds 2^-24 of at most 6.
template <typename T, int LANES>
QWZ_DEVINL bool k_from_32(const uint4& raw, int c, const float* weight, float w_max, float eps, int freqs,
                          bool neighbours, const float2* cos_sin, uint32_t& code, uint32_t& sbits) {
  float y[8];
  turn_k<T, LANES, float, float2>(raw, c, weight, eps, freqs, neighbours, cos_sin, y);
  float most = 0.f, sum = 0.f, amax = 0.f;
  {
    float x[8];
    to_floats<T>(raw, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      most = fmaxf(most, fabsf(x[i]));
      sum += x[i] * x[i];
      amax = fmaxf(amax, fabsf(y[i]));
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  bool fine = true;
  if (weight != nullptr) {
    const float mean = sum / (8 * LANES) + eps;
    fine = mean > 1e-30f && mean < 1e30f;  // (squares that 32 bits hold)
    most *= w_max * rsqrtf(mean) * 1.0001f;
  }
  const float err = weight != nullptr ? most * 2.1e-6f : c < freqs / 4 ? most * 3.8e-7f : 0.f;
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  const float err2 = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, 1));
  // the scale of the least and of the largest that amax can be (equal where it is exact)
  const float q6 = __fdiv_rn(amax, 6.f), slack = err2 > 0.f ? err2 + q6 * 2.4e-7f : 0.f;
  uint32_t pair, s2, unused;
  asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n cvt.u32.u16 %0, t;\n}\n"
      : "=r"(pair)
      : "f"(q6 - slack), "f"(q6 + slack));
  sbits = pair & 0xffu;
  fine = fine && sbits == pair >> 8 && most < 1e30f;
  e4m3x4_to_f16x2x2(sbits, s2, unused);
  const float s = InTraits<__half>::to_float2(s2).x;
  code = 0u;
  uint32_t high = 0u;
  if (s > 0.f) {
    const float r = __frcp_rn(s), d = err > 0.f ? err * r * 1.0001f + 6e-7f : 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float z[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float q = __fmul_rn(y[i + e], r);
        z[e] = __fmaf_rn(__fmaf_rn(-q, s, y[i + e]), r, q);  // y / s, correctly rounded (Markstein)
      }
      asm("{\n .reg .b8 t, u;\n cvt.rn.satfinite.e2m1x2.f32 t, %3, %2;\n cvt.rn.satfinite.e2m1x2.f32 u, %5, %4;\n"
          " cvt.u32.u8 %0, t;\n cvt.u32.u8 %1, u;\n}\n"
          : "=r"(pair), "=r"(unused)
          : "f"(z[0] - d), "f"(z[1] - d), "f"(z[0] + d), "f"(z[1] + d));
      code |= pair << (4 * i);
      high |= unused << (4 * i);
    }
    const uint32_t m = code & 0x77777777u, some = (m | (m >> 1) | (m >> 2)) & 0x11111111u;
    code = m | (code & (some << 3));  // a zero magnitude carries no sign
    const uint32_t mh = high & 0x77777777u, someh = (mh | (mh >> 1) | (mh >> 2)) & 0x11111111u;
    fine = fine && code == (mh | (high & (someh << 3)));
  }
  return fine;
}

constexpr int kRotThreads = 128;

}  // namespace

// A CTA has ROWS rows: their angles' cosines and sines first, then tasks of one warp
// each: q_units warp loads of a row's Q heads, kv_units of its K heads, of its V heads.
// grid.y CTAs share the tasks of the same rows.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kRotThreads, 5) batch_rotate_kernel(const __grid_constant__ BatchRotateParams p, int q_units, int kv_units) {
  constexpr int kLanes = D / 8, kHeads = 32 / kLanes;     // K, V: lanes a head, heads a warp
  constexpr int kQLanes = D / 16, kQHeads = 32 / kQLanes;  // Q
  constexpr int kLoads = 2;                                // warp loads of Q that are under way together
  __shared__ double2 table[ROWS][128];                     // (cos, sin) of a row's angles
  __shared__ float2 narrow[ROWS][128];
  constexpr int kWords = kRotMaxHeads / 32;
  __shared__ uint32_t late[kWide<T> ? ROWS * kWords : 1];  // a bit a Q head that q_from_64 does at the end
  __shared__ int some_late;
  griddep_wait();
  const BatchAppendParams& a = p.kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool neighbours = p.neighbours != 0;
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
    table[r][f] = make_double2(co, s);
    narrow[r][f] = make_float2((float)co, (float)s);
  }
  if (tid == 0) some_late = 0;
  if constexpr (kWide<T>)  // (the words of heads that there are)
    for (int i = tid; i < ROWS * ((p.q_heads + 31) / 32); i += kRotThreads) late[i % ROWS * kWords + i / ROWS] = 0u;
  __syncthreads();
  const int q_tasks = (p.q_heads + q_units * kQHeads - 1) / (q_units * kQHeads);
  const int kv_tasks = (a.kv_heads + kv_units * kHeads - 1) / (kv_units * kHeads), per_row = q_tasks + 2 * kv_tasks;
  for (int task = blockIdx.y * (kRotThreads / 32) + warp; task < rows * per_row; task += gridDim.y * (kRotThreads / 32)) {
    const int r = task / per_row, v = task % per_row;
    const long long row = row0 + r;
    if (v < q_tasks) {
      const int l = lane % kQLanes, sub = lane / kQLanes;
      const int first = v * q_units * kQHeads, end = min(p.q_heads, first + q_units * kQHeads);
      TurnQ turn;
      turn.set(l, p.q_weight, p.freqs, neighbours, narrow[r]);
      const T* src = reinterpret_cast<const T*>(p.q) + row * p.q_stride;
      T* dst = reinterpret_cast<T*>(p.q_out) + row * p.q_out_stride;
#pragma unroll 1
      for (int h0 = first; h0 < end; h0 += kLoads * kQHeads) {
        uint4 raw[kLoads][2];
        bool fine[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int head = h0 + u * kQHeads + sub;
            raw[u][k] = make_uint4(0u, 0u, 0u, 0u);
            if (head < end) raw[u][k] = *reinterpret_cast<const uint4*>(src + head * D + 8 * turn.chunk[k]);
          }
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          fine[u] = neighbours ? turn.template apply<T, kQLanes, true>(raw[u], p.q_weight != nullptr, p.eps)
                               : turn.template apply<T, kQLanes, false>(raw[u], p.q_weight != nullptr, p.eps);
          const int head = h0 + u * kQHeads + sub;
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (fine[u] && head < end) *reinterpret_cast<uint4*>(dst + head * D + 8 * turn.chunk[k]) = raw[u][k];
        }
        if constexpr (kWide<T>)
          if (!(fine[0] && fine[1])) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
              const int head = h0 + u * kQHeads + sub;
              if (!fine[u] && head < end) {
                atomicOr(late + r * kWords + head / 32, 1u << head % 32);
                some_late = 1;
              }
            }
          }
      }
      continue;
    }
    const int c = lane % kLanes, sub = lane / kLanes;
    const bool is_k = v < q_tasks + kv_tasks;
    const int first = (v - q_tasks - (is_k ? 0 : kv_tasks)) * kv_units * kHeads, end = min(a.kv_heads, first + kv_units * kHeads);
    const int slot = __ldg(a.slots + row);
    const bool stored = slot >= 0 && (slot >> 8) < a.num_pages;
    if (slot >= 0 && !stored) flag_error(kErrSlotRange);
    const T* src = reinterpret_cast<const T*>(is_k ? a.k : a.v) + row * (is_k ? a.k_stride : a.v_stride) + sub * D + 8 * c;
    float w_max = 1.f;
    if (is_k && p.k_weight != nullptr) {
      w_max = 0.f;
      for (int i = 0; i < 8; ++i) w_max = fmaxf(w_max, fabsf(__ldg(p.k_weight + 8 * c + i)));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) w_max = fmaxf(w_max, __shfl_xor_sync(0xffffffffu, w_max, o));
    }
    uint4 next = first + sub < end ? *reinterpret_cast<const uint4*>(src + first * D) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
    for (int h0 = first; h0 < end; h0 += kHeads) {
      const int head = h0 + sub;
      const uint4 raw = next;
      next = make_uint4(0u, 0u, 0u, 0u);
      if (head + kHeads < end) next = *reinterpret_cast<const uint4*>(src + (h0 + kHeads) * D);
      uint32_t code, sbits;
      if (is_k) {
        const bool fine = k_from_32<T, kLanes>(raw, c, p.k_weight, w_max, p.eps, p.freqs, neighbours, narrow[r], code, sbits);
        if (!__all_sync(0xffffffffu, fine))
          k_from_64<T, kLanes>(raw, c, p.k_weight, p.eps, p.freqs, neighbours, table[r], code, sbits);
      } else {
        float x[8];
        to_floats<T>(raw, x);
        quantise8<false>(x, code, sbits);
      }
      if (head >= end) continue;
      if (stored) {
        const size_t at = (size_t)slot * a.kv_heads + head;
        reinterpret_cast<uint32_t*>(is_k ? a.k_cache : a.v_cache)[at * kLanes + c] = code;
        if ((c & 1) == 0) (is_k ? a.k_scales : a.v_scales)[at * (D / 16) + c / 2] = (uint8_t)sbits;
      }
      void* held = is_k ? a.k_held : a.v_held;
      if (held != nullptr)
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(held) + (row * a.kv_heads + head) * D + 8 * c) = held8<T>(code, sbits);
    }
  }
  if constexpr (kWide<T>) {
    // (Here, where no task holds registers: in the loop, inlined or called, the path made them
    // spill, 156 to 162 us for 16,384 rows of 24/4/256 against 149 so and 144 without it.)
    __syncthreads();
    if (some_late == 0) return;
    const int steps = (p.q_heads + kQHeads - 1) / kQHeads;
#pragma unroll 1
    for (int i = warp; i < rows * steps; i += kRotThreads / 32) {
      const int r = i / steps, head = i % steps * kQHeads + lane / kQLanes;
      const bool mine = head < p.q_heads && (late[r * kWords + head / 32] >> head % 32 & 1u) != 0u;
      if (__any_sync(0xffffffffu, mine)) q_from_64<T, D>(p, row0 + r, head, mine, table[r]);
    }
  }
  griddep_launch_dependents();
}

namespace {

template <typename T, int D>
cudaError_t launch_rotate(const BatchRotateParams& p, cudaStream_t stream) {
  constexpr int kQHeads = 512 / D, kHeads = 256 / D;  // a warp load's
  const int rows = (int)p.kv.rows, kv_heads = p.kv.kv_heads;
  const int tasks = (p.q_heads + kQHeads - 1) / kQHeads + 2 * ((kv_heads + kHeads - 1) / kHeads);
  // Few rows: short tasks, a row's over several CTAs, each with the row's angles.  Against the form for many,
  // us: 24/4/256 with norm 512 rows 14.1 and 15.6, 700 17.6 and 17.4, 800 20.0 and 17.5, 1,024 24.6 and 17.9;
  // 32/8/128 9.4 and 11.2, 12.1 and 12.4, 13.9 and 12.4, 16.6 and 12.5; 64/8/128 13.5 and 18.0, 17.2 and 19.2,
  // 19.4 and 19.2, 24.0 and 19.3; 48/8/256 with norm 24.6 and 38.4, 32.6 and 41.9, 36.8 and 41.2, 46.8 and 41.2;
  // 14/2/64 3.8 and 5.3, 4.1 and 5.7, 6.1 and 5.8, 7.1 and 6.4
  if (rows <= 700) {
    return launch_pdl(batch_rotate_kernel<T, D, 1>, dim3((unsigned)rows, (tasks + 3) / 4), dim3(kRotThreads), 0, stream, p,
                      1, 1);
  }
  // Many: the factors of Q are made once for 12 loads (2,048 and 16,384 rows of 24/4/256 in BF16 with norm and
  // held values: 25.4 and 159 us with 4, 29.8 and 171 with 6, 22.9 and 148 with 12); 4 rows a CTA (2 rows 29.4
  // and 190, 8 rows 34.6 and 160).  More than 24 heads of 256, 48 of 128 or 96 of 64 are a second task of a row,
  // which falls to the same warp for each of the four rows: 16,384 rows of 64/8/128 199 us, 156 with 6 loads.
  constexpr int kRows = 4;
  return launch_pdl(batch_rotate_kernel<T, D, kRows>, dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(kRotThreads), 0,
                    stream, p, 12, (kv_heads + kHeads - 1) / kHeads);
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
