// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits (sm_100a): what a verify step or a sampler takes from the logits
// that follow the attention.  For a row x of V logits, M = max x:
//   s = sum e^(x - M),  t = sum (x - M) e^(x - M)
//   log p(id) = (x_id - M) - ln s,  H = ln s - t / s,
//   top K by (value, then lowest index).
//
// One pass over the logits; bound by HBM (and, for 16-bit logits, by the
// exponentials: 16 a cycle and SM allow 1.4 times the rate at which the logits
// arrive).  A CTA streams a part of one row, four 16-byte loads a thread in
// flight while the four before them are summed; the sums are FP32, relative to
// a maximum of the thread's own that moves only when a logit exceeds it by more
// than 8, so nothing waits inside the loop.  Top K: the K-th largest of 64 group
// maxima (four threads each) of the part's first tile is a lower bound tau of the
// part's K-th largest value; whatever reaches it (about K times the number of
// tiles) goes to a list in shared memory that is ranked by counting at the end.
// A list that overflows is made again with the tau of the whole part's maxima,
// and where equal values overflow that, K rounds of a maximum find the K.  A
// second kernel, one CTA a row, joins the parts in order; no result depends on
// the order of atomics.
#include "qwz_common.cuh"
#include "batch_kernels.h"
#include "qwz_kernels.h"

#include <math_constants.h>

namespace qwz {

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpVecs = 4;                              // 16-byte loads of a tile a thread
constexpr int kLpTileVecs = kLpThreads * kLpVecs;       // 16 KB
constexpr int kLpCand = 1024;                           // candidates ranked by counting
constexpr int kLpParts = 16 * 148;                      // parts of all rows that a launch aims at
constexpr float kLpMove = 8.f;                          // a thread's reference moves past this
constexpr int kLpMergeCand = 1024;

template <typename T>
struct LpTraits;
template <>
struct LpTraits<float> {
  static constexpr int E = 4;
  static constexpr uint32_t kAbsent = 0xff800000u;  // -inf
  static QWZ_DEVINL void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  static QWZ_DEVINL float one(const float* p) { return *p; }
};
QWZ_DEVINL uint32_t lp_max2(uint32_t a, uint32_t b, __half) {
  const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
QWZ_DEVINL uint32_t lp_max2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 m =
      __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T, uint32_t ABSENT>
struct Lp16 {
  static constexpr int E = 8;
  static constexpr uint32_t kAbsent = ABSENT;
  static QWZ_DEVINL void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = InTraits<T>::to_float2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static QWZ_DEVINL float one(const T* p) {
    return InTraits<T>::to_float2((uint32_t)*reinterpret_cast<const uint16_t*>(p)).x;
  }
};
template <>
struct LpTraits<__half> : Lp16<__half, 0xfc00fc00u> {};
template <>
struct LpTraits<__nv_bfloat16> : Lp16<__nv_bfloat16, 0xff80ff80u> {};

// Orders by value, then by lowest index; NaN below -inf, 0 below everything.
QWZ_DEVINL unsigned long long lp_key(float x, uint32_t idx) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 counts as +0
  const uint32_t u = x != x ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xffffffffu - idx);
}
QWZ_DEVINL float lp_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0) return CUDART_NAN_F;
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
QWZ_DEVINL uint32_t lp_index(unsigned long long key) { return 0xffffffffu - (uint32_t)key; }

QWZ_DEVINL float max_nan(float a, float b) {  // NaN wins
  float d;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

constexpr float kLog2eF = 1.4426950408889634f;

// (d0, d1) += (a0, a1) * (b0, b1)
QWZ_DEVINL void lp_ffma2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  uint64_t d;
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n mov.b64 c, {%5, %6};\n"
      " fma.rn.f32x2 %0, a, b, c;\n}\n"
      : "=l"(d)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(d0), "f"(d1));
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(d0), "=f"(d1) : "l"(d));
}

// Bytes of one chunk's record: m, s, t, (pad), K keys.
QWZ_DEVINL size_t lp_record(int top) { return 16 + 8 * (size_t)top; }

}  // namespace

// The K-th largest (1 <= K <= 64) of 64 values in shared memory, by one warp.
QWZ_DEVINL void lp_kth(const float* v64, int K, int lane, float* out) {
  const float a = v64[lane], b = v64[lane + 32];
  int ra = 0, rb = 0;
#pragma unroll 4
  for (int i = 0; i < 64; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(v64 + i);
    const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ra += (w[j] > a || (w[j] == a && i + j < lane)) ? 1 : 0;
      rb += (w[j] > b || (w[j] == b && i + j < lane + 32)) ? 1 : 0;
    }
  }
  if (ra == K - 1) *out = a;
  if (rb == K - 1) *out = b;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) lp_part_kernel(const __grid_constant__ LogprobParams p) {
  using L = LpTraits<T>;
  constexpr int E = L::E;
  __shared__ float red[3][kLpThreads / 32];
  __shared__ __align__(16) float gmax[64];
  __shared__ unsigned long long cand[kLpCand];
  __shared__ unsigned long long best;
  __shared__ float tau_s;
  __shared__ int n_cand;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / p.chunks, part = blockIdx.x % p.chunks;
  const int K = p.top;
  griddep_wait();

  const T* x0 = reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(x0) / sizeof(T)) % E);  // elements past a 16-byte boundary
  const int v0 = part * p.chunk_tiles * kLpTileVecs;
  const int vecs = (p.vocab + skew + E - 1) / E;
  const int tiles = max(0, min(p.chunk_tiles, (vecs - v0 + kLpTileVecs - 1) / kLpTileVecs));
  // places of the part
  const int first = max(0, v0 * E - skew), last_pos = min(p.vocab, (v0 + p.chunk_tiles * kLpTileVecs) * E - skew);

  // this thread's vectors of a tile, absent places as -inf
  auto load = [&](int tile, uint4(&raw)[kLpVecs]) {
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      const int pos = (v0 + tile * kLpTileVecs + i * kLpThreads + tid) * E - skew;
      if (pos >= 0 && pos + E <= p.vocab) {
        raw[i] = __ldg(reinterpret_cast<const uint4*>(x0 + pos));
      } else {
        raw[i] = make_uint4(L::kAbsent, L::kAbsent, L::kAbsent, L::kAbsent);
        if (pos < p.vocab && pos > -E) {  // an end of the row
          T e[E];
          *reinterpret_cast<uint4*>(e) = raw[i];
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (pos + j >= 0 && pos + j < p.vocab) e[j] = x0[pos + j];
          raw[i] = *reinterpret_cast<uint4*>(e);
        }
      }
    }
  };
  auto vec_max = [&](const uint4& v) {
    float x[E], m = -CUDART_INF_F;
    if constexpr (E == 8) {
      const uint32_t h = lp_max2(lp_max2(v.x, v.y, T()), lp_max2(v.z, v.w, T()), T());
      const float2 f = InTraits<T>::to_float2(h);
      m = fmaxf(f.x, f.y);  // NaN loses
      m = fmaxf(m, -CUDART_INF_F);
    } else {
      L::unpack(v, x);
#pragma unroll
      for (int j = 0; j < E; ++j) m = fmaxf(m, x[j]);
    }
    return m;
  };
  // group maxima of `v` and the K-th largest of them, for the whole CTA
  auto threshold = [&](float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
    if ((lane & 3) == 0) gmax[tid >> 2] = v;
    if (tid == 0) n_cand = 0;
    __syncthreads();
    if (warp == 0) lp_kth(gmax, K, lane, &tau_s);
    __syncthreads();
    return tau_s;
  };
  // Candidates of a vector: at or above tau; where tau is -inf (fewer than K
  // groups hold anything above it), all that is above -inf and the first K
  // places (the lowest indices).
  auto collect = [&](const uint4& v, int pos, float tau) {
    float x[E];
    L::unpack(v, x);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const bool take = tau == -CUDART_INF_F ? x[j] > -CUDART_INF_F || pos + j < first + K : x[j] >= tau;
      if (take && pos + j >= first && pos + j < last_pos) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < kLpCand) cand[at] = lp_key(x[j], (uint32_t)(pos + j));
      }
    }
  };

  uint4 raw[kLpVecs];
  load(0, raw);
  float r = -CUDART_INF_F, tmax = -CUDART_INF_F, tau = CUDART_INF_F;
  if (K > 0) {
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) tmax = fmaxf(tmax, vec_max(raw[i]));
    tau = threshold(tmax);
  }
  float s = 0.f, t = 0.f, s1 = 0.f, t1 = 0.f;
  for (int tile = 0; tile < tiles; ++tile) {
    uint4 cur[kLpVecs];
    float vm[kLpVecs], m = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) cur[i] = raw[i];
    if (tile + 1 < tiles) load(tile + 1, raw);
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      vm[i] = vec_max(cur[i]);
      m = fmaxf(m, vm[i]);
    }
    if (m > r + kLpMove || (r == -CUDART_INF_F && m > r)) {  // a new reference
      const float d = r - m, w = r == -CUDART_INF_F ? 0.f : exp2_approx(d * kLog2eF);
      t = r == -CUDART_INF_F ? t : w * (t + t1 + d * (s + s1));  // (sums without a reference are 0 or NaN)
      s = r == -CUDART_INF_F ? s : w * (s + s1);
      s1 = t1 = 0.f;
      r = m;
    }
    tmax = fmaxf(tmax, m);
    const float mu = r == -CUDART_INF_F ? 0.f : r;
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      float x[E];
      L::unpack(cur[i], x);
#pragma unroll
      for (int j = 0; j < E; j += 2) {  // packed FP32 pairs
        pf_fadd2(x[j], x[j + 1], -mu, -mu);
        const float d0 = max_nan(x[j], -1000.f), d1 = max_nan(x[j + 1], -1000.f);  // -inf: e = 0 and d e = 0
        float e0, e1;
        pf_ffma2(e0, e1, d0, d1, kLog2eF, 0.f);
        e0 = exp2_approx(e0);
        e1 = exp2_approx(e1);
        pf_fadd2(s, s1, e0, e1);
        lp_ffma2(t, t1, d0, d1, e0, e1);
      }
    }
    if (K > 0 && (m >= tau || tau == -CUDART_INF_F)) {
#pragma unroll 1
      for (int i = 0; i < kLpVecs; ++i) {
        const uint4 v = i == 0 ? cur[0] : i == 1 ? cur[1] : i == 2 ? cur[2] : cur[3];
        const float best_of = i == 0 ? vm[0] : i == 1 ? vm[1] : i == 2 ? vm[2] : vm[3];
        if (best_of >= tau || tau == -CUDART_INF_F)
          collect(v, (v0 + tile * kLpTileVecs + i * kLpThreads + tid) * E - skew, tau);
      }
    }
  }
  s += s1;
  t += t1;

  // the part's maximum, and the threads' sums relative to it
  float M = r;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
  M = red[0][0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 32; ++i) M = fmaxf(M, red[0][i]);
  if (r != -CUDART_INF_F) {
    const float d = r - M, w = exp2_approx(d * kLog2eF);
    t = w * (t + d * s);
    s = w * s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) {
    red[1][warp] = s;
    red[2][warp] = t;
  }
  __syncthreads();
  uint8_t* rec = reinterpret_cast<uint8_t*>(p.workspace) + ((size_t)row * p.chunks + part) * lp_record(K);
  if (tid == 0) {
    s = t = 0.f;
#pragma unroll
    for (int i = 0; i < kLpThreads / 32; ++i) {
      s += red[1][i];
      t += red[2][i];
    }
    float* f = reinterpret_cast<float*>(rec);
    f[0] = M;
    f[1] = s;
    f[2] = t;
  }
  if (K > 0) {
    if (n_cand > kLpCand) {  // (the same for all threads: the list is complete)
      __syncthreads();
      tau = threshold(tmax);
#pragma unroll 1
      for (int tile = 0; tile < tiles; ++tile) {
        load(tile, raw);
#pragma unroll 1
        for (int i = 0; i < kLpVecs; ++i) {
          const uint4 v = i == 0 ? raw[0] : i == 1 ? raw[1] : i == 2 ? raw[2] : raw[3];
          collect(v, (v0 + tile * kLpTileVecs + i * kLpThreads + tid) * E - skew, tau);
        }
      }
      __syncthreads();
    }
    const int n = n_cand;
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(rec + 16);
    if (n <= kLpCand) {
      for (int c = tid; c < max(n, K); c += kLpThreads) {
        if (c < n) {
          const unsigned long long mine = cand[c];
          int rank = 0;
          for (int i = 0; i < n; ++i) rank += cand[i] > mine ? 1 : 0;
          if (rank < K) keys[rank] = mine;
        } else {
          keys[c] = 0ull;  // a part with fewer than K elements
        }
      }
    } else {
      // many equal values: K rounds of the largest key below the last one
      unsigned long long last = ~0ull;
      for (int k = 0; k < K; ++k) {
        unsigned long long top = 0ull;
#pragma unroll 1
        for (int i = first + tid; i < last_pos; i += kLpThreads) {
          const unsigned long long key = lp_key(L::one(x0 + i), (uint32_t)i);
          if (key < last && key > top) top = key;
        }
        __syncthreads();
        if (tid == 0) best = 0ull;
        __syncthreads();
        atomicMax(&best, top);
        __syncthreads();
        last = best;
        if (tid == 0) keys[k] = last;
      }
    }
  }
  griddep_launch_dependents();
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) lp_merge_kernel(const __grid_constant__ LogprobParams p) {
  __shared__ unsigned long long cand[kLpMergeCand];
  __shared__ unsigned long long sorted[32];
  __shared__ float red[2][kLpThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x;
  const int K = p.top;
  griddep_wait();
  griddep_launch_dependents();
  const uint8_t* recs = reinterpret_cast<const uint8_t*>(p.workspace) + (size_t)row * p.chunks * lp_record(K);
  auto stat = [&](int c) { return reinterpret_cast<const float*>(recs + c * lp_record(K)); };

  float M = -CUDART_INF_F;
  for (int c = tid; c < p.chunks; c += kLpThreads) M = fmaxf(M, __ldcg(stat(c)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
  M = red[0][0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 32; ++i) M = fmaxf(M, red[0][i]);
  __syncthreads();
  float s = 0.f, t = 0.f;
  for (int c = tid; c < p.chunks; c += kLpThreads) {
    const float m = __ldcg(stat(c)), sc = __ldcg(stat(c) + 1), tc = __ldcg(stat(c) + 2);
    if (m == -CUDART_INF_F) {
      s += sc;  // 0, or NaN
      continue;
    }
    const float d = m - M, w = exp2_approx(d * kLog2eF);
    s += w * sc;
    t += w > 0.f ? w * (tc + d * sc) : 0.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) {
    red[0][warp] = s;
    red[1][warp] = t;
  }
  __syncthreads();
  s = t = 0.f;
#pragma unroll
  for (int i = 0; i < kLpThreads / 32; ++i) {
    s += red[0][i];
    t += red[1][i];
  }
  const float ln_s = logf(s);
  const bool none = M == -CUDART_INF_F && s == 0.f;  // no token is possible
  auto logprob = [&](float x) { return none ? (x != x ? x : -CUDART_INF_F) : (x - M) - ln_s; };

  if (tid == 0) {
    p.entropy[row] = none ? 0.f : ln_s - t / s;
    const long long id = p.ids64 ? __ldg(reinterpret_cast<const long long*>(p.ids) + row)
                                 : (long long)__ldg(reinterpret_cast<const int*>(p.ids) + row);
    float lp = 0.f;  // id < 0: no token
    if (id >= p.vocab) {
      flag_error(kErrSlotRange);
      lp = CUDART_NAN_F;
    } else if (id >= 0) {
      lp = logprob(LpTraits<T>::one(reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride + id));
    }
    p.logprob[row] = lp;
  }
  if (K == 0) return;

  // the best K so far, then as many chunks' lists as fit beside them
  int have = 0;
  const int lists = (kLpMergeCand - 32) / K;
  for (int c0 = 0; c0 < p.chunks; c0 += lists) {
    const int n_lists = min(lists, p.chunks - c0), n = have + n_lists * K;
    if (tid < have) cand[tid] = sorted[tid];
    for (int i = tid; i < n_lists * K; i += kLpThreads)
      cand[have + i] = __ldcg(reinterpret_cast<const unsigned long long*>(recs + (c0 + i / K) * lp_record(K) + 16) + i % K);
    __syncthreads();
    if (tid < K) sorted[tid] = 0ull;
    __syncthreads();
    for (int i = tid; i < n; i += kLpThreads) {
      const unsigned long long mine = cand[i];
      if (mine == 0ull) continue;
      int rank = 0;
      for (int j = 0; j < n && rank < K; ++j) rank += cand[j] > mine ? 1 : 0;
      if (rank < K) sorted[rank] = mine;
    }
    __syncthreads();
    have = K;
  }
  if (tid < K) {
    const unsigned long long key = sorted[tid];
    p.top_ids[(size_t)row * K + tid] = (int32_t)lp_index(key);
    p.top_logprobs[(size_t)row * K + tid] = logprob(lp_value(key));
  }
}

namespace {

int lp_tiles(int vocab, int itemsize) {
  const int e = 16 / itemsize;
  const long long vecs = ((long long)vocab + 2 * e - 2) / e;  // with the worst skew
  return (int)((vecs + kLpTileVecs - 1) / kLpTileVecs);
}

}  // namespace

// Parts of a row: about kLpParts of all rows (16 an SM, four rounds of the
// resident CTAs: 448 rows of 151,000 take five of four tiles), a tile at least.
void logprob_parts(int rows, int vocab, int itemsize, int* parts, int* tiles_each) {
  const int tiles = lp_tiles(vocab, itemsize);
  const int want = max(1, min(tiles, (kLpParts + rows - 1) / max(rows, 1)));
  *tiles_each = (tiles + want - 1) / want;
  *parts = (tiles + *tiles_each - 1) / *tiles_each;
}

// Records that any call of up to `rows` rows needs.
long long logprob_records(int rows, int vocab, int itemsize) {
  return min((long long)rows * lp_tiles(vocab, itemsize), (long long)kLpParts + rows);
}

size_t logprob_record_bytes(int top) { return 16 + 8 * (size_t)top; }

namespace {

template <typename T>
cudaError_t launch_lp(const LogprobParams& p, cudaStream_t stream) {
  cudaError_t e = launch_pdl(lp_part_kernel<T>, dim3((unsigned)p.chunks * p.rows), dim3(kLpThreads), 0, stream, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(lp_merge_kernel<T>, dim3(p.rows), dim3(kLpThreads), 0, stream, p);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobParams& p, int dtype, cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  switch (dtype) {
    case kDtypeF16: return launch_lp<__half>(p, stream);
    case kDtypeBF16: return launch_lp<__nv_bfloat16>(p, stream);
    default: return launch_lp<float>(p, stream);
  }
}

}  // namespace qwz
