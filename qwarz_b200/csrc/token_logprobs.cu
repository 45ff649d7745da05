// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits (sm_100a): what a verify step or a sampler takes from the logits
// that follow the attention.  For a row x of V logits, M = max x:
//   s = sum e^(x - M),  t = sum (x - M) e^(x - M)
//   log p(id) = (x_id - M) - ln s,  H = ln s - t / s,
//   top K by (value, then lowest index).
//
// One pass over the logits; bound by HBM (and, for 16-bit logits, by the
// exponentials: 16 a cycle and SM allow 1.4 times the rate at which the logits
// arrive).  A CTA takes 32 KB of one row into registers (eight 16-byte loads a
// thread, all in flight at once), so maximum, sums and candidates come from one
// read.  Sums are FP32, relative to the chunk's own maximum.  The candidates:
// the K-th largest of 64 group maxima (four threads each) is a lower bound of
// the chunk's K-th largest value, so only elements at or above it (a few more
// than K) are collected and ranked by counting.  A second kernel, one CTA a
// row, joins the chunks in order; no result depends on the order of atomics.
#include "qwz_common.cuh"
#include "batch_kernels.h"
#include "qwz_kernels.h"

#include <math_constants.h>

namespace qwz {

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpVecs = 8;                              // 16-byte loads a thread
constexpr int kLpChunkVecs = kLpThreads * kLpVecs;      // 32 KB
constexpr int kLpCand = 512;                            // candidates ranked by counting
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

// Makes the raw words opaque between two passes over them: otherwise the
// compiler keeps every unpacked FP32 value of the first pass (64 registers)
// for the second instead of unpacking again.
QWZ_DEVINL void lp_opaque(uint4 (&raw)[kLpVecs]) {
#pragma unroll
  for (int i = 0; i < kLpVecs; ++i) asm volatile("" : "+r"(raw[i].x), "+r"(raw[i].y), "+r"(raw[i].z), "+r"(raw[i].w));
}

// Bytes of one chunk's record: m, s, t, (pad), K keys.
QWZ_DEVINL size_t lp_record(int top) { return 16 + 8 * (size_t)top; }

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) lp_chunk_kernel(const __grid_constant__ LogprobParams p) {
  using L = LpTraits<T>;
  constexpr int E = L::E;
  __shared__ float red[3][kLpThreads / 32];
  __shared__ __align__(16) float gmax[64];
  __shared__ unsigned long long cand[kLpCand];
  __shared__ unsigned long long best;
  __shared__ float tau_s;
  __shared__ int n_cand;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  griddep_wait();

  const T* x0 = reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(x0) / sizeof(T)) % E);  // elements past a 16-byte boundary
  const int v0 = chunk * kLpChunkVecs;
  uint4 raw[kLpVecs];
#pragma unroll
  for (int i = 0; i < kLpVecs; ++i) {
    const int pos = (v0 + i * kLpThreads + tid) * E - skew;
    if (pos >= 0 && pos + E <= p.vocab) {
      raw[i] = __ldcs(reinterpret_cast<const uint4*>(x0 + pos));
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

  float tmax = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < kLpVecs; ++i) {
    float x[E];
    L::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < E; ++j) tmax = fmaxf(tmax, x[j]);
  }
  float g4 = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, 1));
  g4 = fmaxf(g4, __shfl_xor_sync(0xffffffffu, g4, 2));
  if ((lane & 3) == 0) gmax[tid >> 2] = g4;
  float M = g4;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[0][warp] = M;
  if (tid == 0) n_cand = 0;
  __syncthreads();
  M = red[0][0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 32; ++i) M = fmaxf(M, red[0][i]);
  const int K = p.top;
  if (K > 0 && warp == 0) {  // the K-th largest of the 64 group maxima
    const float a = gmax[lane], b = gmax[lane + 32];
    int ra = 0, rb = 0;
#pragma unroll 4
    for (int i = 0; i < 64; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(gmax + i);
      const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ra += (w[j] > a || (w[j] == a && i + j < lane)) ? 1 : 0;
        rb += (w[j] > b || (w[j] == b && i + j < lane + 32)) ? 1 : 0;
      }
    }
    if (ra == K - 1) tau_s = a;
    if (rb == K - 1) tau_s = b;
  }

  lp_opaque(raw);
  const float mu = M == -CUDART_INF_F ? 0.f : M;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < kLpVecs; ++i) {
    float x[E];
    L::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float d = max_nan(x[j] - mu, -1000.f);  // -inf: e = 0 and d e = 0
      const float e = exp2_approx(d * kLog2eF);
      s += e;
      t = fmaf(d, e, t);
    }
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
  uint8_t* rec = reinterpret_cast<uint8_t*>(p.workspace) + ((size_t)row * p.chunks + chunk) * lp_record(K);
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
  if (K == 0) {
    griddep_launch_dependents();
    return;
  }

  // candidates: at or above tau; where fewer than K groups hold anything above
  // -inf, all that is above -inf and the first K places (the lowest indices)
  lp_opaque(raw);
  const float tau = tau_s;
  const bool open = tau == -CUDART_INF_F;
  const int first = max(0, v0 * E - skew);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(rec + 16);
  if (tmax >= tau || open) {
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      float x[E];
      L::unpack(raw[i], x);
      const int pos = (v0 + i * kLpThreads + tid) * E - skew;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const bool take = open ? (x[j] > -CUDART_INF_F || (pos + j >= first && pos + j < first + K)) : x[j] >= tau;
        if (take && pos + j >= 0 && pos + j < p.vocab) {
          const int at = atomicAdd(&n_cand, 1);
          if (at < kLpCand) cand[at] = lp_key(x[j], (uint32_t)(pos + j));
        }
      }
    }
  }
  __syncthreads();
  const int n = n_cand;
  if (n <= kLpCand) {
    for (int c = tid; c < max(n, K); c += kLpThreads) {
      if (c < n) {
        const unsigned long long mine = cand[c];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += cand[i] > mine ? 1 : 0;
        if (rank < K) keys[rank] = mine;
      } else {
        keys[c] = 0ull;  // a chunk with fewer than K elements
      }
    }
  } else {
    // many equal values: K rounds of the largest key below the last one
    unsigned long long last = ~0ull;
    for (int k = 0; k < K; ++k) {
      unsigned long long top = 0ull;
      lp_opaque(raw);
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) {
        float x[E];
        L::unpack(raw[i], x);
        const int pos = (v0 + i * kLpThreads + tid) * E - skew;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          if (pos + j < 0 || pos + j >= p.vocab) continue;
          const unsigned long long key = lp_key(x[j], (uint32_t)(pos + j));
          if (key < last && key > top) top = key;
        }
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

int logprob_chunks(int vocab, int itemsize) {
  const int e = 16 / itemsize;
  const long long vecs = ((long long)vocab + 2 * e - 2) / e;  // with the worst skew
  return (int)((vecs + kLpChunkVecs - 1) / kLpChunkVecs);
}

size_t logprob_record_bytes(int top) { return 16 + 8 * (size_t)top; }

namespace {

template <typename T>
cudaError_t launch_lp(const LogprobParams& p, cudaStream_t stream) {
  cudaError_t e = launch_pdl(lp_chunk_kernel<T>, dim3((unsigned)p.chunks * p.rows), dim3(kLpThreads), 0, stream, p);
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
