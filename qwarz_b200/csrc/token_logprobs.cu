// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits (sm_100a): what a verify step or a sampler takes from the logits
// that follow the attention.  For a row x of V logits, M = max x:
//   s = sum e^(x - M),  t = sum (x - M) e^(x - M)
//   log p(id) = (x_id - M) - ln s,  H = ln s - t / s,
//   top K by (value, then lowest index).
//
// One pass over the logits.  A CTA streams an equal share of all rows' 16 KB
// tiles (a share may end one row and begin others: a part a row), four 16-byte
// loads a thread in flight while the four before them are summed; the sums are
// FP32, relative to a maximum of the thread's own that moves only when a logit
// exceeds it by more than 8, so nothing waits inside the loop.  Top K: the K-th
// largest of 64 group maxima (four threads each) of the part's first tiles is a
// lower bound tau of the part's K-th largest value; the places of the vectors
// that reach it (about K a tile) go to a list, and at the end, with the tau of
// the whole part's maxima, their elements are read again and ranked by counting
// (reading them at once, a warp a vector, took 61 us where this took 53).  If
// the list overflows, the part is read again with that tau, and where equal
// values overflow the candidates, or NaN stands among nothing but -inf, K rounds
// of a maximum find the K.  A second kernel, one CTA a row, joins the parts in
// order; no result depends on the order of atomics.
//
// What bounds it: the exponentials, 16 a cycle and SM, would take 15 us of the
// first case below and HBM 21; with what stands around them (unpack, difference,
// two sums, maxima; two elements an instruction made no difference) the sums alone
// take 39, the search for the top 20 another 12, a part's beginning and end being
// half of that.  2, 3, 5, 6 or 8 CTAs an SM are 1 to 15 us slower than 4.
// Measured: 448 rows of 151,000 BF16 logits, top 20, 51 us (2.6 TB/s, 41 % of
// the measured copy bandwidth); 33 rows of 50,257 FP32, top 5, 8.7 us and 7 rows
// of 131,072 BF16, top 8, 8.8 us: the latency of two launches and of one part's
// ranking.  A CTA a row took 203 us for the first of these.
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
constexpr int kLpList = 1024;                           // vectors that may hold candidates
constexpr int kLpCtasPerSm = 4;
constexpr int kLpMaxCtas = 4 * 256;
constexpr int kLpAgain = 4;                             // a long part's tau is made again after this tile
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

// Bytes of one chunk's record: m, s, t, (pad), K keys.
QWZ_DEVINL size_t lp_record(int top) { return 16 + 8 * (size_t)top; }

}  // namespace

// The K-th largest (1 <= K <= 64) of 64 values in shared memory, by 256 threads:
// four threads rank a value against sixteen others each.
QWZ_DEVINL void lp_kth(const float* v64, int K, int tid, float* out) {
  const int at = tid >> 2, from = (tid & 3) * 16;
  const float a = v64[at];
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(v64 + from + i);
    const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) rank += (w[j] > a || (w[j] == a && from + i + j < at)) ? 1 : 0;
  }
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  rank += __shfl_xor_sync(0xffffffffu, rank, 2);
  if (rank == K - 1 && (tid & 3) == 0) *out = a;
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
  __shared__ int n_cand, n_vec, list[kLpList];  // candidates; places of vectors that may hold some
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int K = p.top;
  griddep_wait();
  // this CTA's tiles of the concatenation of all rows' tiles
  const long long total = (long long)p.rows * p.row_tiles;
  long long at = (long long)blockIdx.x * total / gridDim.x;
  const long long stop = ((long long)blockIdx.x + 1) * total / gridDim.x;
  while (at < stop) {  // a part: tiles of one row
  const int row = (int)(at / p.row_tiles), tile0 = (int)(at % p.row_tiles);
  const int tiles = (int)min(stop - at, (long long)(p.row_tiles - tile0));
  at += tiles;

  const T* x0 = reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(x0) / sizeof(T)) % E);  // elements past a 16-byte boundary
  const int v0 = tile0 * kLpTileVecs;
  // places of the part
  const int first = max(0, v0 * E - skew), last_pos = min(p.vocab, (v0 + tiles * kLpTileVecs) * E - skew);

  // this thread's vectors of a tile, absent places as -inf
  auto load = [&](int tile, uint4(&raw)[kLpVecs]) {
    const int begin = (v0 + tile * kLpTileVecs) * E - skew;
    if (begin >= 0 && begin + kLpTileVecs * E <= p.vocab) {  // wholly inside the row
      const uint4* src = reinterpret_cast<const uint4*>(x0 + begin) + tid;
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) raw[i] = __ldg(src + i * kLpThreads);
      return;
    }
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
    __syncthreads();
    lp_kth(gmax, K, tid, &tau_s);
    __syncthreads();
    return tau_s;
  };
  // Candidates: at or above tau; where tau is -inf (fewer than K groups hold
  // anything above it), all that is above -inf and the first K places (the lowest
  // indices).
  auto wanted = [&](float vmax, int pos, float tau) {
    return tau == -CUDART_INF_F ? vmax > tau || pos < first + K : vmax >= tau;
  };
  auto place = [&](int tile, int i) { return (v0 + tile * kLpTileVecs + i * kLpThreads + tid) * E - skew; };
  // the candidates of the vector at `pos`, which is read again
  auto expand = [&](int pos, float tau) {
    float x[E];
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = pos + j >= first && pos + j < last_pos ? L::one(x0 + pos + j) : CUDART_NAN_F;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (pos + j >= first && pos + j < last_pos && wanted(x[j], pos + j, tau)) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < kLpCand) cand[at] = lp_key(x[j], (uint32_t)(pos + j));
      }
  };

  uint4 raw[kLpVecs], cur[kLpVecs];
  load(0, cur);
  if (tiles > 1) load(1, raw);
  float r = -CUDART_INF_F, tmax = -CUDART_INF_F, tau = CUDART_INF_F;
  if (K > 0) {
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      tmax = fmaxf(tmax, vec_max(cur[i]));
      if (tiles > 1) tmax = fmaxf(tmax, vec_max(raw[i]));
    }
    if (tid == 0) n_cand = n_vec = 0;
    tau = threshold(tmax);
  }
  float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};  // two chains each
  for (int tile = 0; tile < tiles; ++tile) {
    float vm[kLpVecs], m = -CUDART_INF_F;
    if (tile > 0) {
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) cur[i] = raw[i];
      if (tile + 1 < tiles) load(tile + 1, raw);
    }
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      vm[i] = vec_max(cur[i]);
      m = fmaxf(m, vm[i]);
    }
    if (m > r + kLpMove || (r == -CUDART_INF_F && m > r)) {  // a new reference
      if (r != -CUDART_INF_F) {  // (sums without a reference are 0 or NaN)
        const float d = max_nan(r - m, -1000.f), w = exp2_approx(d * kLog2eF);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          t[e] = w * fmaf(d, s[e], t[e]);
          s[e] *= w;
        }
      }
      r = m;
    }
    tmax = fmaxf(tmax, m);
    const float mu = r == -CUDART_INF_F ? 0.f : r;
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      float x[E];
      L::unpack(cur[i], x);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float d = max_nan(x[j] - mu, -1000.f);  // -inf: e = 0 and d e = 0
        const float e = exp2_approx(d * kLog2eF);
        s[j & 1] += e;
        t[j & 1] = fmaf(d, e, t[j & 1]);
      }
    }
    if (K > 0) {
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i)
        if (wanted(vm[i], place(tile, i), tau)) {
          const int at = atomicAdd(&n_vec, 1);
          if (at < kLpList) list[at] = place(tile, i);
        }
      if (tile == kLpAgain && tiles > 2 * kLpAgain) tau = fmaxf(tau, threshold(tmax));
    }
  }

  // the part's reference, and the threads' sums relative to it
  float M = r, sum = s[0] + s[1], tsum = t[0] + t[1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
  M = red[0][0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 32; ++i) M = fmaxf(M, red[0][i]);
  if (r != -CUDART_INF_F) {
    const float d = max_nan(r - M, -1000.f), w = exp2_approx(d * kLog2eF);
    tsum = w * fmaf(d, sum, tsum);
    sum *= w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    tsum += __shfl_xor_sync(0xffffffffu, tsum, o);
  }
  if (lane == 0) {
    red[1][warp] = sum;
    red[2][warp] = tsum;
  }
  __syncthreads();
  // (CTA + row) numbers the parts of the launch without gaps within a row
  uint8_t* rec = reinterpret_cast<uint8_t*>(p.workspace) + ((size_t)blockIdx.x + row) * lp_record(K);
  if (tid == 0) {
    sum = tsum = 0.f;
#pragma unroll
    for (int i = 0; i < kLpThreads / 32; ++i) {
      sum += red[1][i];
      tsum += red[2][i];
    }
    float* f = reinterpret_cast<float*>(rec);
    f[0] = M;
    f[1] = sum;
    f[2] = tsum;
  }
  if (K > 0) {
    // The whole part's maxima give a closer bound, which most of the listed
    // vectors do not reach.
    if (tiles > 2) tau = threshold(tmax);
    // Without a bound the first K places stand for the -inf tokens, which holds
    // as long as none of them is NaN (a NaN, or +inf, is in the part's sum).
    bool nan = false;
    if (tau == -CUDART_INF_F) {
#pragma unroll 1
      for (int i = 0; i < kLpThreads / 32; ++i) nan |= red[1][i] != red[1][i];
    }
    if (nan) {
      // ranked below without a list
    } else if (n_vec <= kLpList) {
      for (int c = tid; c < n_vec; c += kLpThreads) expand(list[c], tau);
    } else {  // the list overflowed
#pragma unroll 1
      for (int tile = 0; tile < tiles; ++tile) {
        load(tile, raw);
#pragma unroll
        for (int i = 0; i < kLpVecs; ++i)
          if (wanted(vec_max(raw[i]), place(tile, i), tau)) expand(place(tile, i), tau);
      }
    }
    __syncthreads();
    const int n = n_cand;
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(rec + 16);
    if (!nan && n <= kLpCand) {
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
      // many equal values, or NaN among -inf: K rounds of the largest key below the last one
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
  __syncthreads();  // the next part's list takes the place of this one's
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
  // the parts of this row: those of CTAs c0 .. c1
  const long long total = (long long)p.rows * p.row_tiles, t0 = (long long)row * p.row_tiles, t1 = t0 + p.row_tiles - 1;
  const int c0 = (int)(((t0 + 1) * p.ctas - 1) / total), c1 = (int)(((t1 + 1) * p.ctas - 1) / total);
  const int parts = c1 - c0 + 1;
  const uint8_t* recs = reinterpret_cast<const uint8_t*>(p.workspace) + ((size_t)c0 + row) * lp_record(K);
  auto stat = [&](int c) { return reinterpret_cast<const float*>(recs + c * lp_record(K)); };
  // the given token's logit and the first lists, on their way while the sums are joined
  long long id = -1;
  float x_id = 0.f;
  if (tid == 0) {
    id = p.ids64 ? __ldg(reinterpret_cast<const long long*>(p.ids) + row)
                 : (long long)__ldg(reinterpret_cast<const int*>(p.ids) + row);
    if (id >= 0 && id < p.vocab)
      x_id = LpTraits<T>::one(reinterpret_cast<const T*>(p.logits) + (long long)row * p.stride + id);
  }
  if (K > 0 && tid < parts * K)
    cand[tid] = __ldcg(reinterpret_cast<const unsigned long long*>(recs + tid / K * lp_record(K) + 16) + tid % K);

  float M = -CUDART_INF_F;
  for (int c = tid; c < parts; c += kLpThreads) M = fmaxf(M, __ldcg(stat(c)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
  M = red[0][0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 32; ++i) M = fmaxf(M, red[0][i]);
  __syncthreads();
  float s = 0.f, t = 0.f;
  for (int c = tid; c < parts; c += kLpThreads) {
    const float m = __ldcg(stat(c)), sc = __ldcg(stat(c) + 1), tc = __ldcg(stat(c) + 2);
    if (m == -CUDART_INF_F) {
      s += sc;  // 0, or NaN
      continue;
    }
    const float d = max_nan(m - M, -1000.f), w = exp2_approx(d * kLog2eF);
    s += w * sc;
    t += w * fmaf(d, sc, tc);
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
    float lp = 0.f;  // id < 0: no token
    if (id >= p.vocab) {
      flag_error(kErrSlotRange);
      lp = CUDART_NAN_F;
    } else if (id >= 0) {
      lp = logprob(x_id);
    }
    p.logprob[row] = lp;
  }
  if (K == 0) return;

  // the best K so far, then as many chunks' lists as fit beside them
  int have = 0;
  const int lists = (kLpMergeCand - 32) / K;
  for (int l0 = 0; l0 < parts; l0 += lists) {
    const int n_lists = min(lists, parts - l0), n = have + n_lists * K;
    if (tid < have) cand[tid] = sorted[tid];
    for (int i = tid + (l0 == 0 ? kLpThreads : 0); i < n_lists * K; i += kLpThreads)
      cand[have + i] = __ldcg(reinterpret_cast<const unsigned long long*>(recs + (l0 + i / K) * lp_record(K) + 16) + i % K);
    __syncthreads();
    if (tid < K) sorted[tid] = 0ull;
    if (tid < 16 && n + tid < kLpMergeCand) cand[n + tid] = 0ull;  // the last sixteen are whole
    __syncthreads();
    for (int i = tid; i < n; i += kLpThreads) {
      const unsigned long long mine = cand[i];
      if (mine == 0ull) continue;
      int rank = 0;  // looked at every sixteen: every one costs 4 us of a 13 us call
      for (int j = 0; j < n && rank < K; j += 16) {
#pragma unroll
        for (int e = 0; e < 16; ++e) rank += cand[j + e] > mine ? 1 : 0;
      }
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

// Records that any call of up to `rows` rows needs: a part begins with a CTA or
// with a row.
long long logprob_records(int rows) { return (long long)kLpMaxCtas + rows; }

size_t logprob_record_bytes(int top) { return 16 + 8 * (size_t)top; }

namespace {

template <typename T>
cudaError_t launch_lp(const LogprobParams& p, cudaStream_t stream) {
  cudaError_t e = launch_pdl(lp_part_kernel<T>, dim3(p.ctas), dim3(kLpThreads), 0, stream, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(lp_merge_kernel<T>, dim3(p.rows), dim3(kLpThreads), 0, stream, p);
}

}  // namespace

cudaError_t launch_token_logprobs(LogprobParams p, int dtype, int sms, cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  p.row_tiles = lp_tiles(p.vocab, dtype == kDtypeF32 ? 4 : 2);
  p.ctas = (int)min((long long)p.rows * p.row_tiles, (long long)min(kLpMaxCtas, sms * kLpCtasPerSm));
  switch (dtype) {
    case kDtypeF16: return launch_lp<__half>(p, stream);
    case kDtypeBF16: return launch_lp<__nv_bfloat16>(p, stream);
    default: return launch_lp<float>(p, stream);
  }
}

}  // namespace qwz
