// Softmax statistics and softmax-shaped gradients of one row of logits, shared
// by the token scores (token_scores.cu) and the distillation loss
// (distill.cu).
//
// A row of V logits (FP32 or BF16, any alignment) is walked as a scalar head
// up to the first 16-byte boundary, 16-byte vectors, and a scalar tail, so odd
// vocabularies and padded row strides take the same path.  With c = log2(e) /
// temperature the statistics are
//   m  = max x,   s = sum 2^d,   sd = sum d 2^d,   d = (x - m) c,
// all FP32; (x - m) is formed first, so a row far from zero loses nothing.
// d is clamped from below at -150, where 2^d flushes to zero: a masked logit
// (-inf, or the type's lowest value) adds 0 to both sums instead of 0 * -inf.
// The maximum is clamped at -FLT_MAX, so that s == 0 exactly when every logit
// is -inf.  NaN and +inf make s NaN.
#pragma once

#include <cfloat>

#include "common.cuh"

namespace dabsn {
namespace rowsm {

typedef __nv_bfloat16 bf16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -150.f;  // 2^kFloor is zero in FP32

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// max(a, b) that keeps a NaN of a (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float scaled_gap(float x, float m, float c) {
  return max_nan((x - m) * c, kFloor);
}

// 16-byte vectors of T.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr unsigned kNegInf = 0xff800000u;
};
template <>
struct Vec<bf16> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xff80ff80u;
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[Vec<T>::N]);
template <>
__device__ __forceinline__ void unpack<float>(const uint4& u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x);
  v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z);
  v[3] = __uint_as_float(u.w);
}
template <>
__device__ __forceinline__ void unpack<bf16>(const uint4& u, float (&v)[8]) {
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[Vec<T>::N]);
template <>
__device__ __forceinline__ uint4 pack<float>(const float (&v)[4]) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                    __float_as_uint(v[3]));
}
template <>
__device__ __forceinline__ uint4 pack<bf16>(const float (&v)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  return u;
}

// Head, vectors and tail of n elements at p.
struct RowShape {
  int head, nv, tail0, tail;
};
template <typename T>
__device__ __forceinline__ RowShape row_shape(const T* p, int n) {
  constexpr int VW = Vec<T>::N;
  RowShape r;
  const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
  r.head = off == 0 ? 0 : VW - off;
  if (r.head > n) r.head = n;
  r.nv = (n - r.head) / VW;
  r.tail0 = r.head + r.nv * VW;
  r.tail = n - r.tail0;
  return r;
}

// ---------------------------------------------------------------------------
// Statistics
// ---------------------------------------------------------------------------
struct Stats {
  float mx = -INFINITY;  // maximum as it stands in the row
  float s = 0.f, sd = 0.f;
};

__device__ __forceinline__ float finite_max(float mx) { return fmaxf(mx, -FLT_MAX); }

// Moves the sums of st to a maximum mx >= st.mx.
__device__ __forceinline__ void rescale(Stats& st, float mx, float c) {
  const float g = scaled_gap(finite_max(st.mx), finite_max(mx), c);
  const float f = ex2(g);
  st.sd = f * fmaf(st.s, g, st.sd);
  st.s *= f;
  st.mx = mx;
}

__device__ __forceinline__ void merge(Stats& a, Stats b, float c) {
  const float mx = fmaxf(a.mx, b.mx);
  rescale(a, mx, c);
  rescale(b, mx, c);
  a.s += b.s;
  a.sd += b.sd;
}

template <int N>
__device__ __forceinline__ void add_values(Stats& st, const float (&v)[N], float c) {
  float mx = st.mx;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmaxf(mx, v[i]);
  rescale(st, mx, c);
  const float m = finite_max(mx);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = scaled_gap(v[i], m, c);
    const float e = ex2(d);
    st.s += e;
    st.sd = fmaf(e, d, st.sd);
  }
}

// The part of a row of n elements that belongs to thread `t` of THREADS:
// vectors t, t + THREADS, ...; one head and one tail element for the first
// threads.  Four vectors are in flight at a time.
template <typename T, int THREADS>
__device__ __forceinline__ Stats sweep(const T* p, int n, int t, float c) {
  constexpr int VW = Vec<T>::N, U = 4;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  Stats st;
  for (int i = t; i < r.nv; i += THREADS * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = i + u * THREADS;
      constexpr unsigned ni = Vec<T>::kNegInf;
      raw[u] = k < r.nv ? __ldg(pv + k) : make_uint4(ni, ni, ni, ni);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[VW];
      unpack<T>(raw[u], v);
      add_values<VW>(st, v, c);
    }
  }
  float edge[2] = {-INFINITY, -INFINITY};
  if (t < r.head) edge[0] = to_f<T>(p[t]);
  if (t < r.tail) edge[1] = to_f<T>(p[r.tail0 + t]);
  add_values<2>(st, edge, c);
  return st;
}

// Merges the threads' statistics of a CTA in a fixed order; every thread gets
// the result.  `sh` holds three floats a warp.  Ends with a barrier before the
// next use of `sh` being the caller's business.
template <int THREADS>
__device__ __forceinline__ Stats block_merge(Stats st, float (*sh)[3], float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats b;
    b.mx = __shfl_xor_sync(0xffffffffu, st.mx, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    b.sd = __shfl_xor_sync(0xffffffffu, st.sd, o);
    merge(st, b, c);
  }
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    sh[warp][0] = st.mx;
    sh[warp][1] = st.s;
    sh[warp][2] = st.sd;
  }
  __syncthreads();
  Stats all;
  for (int w = 0; w < THREADS / 32; ++w) {
    Stats b;
    b.mx = sh[w][0];
    b.s = sh[w][1];
    b.sd = sh[w][2];
    merge(all, b, c);
  }
  return all;
}

// ---------------------------------------------------------------------------
// Gradient of a row: out_j = 2^d_j (A + B d_j), in the logits' type.  With
// A = a / s and B = b ln2 / s that is p_j (a + b d_j ln2).
// ---------------------------------------------------------------------------
template <bool HAS_B>
__device__ __forceinline__ float grad_value(float x, float m, float c, float A, float B) {
  if (HAS_B) {
    const float d = scaled_gap(x, m, c);
    return ex2(d) * fmaf(B, d, A);
  }
  return ex2((x - m) * c) * A;
}

// Whether 16-byte vectors of a logits row and of its gradient row start at the
// same element in every row (else the gradient is stored by element).
inline bool same_phase(const void* x, long long ld, const void* dx, long long ldd, size_t size) {
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0 &&
         (((ld - ldd) * (long long)size) & 15) == 0;
}

template <typename T, int THREADS, bool HAS_B, bool SAME>
__device__ __forceinline__ void grad_sweep(const T* p, T* q, int n, int t, float m, float c,
                                           float A, float B) {
  constexpr int VW = Vec<T>::N, U = 4;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  for (int i = t; i < r.nv; i += THREADS * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * THREADS < r.nv) raw[u] = __ldg(pv + i + u * THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = i + u * THREADS;
      if (k >= r.nv) break;
      float v[VW];
      unpack<T>(raw[u], v);
#pragma unroll
      for (int j = 0; j < VW; ++j) v[j] = grad_value<HAS_B>(v[j], m, c, A, B);
      T* dst = q + r.head + (size_t)k * VW;
      if (SAME) {
        *reinterpret_cast<uint4*>(dst) = pack<T>(v);
      } else {
#pragma unroll
        for (int j = 0; j < VW; ++j) dst[j] = from_f<T>(v[j]);
      }
    }
  }
  if (t < r.head) q[t] = from_f<T>(grad_value<HAS_B>(to_f<T>(p[t]), m, c, A, B));
  if (t < r.tail)
    q[r.tail0 + t] = from_f<T>(grad_value<HAS_B>(to_f<T>(p[r.tail0 + t]), m, c, A, B));
}

template <typename T, int THREADS>
__device__ __forceinline__ void zero_row(T* q, int n, int t) {
  const RowShape r = row_shape(q, n);
  uint4* qv = reinterpret_cast<uint4*>(q + r.head);
  for (int i = t; i < r.nv; i += THREADS) qv[i] = make_uint4(0u, 0u, 0u, 0u);
  if (t < r.head) q[t] = from_f<T>(0.f);
  if (t < r.tail) q[r.tail0 + t] = from_f<T>(0.f);
}

}  // namespace rowsm
}  // namespace dabsn
