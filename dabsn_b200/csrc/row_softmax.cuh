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
// d is clamped from below at -127, where 2^d flushes to zero: a masked logit
// (-inf, or the type's lowest value) adds 0 to both sums instead of 0 * -inf.
// The maximum is clamped at -FLT_MAX, so that s == 0 exactly when every logit
// is -inf.  NaN and +inf make s NaN.
#pragma once

#include <cfloat>

#include "../../include/dabsn_b200.h"
#include "common.cuh"

namespace dabsn {
namespace rowsm {

typedef __nv_bfloat16 bf16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -127.f;  // 2^kFloor is flushed to zero

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

// Two FP32 lanes in one register pair: one instruction does both.  BF16 rows
// arrive at 11.6 elements a clock and SM at the memory's rate, which leaves 11
// issue slots an element and keeps the exponential unit (16 a clock) busy for
// 73 % of the time; with scalar arithmetic and a rescaling per vector the sweep
// of token_scores took 194 us where it takes 155.  (A quarter of the exponentials
// as a polynomial on the FMA pipes: 179 us where it took 170.)
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ f32x2 clamp2(f32x2 d) {
  const float2 v = split(d);
  return pair(max_nan(v.x, kFloor), max_nan(v.y, kFloor));
}

__device__ __forceinline__ f32x2 ex2_pair(f32x2 d) {
  const float2 v = split(d);
  return pair(ex2(v.x), ex2(v.y));
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

// The vector's elements as FP32 pairs.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, f32x2 (&v)[Vec<T>::N / 2]);
template <>
__device__ __forceinline__ void unpack<float>(const uint4& u, f32x2 (&v)[2]) {
  v[0] = pair(__uint_as_float(u.x), __uint_as_float(u.y));
  v[1] = pair(__uint_as_float(u.z), __uint_as_float(u.w));
}
template <>
__device__ __forceinline__ void unpack<bf16>(const uint4& u, f32x2 (&v)[4]) {
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ uint4 pack(const f32x2 (&v)[Vec<T>::N / 2]);
template <>
__device__ __forceinline__ uint4 pack<float>(const f32x2 (&v)[2]) {
  const float2 a = split(v[0]), b = split(v[1]);
  return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x),
                    __float_as_uint(b.y));
}
template <>
__device__ __forceinline__ uint4 pack<bf16>(const f32x2 (&v)[4]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = split(v[i]);
    h[i] = __floats2bfloat162_rn(f.x, f.y);
  }
  return u;
}

// Largest element of U vectors (NaN is passed over; the sums carry it).
template <typename T, int U>
__device__ __forceinline__ float vector_max(const uint4 (&raw)[U]);
template <>
__device__ __forceinline__ float vector_max<float, 1>(const uint4 (&r)[1]) {
  return fmaxf(fmaxf(__uint_as_float(r[0].x), __uint_as_float(r[0].y)),
               fmaxf(__uint_as_float(r[0].z), __uint_as_float(r[0].w)));
}
__device__ __forceinline__ unsigned max_bf16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ unsigned vector_max2(const uint4& u) {
  return max_bf16x2(max_bf16x2(u.x, u.y), max_bf16x2(u.z, u.w));
}
__device__ __forceinline__ float pair_max(unsigned w) {
  return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float vector_max<bf16, 1>(const uint4 (&r)[1]) {
  return pair_max(vector_max2(r[0]));
}
template <>
__device__ __forceinline__ float vector_max<float, 4>(const uint4 (&r)[4]) {
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(r[u].x), __uint_as_float(r[u].y)),
                       fmaxf(__uint_as_float(r[u].z), __uint_as_float(r[u].w))));
  return m;
}
template <>
__device__ __forceinline__ float vector_max<bf16, 4>(const uint4 (&r)[4]) {
  return pair_max(max_bf16x2(max_bf16x2(vector_max2(r[0]), vector_max2(r[1])),
                             max_bf16x2(vector_max2(r[2]), vector_max2(r[3]))));
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

// Moves the sums of st to a maximum mx >= st.mx.  The products are rounded by
// themselves (not contracted with the sums that follow), so that merging is
// symmetric and all lanes of a butterfly end with the same bits.
__device__ __forceinline__ void rescale(Stats& st, float mx, float c) {
  const float g = scaled_gap(finite_max(st.mx), finite_max(mx), c);
  const float f = ex2(g);
  st.sd = __fmul_rn(f, fmaf(st.s, g, st.sd));
  st.s = __fmul_rn(st.s, f);
  st.mx = mx;
}

// Adds one element.
__device__ __forceinline__ void add_value(Stats& st, float x, float c) {
  rescale(st, fmaxf(st.mx, x), c);
  const float d = scaled_gap(x, finite_max(st.mx), c);
  const float e = ex2(d);
  st.s += e;
  st.sd = fmaf(e, d, st.sd);
}

// Adds U vectors, moving the sums to a new maximum once.  SD: with the sum that
// the entropy needs (without it -inf needs no clamp: 2^-inf is 0).
template <typename T, int U, bool SD>
__device__ __forceinline__ void add_vectors(Stats& st, const uint4 (&raw)[U], float c) {
  constexpr int P = Vec<T>::N / 2;
  rescale(st, fmaxf(st.mx, vector_max<T, U>(raw)), c);
  const float m = finite_max(st.mx);
  const f32x2 m2 = pair(-m, -m), c2 = pair(c, c);
  f32x2 s2 = pair(st.s, 0.f), sd2 = pair(st.sd, 0.f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    f32x2 v[P];
    unpack<T>(raw[u], v);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      f32x2 d = mul2(add2(v[i], m2), c2);
      if (SD) d = clamp2(d);
      const f32x2 e = ex2_pair(d);
      s2 = add2(s2, e);
      if (SD) sd2 = fma2(e, d, sd2);
    }
  }
  const float2 s = split(s2), sd = split(sd2);
  st.s = s.x + s.y;
  if (SD) st.sd = sd.x + sd.y;
}

template <bool ONCE>
__device__ __forceinline__ uint4 load_vector(const uint4* p) {
  return ONCE ? __ldcs(p) : __ldg(p);
}

// The part of a row of n elements that belongs to thread `t` of THREADS:
// vectors t, t + THREADS, ...; one head and one tail element for the first
// threads.  Four vectors are in flight at a time.  ONCE: the kernel does not
// come back to the row, so its lines may leave L2 first (4096 BF16 rows of 32000
// in 51 us instead of 56; a kernel that reads the row again loses 10 % by it).
template <typename T, int THREADS, bool SD, bool ONCE>
__device__ __forceinline__ Stats sweep(const T* p, int n, int t, float c) {
  constexpr int U = 4;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  Stats st;
  int i = t;
  for (; i + (U - 1) * THREADS < r.nv; i += THREADS * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_vector<ONCE>(pv + i + u * THREADS);
    add_vectors<T, U, SD>(st, raw, c);
  }
  if (i < r.nv) {  // one to three more, loaded together
    uint4 raw[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (i + u * THREADS < r.nv) raw[u] = load_vector<ONCE>(pv + i + u * THREADS);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (i + u * THREADS < r.nv) {
        const uint4 one[1] = {raw[u]};
        add_vectors<T, 1, SD>(st, one, c);
      }
  }
  if (t < r.head) add_value(st, to_f<T>(p[t]), c);
  if (t < r.tail) add_value(st, to_f<T>(p[r.tail0 + t]), c);
  return st;
}

// The merged statistics of groups of LANES lanes, the same bits in each: the
// maximum first, one rescaling, then plain sums.
template <int LANES = 32>
__device__ __forceinline__ Stats warp_merge(Stats st, float c) {
  float mx = st.mx;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  rescale(st, mx, c);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    st.sd += __shfl_xor_sync(0xffffffffu, st.sd, o);
  }
  return st;
}

// Merges the threads' statistics of a CTA in a fixed order; every thread gets
// the result.  `sh` holds three floats a warp; a barrier must come between this
// call and the next.
template <int THREADS>
__device__ __forceinline__ Stats block_merge(Stats st, float (*sh)[3], float c) {
  constexpr int WARPS = THREADS / 32;
  static_assert((WARPS & (WARPS - 1)) == 0 && WARPS <= 32, "a power of two");
  st = warp_merge(st, c);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    sh[warp][0] = st.mx;
    sh[warp][1] = st.s;
    sh[warp][2] = st.sd;
  }
  __syncthreads();
  Stats all;
  all.mx = sh[lane % WARPS][0];
  all.s = sh[lane % WARPS][1];
  all.sd = sh[lane % WARPS][2];
  return warp_merge<WARPS>(all, c);
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

template <typename T, bool HAS_B>
__device__ __forceinline__ uint4 grad_vector(const uint4& raw, f32x2 m2, f32x2 c2, f32x2 A2,
                                             f32x2 B2) {
  constexpr int P = Vec<T>::N / 2;
  f32x2 v[P];
  unpack<T>(raw, v);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    f32x2 d = mul2(add2(v[i], m2), c2);
    if (HAS_B) d = clamp2(d);
    v[i] = mul2(ex2_pair(d), HAS_B ? fma2(B2, d, A2) : A2);
  }
  return pack<T>(v);
}

template <typename T, int THREADS, bool HAS_B>
__device__ __forceinline__ void grad_sweep(const T* p, T* q, int n, int t, float m, float c,
                                           float A, float B) {
  constexpr int U = 4;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  uint4* qv = reinterpret_cast<uint4*>(q + r.head);
  const f32x2 m2 = pair(-m, -m), c2 = pair(c, c), A2 = pair(A, A), B2 = pair(B, B);
  for (int i = t; i < r.nv; i += THREADS * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * THREADS < r.nv) raw[u] = __ldg(pv + i + u * THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = i + u * THREADS;
      if (k >= r.nv) break;
      qv[k] = grad_vector<T, HAS_B>(raw[u], m2, c2, A2, B2);
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

// The gradient kernels store the vectors they loaded, so a gradient row starts
// at the 16-byte phase of its logits row.
inline int check_gradient_rows(const char* what, int dtype, int64_t rows, int64_t V, int64_t ld,
                               const void* x, int64_t ldd, const void* dx) {
  const int64_t size = dtype == DABSN_BF16 ? 2 : 4;
  if (ldd < V) {
    set_error("%s: gradient rows %lld apart overlap (V=%lld)", what, (long long)ldd,
              (long long)V);
    return DABSN_ERR_SHAPE;
  }
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) != 0 ||
      (rows > 1 && ((ld - ldd) * size & 15) != 0)) {
    set_error("%s: gradient rows must start at the 16-byte phase of the logits rows", what);
    return DABSN_ERR_UNSUPPORTED;
  }
  return DABSN_OK;
}

}  // namespace rowsm
}  // namespace dabsn
