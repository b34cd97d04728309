// Log-probabilities of given tokens, with the entropy and the top alternatives
// of every row, and the reverse of the first two.
//
//   x = logits / temperature, p = softmax(x), t = the row's token
//   log_prob = log p_t,  entropy = -sum p log p,
//   alternatives: the k largest logits (ties to the lowest index), as log p;
//   dlogits_j = (1 / temperature) [g (1[j = t] - p_j) - h p_j (log p_j + entropy)]
//   for the gradients g of log_prob and h of entropy.
//
// Forward: one CTA per row, one pass over the logits for the maximum, the sum
// of exponentials and the sum that the entropy needs (row_softmax.cuh).  What
// bounds it is HBM, with the exponential unit at three quarters: 16384 BF16 rows
// of 32000 (a tenth of them ignored) in 155 us, 6.1 TB/s.  A row whose token is
// ignore_index is not read.
//
// The alternatives come out of the same pass: every thread knows the maximum of
// the part of the row it read, the k-th largest of those maxima bounds the
// row's k-th largest logit from below, and only the parts whose maximum
// reaches that bound (about k of 256) are read again, out of L2.  20 of 16384
// rows of 32000: 233 us.  The selection adds two fifths to a row's instructions
// in short steps between barriers, so it wants many rows on an SM: 256 threads a
// row and eight CTAs an SM took 232 us, six 240 us, 128 threads a row 253 us, and
// the selection left to one warp of the CTA 411 us.
//
// Reverse: one sweep that reads the logits and writes their gradient, 6.8 TB/s
// at the same size (294 to 299 us).
#include <algorithm>

#include "../../include/dabsn_b200.h"
#include "common.cuh"
#include "row_softmax.cuh"

namespace dabsn {
namespace {

using namespace rowsm;
typedef unsigned long long u64;

constexpr int TS_THREADS = 256;
// Up to three rows an SM, long rows go to 512 threads each: those of more than
// 24 KB, or with alternatives, whose selection takes longer among more threads, of
// more than 96 KB.  Device us with 256 threads a row and with 512:
//   rows                         8        148        444        592
//   BF16 x 8000 (16 KB)     4.0  3.2   4.7  4.1   6.2  5.7   6.6  7.9
//   FP32 x 8000 (32 KB)     4.6  4.0   5.7  5.2   7.1  7.2   7.9  9.9
//   BF16 x 32000            6.2  4.9   7.3  6.2  10.2 10.1  11.6 13.7
//   FP32 x 128000          25.9 15.8  28.6 19.8  42.9 41.4  53.9 60.1
// and with 20 alternatives:
//   BF16 x 32000 (64 KB)   10.3 10.5  11.8 12.2  15.1 16.2  17.4 19.1
//   FP32 x 32000 (128 KB)  13.0 11.7  15.4 14.0  22.7 21.8  27.5 26.3
//   BF16 x 128000          23.1 17.8  25.8 20.8  41.7 36.6  48.6 45.3
//   FP32 x 128000          33.0 22.2  43.9 32.1  69.9 59.8  87.5 77.8
// (888 rows: 67.2 and 74.6 for BF16 x 128000, 37.0 and 41.1 for FP32 x 32000.)
constexpr int TS_FEW_THREADS = 512;
constexpr int TS_FEW_ROWS = 444;
constexpr int TS_FEW_BYTES = 24 * 1024;
constexpr int TS_FEW_TOP_BYTES = 96 * 1024;
constexpr int TS_MAX_K = 128;
constexpr int TS_CAP = 1024;  // candidates of a row
constexpr int STATUS_BAD_TOKEN = 8;

// Order of the alternatives as unsigned keys: larger logit, larger key; -0
// equals +0; 0 is below every logit.  (A row with NaN has no order: it takes
// another way.)
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x + 0.f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// One candidate: larger is better; equal logits rank by the lower index.
__device__ __forceinline__ u64 candidate(unsigned key, int index) {
  return ((u64)key << 32) | (unsigned)~index;
}
__device__ __forceinline__ int candidate_index(u64 c) { return ~(int)(unsigned)c; }

// Shared memory of a CTA of THREADS threads that selects.
template <int THREADS>
struct TopkShared {
  unsigned keys[THREADS];
  short hot[THREADS];
  u64 found[TS_CAP];
  int n_found, n_hot;
  unsigned bound;
  int warp_count[THREADS / 32];
};

// One warp: a bound that at least k of the threads' keys reach, and the list of
// the threads whose key reaches it.  The bound is found two bits at a time below
// the bits that all keys share: the k-th largest key, or (unless `exact`) the
// first prefix of it that few more than k reach; 0 when fewer than k threads
// have any element.  A BF16 key is its upper half.
template <typename T, int THREADS>
__device__ __forceinline__ void find_bound(TopkShared<THREADS>& sh, int k, bool exact) {
  constexpr int PER = THREADS / 32, LAST = sizeof(T) == 2 ? 16 : 0;
  const int lane = threadIdx.x & 31;
  unsigned own[PER], hi = 0u, lo = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    own[i] = sh.keys[lane + 32 * i];
    hi = max(hi, own[i]);
    lo = min(lo, own[i]);
  }
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo);
  const int open = (33 - __clz((int)(hi ^ lo))) & ~1;  // lower bits that differ, rounded up
  unsigned t = open >= 32 ? 0u : hi >> open << open;
  for (int bit = open - 2; bit >= LAST; bit -= 2) {
    // how many keys reach each of the three next steps, in one sum
    const unsigned step = 1u << bit;
    unsigned n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      n += (own[i] >= t + step) + ((own[i] >= t + 2 * step) << 10) +
           ((own[i] >= t + 3 * step) << 20);
    n = __reduce_add_sync(0xffffffffu, n);
    const int n1 = n & 1023, n2 = n >> 10 & 1023, n3 = n >> 20;
    const int took = n3 >= k ? 3 : n2 >= k ? 2 : n1 >= k ? 1 : 0;
    t += took * step;
    if (!exact && took > 0 && (took == 3 ? n3 : took == 2 ? n2 : n1) <= k + 8) break;
  }
  // the lower half of a BF16 key: zeros from zero up, ones below
  if (LAST == 16 && exact) {
    t &= 0xffff0000u;
    if (t != 0u && !(t & 0x80000000u)) t |= 0xffffu;
  }
  int count = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool hot = own[i] != 0u && own[i] >= t;
    const unsigned votes = __ballot_sync(0xffffffffu, hot);
    if (hot) sh.hot[count + __popc(votes & ((1u << lane) - 1))] = (short)(lane + 32 * i);
    count += __popc(votes);
  }
  if (lane == 0) {
    sh.bound = t;
    sh.n_hot = count;
  }
}

// Visits every element of the row that a thread of `hot` read in the sweep, a
// vector to a thread at a time: visit(x, index) for the elements from `low` on;
// vectors below it cost their maximum.
template <typename T, int THREADS, typename Visit>
__device__ __forceinline__ void visit_parts(const TopkShared<THREADS>& sh, const T* p, int n,
                                            int n_hot, float low, Visit visit) {
  constexpr int VW = Vec<T>::N;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  const int per = (r.nv + THREADS - 1) / THREADS;
  for (int e = threadIdx.x; e < n_hot * per; e += THREADS) {
    const int h = e / per, k = sh.hot[h] + (e - h * per) * THREADS;
    if (k >= r.nv) continue;
    const uint4 raw[1] = {__ldg(pv + k)};
    if (vector_max<T, 1>(raw) < low) continue;
    f32x2 v[VW / 2];
    unpack<T>(raw[0], v);
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) {
      const float2 x = split(v[j]);
      if (x.x >= low) visit(x.x, r.head + k * VW + 2 * j);
      if (x.y >= low) visit(x.y, r.head + k * VW + 2 * j + 1);
    }
  }
  for (int h = threadIdx.x; h < n_hot; h += THREADS) {
    const int t = sh.hot[h];
#pragma unroll
    for (int side = 0; side < 2; ++side) {  // the part's head and tail element
      if (t >= (side == 0 ? r.head : r.tail)) continue;
      const int i = side == 0 ? t : r.tail0 + t;
      const float x = to_f<T>(p[i]);
      if (x >= low) visit(x, i);
    }
  }
}

template <int THREADS>
__device__ __forceinline__ void keep(TopkShared<THREADS>& sh, unsigned key, int index) {
  const int at = atomicAdd(&sh.n_found, 1);
  if (at < TS_CAP) sh.found[at] = candidate(key, index);
}

// visit(x, index) for the row's elements from `low` on; four vectors of a
// thread in flight, those below `low` cost their maximum.
template <typename T, int THREADS, typename Visit>
__device__ __forceinline__ void visit_row(const T* p, int n, float low, Visit visit) {
  constexpr int VW = Vec<T>::N, U = 4;
  const int t = threadIdx.x;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  for (int k0 = t; k0 < r.nv; k0 += U * THREADS) {
    float top[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * THREADS;
      constexpr unsigned ni = Vec<T>::kNegInf;
      const uint4 raw[1] = {k < r.nv ? __ldg(pv + k) : make_uint4(ni, ni, ni, ni)};
      top[u] = vector_max<T, 1>(raw);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * THREADS;
      if (k >= r.nv || top[u] < low) continue;
      for (int j = 0; j < VW; ++j) {
        const int i = r.head + k * VW + j;
        const float x = to_f<T>(p[i]);
        if (x >= low) visit(x, i);
      }
    }
  }
  if (t < r.head && to_f<T>(p[t]) >= low) visit(to_f<T>(p[t]), t);
  if (t < r.tail && to_f<T>(p[r.tail0 + t]) >= low) visit(to_f<T>(p[r.tail0 + t]), r.tail0 + t);
}

// More logits reach the bound than are kept (a flat row, one built against the
// bound), or fewer than k threads have any left in a masked row.  With the k-th
// largest key of the threads (or, where too many lie above that too, of the row;
// -inf for the masked row): what lies above it, and of the logits equal to it the
// lowest indices, in order.
template <typename T, int THREADS>
__device__ __noinline__ void select_top_slow(TopkShared<THREADS>& sh, const T* p, int n, int k,
                                             bool masked) {
  const int t = threadIdx.x;
  unsigned bound = order_key(-INFINITY);
  auto above = [&](float x, int index) {
    const unsigned key = order_key(x);
    if (key > bound && *(volatile int*)&sh.n_found <= TS_CAP) keep(sh, key, index);
  };
  if (t == 0) sh.n_found = sh.n_hot = 0;
  if (masked) {
    __syncthreads();
    if (sh.keys[t] > bound) sh.hot[atomicAdd(&sh.n_hot, 1)] = (short)t;
    __syncthreads();
    visit_parts<T, THREADS>(sh, p, n, sh.n_hot, -FLT_MAX, above);
  } else {
    if (t < 32) find_bound<T, THREADS>(sh, k, true);
    __syncthreads();
    bound = sh.bound;
    // strictly above, so the next number is where the visit starts
    visit_row<T, THREADS>(p, n, bound == 0u ? -INFINITY : key_value(bound + 1u), above);
  }
  __syncthreads();
  if (sh.n_found > TS_CAP) {
    bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned cand = bound | (1u << bit);
      __syncthreads();
      if (t == 0) sh.n_found = 0;
      __syncthreads();
      int c = 0;
      for (int i = t; i < n; i += THREADS) c += order_key(to_f<T>(p[i])) >= cand;
      c = __reduce_add_sync(0xffffffffu, c);
      if ((t & 31) == 0) atomicAdd(&sh.n_found, c);
      __syncthreads();
      if (sh.n_found >= k) bound = cand;
    }
    __syncthreads();
    if (t == 0) sh.n_found = 0;
    __syncthreads();
    visit_row<T, THREADS>(p, n, bound == 0u ? -INFINITY : key_value(bound + 1u), above);
    __syncthreads();
  }
  const int have = sh.n_found, need = k - have;
  int got = 0;
  for (int base = 0; base < n && got < need; base += THREADS) {
    const int i = base + t;
    const bool hit = i < n && order_key(to_f<T>(p[i])) == bound;
    const unsigned votes = __ballot_sync(0xffffffffu, hit);
    __syncthreads();
    if ((t & 31) == 0) sh.warp_count[t >> 5] = __popc(votes);
    __syncthreads();
    int at = got + __popc(votes & ((1u << (t & 31)) - 1));
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < (t >> 5)) at += sh.warp_count[w];
      got += sh.warp_count[w];
    }
    if (hit && at < need) sh.found[have + at] = candidate(bound, i);
  }
  __syncthreads();
  if (t == 0 && need > 0) sh.n_found = k;
  __syncthreads();
}

// This thread's key: the maximum of its part of the row.  A barrier comes
// between this and select_top.
template <typename T, int THREADS>
__device__ __forceinline__ void offer_part(TopkShared<THREADS>& sh, const T* p, int n, float mx) {
  const int t = threadIdx.x;
  const RowShape r = row_shape(p, n);
  const bool any = t < r.nv || t < r.head || t < r.tail;
  sh.keys[t] = any ? order_key(mx) : 0u;
  if (t == 0) sh.n_found = 0;
}

// Candidates for the k largest of the row's n logits (no NaN, not all -inf)
// into sh.found, sh.n_found of them (k at least).
template <typename T, int THREADS>
__device__ __forceinline__ void select_top(TopkShared<THREADS>& sh, const T* p, int n, int k) {
  if (threadIdx.x < 32) find_bound<T, THREADS>(sh, k, false);
  __syncthreads();
  const unsigned bound = sh.bound;
  // Below the key of -inf the bound admits masked logits: the other way takes
  // those in order.
  const bool masked = bound <= order_key(-INFINITY);
  if (!masked) {
    visit_parts<T, THREADS>(sh, p, n, sh.n_hot, key_value(bound), [&](float x, int index) {
      if (*(volatile int*)&sh.n_found <= TS_CAP) keep(sh, order_key(x), index);
    });
    __syncthreads();
    if (sh.n_found <= TS_CAP) return;
  }
  __syncthreads();
  select_top_slow<T, THREADS>(sh, p, n, k, masked);
}

// Calls put(rank, candidate) for the k best candidates.
template <int THREADS, typename Put>
__device__ __forceinline__ void rank_found(const TopkShared<THREADS>& sh, int k, Put put) {
  const int n = sh.n_found;
  for (int c = threadIdx.x; c < n; c += THREADS) {
    const u64 mine = sh.found[c];
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += sh.found[o] > mine;
    if (rank < k) put(rank, mine);
  }
}

// One thread: the numbers of a row from its merged statistics.
template <typename T>
__device__ __forceinline__ void write_scores(const Stats& all, const T* row, long long t, int V,
                                             bool ignored, float inv_t, float* log_prob,
                                             float* entropy, float2* stats, int* status) {
  const float m = finite_max(all.mx);
  float lp = 0.f, h = 0.f;
  if (!ignored) {
    const float log_s = logf(all.s);
    const bool empty = all.s == 0.f;
    if (!empty) h = fmaf(-kLn2, all.sd / all.s, log_s);
    if (t < 0 || t >= V) {
      lp = __int_as_float(0x7fc00000);
      if (status) atomicExch(status, STATUS_BAD_TOKEN);
    } else {
      lp = empty ? -INFINITY : (to_f<T>(row[t]) - m) * inv_t - log_s;
    }
  }
  *log_prob = lp;
  *entropy = h;
  if (stats) *stats = make_float2(m, all.s);
}

template <typename T, int THREADS, bool TOP>
__device__ __forceinline__ void token_scores_rows(
    long long rows, int V, long long ld, const T* __restrict__ logits,
    const int64_t* __restrict__ tokens, long long ignore_index, float inv_t, int k,
    float* __restrict__ log_prob, float* __restrict__ entropy, float2* __restrict__ stats,
    float* __restrict__ top_values, int64_t* __restrict__ top_ids, int* status) {
  __shared__ float part[THREADS / 32][3];
  __shared__ TopkShared<THREADS> top;
  const float c = kLog2e * inv_t;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const long long t = tokens[r];
    if (t == ignore_index) {
      if (threadIdx.x == 0)
        write_scores(Stats(), logits, t, V, true, inv_t, log_prob + r, entropy + r,
                     stats ? stats + r : nullptr, status);
      if (TOP)
        for (int i = threadIdx.x; i < k; i += THREADS) {
          top_values[r * k + i] = -INFINITY;
          top_ids[r * k + i] = -1;
        }
      continue;
    }
    const T* row = logits + (size_t)r * ld;
    const Stats own = sweep<T, THREADS, true, !TOP>(row, V, threadIdx.x, c);
    if (TOP) offer_part<T, THREADS>(top, row, V, own.mx);
    const Stats all = block_merge<THREADS>(own, part, c);
    if (threadIdx.x == 0)
      write_scores(all, row, t, V, false, inv_t, log_prob + r, entropy + r,
                   stats ? stats + r : nullptr, status);
    if (TOP) {
      const float m = finite_max(all.mx), log_s = logf(all.s);
      float* values = top_values + r * k;
      int64_t* ids = top_ids + r * k;
      if (all.s > 0.f) {
        select_top<T, THREADS>(top, row, V, k);
        rank_found<THREADS>(top, k, [&](int rank, u64 best) {
          values[rank] = (key_value((unsigned)(best >> 32)) - m) * inv_t - log_s;
          ids[rank] = candidate_index(best);
        });
      } else {  // all -inf (s == 0), or no order (s is NaN): the first ids
        for (int i = threadIdx.x; i < k; i += THREADS) {
          values[i] = all.s == 0.f ? -INFINITY : all.s;
          ids[i] = i;
        }
      }
    }
    __syncthreads();
  }
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) token_scores_fwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits,
    const int64_t* __restrict__ tokens, long long ignore_index, float inv_t,
    float* __restrict__ log_prob, float* __restrict__ entropy, float2* __restrict__ stats,
    int* status) {
  token_scores_rows<T, THREADS, false>(rows, V, ld, logits, tokens, ignore_index, inv_t, 0,
                                       log_prob, entropy, stats, nullptr, nullptr, status);
}

// 2048 threads an SM: the selection is a chain of short steps between barriers,
// which only other rows can fill.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 2048 / THREADS) token_scores_top_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits,
    const int64_t* __restrict__ tokens, long long ignore_index, float inv_t, int k,
    float* __restrict__ log_prob, float* __restrict__ entropy, float2* __restrict__ stats,
    float* __restrict__ top_values, int64_t* __restrict__ top_ids, int* status) {
  token_scores_rows<T, THREADS, true>(rows, V, ld, logits, tokens, ignore_index, inv_t, k,
                                      log_prob, entropy, stats, top_values, top_ids, status);
}

// Rows short enough for one warp: eight a CTA, no barriers.  2048 FP32 rows of 64
// in 3.4 us forward and 3.2 us back, against 7.4 and 7.2 us with a CTA a row.
constexpr int TS_WARP_BYTES = 2048;

template <typename T>
__global__ void __launch_bounds__(TS_THREADS) token_scores_warp_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits,
    const int64_t* __restrict__ tokens, long long ignore_index, float inv_t,
    float* __restrict__ log_prob, float* __restrict__ entropy, float2* __restrict__ stats,
    int* status) {
  const int lane = threadIdx.x & 31;
  const long long r = (long long)blockIdx.x * (TS_THREADS / 32) + (threadIdx.x >> 5);
  if (r >= rows) return;
  const float c = kLog2e * inv_t;
  const long long t = tokens[r];
  Stats all;
  const T* row = logits + (size_t)r * ld;
  if (t != ignore_index) all = warp_merge(sweep<T, 32, true, true>(row, V, lane, c), c);
  if (lane == 0)
    write_scores(all, row, t, V, t == ignore_index, inv_t, log_prob + r, entropy + r,
                 stats ? stats + r : nullptr, status);
}

// A row to every THREADS threads (a warp or the CTA).
template <typename T, int THREADS, bool HAS_B>
__global__ void __launch_bounds__(TS_THREADS) token_scores_bwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits,
    const int64_t* __restrict__ tokens, long long ignore_index, float inv_t,
    const float2* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ g_log_prob, const float* __restrict__ g_entropy,
    T* __restrict__ dlogits, long long ldd) {
  constexpr int GROUPS = TS_THREADS / THREADS;
  const float c = kLog2e * inv_t;
  const int lane = threadIdx.x % THREADS;
  for (long long r = (long long)blockIdx.x * GROUPS + threadIdx.x / THREADS; r < rows;
       r += (long long)gridDim.x * GROUPS) {
    const T* row = logits + (size_t)r * ld;
    T* drow = dlogits + (size_t)r * ldd;
    const long long t = tokens[r];
    const float2 ms = stats[r];
    const float g = g_log_prob ? g_log_prob[r] * inv_t : 0.f;
    // the log-probability of a token outside the vocabulary is NaN, and so is
    // its gradient
    const bool undefined = t != ignore_index && (t < 0 || t >= V) && g != 0.f;
    if (t == ignore_index || (ms.y == 0.f && !undefined)) {
      // padding, or a row with every logit masked: nothing to learn
      zero_row<T, THREADS>(drow, V, lane);
      continue;
    }
    const float h = HAS_B ? g_entropy[r] * inv_t : 0.f;
    // p_j (log p_j + entropy) = 2^d_j (d_j ln2 - log s + entropy) / s
    const float B = HAS_B ? -h * kLn2 / ms.y : 0.f;
    const float A = undefined ? __int_as_float(0x7fc00000)
                              : -(HAS_B ? fmaf(h, entropy[r] - logf(ms.y), g) : g) / ms.y;
    grad_sweep<T, THREADS, HAS_B>(row, drow, V, lane, ms.x, c, A, B);
    if (t >= 0 && t < V) {
      // the token's element is rounded once, with its own term
      if (THREADS == 32)
        __syncwarp();
      else
        __syncthreads();
      if (lane == 0)
        drow[t] = from_f<T>(grad_value<HAS_B>(to_f<T>(row[t]), ms.x, c, A, B) + g);
    }
  }
}

unsigned row_grid(long long rows) {
  return (unsigned)std::min<long long>(rows, 0x7fffffffLL);
}

unsigned warp_grid(long long rows) {
  return row_grid((rows + TS_THREADS / 32 - 1) / (TS_THREADS / 32));
}

int check_rows(const char* what, int dtype, int64_t rows, int64_t V, int64_t ld,
               float temperature) {
  if (rows < 0 || V <= 0 || V >= INT32_MAX || ld < V) {
    set_error("%s: unsupported sizes rows=%lld V=%lld ld=%lld", what, (long long)rows,
              (long long)V, (long long)ld);
    return DABSN_ERR_SHAPE;
  }
  if (dtype != DABSN_F32 && dtype != DABSN_BF16) {
    set_error("%s: logits must be FP32 or BF16", what);
    return DABSN_ERR_DTYPE;
  }
  if (!(temperature >= 1e-6f && temperature <= 1e6f)) {
    set_error("%s: the temperature must lie in [1e-6, 1e6]", what);
    return DABSN_ERR_UNSUPPORTED;
  }
  return DABSN_OK;
}

template <typename T, int THREADS>
void launch_rows(int64_t rows, int64_t V, int64_t ld, const void* logits, const int64_t* tokens,
                 int64_t ignore_index, float inv_t, int64_t k, float* log_prob, float* entropy,
                 float* stats, float* top_values, int64_t* top_ids, int* status,
                 cudaStream_t st) {
  if (k > 0)
    token_scores_top_kernel<T, THREADS><<<row_grid(rows), THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, (int)k, log_prob,
        entropy, (float2*)stats, top_values, top_ids, status);
  else
    token_scores_fwd_kernel<T, THREADS><<<row_grid(rows), THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, log_prob, entropy,
        (float2*)stats, status);
}

template <typename T>
int launch_fwd(int64_t rows, int64_t V, int64_t ld, const void* logits, const int64_t* tokens,
               int64_t ignore_index, float temperature, int64_t k, float* log_prob,
               float* entropy, float* stats, float* top_values, int64_t* top_ids,
               cudaStream_t st) {
  const float inv_t = 1.f / temperature;
  int* status = device_status();
  if (k == 0 && V * (int64_t)sizeof(T) <= TS_WARP_BYTES)
    token_scores_warp_kernel<T><<<warp_grid(rows), TS_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, log_prob, entropy,
        (float2*)stats, status);
  else if (rows <= TS_FEW_ROWS &&
           V * (int64_t)sizeof(T) > (k > 0 ? TS_FEW_TOP_BYTES : TS_FEW_BYTES))
    launch_rows<T, TS_FEW_THREADS>(rows, V, ld, logits, tokens, ignore_index, inv_t, k,
                                   log_prob, entropy, stats, top_values, top_ids, status, st);
  else
    launch_rows<T, TS_THREADS>(rows, V, ld, logits, tokens, ignore_index, inv_t, k, log_prob,
                               entropy, stats, top_values, top_ids, status, st);
  return launch_status("token_scores_fwd");
}

template <typename T, bool HAS_B>
int launch_bwd(int64_t rows, int64_t V, int64_t ld, const void* logits, const int64_t* tokens,
               int64_t ignore_index, float temperature, const float* stats, const float* entropy,
               const float* g_log_prob, const float* g_entropy, void* dlogits, int64_t ldd,
               cudaStream_t st) {
  const float inv_t = 1.f / temperature;
  if (V * (int64_t)sizeof(T) <= TS_WARP_BYTES)
    token_scores_bwd_kernel<T, 32, HAS_B><<<warp_grid(rows), TS_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, (const float2*)stats,
        entropy, g_log_prob, g_entropy, (T*)dlogits, ldd);
  else
    token_scores_bwd_kernel<T, TS_THREADS, HAS_B><<<row_grid(rows), TS_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, (const float2*)stats,
        entropy, g_log_prob, g_entropy, (T*)dlogits, ldd);
  return launch_status("token_scores_bwd");
}

}  // namespace
}  // namespace dabsn

using namespace dabsn;

extern "C" int dabsn_token_scores_fwd(int dtype, int64_t rows, int64_t V, int64_t ld,
                                      const void* logits, const int64_t* tokens,
                                      int64_t ignore_index, float temperature, int64_t top_k,
                                      float* log_prob, float* entropy, float* stats,
                                      float* top_values, int64_t* top_ids, void* stream) {
  const int bad = check_rows("token_scores_fwd", dtype, rows, V, ld, temperature);
  if (bad) return bad;
  if (top_k < 0 || top_k > TS_MAX_K || top_k > V) {
    set_error("token_scores_fwd: top_k=%lld must lie in [0, min(%d, V)]", (long long)top_k,
              TS_MAX_K);
    return DABSN_ERR_UNSUPPORTED;
  }
  // the selection's scans of a row step past its end by up to a CTA's threads
  if (top_k > 0 && V > INT32_MAX - TS_FEW_THREADS) {
    set_error("token_scores_fwd: V=%lld is too long for alternatives", (long long)V);
    return DABSN_ERR_SHAPE;
  }
  if (rows == 0) return DABSN_OK;
  int null = check_pointers("token_scores_fwd", {logits, tokens, log_prob, entropy});
  if (!null && top_k > 0) null = check_pointers("token_scores_fwd", {top_values, top_ids});
  if (null) return null;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == DABSN_BF16
             ? launch_fwd<bf16>(rows, V, ld, logits, tokens, ignore_index, temperature, top_k,
                                log_prob, entropy, stats, top_values, top_ids, st)
             : launch_fwd<float>(rows, V, ld, logits, tokens, ignore_index, temperature, top_k,
                                 log_prob, entropy, stats, top_values, top_ids, st);
}

extern "C" int dabsn_token_scores_bwd(int dtype, int64_t rows, int64_t V, int64_t ld,
                                      const void* logits, const int64_t* tokens,
                                      int64_t ignore_index, float temperature,
                                      const float* stats, const float* entropy,
                                      const float* g_log_prob, const float* g_entropy,
                                      void* dlogits, int64_t ldd, void* stream) {
  int bad = check_rows("token_scores_bwd", dtype, rows, V, ld, temperature);
  if (!bad)
    bad = check_gradient_rows("token_scores_bwd", dtype, rows, V, ld, logits, ldd, dlogits);
  if (bad) return bad;
  if (rows == 0) return DABSN_OK;
  bad = check_pointers("token_scores_bwd", {logits, tokens, stats, entropy, dlogits});
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DABSN_BF16)
    return g_entropy ? launch_bwd<bf16, true>(rows, V, ld, logits, tokens, ignore_index,
                                              temperature, stats, entropy, g_log_prob, g_entropy,
                                              dlogits, ldd, st)
                     : launch_bwd<bf16, false>(rows, V, ld, logits, tokens, ignore_index,
                                               temperature, stats, entropy, g_log_prob,
                                               g_entropy, dlogits, ldd, st);
  return g_entropy ? launch_bwd<float, true>(rows, V, ld, logits, tokens, ignore_index,
                                             temperature, stats, entropy, g_log_prob, g_entropy,
                                             dlogits, ldd, st)
                   : launch_bwd<float, false>(rows, V, ld, logits, tokens, ignore_index,
                                              temperature, stats, entropy, g_log_prob, g_entropy,
                                              dlogits, ldd, st);
}
