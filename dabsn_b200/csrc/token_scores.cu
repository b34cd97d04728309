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
// of exponentials and the sum that the entropy needs (row_softmax.cuh).  The
// alternatives come out of the same pass: every thread knows the maximum of
// the part of the row it read, the k-th largest of those maxima bounds the
// row's k-th largest logit from below, and only the parts whose maximum
// reaches that bound (about k of THREADS) are read again, out of L2.
// A row whose token is ignore_index is not read.
#include <algorithm>

#include "../../include/dabsn_b200.h"
#include "common.cuh"
#include "row_softmax.cuh"

namespace dabsn {
namespace {

using namespace rowsm;
typedef unsigned long long u64;

constexpr int TS_THREADS = 256;
constexpr int TS_MAX_K = 128;
constexpr int TS_CAP = 512;  // candidates above the bound, and as many equal to it
constexpr int STATUS_BAD_TOKEN = 8;

// Order of the alternatives as unsigned keys: larger logit, larger key; -0
// equals +0; NaN is above everything; 0 is below every logit.
__device__ __forceinline__ unsigned order_key(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __float_as_uint(x + 0.f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
  if (k == 0xffffffffu) return __int_as_float(0x7fc00000);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// One candidate: larger is better; equal logits rank by the lower index.
__device__ __forceinline__ u64 candidate(unsigned key, int index) {
  return ((u64)key << 32) | (unsigned)~index;
}

struct TopkShared {
  unsigned keys[TS_THREADS];
  short hot[TS_THREADS];
  u64 above[TS_CAP], equal[TS_CAP];
  int n_above, n_equal, n_hot;
  unsigned bound;
  int warp_count[TS_THREADS / 32];
};

// The k-th largest of the threads' keys, found bit by bit by one warp (0 when
// fewer than k threads have any element: everything is a candidate then).
__device__ __forceinline__ unsigned kth_key(const unsigned* keys, int k) {
  constexpr int PER = TS_THREADS / 32;
  const int lane = threadIdx.x & 31;
  unsigned own[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) own[i] = keys[lane + 32 * i];
  unsigned t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned cand = t | (1u << bit);
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += own[i] >= cand;
    if (__reduce_add_sync(0xffffffffu, n) >= k) t = cand;
  }
  return t;
}

__device__ __forceinline__ void offer(TopkShared& sh, unsigned bound, float x, int index) {
  const unsigned key = order_key(x);
  if (key > bound) {
    const int at = atomicAdd(&sh.n_above, 1);
    if (at < TS_CAP) sh.above[at] = candidate(key, index);
  } else if (key == bound) {
    if (*(volatile int*)&sh.n_equal <= TS_CAP) {
      const int at = atomicAdd(&sh.n_equal, 1);
      if (at < TS_CAP) sh.equal[at] = candidate(key, index);
    }
  }
}

// Offers every element of the row that a thread of `hot` read in the sweep.
template <typename T>
__device__ __forceinline__ void offer_parts(TopkShared& sh, unsigned bound, const T* p, int n,
                                            int n_hot) {
  constexpr int VW = Vec<T>::N;
  const RowShape r = row_shape(p, n);
  const uint4* pv = reinterpret_cast<const uint4*>(p + r.head);
  const int per = (r.nv + TS_THREADS - 1) / TS_THREADS;
  for (int e = threadIdx.x; e < n_hot * per; e += TS_THREADS) {
    const int k = sh.hot[e / per] + (e % per) * TS_THREADS;
    if (k >= r.nv) continue;
    f32x2 v[VW / 2];
    unpack<T>(__ldg(pv + k), v);
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) {
      const float2 x = split(v[j]);
      offer(sh, bound, x.x, r.head + k * VW + 2 * j);
      offer(sh, bound, x.y, r.head + k * VW + 2 * j + 1);
    }
  }
  for (int e = threadIdx.x; e < n_hot; e += TS_THREADS) {
    const int t = sh.hot[e];
    if (t < r.head) offer(sh, bound, to_f<T>(p[t]), t);
    if (t < r.tail) offer(sh, bound, to_f<T>(p[r.tail0 + t]), r.tail0 + t);
  }
}

// The row's k largest logits into sh.above / sh.equal (n_above and n_equal of
// them, at least k together); `mx` is the maximum of this thread's part.
template <typename T>
__device__ void select_top(TopkShared& sh, const T* p, int n, int k, float mx) {
  const int t = threadIdx.x;
  const RowShape r = row_shape(p, n);
  const bool any = t < r.nv || t < r.head || t < r.tail;
  const unsigned key = any ? order_key(mx) : 0u;
  sh.keys[t] = key;
  if (t == 0) sh.n_above = sh.n_equal = sh.n_hot = 0;
  __syncthreads();
  if (t < 32) {
    const unsigned b = kth_key(sh.keys, k);
    if (t == 0) sh.bound = b;
  }
  __syncthreads();
  unsigned bound = sh.bound;
  if (any && key >= bound) sh.hot[atomicAdd(&sh.n_hot, 1)] = (short)t;
  __syncthreads();
  offer_parts<T>(sh, bound, p, n, sh.n_hot);
  __syncthreads();
  if (sh.n_above > TS_CAP) {
    // A row built against the bound: find its exact k-th largest key, by bits,
    // over the whole row, and take what lies above it (fewer than k).
    bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned cand = bound | (1u << bit);
      __syncthreads();
      if (t == 0) sh.n_above = 0;
      __syncthreads();
      int c = 0;
      for (int i = t; i < n; i += TS_THREADS) c += order_key(to_f<T>(p[i])) >= cand;
      c = __reduce_add_sync(0xffffffffu, c);
      if ((t & 31) == 0) atomicAdd(&sh.n_above, c);
      __syncthreads();
      if (sh.n_above >= k) bound = cand;
    }
    __syncthreads();
    if (t == 0) sh.n_above = sh.n_equal = 0;
    __syncthreads();
    for (int i = t; i < n; i += TS_THREADS) offer(sh, bound, to_f<T>(p[i]), i);
    __syncthreads();
  }
  const int need = k - sh.n_above;
  if (need > 0 && sh.n_equal > TS_CAP) {
    // More logits equal to the bound than were kept (a masked row with fewer
    // than k logits left, a flat row): the lowest indices, in order.
    int found = 0;
    for (int base = 0; base < n && found < need; base += TS_THREADS) {
      const int i = base + t;
      const bool hit = i < n && order_key(to_f<T>(p[i])) == bound;
      const unsigned votes = __ballot_sync(0xffffffffu, hit);
      __syncthreads();
      if ((t & 31) == 0) sh.warp_count[t >> 5] = __popc(votes);
      __syncthreads();
      int at = found + __popc(votes & ((1u << (t & 31)) - 1));
      for (int w = 0; w < TS_THREADS / 32; ++w) {
        if (w < (t >> 5)) at += sh.warp_count[w];
        found += sh.warp_count[w];
      }
      if (hit && at < need) sh.equal[at] = candidate(bound, i);
    }
    __syncthreads();
    if (t == 0) sh.n_equal = need;
    __syncthreads();
  }
}

// Ranks the candidates and stores the first k: ids, and log-probabilities
// (x - m) inv_t - log_s.
__device__ __forceinline__ void store_top(const TopkShared& sh, int k, float m, float inv_t,
                                          float log_s, bool empty, float* values, int64_t* ids) {
  const int na = sh.n_above, ne = na >= k ? 0 : sh.n_equal;
  for (int c = threadIdx.x; c < na + ne; c += TS_THREADS) {
    const u64 mine = c < na ? sh.above[c] : sh.equal[c - na];
    int rank = 0;
    for (int o = 0; o < na; ++o) rank += sh.above[o] > mine;
    for (int o = 0; o < ne; ++o) rank += sh.equal[o] > mine;
    if (rank < k) {
      const float x = key_value((unsigned)(mine >> 32));
      values[rank] = empty ? -INFINITY : (x - m) * inv_t - log_s;
      ids[rank] = (int64_t)(unsigned)~(unsigned)mine;
    }
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

template <typename T, bool TOP>
__global__ void __launch_bounds__(TS_THREADS) token_scores_fwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits,
    const int64_t* __restrict__ tokens, long long ignore_index, float inv_t, int k,
    float* __restrict__ log_prob, float* __restrict__ entropy, float2* __restrict__ stats,
    float* __restrict__ top_values, int64_t* __restrict__ top_ids, int* status) {
  __shared__ float part[TS_THREADS / 32][3];
  __shared__ TopkShared top;
  const float c = kLog2e * inv_t;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const long long t = tokens[r];
    if (t == ignore_index) {
      if (threadIdx.x == 0)
        write_scores(Stats(), logits, t, V, true, inv_t, log_prob + r, entropy + r,
                     stats ? stats + r : nullptr, status);
      if (TOP)
        for (int i = threadIdx.x; i < k; i += TS_THREADS) {
          top_values[r * k + i] = -INFINITY;
          top_ids[r * k + i] = -1;
        }
      continue;
    }
    const T* row = logits + (size_t)r * ld;
    const Stats own = sweep<T, TS_THREADS, true>(row, V, threadIdx.x, c);
    const Stats all = block_merge<TS_THREADS>(own, part, c);
    if (threadIdx.x == 0)
      write_scores(all, row, t, V, false, inv_t, log_prob + r, entropy + r,
                   stats ? stats + r : nullptr, status);
    if (TOP) {
      select_top<T>(top, row, V, k, own.mx);
      store_top(top, k, finite_max(all.mx), inv_t, logf(all.s), all.s == 0.f,
                top_values + r * k, top_ids + r * k);
    }
    __syncthreads();
  }
}

// Rows short enough for one warp: eight a CTA, no barriers.
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
  if (t != ignore_index) all = warp_merge(sweep<T, 32, true>(row, V, lane, c), c);
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
    if (t == ignore_index || ms.y == 0.f) {
      // padding, or a row with every logit masked: nothing to learn
      zero_row<T, THREADS>(drow, V, lane);
      continue;
    }
    const float g = g_log_prob ? g_log_prob[r] * inv_t : 0.f;
    const float h = HAS_B ? g_entropy[r] * inv_t : 0.f;
    // p_j (log p_j + entropy) = 2^d_j (d_j ln2 - log s + entropy) / s
    const float B = HAS_B ? -h * kLn2 / ms.y : 0.f;
    const float A = -(HAS_B ? fmaf(h, entropy[r] - logf(ms.y), g) : g) / ms.y;
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
  if (!(temperature > 0.f) || temperature == INFINITY) {
    set_error("%s: the temperature must be positive and finite", what);
    return DABSN_ERR_UNSUPPORTED;
  }
  return DABSN_OK;
}

template <typename T>
int launch_fwd(int64_t rows, int64_t V, int64_t ld, const void* logits, const int64_t* tokens,
               int64_t ignore_index, float temperature, int64_t k, float* log_prob,
               float* entropy, float* stats, float* top_values, int64_t* top_ids,
               cudaStream_t st) {
  const float inv_t = 1.f / temperature;
  int* status = device_status();
  if (k > 0)
    token_scores_fwd_kernel<T, true><<<row_grid(rows), TS_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, (int)k, log_prob,
        entropy, (float2*)stats, top_values, top_ids, status);
  else if (V * sizeof(T) <= TS_WARP_BYTES)
    token_scores_warp_kernel<T><<<warp_grid(rows), TS_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, log_prob, entropy,
        (float2*)stats, status);
  else
    token_scores_fwd_kernel<T, false><<<row_grid(rows), TS_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, tokens, ignore_index, inv_t, 0, log_prob, entropy,
        (float2*)stats, nullptr, nullptr, status);
  return launch_status("token_scores_fwd");
}

template <typename T, bool HAS_B>
int launch_bwd(int64_t rows, int64_t V, int64_t ld, const void* logits, const int64_t* tokens,
               int64_t ignore_index, float temperature, const float* stats, const float* entropy,
               const float* g_log_prob, const float* g_entropy, void* dlogits, int64_t ldd,
               cudaStream_t st) {
  const float inv_t = 1.f / temperature;
  if (V * sizeof(T) <= TS_WARP_BYTES)
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
  if (rows == 0) return DABSN_OK;
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
