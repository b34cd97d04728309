// Distillation from a teacher's top logits, loss and gradient.
//
//   q = softmax(teacher_logits / T) over the entries a row lists,
//   p = softmax(logits / T) over the vocabulary,
//   loss_r = T^2 sum_k q_k (log q_k - log p_id_k),
//   dlogits_j = w_r T (p_j - sum over the entries with id_k = j of q_k)
// for the weight w_r with which the row's loss enters the result.
//
// An entry whose id is ignore_index is absent, so rows may list fewer than K
// entries; a row without any (or with -inf teacher logits throughout) has no
// loss, no gradient and no part in the mean.  The lists are small: one warp a
// row turns them into probabilities once (distill_prep), merges an id that is
// listed twice, and counts the rows.  What costs is the sweep over the student's logits
// (row_softmax.cuh), one CTA per row.
#include <algorithm>

#include "../../include/dabsn_b200.h"
#include "common.cuh"
#include "row_softmax.cuh"

namespace dabsn {
namespace {

using namespace rowsm;

constexpr int DT_THREADS = 256;
constexpr int DT_MAX_K = 256;
constexpr int DT_PREP_THREADS = 512;
constexpr int DT_STATUS_BAD_TOKEN = 8;

// Entry of a row's list after preparation: id (-1: absent), q, and q summed
// over the entries with the same id (at the first of them; 0 at the others).
struct Entries {
  int* id;
  float2* q;
  int* live;    // [rows] 1 where the row has a loss
  int* counts;  // [blocks] live rows of each preparation block
};

int prep_blocks(int64_t rows) {
  const int64_t warps = DT_PREP_THREADS / 32;
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + warps - 1) / warps, 148));
}

Entries entries_of(void* ws, int64_t rows, int64_t K) {
  Entries e;
  e.q = (float2*)ws;
  e.id = (int*)(e.q + rows * K);
  e.live = e.id + rows * K;
  e.counts = e.live + rows;
  return e;
}

template <typename T>
__global__ void __launch_bounds__(DT_PREP_THREADS) distill_prep_kernel(
    long long rows, int V, int K, const int64_t* __restrict__ ids, const T* __restrict__ logits,
    float inv_t, long long ignore_index, Entries out, int* status) {
  constexpr int PER = DT_MAX_K / 32;
  __shared__ int live_rows[DT_PREP_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long nwarps = (long long)gridDim.x * (DT_PREP_THREADS / 32);
  const int per = (K + 31) / 32;
  int counted = 0;
  for (long long r = (long long)blockIdx.x * (DT_PREP_THREADS / 32) + warp; r < rows;
       r += nwarps) {
    int id[PER];
    float q[PER];
    float m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      id[i] = -1;
      q[i] = -INFINITY;
      const int k = lane + 32 * i;
      if (i < per && k < K) {
        const long long t = ids[r * K + k];
        if (t != ignore_index) {
          if (t >= 0 && t < V) {
            id[i] = (int)t;
            q[i] = to_f<T>(logits[r * K + k]);
            m = fmaxf(m, q[i]);
          } else {
            bad = true;
          }
        }
      }
    }
    m = finite_max(warp_max(m));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      q[i] = id[i] < 0 ? 0.f : expf((q[i] - m) * inv_t);
      sum += q[i];
    }
    sum = warp_sum(sum);
    bad = __any_sync(0xffffffffu, bad);
    const bool live = bad || !(sum == 0.f);
    counted += live;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (bad && status && lane == 0) atomicExch(status, DT_STATUS_BAD_TOKEN);
#pragma unroll
    for (int i = 0; i < PER; ++i) q[i] *= inv;
    // merge equal ids into the first of them
    float all[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) all[i] = 0.f;
    unsigned later = 0u;  // bit i: an earlier entry has id[i]
    for (int k = 0; k < K; ++k) {
      int other = 0;
      float oq = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int v = __shfl_sync(0xffffffffu, id[i], k & 31);
        const float w = __shfl_sync(0xffffffffu, q[i], k & 31);
        if (i == (k >> 5)) {
          other = v;
          oq = w;
        }
      }
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (id[i] == other) {
          all[i] += oq;
          if (k < lane + 32 * i) later |= 1u << i;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = lane + 32 * i;
      if (i < per && k < K) {
        // a list that names a token outside the vocabulary makes its loss NaN
        const float mine = bad ? __int_as_float(0x7fc00000) : q[i];
        out.id[r * K + k] = id[i];
        out.q[r * K + k] = make_float2(mine, (later >> i) & 1u ? 0.f : all[i]);
      }
    }
    if (lane == 0) out.live[r] = live;
  }
  if (lane == 0) live_rows[warp] = counted;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int w = 0; w < DT_PREP_THREADS / 32; ++w) n += live_rows[w];
    out.counts[blockIdx.x] = n;
  }
}

// sum_k q_k (log q_k - log p_id_k) over the entries of this thread.
template <typename T, int THREADS>
__device__ __forceinline__ float list_loss(const T* row, const int* id, const float2* q, int K,
                                           int t, float m, float inv_t, float log_s, bool empty) {
  float loss = 0.f;
  for (int k = t; k < K; k += THREADS) {
    const float w = q[k].x;
    if (w != w) loss = w;
    if (id[k] < 0 || !(w > 0.f)) continue;
    const float lp = empty ? -INFINITY : (to_f<T>(row[id[k]]) - m) * inv_t - log_s;
    loss += w * (logf(w) - lp);
  }
  return loss;
}

template <typename T>
__global__ void __launch_bounds__(DT_THREADS) distill_fwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    float temperature, float* __restrict__ loss, float2* __restrict__ stats) {
  __shared__ float part[DT_THREADS / 32][3];
  const float inv_t = 1.f / temperature, c = kLog2e * inv_t;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    if (!list.live[r]) {
      if (threadIdx.x == 0) {
        loss[r] = 0.f;
        if (stats) stats[r] = make_float2(0.f, 0.f);
      }
      continue;
    }
    const T* row = logits + (size_t)r * ld;
    const Stats all =
        block_merge<DT_THREADS>(sweep<T, DT_THREADS>(row, V, threadIdx.x, c), part, c);
    const float m = finite_max(all.mx);
    if (threadIdx.x < 32) {
      const float l = warp_sum(list_loss<T, 32>(row, list.id + r * K, list.q + r * K, K,
                                                threadIdx.x, m, inv_t, logf(all.s),
                                                all.s == 0.f));
      if (threadIdx.x == 0) {
        loss[r] = temperature * temperature * l;
        if (stats) stats[r] = make_float2(m, all.s);
      }
    }
    __syncthreads();
  }
}

// weight[r * wstride] * (1 / live rows if `mean`) is the weight of row r.
__device__ __forceinline__ float mean_scale(const int* counts, int blocks) {
  int n = 0;
  for (int i = threadIdx.x & 31; i < blocks; i += 32) n += counts[i];
  n = __reduce_add_sync(0xffffffffu, n);
  return 1.f / (float)max(n, 1);
}

template <typename T, bool SAME>
__global__ void __launch_bounds__(DT_THREADS) distill_bwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    int mean_blocks, float temperature, const float2* __restrict__ stats,
    const float* __restrict__ weight, long long wstride, T* __restrict__ dlogits) {
  const float inv_t = 1.f / temperature, c = kLog2e * inv_t;
  const float scale = temperature * (mean_blocks ? mean_scale(list.counts, mean_blocks) : 1.f);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = logits + (size_t)r * ld;
    T* drow = dlogits + (size_t)r * V;
    const float2 ms = stats[r];
    if (!list.live[r] || ms.y == 0.f) {
      zero_row<T, DT_THREADS>(drow, V, threadIdx.x);
      continue;
    }
    const float w = scale * weight[r * wstride];
    const float A = w / ms.y;
    grad_sweep<T, DT_THREADS, false, SAME>(row, drow, V, threadIdx.x, ms.x, c, A, 0.f);
    __syncthreads();  // listed elements are rounded once, with their own term
    for (int k = threadIdx.x; k < K; k += DT_THREADS) {
      const int id = list.id[r * K + k];
      const float q = list.q[r * K + k].y;
      if (id >= 0 && q > 0.f)
        drow[id] = from_f<T>(grad_value<false>(to_f<T>(row[id]), ms.x, c, A, 0.f) - w * q);
    }
  }
}

// result = sum of the row losses (times 1 / live rows if mean_blocks), in a
// fixed order.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(long long rows,
                                                              const float* __restrict__ loss,
                                                              const int* __restrict__ counts,
                                                              int mean_blocks,
                                                              float* __restrict__ result) {
  __shared__ double sh[32];
  double s = 0.;
  for (long long r = threadIdx.x; r < rows; r += 1024) s += (double)loss[r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = sh[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float scale = mean_blocks ? mean_scale(counts, mean_blocks) : 1.f;
    if (threadIdx.x == 0) *result = (float)(s * (double)scale);
  }
}

int check_distill(const char* what, int dtype, int64_t rows, int64_t V, int64_t ld, int64_t K,
                  float temperature) {
  if (rows < 0 || V <= 0 || V >= INT32_MAX || ld < V) {
    set_error("%s: unsupported sizes rows=%lld V=%lld ld=%lld", what, (long long)rows,
              (long long)V, (long long)ld);
    return DABSN_ERR_SHAPE;
  }
  if (K < 1 || K > DT_MAX_K) {
    set_error("%s: %lld entries a row; supported are 1 to %d", what, (long long)K, DT_MAX_K);
    return DABSN_ERR_UNSUPPORTED;
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

unsigned row_grid(long long rows) { return (unsigned)std::min<long long>(rows, 0x7fffffffLL); }

}  // namespace
}  // namespace dabsn

using namespace dabsn;

extern "C" size_t dabsn_distill_list_bytes(int64_t rows, int64_t K) {
  if (rows < 0 || K < 1) return 0;
  return (size_t)rows * K * 12 + (size_t)rows * 4 + (size_t)prep_blocks(rows) * 4;
}

extern "C" int dabsn_distill_prep(int teacher_dtype, int64_t rows, int64_t V, int64_t K,
                                  const int64_t* teacher_tokens, const void* teacher_logits,
                                  float temperature, int64_t ignore_index, void* list,
                                  void* stream) {
  const int bad = check_distill("distill_prep", teacher_dtype, rows, V, V, K, temperature);
  if (bad) return bad;
  if (rows == 0) {
    const Entries e = entries_of(list, 0, K);
    cudaMemsetAsync(e.counts, 0, sizeof(int), (cudaStream_t)stream);
    return launch_status("distill_prep");
  }
  const Entries e = entries_of(list, rows, K);
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = prep_blocks(rows);
  if (teacher_dtype == DABSN_BF16)
    distill_prep_kernel<bf16><<<grid, DT_PREP_THREADS, 0, st>>>(
        rows, (int)V, (int)K, teacher_tokens, (const bf16*)teacher_logits, 1.f / temperature,
        ignore_index, e, device_status());
  else
    distill_prep_kernel<float><<<grid, DT_PREP_THREADS, 0, st>>>(
        rows, (int)V, (int)K, teacher_tokens, (const float*)teacher_logits, 1.f / temperature,
        ignore_index, e, device_status());
  return launch_status("distill_prep");
}

extern "C" int dabsn_distill_fwd(int dtype, int64_t rows, int64_t V, int64_t ld,
                                 const void* logits, int64_t K, const void* list,
                                 float temperature, float* row_loss, float* stats, void* stream) {
  const int bad = check_distill("distill_fwd", dtype, rows, V, ld, K, temperature);
  if (bad) return bad;
  if (rows == 0) return DABSN_OK;
  const Entries e = entries_of(const_cast<void*>(list), rows, K);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DABSN_BF16)
    distill_fwd_kernel<bf16><<<row_grid(rows), DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const bf16*)logits, (int)K, e, temperature, row_loss, (float2*)stats);
  else
    distill_fwd_kernel<float><<<row_grid(rows), DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const float*)logits, (int)K, e, temperature, row_loss,
        (float2*)stats);
  return launch_status("distill_fwd");
}

extern "C" int dabsn_distill_bwd(int dtype, int64_t rows, int64_t V, int64_t ld,
                                 const void* logits, int64_t K, const void* list,
                                 float temperature, const float* stats, int mean,
                                 const float* weight, int64_t weight_stride, void* dlogits,
                                 void* stream) {
  const int bad = check_distill("distill_bwd", dtype, rows, V, ld, K, temperature);
  if (bad) return bad;
  if (rows == 0) return DABSN_OK;
  const Entries e = entries_of(const_cast<void*>(list), rows, K);
  cudaStream_t st = (cudaStream_t)stream;
  const int mb = mean ? prep_blocks(rows) : 0;
  const unsigned grid = row_grid(rows);
  const bool bf = dtype == DABSN_BF16;
  const bool same = same_phase(logits, ld, dlogits, V, bf ? 2 : 4);
#define DISTILL_BWD(T, SAME)                                                                  \
  distill_bwd_kernel<T, SAME><<<grid, DT_THREADS, 0, st>>>(                                   \
      rows, (int)V, ld, (const T*)logits, (int)K, e, mb, temperature, (const float2*)stats,   \
      weight, weight_stride, (T*)dlogits)
  if (bf && same) DISTILL_BWD(bf16, true);
  else if (bf) DISTILL_BWD(bf16, false);
  else if (same) DISTILL_BWD(float, true);
  else DISTILL_BWD(float, false);
#undef DISTILL_BWD
  return launch_status("distill_bwd");
}

extern "C" int dabsn_distill_reduce(int64_t rows, int64_t K, const float* row_loss,
                                    const void* list, int mean, float* result, void* stream) {
  if (rows < 0 || K < 1 || K > DT_MAX_K) {
    set_error("distill_reduce: bad sizes rows=%lld K=%lld", (long long)rows, (long long)K);
    return DABSN_ERR_SHAPE;
  }
  const Entries e = entries_of(const_cast<void*>(list), rows, K);
  distill_reduce_kernel<<<1, 1024, 0, (cudaStream_t)stream>>>(
      rows, row_loss, e.counts, mean ? prep_blocks(rows) : 0, result);
  return launch_status("distill_reduce");
}
