// Distillation from a teacher's top logits, loss and gradient.
//
//   q = softmax(teacher_logits / T) over the entries a row lists,
//   p = softmax(logits / T) over the vocabulary,
//   loss_r = T^2 sum_k q_k (log q_k - log p_id_k),
//   dlogits_j = w_r T (p_j - sum over the entries with id_k = j of q_k)
// for the factor w_r with which the row's loss enters the result.
//
// An entry whose id is ignore_index is absent, so rows may list fewer than K
// entries, and so is one of id -1 with a logit of -inf, which is how token_scores
// leaves the alternatives of a row it ignored; a row without any (or with -inf
// teacher logits throughout) has no loss, no gradient and no part in the mean.
// The lists are small: one warp a row turns them into probabilities once
// (distill_prep), merges an id that is listed twice, and counts the rows: 32768
// lists of 64 in 15 us (8 us of traffic; what it waits for is a list's chain of
// short steps).  What costs is
// the sweep over the student's logits (row_softmax.cuh), one CTA per row: the
// loss alone, of 32768 BF16 rows of 32000 with a twentieth ignored, in 315 us,
// 6.3 TB/s.
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
constexpr int DT_BAD_LIST = 2;  // of Entries::live

// Entry of a row's list after preparation: id (-1: absent), q, and q summed
// over the entries with the same id (at the first of them; 0 at the others; NaN
// among the teacher's logits makes both NaN, and with them loss and gradient).
// A list that names an id outside the vocabulary has no right gradient: its loss
// is NaN and so is its whole row of the gradient, unless the factor with which
// the row enters is 0.
struct Entries {
  int* id;
  float2* q;
  float2* stats;  // [rows] maximum and sum of exponentials of the student's row
  int* live;      // [rows] 0 no loss, 1 a loss, 2 a NaN loss for an id outside
  float* loss;    // [rows] losses, where the caller has no place for them
  int* counts;    // [blocks] live rows of each preparation block
};

int prep_blocks(int64_t rows) {
  const int64_t warps = DT_PREP_THREADS / 32;
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + warps - 1) / warps, 148 * 4));
}

// The workspace of a call, read again by its reverse.
Entries entries_of(void* ws, int64_t rows, int64_t K) {
  Entries e;
  e.q = (float2*)ws;
  e.stats = e.q + rows * K;
  e.id = (int*)(e.stats + rows);
  e.live = e.id + rows * K;
  e.loss = (float*)(e.live + rows);
  e.counts = (int*)(e.loss + rows);
  return e;
}

// One warp a row, PER entries a lane.
template <typename T, int PER>
__global__ void __launch_bounds__(DT_PREP_THREADS) distill_prep_kernel(
    long long rows, int V, int K, const int64_t* __restrict__ ids, const T* __restrict__ logits,
    float inv_t, long long ignore_index, Entries out, int* status) {
  __shared__ int live_rows[DT_PREP_THREADS / 32];
  constexpr int TABLE = 64 * PER;  // two slots an entry
  __shared__ int table[DT_PREP_THREADS / 32][TABLE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long nwarps = (long long)gridDim.x * (DT_PREP_THREADS / 32);
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
      if (k < K) {
        const long long t = ids[r * K + k];
        const float x = to_f<T>(logits[r * K + k]);
        if (t != ignore_index && !(t == -1 && x == -INFINITY)) {
          if (t >= 0 && t < V) {
            id[i] = (int)t;
            q[i] = x;
          } else {
            bad = true;
          }
        }
      }
      m = fmaxf(m, q[i]);
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
    // An id listed twice is rare: a hash table of the row's ids finds out
    // whether there is one, and only then are they merged.
#pragma unroll
    for (int i = 0; i < TABLE / 32; ++i) table[warp][lane + 32 * i] = -1;
    __syncwarp();
    bool twice = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (id[i] < 0) continue;
      unsigned slot = (unsigned)id[i] * 2654435761u >> 16;
      for (int probe = 0; probe < TABLE; ++probe, ++slot) {
        const int had = atomicCAS(&table[warp][slot % TABLE], -1, id[i]);
        if (had == id[i]) twice = true;
        if (had == -1 || had == id[i]) break;
      }
    }
    __syncwarp();
    float all[PER];
    unsigned later = 0u;  // bit i: an earlier entry has id[i]
#pragma unroll
    for (int i = 0; i < PER; ++i) all[i] = q[i];
    if (__any_sync(0xffffffffu, twice)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) all[i] = 0.f;
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
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = lane + 32 * i;
      if (k < K) {
        // a list that names a token outside the vocabulary makes its loss NaN
        const float mine = bad ? __int_as_float(0x7fc00000) : q[i];
        out.id[r * K + k] = id[i];
        out.q[r * K + k] = make_float2(mine, (later >> i) & 1u ? 0.f : all[i]);
      }
    }
    if (lane == 0) out.live[r] = bad ? DT_BAD_LIST : live;
  }
  if (lane == 0) live_rows[warp] = counted;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int w = 0; w < DT_PREP_THREADS / 32; ++w) n += live_rows[w];
    out.counts[blockIdx.x] = n;
  }
}

template <typename T>
void launch_prep(int64_t rows, int64_t V, int64_t K, const int64_t* ids, const void* logits,
                 float inv_t, int64_t ignore_index, const Entries& e, cudaStream_t st) {
  const int grid = prep_blocks(rows);
  int* status = device_status();
#define DISTILL_PREP(PER)                                                          \
  distill_prep_kernel<T, PER><<<grid, DT_PREP_THREADS, 0, st>>>(                   \
      rows, (int)V, (int)K, ids, (const T*)logits, inv_t, ignore_index, e, status)
  if (K <= 32) DISTILL_PREP(1);
  else if (K <= 64) DISTILL_PREP(2);
  else if (K <= 128) DISTILL_PREP(4);
  else DISTILL_PREP(8);
#undef DISTILL_PREP
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

// 1 / the number of rows with a loss.
__device__ __forceinline__ float mean_scale(const int* counts, int blocks) {
  int n = 0;
  for (int i = threadIdx.x & 31; i < blocks; i += 32) n += counts[i];
  n = __reduce_add_sync(0xffffffffu, n);
  return 1.f / (float)max(n, 1);
}

// result = sum of the row losses, in a fixed order and in 64 bits, or their mean
// over the live rows if mean_blocks.  A launch of its own: at the end of the
// persistent kernel below, in its last CTA, the same sum cost that kernel's main
// loop 100 us of 705.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(long long rows,
                                                              const float* __restrict__ loss,
                                                              const int* __restrict__ counts,
                                                              int mean_blocks,
                                                              float* __restrict__ result) {
  __shared__ double sums[32];
  const int t = threadIdx.x;
  double s = 0.;
  for (long long r = t; r < rows; r += 8 * 1024) {
    float v[8];
#pragma unroll
    for (int a = 0; a < 8; ++a) v[a] = r + a * 1024 < rows ? loss[r + a * 1024] : 0.f;
#pragma unroll
    for (int a = 0; a < 8; ++a) s += (double)v[a];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((t & 31) == 0) sums[t >> 5] = s;
  __syncthreads();
  if (t < 32) {
    s = sums[t];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float scale = mean_blocks ? mean_scale(counts, mean_blocks) : 1.f;
    if (t == 0) *result = (float)(s * (double)scale);
  }
}

// What the divergence and its gradient in the logits are multiplied by.
struct Scaling {
  float temperature, weight;
  __device__ __forceinline__ float loss() const { return temperature * temperature * weight; }
  __device__ __forceinline__ float gradient() const { return temperature * weight; }
};

// A of grad_value for a row with the factor w and the sum of exponentials s: p_j w
// is 2^d_j A.  A row with every logit masked (s == 0) has no gradient.
__device__ __forceinline__ float gradient_factor(int live, float w, float s) {
  if (live == DT_BAD_LIST && w != 0.f) return __int_as_float(0x7fc00000);
  return s == 0.f ? 0.f : w / s;
}

// Whether a listed entry changes its element: it has a probability or is NaN.
// In a row with every logit masked NaN alone reaches the gradient.
__device__ __forceinline__ bool entry_counts(int id, float q, bool empty) {
  return id >= 0 && !(q <= 0.f) && (!empty || q != q);
}

template <typename T>
__global__ void __launch_bounds__(DT_THREADS) distill_fwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    Scaling by, float* __restrict__ loss) {
  __shared__ float part[DT_THREADS / 32][3];
  const float inv_t = 1.f / by.temperature, c = kLog2e * inv_t;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    if (!list.live[r]) {
      if (threadIdx.x == 0) {
        loss[r] = 0.f;
        list.stats[r] = make_float2(0.f, 0.f);
      }
      continue;
    }
    const T* row = logits + (size_t)r * ld;
    const Stats all = block_merge<DT_THREADS>(
        sweep<T, DT_THREADS, false, true>(row, V, threadIdx.x, c), part, c);
    const float m = finite_max(all.mx);
    if (threadIdx.x < 32) {
      const float l = warp_sum(list_loss<T, 32>(row, list.id + r * K, list.q + r * K, K,
                                                threadIdx.x, m, inv_t, logf(all.s),
                                                all.s == 0.f));
      if (threadIdx.x == 0) {
        loss[r] = by.loss() * l;
        list.stats[r] = make_float2(m, all.s);
      }
    }
    __syncthreads();
  }
}

// `unless_one`: dlogits holds the gradient for an upstream gradient of 1 already,
// and that (the usual one: nothing behind a mean but backward()) leaves it as it
// is.  Any other starts from the logits again, so that every element is rounded
// once.
template <typename T>
__global__ void __launch_bounds__(DT_THREADS) distill_bwd_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    int mean_blocks, Scaling by, const float* __restrict__ upstream,
    long long ustride, bool unless_one, T* __restrict__ dlogits, long long ldd) {
  if (unless_one && *upstream == 1.f) return;
  const float inv_t = 1.f / by.temperature, c = kLog2e * inv_t;
  const float scale = by.gradient() * (mean_blocks ? mean_scale(list.counts, mean_blocks) : 1.f);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = logits + (size_t)r * ld;
    T* drow = dlogits + (size_t)r * ldd;
    const float2 ms = list.stats[r];
    const int live = list.live[r];
    if (!live) {
      zero_row<T, DT_THREADS>(drow, V, threadIdx.x);
      continue;
    }
    const float w = scale * upstream[r * ustride];
    const float A = gradient_factor(live, w, ms.y);
    grad_sweep<T, DT_THREADS, false>(row, drow, V, threadIdx.x, ms.x, c, A, 0.f);
    __syncthreads();  // listed elements are rounded once, with their own term
    for (int k = threadIdx.x; k < K; k += DT_THREADS) {
      const int id = list.id[r * K + k];
      const float q = list.q[r * K + k].y;
      if (entry_counts(id, q, ms.y == 0.f))
        drow[id] = from_f<T>(fmaf(-w, q, grad_value<false>(to_f<T>(row[id]), ms.x, c, A, 0.f)));
    }
  }
}

// ---------------------------------------------------------------------------
// Small vocabularies: a warp holds a row in registers (four vectors a lane), so
// loss and gradient take one read, and a CTA eight rows.
// ---------------------------------------------------------------------------
template <typename T>
constexpr int warp_row() {
  return 4 * 32 * Vec<T>::N;
}

template <typename T, bool GRAD>
__device__ __forceinline__ void distill_warp_row(long long r, int V, const T* row, int K,
                                                 const Entries& list, Scaling by, float w,
                                                 float* loss, T* drow) {
  const int lane = threadIdx.x & 31;
  const float inv_t = 1.f / by.temperature, c = kLog2e * inv_t;
  const int live = list.live[r];
  if (!live) {
    if (GRAD) zero_row<T, 32>(drow, V, lane);
    if (lane == 0) {
      loss[r] = 0.f;
      list.stats[r] = make_float2(0.f, 0.f);
    }
    return;
  }
  const RowShape s = row_shape(row, V);
  const uint4* pv = reinterpret_cast<const uint4*>(row + s.head);
  uint4 raw[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    constexpr unsigned ni = Vec<T>::kNegInf;
    raw[u] = lane + 32 * u < s.nv ? __ldg(pv + lane + 32 * u) : make_uint4(ni, ni, ni, ni);
  }
  const float head = lane < s.head ? to_f<T>(row[lane]) : -INFINITY;
  const float tail = lane < s.tail ? to_f<T>(row[s.tail0 + lane]) : -INFINITY;
  Stats st;
  add_vectors<T, 4, false>(st, raw, c);
  add_value(st, head, c);
  add_value(st, tail, c);
  st.sd = 0.f;
  st = warp_merge(st, c);
  const float m = finite_max(st.mx);
  const bool empty = st.s == 0.f;
  const float l = warp_sum(list_loss<T, 32>(row, list.id + r * K, list.q + r * K, K, lane, m,
                                            inv_t, logf(st.s), empty));
  if (lane == 0) {
    loss[r] = by.loss() * l;
    list.stats[r] = make_float2(m, st.s);
  }
  if (!GRAD) return;
  const float A = gradient_factor(live, w, st.s);
  const f32x2 m2 = pair(-m, -m), c2 = pair(c, c), A2 = pair(A, A);
  uint4* dv = reinterpret_cast<uint4*>(drow + s.head);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 32 * u < s.nv)
      dv[lane + 32 * u] = grad_vector<T, false>(raw[u], m2, c2, A2, A2);
  if (lane < s.head) drow[lane] = from_f<T>(grad_value<false>(head, m, c, A, 0.f));
  if (lane < s.tail) drow[s.tail0 + lane] = from_f<T>(grad_value<false>(tail, m, c, A, 0.f));
  __syncwarp();  // listed elements are rounded once, with their own term
  for (int k = lane; k < K; k += 32) {
    const int id = list.id[r * K + k];
    const float q = list.q[r * K + k].y;
    if (entry_counts(id, q, empty))
      drow[id] = from_f<T>(fmaf(-w, q, grad_value<false>(to_f<T>(row[id]), m, c, A, 0.f)));
  }
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(DT_THREADS) distill_warp_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    int mean_blocks, Scaling by, float* __restrict__ loss, T* __restrict__ dlogits,
    long long ldd) {
  const long long r = (long long)blockIdx.x * (DT_THREADS / 32) + (threadIdx.x >> 5);
  const float w =
      GRAD ? by.gradient() * (mean_blocks ? mean_scale(list.counts, mean_blocks) : 1.f) : 0.f;
  if (r < rows)
    distill_warp_row<T, GRAD>(r, V, logits + (size_t)r * ld, K, list, by, w, loss,
                              GRAD ? dlogits + (size_t)r * ldd : nullptr);
}

// ---------------------------------------------------------------------------
// Loss and gradient with one read of the logits from memory (weights known
// beforehand: the sum or the mean of the rows' losses, upstream gradient 1).
// What bounds it is HBM: V read and V written a row.
//
// Rows of up to 72 KB stay in shared memory between their statistics and their
// gradient, three CTAs an SM: every thread copies its own vectors into its own
// slots (cp.async), so neither sweep waits for another thread's copies, and the
// copies of the next row are issued slot by slot as the gradient of this one
// leaves them: reads, arithmetic and writes of neighbouring rows overlap.
// Longer rows, and rows too few to fill the SMs that way, are read a second
// time out of L2 (distill_long_kernel): two CTAs of 1024 threads an SM keep at
// most 296 rows in flight, 76 MB of BF16 rows of 128000.  32768 BF16 rows of
// 32000: 700 us the first way (630 us of traffic at the copy rate), 715 us the
// second; 515 of 128000: 70 us the second way, 87 us with a row shared by the
// shared memory of a cluster of four CTAs.
// ---------------------------------------------------------------------------
constexpr int DF_THREADS = 256;
constexpr int DF_ROW_BYTES = 72 * 1024;
static_assert(DT_MAX_K <= DF_THREADS, "a thread holds at most one entry");

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}

// Waits until at most `pending` of this thread's latest groups of copies are
// under way (more strictly where that is over 7).
__device__ __forceinline__ void cp_async_wait_for(int pending) {
  switch (pending) {
    case 0: cp_async_wait<0>(); break;
    case 1: cp_async_wait<1>(); break;
    case 2: cp_async_wait<2>(); break;
    case 3: cp_async_wait<3>(); break;
    case 4: cp_async_wait<4>(); break;
    case 5: cp_async_wait<5>(); break;
    case 6: cp_async_wait<6>(); break;
    default: cp_async_wait<7>(); break;
  }
}

// A bound of two CTAs an SM leaves the compiler 64 and 74 registers, with which
// three still fit (697 us; 703 us with 58 and 66).  Handing the rows out one at a
// time instead of in equal shares changed nothing (705 us).
template <typename T>
__global__ void __launch_bounds__(DF_THREADS, 2) distill_grad_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    int mean_blocks, Scaling by, float* __restrict__ loss, T* __restrict__ dlogits,
    long long ldd) {
  extern __shared__ uint4 slots[];  // [vectors of a thread][DF_THREADS]
  __shared__ float part[DF_THREADS / 32][3];
  __shared__ float loss_part[DF_THREADS / 32];
  const int t = threadIdx.x;
  const long long stride = gridDim.x;
  const float inv_t = 1.f / by.temperature, c = kLog2e * inv_t;
  const float w = by.gradient() * (mean_blocks ? mean_scale(list.counts, mean_blocks) : 1.f);
  // Vectors of a row at most (rows of other alignments have one less).  Copies
  // are committed in groups of four vectors a thread, as many for every row, so
  // that the statistics start on the first while the last are under way.
  const int most = V / Vec<T>::N;
  const int groups = (most + 4 * DF_THREADS - 1) / (4 * DF_THREADS);

  // The next row from r on that has a loss; the others' gradient is zero.
  auto next_live = [&](long long r) {
    while (r < rows && !list.live[r]) {
      zero_row<T, DF_THREADS>(dlogits + (size_t)r * ldd, V, t);
      if (t == 0) {
        loss[r] = 0.f;
        list.stats[r] = make_float2(0.f, 0.f);
      }
      r += stride;
    }
    return r;
  };

  long long r = next_live(blockIdx.x);
  float edge[2] = {0.f, 0.f};  // this thread's head and tail element
  auto load_edges = [&](const T* p, const RowShape& s) {
    if (t < s.head) edge[0] = to_f<T>(p[t]);
    if (t < s.tail) edge[1] = to_f<T>(p[s.tail0 + t]);
  };
  if (r < rows) {
    const T* p = logits + (size_t)r * ld;
    const RowShape s = row_shape(p, V);
    const uint4* v = reinterpret_cast<const uint4*>(p + s.head);
    for (int k0 = 0; k0 < most; k0 += 4 * DF_THREADS) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = k0 + u * DF_THREADS + t;
        if (k < s.nv) cp_async16(&slots[k], v + k);
      }
      cp_async_commit();
    }
    load_edges(p, s);
  }
  while (r < rows) {
    const T* row = logits + (size_t)r * ld;
    const RowShape s = row_shape(row, V);
    const int live = list.live[r];
    int id = -1;
    float2 q = make_float2(0.f, 0.f);
    float x = 0.f;
    if (t < K) {
      id = list.id[r * K + t];
      q = list.q[r * K + t];
      if (id >= 0) x = to_f<T>(row[id]);
    }
    Stats st;
    for (int g = 0; g < groups; ++g) {
      cp_async_wait_for(groups - 1 - g);
      const int k = g * 4 * DF_THREADS + t;
      if (k + 3 * DF_THREADS < s.nv) {
        const uint4 raw[4] = {slots[k], slots[k + DF_THREADS], slots[k + 2 * DF_THREADS],
                              slots[k + 3 * DF_THREADS]};
        add_vectors<T, 4, false>(st, raw, c);
      } else {
        for (int i = k; i < s.nv; i += DF_THREADS) {
          const uint4 raw[1] = {slots[i]};
          add_vectors<T, 1, false>(st, raw, c);
        }
      }
    }
    if (t < s.head) add_value(st, edge[0], c);
    if (t < s.tail) add_value(st, edge[1], c);
    st.sd = 0.f;
    st = block_merge<DF_THREADS>(st, part, c);
    const float m = finite_max(st.mx);
    const bool empty = st.s == 0.f;
    float l = 0.f;
    if (q.x != q.x) l = q.x;
    if (id >= 0 && q.x > 0.f)
      l = q.x * (logf(q.x) - (empty ? -INFINITY : (x - m) * inv_t - logf(st.s)));
    l = warp_sum(l);
    if ((t & 31) == 0) loss_part[t >> 5] = l;

    // gradient, and the next row's copies
    const float A = gradient_factor(live, w, st.s);
    const long long rn = next_live(r + stride);
    const T* pn = logits + (size_t)(rn < rows ? rn : r) * ld;
    RowShape sn = row_shape(pn, V);
    if (rn >= rows) sn.nv = sn.head = sn.tail = 0;
    const uint4* nv = reinterpret_cast<const uint4*>(pn + sn.head);
    T* drow = dlogits + (size_t)r * ldd;
    uint4* dv = reinterpret_cast<uint4*>(drow + s.head);
    {
      const f32x2 m2 = pair(-m, -m), c2 = pair(c, c), A2 = pair(A, A);
      const int least = min(s.nv, sn.nv);
      for (int g = 0; g < groups; ++g) {
        const int k = g * 4 * DF_THREADS + t;
        if (k + 3 * DF_THREADS < least) {
          uint4 raw[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) raw[u] = slots[k + u * DF_THREADS];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = k + u * DF_THREADS;
            dv[i] = grad_vector<T, false>(raw[u], m2, c2, A2, A2);
            cp_async16(&slots[i], nv + i);
          }
        } else {
          for (int i = k; i < min(k + 4 * DF_THREADS, most); i += DF_THREADS) {
            if (i < s.nv) dv[i] = grad_vector<T, false>(slots[i], m2, c2, A2, A2);
            if (i < sn.nv) cp_async16(&slots[i], nv + i);
          }
        }
        cp_async_commit();
      }
      if (t < s.head)
        drow[t] = from_f<T>(grad_value<false>(edge[0], m, c, A, 0.f));
      if (t < s.tail)
        drow[s.tail0 + t] = from_f<T>(grad_value<false>(edge[1], m, c, A, 0.f));
      load_edges(pn, sn);
    }
    __syncthreads();  // listed elements are rounded once, with their own term
    if (entry_counts(id, q.y, empty))
      drow[id] = from_f<T>(fmaf(-w, q.y, grad_value<false>(x, m, c, A, 0.f)));
    if (t == 0) {
      l = 0.f;
      for (int i = 0; i < DF_THREADS / 32; ++i) l += loss_part[i];
      loss[r] = by.loss() * l;
      list.stats[r] = make_float2(m, st.s);
    }
    r = rn;
  }
}

constexpr int DF_LONG_THREADS = 1024;

template <typename T>
__global__ void __launch_bounds__(DF_LONG_THREADS, 2) distill_long_kernel(
    long long rows, int V, long long ld, const T* __restrict__ logits, int K, Entries list,
    int mean_blocks, Scaling by, float* __restrict__ loss, T* __restrict__ dlogits,
    long long ldd) {
  __shared__ float part[DF_LONG_THREADS / 32][3];
  const int t = threadIdx.x;
  const float inv_t = 1.f / by.temperature, c = kLog2e * inv_t;
  const long long r = blockIdx.x;
  const T* row = logits + (size_t)r * ld;
  T* drow = dlogits + (size_t)r * ldd;
  const int live = list.live[r];
  if (!live) {
    zero_row<T, DF_LONG_THREADS>(drow, V, t);
    if (t == 0) {
      loss[r] = 0.f;
      list.stats[r] = make_float2(0.f, 0.f);
    }
    return;
  }
  const Stats all = block_merge<DF_LONG_THREADS>(
      sweep<T, DF_LONG_THREADS, false, false>(row, V, t, c), part, c);
  const float m = finite_max(all.mx);
  const bool empty = all.s == 0.f;
  const float w = by.gradient() * (mean_blocks ? mean_scale(list.counts, mean_blocks) : 1.f);
  const float A = gradient_factor(live, w, all.s);
  grad_sweep<T, DF_LONG_THREADS, false>(row, drow, V, t, m, c, A, 0.f);
  if (t < 32) {
    const float l = warp_sum(list_loss<T, 32>(row, list.id + r * K, list.q + r * K, K, t, m,
                                              inv_t, logf(all.s), empty));
    if (t == 0) {
      loss[r] = by.loss() * l;
      list.stats[r] = make_float2(m, all.s);
    }
  }
  __syncthreads();  // listed elements are rounded once, with their own term
  for (int k = t; k < K; k += DF_LONG_THREADS) {
    const int id = list.id[r * K + k];
    const float q = list.q[r * K + k].y;
    if (entry_counts(id, q, empty))
      drow[id] = from_f<T>(fmaf(-w, q, grad_value<false>(to_f<T>(row[id]), m, c, A, 0.f)));
  }
}

int check_distill(const char* what, int dtype, int64_t rows, int64_t V, int64_t ld, int64_t K,
                  float temperature) {
  if (rows < 0 || rows > INT32_MAX || V <= 0 || V >= INT32_MAX || ld < V) {
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
  if (!(temperature >= 1e-6f && temperature <= 1e6f)) {
    set_error("%s: the temperature must lie in [1e-6, 1e6]", what);
    return DABSN_ERR_UNSUPPORTED;
  }
  return DABSN_OK;
}

unsigned row_grid(long long rows) { return (unsigned)std::min<long long>(rows, 0x7fffffffLL); }

}  // namespace
}  // namespace dabsn

using namespace dabsn;

namespace {

template <typename T>
int fwd(int64_t rows, int64_t V, int64_t ld, const void* logits, int64_t K, const Entries& e,
        Scaling by, float* row_loss, cudaStream_t st) {
  if (V <= warp_row<T>()) {
    const int64_t grid = (rows + DT_THREADS / 32 - 1) / (DT_THREADS / 32);
    distill_warp_kernel<T, false><<<(unsigned)grid, DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, (int)K, e, 0, by, row_loss, nullptr, 0);
  } else {
    distill_fwd_kernel<T><<<row_grid(rows), DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, (int)K, e, by, row_loss);
  }
  return launch_status("distill_fwd");
}

template <typename T>
int grad(int64_t rows, int64_t V, int64_t ld, const void* logits, int64_t K, const Entries& e,
         Scaling by, int mean_blocks, float* row_loss, void* dlogits, int64_t ldd,
         cudaStream_t st) {
  if (V <= warp_row<T>()) {
    const int64_t grid = (rows + DT_THREADS / 32 - 1) / (DT_THREADS / 32);
    distill_warp_kernel<T, true><<<(unsigned)grid, DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, (int)K, e, mean_blocks, by, row_loss,
        (T*)dlogits, ldd);
    return launch_status("distill_grad");
  }
  const int64_t unit = DF_THREADS * 16;
  const int64_t smem = (V * (int64_t)sizeof(T) + unit - 1) / unit * unit;
  if (smem > DF_ROW_BYTES || rows <= 2 * 148) {
    distill_long_kernel<T><<<row_grid(rows), DF_LONG_THREADS, 0, st>>>(
        rows, (int)V, ld, (const T*)logits, (int)K, e, mean_blocks, by, row_loss,
        (T*)dlogits, ldd);
    return launch_status("distill_grad");
  }
  if (!kernel_prepared((const void*)distill_grad_kernel<T>, DF_ROW_BYTES))
    return DABSN_ERR_LAUNCH;
  const int64_t grid = std::min<int64_t>(rows, 3 * 148);
  distill_grad_kernel<T><<<(unsigned)grid, DF_THREADS, smem, st>>>(
      rows, (int)V, ld, (const T*)logits, (int)K, e, mean_blocks, by, row_loss,
      (T*)dlogits, ldd);
  return launch_status("distill_grad");
}

}  // namespace

extern "C" size_t dabsn_distill_workspace(int64_t rows, int64_t K) {
  if (rows < 0 || K < 1) return 0;
  return (size_t)rows * K * 12 + (size_t)rows * 16 + (size_t)prep_blocks(rows) * 4;
}

extern "C" int dabsn_distill_fwd(int dtype, int64_t rows, int64_t V, int64_t ld,
                                 const void* logits, int teacher_dtype, int64_t K,
                                 const int64_t* teacher_tokens, const void* teacher_logits,
                                 int64_t ignore_index, float temperature, float weight, int mean,
                                 void* workspace, float* row_loss, float* result, void* dlogits,
                                 int64_t ldd, void* stream) {
  int bad = check_distill("distill_fwd", dtype, rows, V, ld, K, temperature);
  if (!bad && teacher_dtype != DABSN_F32 && teacher_dtype != DABSN_BF16) {
    set_error("distill_fwd: the teacher's logits must be FP32 or BF16");
    bad = DABSN_ERR_DTYPE;
  }
  if (!bad && dlogits) {
    bad = check_gradient_rows("distill_fwd", dtype, rows, V, ld, logits, ldd, dlogits);
    if (!bad && !result) {
      set_error("distill_fwd: a gradient needs the result it belongs to");
      bad = DABSN_ERR_UNSUPPORTED;
    }
  }
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (result) cudaMemsetAsync(result, 0, sizeof(float), st);
    return result ? launch_status("distill_fwd") : DABSN_OK;
  }
  bad = check_pointers("distill_fwd", {logits, teacher_tokens, teacher_logits, workspace});
  if (bad) return bad;
  const Entries e = entries_of(workspace, rows, K);
  if (!row_loss) row_loss = e.loss;
  if (teacher_dtype == DABSN_BF16)
    launch_prep<bf16>(rows, V, K, teacher_tokens, teacher_logits, 1.f / temperature,
                      ignore_index, e, st);
  else
    launch_prep<float>(rows, V, K, teacher_tokens, teacher_logits, 1.f / temperature,
                       ignore_index, e, st);
  int status = launch_status("distill_prep");
  if (status) return status;
  const int mb = mean ? prep_blocks(rows) : 0;
  const bool bf = dtype == DABSN_BF16;
  const Scaling by = {temperature, weight};
  if (dlogits)
    status = bf ? grad<bf16>(rows, V, ld, logits, K, e, by, mb, row_loss, dlogits, ldd, st)
                : grad<float>(rows, V, ld, logits, K, e, by, mb, row_loss, dlogits, ldd, st);
  else
    status = bf ? fwd<bf16>(rows, V, ld, logits, K, e, by, row_loss, st)
                : fwd<float>(rows, V, ld, logits, K, e, by, row_loss, st);
  if (status || !result) return status;
  distill_reduce_kernel<<<1, 1024, 0, st>>>(rows, row_loss, e.counts, mb, result);
  return launch_status("distill_reduce");
}

extern "C" int dabsn_distill_bwd(int dtype, int64_t rows, int64_t V, int64_t ld,
                                 const void* logits, int64_t K, const void* workspace,
                                 float temperature, float weight, int mean,
                                 const float* upstream, int64_t upstream_stride, int unless_one,
                                 void* dlogits, int64_t ldd, void* stream) {
  int bad = check_distill("distill_bwd", dtype, rows, V, ld, K, temperature);
  if (!bad) bad = check_gradient_rows("distill_bwd", dtype, rows, V, ld, logits, ldd, dlogits);
  if (bad) return bad;
  if (unless_one && upstream_stride != 0) {
    set_error("distill_bwd: unless_one takes one upstream gradient for all rows");
    return DABSN_ERR_UNSUPPORTED;
  }
  if (rows == 0) return DABSN_OK;
  bad = check_pointers("distill_bwd", {logits, workspace, upstream, dlogits});
  if (bad) return bad;
  const Entries e = entries_of(const_cast<void*>(workspace), rows, K);
  cudaStream_t st = (cudaStream_t)stream;
  const int mb = mean ? prep_blocks(rows) : 0;
  // a launch that mostly finds nothing to do stays one wave of CTAs
  const unsigned grid =
      unless_one ? (unsigned)std::min<int64_t>(rows, 148 * 8) : row_grid(rows);
  const Scaling by = {temperature, weight};
  if (dtype == DABSN_BF16)
    distill_bwd_kernel<bf16><<<grid, DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const bf16*)logits, (int)K, e, mb, by, upstream, upstream_stride,
        unless_one != 0, (bf16*)dlogits, ldd);
  else
    distill_bwd_kernel<float><<<grid, DT_THREADS, 0, st>>>(
        rows, (int)V, ld, (const float*)logits, (int)K, e, mb, by, upstream, upstream_stride,
        unless_one != 0, (float*)dlogits, ldd);
  return launch_status("distill_bwd");
}
