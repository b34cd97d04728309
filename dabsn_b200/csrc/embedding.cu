// Scaled embedding lookup and the gradient of its table.
//
//   out[i, :] = scale * weight[token_i, :]            (rounded once, to out's type)
//   dweight[v, :] = scale * sum over i with token_i = v of dout[i, :]
//
// Both are bound by memory: the lookup writes N x D and reads the rows used,
// the gradient reads N x D and writes the whole table (zeros where no token
// points).  The gradient's sums run over the tokens sorted by id, positions
// ascending inside an id, so no atomics are needed: a stable radix sort of (id,
// position), digits of at most eight bits, then one sum per run of equal ids in
// FP32, rounded once to the table's type.  A long run is summed in pieces, which
// are added up in an order of their own; the tokens alone fix it, so the result is
// the same every time.
//
// Tokens outside [0, V) give NaN rows and status 8, and take no part in the
// gradient; nor do tokens equal to the padding id.
#include <algorithm>

#include "../../include/dabsn_b200.h"
#include "common.cuh"

namespace dabsn {
namespace {

typedef __nv_bfloat16 bf16;

constexpr int EM_THREADS = 256;
constexpr int EM_STATUS_BAD_TOKEN = 8;
constexpr int64_t EM_MAX_N = INT32_MAX - (1 << 16);  // positions are 32-bit, with a chunk to spare

// Eight consecutive elements as FP32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<bf16>(const bf16* p, float (&v)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<bf16>(bf16* p, const float (&v)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = u;
}

// W elements at p: an aligned vector (W = 8, or 4) or one element (W = 1).
template <int W, typename T>
__device__ __forceinline__ void load_w(const T* p, float (&v)[W]) {
  if constexpr (W == 8) {
    load8<T>(p, v);
  } else if constexpr (W == 4) {
    static_assert(sizeof(T) == 4, "16 bytes");
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    v[0] = to_f<T>(__ldg(p));
  }
}
template <int W, typename T>
__device__ __forceinline__ void store_w(T* p, const float (&v)[W]) {
  if constexpr (W == 8) {
    store8<T>(p, v);
  } else if constexpr (W == 4 && sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else if constexpr (W == 4) {
    uint2 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
    h[0] = __floats2bfloat162_rn(v[0], v[1]);
    h[1] = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = u;
  } else {
    p[0] = from_f<T>(v[0]);
  }
}

// A 16-byte vector (or one element) as it was loaded, and as FP32.
template <int W, typename T>
struct Raw {
  alignas(W * sizeof(T)) T v[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (W > 1) {
      static_assert(W * sizeof(T) == 16, "16 bytes");
      *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(p));  // read once
    } else {
      v[0] = __ldg(p);
    }
  }
  __device__ __forceinline__ float at(int i) const { return to_f<T>(v[i]); }
};
static_assert(alignof(Raw<4, float>) == 16 && alignof(Raw<8, bf16>) == 16,
              "written as one vector, wherever the compiler keeps it");

// ---------------------------------------------------------------------------
// Lookup: each CTA copies a group of rows, a thread per unit.  131072 Zipf rows
// of 2048, FP32 to BF16, in 121 us (100 us of traffic at the copy rate) with one
// unit in flight a thread, eight CTAs an SM and eight units a thread; 127 us with
// four units a thread, 178 us with one, and 158 us with two or four in flight at
// four CTAs an SM.
// ---------------------------------------------------------------------------
template <typename TW, typename TO, int W>
__global__ void __launch_bounds__(EM_THREADS) embedding_fwd_kernel(
    long long N, int V, int units, int group, const int64_t* __restrict__ tokens,
    const TW* __restrict__ weight, long long ldw, float scale, TO* __restrict__ out,
    int* status) {
  const long long r0 = (long long)blockIdx.x * group;
  const int here = (int)min((long long)group, N - r0);
  for (int e = threadIdx.x; e < here * units; e += EM_THREADS) {
    const int i = e / units, u = e - i * units;
    const long long r = r0 + i;
    const long long t = tokens[r];
    float v[W];
    if (t >= 0 && t < V) {
      load_w<W, TW>(weight + (size_t)t * ldw + (size_t)u * W, v);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] *= scale;
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = __int_as_float(0x7fc00000);
      if (u == 0 && status) atomicExch(status, EM_STATUS_BAD_TOKEN);
    }
    store_w<W, TO>(out + ((size_t)r * units + u) * W, v);
  }
}

// ---------------------------------------------------------------------------
// Stable radix sort of (id, position).  A block owns a contiguous tile of the
// input; one launch counts its digits, the next places its elements after
// those of smaller digits and of earlier blocks.
// ---------------------------------------------------------------------------
constexpr int RS_ITEMS = 4;  // 131072 tokens in 18 us; 20 us with 8, 27 us with 16
constexpr int RS_UNIT = EM_THREADS * RS_ITEMS;  // elements ranked at a time
constexpr int RS_MAX_BLOCKS = 256;
constexpr int RS_DIGITS = 256;
constexpr int RS_WARPS = EM_THREADS / 32;

struct SortPlan {
  int blocks, tile, passes, bits;
};

SortPlan sort_plan(int64_t N, int64_t V) {
  SortPlan p;
  const int64_t units = std::max<int64_t>(1, (N + RS_UNIT - 1) / RS_UNIT);
  const int64_t per = (units + RS_MAX_BLOCKS - 1) / RS_MAX_BLOCKS;
  p.tile = (int)std::min<int64_t>(per * RS_UNIT, 0x7fffffff / RS_UNIT * RS_UNIT);
  p.blocks = (int)((units + per - 1) / per);
  int nbits = 1;
  while ((int64_t(1) << nbits) <= V) ++nbits;  // ids 0 .. V, V for those left out
  p.passes = (nbits + 7) / 8;
  p.bits = (nbits + p.passes - 1) / p.passes;
  return p;
}

struct SortSpace {
  int* key[2];
  int* pos[2];
  int* hist;  // [blocks][RS_DIGITS]
};

SortSpace sort_space(void* ws, int64_t N) {
  SortSpace s;
  int* p = (int*)ws;
  for (int i = 0; i < 2; ++i) {
    s.key[i] = p;
    s.pos[i] = p + N;
    p += 2 * N;
  }
  s.hist = p;
  return s;
}

// What the first pass sorts by: the id, or V for an element left out.
__device__ __forceinline__ int sort_key(long long t, int V, long long padding) {
  return t < 0 || t >= V || t == padding ? V : (int)t;
}

// The lanes whose digit (of `bits` bits) is this lane's, of those that have one,
// by a ballot a bit: sorting 8192 tokens in one CTA takes 16 us with it and 20 us
// with __match_any_sync.
__device__ __forceinline__ unsigned same_digit(int digit, int bits, bool in) {
  unsigned peers = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    if (b >= bits) break;
    const bool one = digit >> b & 1;
    const unsigned votes = __ballot_sync(0xffffffffu, one);
    peers &= one ? votes : ~votes;
  }
  return peers;
}

template <bool FIRST>
__global__ void __launch_bounds__(EM_THREADS) sort_count_kernel(
    int N, int V, long long padding, int tile, int shift, int mask,
    const int64_t* __restrict__ tokens, const int* __restrict__ key, int* __restrict__ hist) {
  __shared__ int count[RS_DIGITS];
  for (int d = threadIdx.x; d < RS_DIGITS; d += EM_THREADS) count[d] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * tile;
  const long long last = min(first + tile, (long long)N);
  for (long long i = first + threadIdx.x; i < last; i += EM_THREADS) {
    const int k = FIRST ? sort_key(tokens[i], V, padding) : key[i];
    atomicAdd(&count[(k >> shift) & mask], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < RS_DIGITS; d += EM_THREADS)
    hist[blockIdx.x * RS_DIGITS + d] = count[d];
}

template <bool FIRST>
__global__ void __launch_bounds__(EM_THREADS) sort_place_kernel(
    int N, int V, long long padding, int tile, int shift, int bits,
    const int64_t* __restrict__ tokens, const int* __restrict__ key, const int* __restrict__ pos,
    const int* __restrict__ hist, int* __restrict__ key_out, int* __restrict__ pos_out) {
  static_assert(RS_DIGITS == EM_THREADS, "one digit per thread");
  __shared__ int next[RS_DIGITS];              // where the digit's next element goes
  __shared__ int offset[RS_WARPS][RS_DIGITS];  // counts, then places, of each warp
  __shared__ int warp_total[RS_WARPS];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, mask = (1 << bits) - 1;
  {
    int before = 0, total = 0;
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int n = hist[b * RS_DIGITS + t];
      if (b < (int)blockIdx.x) before += n;
      total += n;
    }
    int scan = total;  // inclusive over the digits of this warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    int base = scan - total;
    for (int w = 0; w < warp; ++w) base += warp_total[w];
    next[t] = base + before;
  }
  const long long first = (long long)blockIdx.x * tile;
  const long long last = min(first + tile, (long long)N);
  for (long long unit = first; unit < last; unit += RS_UNIT) {
    for (int w = 0; w < RS_WARPS; ++w) offset[w][t] = 0;
    __syncthreads();
    // a warp ranks 32 * RS_ITEMS consecutive elements, 32 at a time, in order
    int k[RS_ITEMS], rank[RS_ITEMS];
#pragma unroll
    for (int j = 0; j < RS_ITEMS; ++j) {
      const long long i = unit + warp * (32 * RS_ITEMS) + j * 32 + lane;
      k[j] = i < last ? (FIRST ? sort_key(tokens[i], V, padding) : key[i]) : -1;
    }
#pragma unroll
    for (int j = 0; j < RS_ITEMS; ++j) {
      const bool in = k[j] >= 0;
      const int digit = (k[j] >> shift) & mask;
      const unsigned peers = same_digit(digit, bits, in);
      const int seen = in ? offset[warp][digit] : 0;
      rank[j] = seen + __popc(peers & ((1u << lane) - 1));
      __syncwarp();
      if (in && (peers >> lane) == 1u) offset[warp][digit] = seen + __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    {
      int at = next[t];
      for (int w = 0; w < RS_WARPS; ++w) {
        const int n = offset[w][t];
        offset[w][t] = at;
        at += n;
      }
      next[t] = at;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RS_ITEMS; ++j) {
      if (k[j] < 0) continue;
      const long long i = unit + warp * (32 * RS_ITEMS) + j * 32 + lane;
      const int dst = offset[warp][(k[j] >> shift) & mask] + rank[j];
      key_out[dst] = k[j];
      pos_out[dst] = FIRST ? (int)i : pos[i];
    }
    __syncthreads();
  }
}

// The whole sort of up to RS_SMALL tokens in one CTA and one launch, passes
// through shared memory: 4099 tokens of 1009 in 11 us, as long as the four
// launches of two passes take on the device, and three launches' work less for
// the host, which is what calls of this size wait for.
constexpr int RS_SMALL_THREADS = 1024;
constexpr int RS_SMALL_ITEMS = 8;
constexpr int RS_SMALL = RS_SMALL_THREADS * RS_SMALL_ITEMS;
constexpr int RS_SMALL_WARPS = RS_SMALL_THREADS / 32;
constexpr int RS_SMALL_ROW = RS_DIGITS + 1;  // the rows of counts start in other banks
constexpr int RS_SMALL_SMEM = (2 * RS_SMALL + RS_SMALL_WARPS * RS_SMALL_ROW) * (int)sizeof(int);

__global__ void __launch_bounds__(RS_SMALL_THREADS) sort_small_kernel(
    int N, int V, long long padding, int passes, int bits, const int64_t* __restrict__ tokens,
    int* __restrict__ key_out, int* __restrict__ pos_out) {
  extern __shared__ int small[];
  int* key = small;                    // [RS_SMALL]
  int* pos = small + RS_SMALL;         // [RS_SMALL]
  int* offset = small + 2 * RS_SMALL;  // [RS_SMALL_WARPS][RS_SMALL_ROW]
  static_assert(RS_SMALL_THREADS == 4 * RS_DIGITS, "four threads a digit");
  __shared__ int warp_total[RS_SMALL_WARPS];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  // as few items a thread as hold the input, a warp's consecutive
  const int items = (N + RS_SMALL_THREADS - 1) / RS_SMALL_THREADS;
  int* mine = offset + warp * RS_SMALL_ROW;
  int k[RS_SMALL_ITEMS], p[RS_SMALL_ITEMS], rank[RS_SMALL_ITEMS];
#pragma unroll
  for (int j = 0; j < RS_SMALL_ITEMS; ++j) {
    p[j] = (warp * items + j) * 32 + lane;
    k[j] = j < items && p[j] < N ? sort_key(tokens[p[j]], V, padding) : -1;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits, mask = (1 << bits) - 1;
    for (int d = t; d < RS_SMALL_WARPS * RS_SMALL_ROW; d += RS_SMALL_THREADS) offset[d] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RS_SMALL_ITEMS; ++j) {
      if (j >= items) break;
      const bool in = k[j] >= 0;
      const int digit = (k[j] >> shift) & mask;
      const unsigned peers = same_digit(digit, bits, in);
      const int seen = in ? mine[digit] : 0;
      rank[j] = seen + __popc(peers & ((1u << lane) - 1));
      __syncwarp();
      if (in && (peers >> lane) == 1u) mine[digit] = seen + __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    // four threads a digit, each a quarter of the warps
    constexpr int QUARTER = RS_SMALL_WARPS / 4;
    int* column = offset + (t & 3) * QUARTER * RS_SMALL_ROW + (t >> 2);
    int n[QUARTER], sum = 0;
#pragma unroll
    for (int w = 0; w < QUARTER; ++w) {
      n[w] = column[w * RS_SMALL_ROW];
      sum += n[w];
    }
    int scan = sum;  // over the digits and quarters before this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    if (warp == 0) {
      int all = warp_total[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, all, o);
        if (lane >= o) all += v;
      }
      warp_total[lane] = all;
    }
    __syncthreads();
    int at = scan - sum + (warp > 0 ? warp_total[warp - 1] : 0);
#pragma unroll
    for (int w = 0; w < QUARTER; ++w) {
      column[w * RS_SMALL_ROW] = at;
      at += n[w];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RS_SMALL_ITEMS; ++j) {
      if (j >= items || k[j] < 0) continue;
      const int dst = mine[(k[j] >> shift) & mask] + rank[j];
      key[dst] = k[j];
      pos[dst] = p[j];
    }
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int j = 0; j < RS_SMALL_ITEMS; ++j) {
        const int i = (warp * items + j) * 32 + lane;
        const bool in = j < items && i < N;
        k[j] = in ? key[i] : -1;
        p[j] = in ? pos[i] : 0;
      }
      __syncthreads();
    }
  }
  for (int i = t; i < N; i += RS_SMALL_THREADS) {
    key_out[i] = key[i];
    pos_out[i] = pos[i];
  }
}

// First sorted element whose key is not below v.
__device__ __forceinline__ int lower_bound(const int* key, int N, int v) {
  int lo = 0, hi = N;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (key[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// Sums over runs of equal ids.  Token frequencies are skewed (the first of
// 32000 Zipf tokens has a seventh of all positions), so the work is cut along
// the sorted positions, not along the ids: a group of threads sums the runs that
// begin in a chunk of them, one 16-byte unit of the columns a thread.  A run that
// ends in the next chunk is summed to its end by the chunk it begins in.  A
// longer one, which covers a chunk whole, leaves an FP32 partial sum in each
// chunk it touches, and the join adds those up in order.
// ---------------------------------------------------------------------------
// 131072 Zipf tokens of 32000, width 2048, BF16 gradients into an FP32 table:
// 141 us for the runs and the absent rows, 17 us for the join (122 us of traffic
// at the copy rate), 18 us for the sort.  One CTA per table row took 7000 us.
struct GradPlan {
  int chunk, chunks;   // sorted positions in a chunk, number of chunks
  int units;           // of the columns
  int wide, tiles;     // units that a group covers, column tiles
  int groups;          // chunks that a CTA works on side by side
  int blocks;          // CTAs for the chunks (x tiles), before those for absent rows
  int zero_blocks;
};

constexpr int GR_CHUNK_MAX = 64;
constexpr int GR_ZERO_ROWS = 32;
constexpr int GR_JOIN_UNITS = 32;
constexpr int GR_JOIN_CHUNKS = 8;
constexpr int GR_JOIN_AHEAD = 4;  // partial sums in flight a thread
constexpr int GR_POSITIONS = 2048;  // of the chunks of a CTA, at most

GradPlan grad_plan(int64_t N, int64_t V, int units) {
  GradPlan g;
  g.units = units;
  g.tiles = (units + EM_THREADS - 1) / EM_THREADS;
  g.wide = (units + g.tiles - 1) / g.tiles;
  // Longer chunks leave fewer partial sums, shorter ones more groups for a small
  // call.  Runs and join with 32 and 64, Zipf tokens: 32000 x 2048 BF16, 61 and 69
  // us for 8192 tokens, 65 and 67 for 16384, 80 and 76 for 32768, 169 and 161 for
  // 131072; 32000 x 512 FP32, 25 and 35, 28 and 37, 35 and 38, 80 and 70; 1009 x
  // 515 FP32, 21 and 28, 30 and 35, 48 and 46, 154 and 131.
  g.chunk = N >= 32768 ? GR_CHUNK_MAX : 32;
  g.groups = std::min(EM_THREADS / g.wide, GR_POSITIONS / GR_CHUNK_MAX);
  g.chunks = (int)((N + g.chunk - 1) / g.chunk);
  g.blocks = (g.chunks + g.groups - 1) / g.groups;
  g.zero_blocks = (int)((V + GR_ZERO_ROWS - 1) / GR_ZERO_ROWS);
  return g;
}

template <typename TG, typename TW, int W>
__global__ void __launch_bounds__(EM_THREADS, 4) embedding_grad_kernel(
    int N, int V, GradPlan g, const int* __restrict__ key, const int* __restrict__ pos,
    const TG* __restrict__ dout, float scale, TW* __restrict__ dweight,
    float* __restrict__ partial) {
  constexpr int AHEAD = 8;  // gradient rows in flight
  const int t = threadIdx.x;
  if ((int)blockIdx.x >= g.blocks) {
    // rows that no token points at
    __shared__ bool absent[GR_ZERO_ROWS];
    const int v0 = ((int)blockIdx.x - g.blocks) * GR_ZERO_ROWS;
    if (t < GR_ZERO_ROWS) {
      const int v = v0 + t;
      const int at = v < V ? lower_bound(key, N, v) : 0;
      absent[t] = v < V && (at >= N || key[at] != v);
    }
    __syncthreads();
    const float zero[W] = {};
    const int u0 = blockIdx.y * g.wide, u1 = min(u0 + g.wide, g.units);
    for (int r = 0; r < GR_ZERO_ROWS; ++r) {
      if (!absent[r]) continue;
      for (int u = u0 + t; u < u1; u += EM_THREADS)
        store_w<W, TW>(dweight + ((size_t)(v0 + r) * g.units + u) * W, zero);
    }
    return;
  }
  // the keys and positions of the CTA's chunks, and of the chunk after them;
  // the keys from a chunk (and one) before them
  __shared__ int keys[GR_POSITIONS + 2 * GR_CHUNK_MAX + 2];
  __shared__ int places[GR_POSITIONS + GR_CHUNK_MAX];
  const int c0 = blockIdx.x * g.groups * g.chunk;
  const int count = min((g.groups + 1) * g.chunk, N - c0);
  for (int i = t; i < (g.groups + 2) * g.chunk + 2; i += EM_THREADS) {
    const int at = c0 - g.chunk - 1 + i;
    keys[i] = at >= 0 && at < N ? key[at] : -1;
  }
  for (int i = t; i < count; i += EM_THREADS) places[i] = pos[c0 + i];
  __syncthreads();
  const int group = t / g.wide;
  const int chunk = blockIdx.x * g.groups + group;
  const int u = blockIdx.y * g.wide + t % g.wide;
  if (group >= g.groups || chunk >= g.chunks || u >= g.units) return;
  const int C = g.chunk;
  const int* k = keys + C + 1 + group * C;  // this chunk's keys; from k[-C - 1] to k[2 * C]
  const int* place = places + group * C;
  const int end = min(C, N - chunk * C);    // of the chunk
  // A run that comes in from the chunk before and began there ends there for
  // this chunk, if it ends here; the same for the run that leaves this chunk.
  int from = 0, to = end;
  bool came = k[0] == k[-1], leaves = k[end - 1] == k[end];  // as a partial sum
  if (came && k[-C - 1] != k[0] && !(k[end - 1] == k[0] && leaves)) {
    came = false;
    while (from < end && k[from] == k[-1]) ++from;
    if (from == end) return;
  }
  if (leaves && !(k[0] == k[end - 1] && k[-1] == k[0])) {
    // it begins here; does it end in the next chunk?
    const int far = min(2 * C, N - chunk * C);
    if (k[far - 1] != k[end - 1] || k[far] != k[end - 1]) {
      leaves = false;
      while (to < far && k[to] == k[end - 1]) ++to;
    }
  }
  int cur = k[from];
  bool first = true;
  float sum[W];
#pragma unroll
  for (int j = 0; j < W; ++j) sum[j] = 0.f;
  auto flush = [&](bool last) {
    if (cur >= V) return;
    if ((first && came) || (last && leaves)) {
      store_w<W, float>(partial + ((size_t)chunk * 2 + (first && came ? 0 : 1)) * g.units * W +
                            (size_t)u * W,
                        sum);
    } else {
      float out[W];
#pragma unroll
      for (int j = 0; j < W; ++j) out[j] = sum[j] * scale;
      store_w<W, TW>(dweight + ((size_t)cur * g.units + u) * W, out);
    }
  };
  const TG* column = dout + (size_t)u * W;
  for (int i = from; i < to && cur < V; i += AHEAD) {
    Raw<W, TG> v[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
      if (i + a < to) v[a].load(column + (size_t)place[i + a] * g.units * W);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a >= to) break;
      if (k[i + a] != cur) {
        flush(false);
        first = false;
        cur = k[i + a];
        if (cur >= V) break;
#pragma unroll
        for (int j = 0; j < W; ++j) sum[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < W; ++j) sum[j] += v[a].at(j);
    }
  }
  flush(true);
}

// One CTA per GR_JOIN_CHUNKS chunks and tile of GR_JOIN_UNITS units: for every
// run that begins in one of the chunks and covers the next one whole, adds up
// its partial sums (slot 1 where it begins, slot 0 where it goes on).  Eight
// threads share a unit, each every eighth partial.
template <typename TW, int W>
__global__ void __launch_bounds__(EM_THREADS) embedding_join_kernel(
    int N, int V, GradPlan g, const int* __restrict__ key, const float* __restrict__ partial,
    float scale, TW* __restrict__ dweight) {
  constexpr int SLICES = EM_THREADS / GR_JOIN_UNITS;
  __shared__ float sh[SLICES][GR_JOIN_UNITS * W];
  __shared__ int begins[GR_JOIN_CHUNKS];  // id of the long run that begins there, or -1
  if (threadIdx.x < GR_JOIN_CHUNKS) {
    const int chunk = blockIdx.x * GR_JOIN_CHUNKS + threadIdx.x;
    int id = -1;
    if (chunk < g.chunks) {
      const long long i0 = (long long)chunk * g.chunk, i1 = i0 + g.chunk, i2 = i1 + g.chunk;
      if (i2 < N) {
        const int first = key[i0], before = i0 > 0 ? key[i0 - 1] : -1;
        const int last = key[i1 - 1], next = key[i1], far = key[i2 - 1], over = key[i2];
        // leaves this chunk, covers the next and goes on, and began here
        if (last < V && last == next && last == far && last == over &&
            !(first == last && before == last))
          id = last;
      }
    }
    begins[threadIdx.x] = id;
  }
  __syncthreads();
  const int lane = threadIdx.x % GR_JOIN_UNITS, slice = threadIdx.x / GR_JOIN_UNITS;
  const int u = blockIdx.y * GR_JOIN_UNITS + lane;
  const bool in = u < g.units;
  for (int b = 0; b < GR_JOIN_CHUNKS; ++b) {
    const int id = begins[b], chunk = blockIdx.x * GR_JOIN_CHUNKS + b;
    if (id < 0) continue;
    // chunks it goes on into: those that begin with its id, EM_THREADS of them
    // looked at in one round trip
    int n = 0;
    for (int c = chunk + 1;; c += EM_THREADS) {
      const long long at = ((long long)c + threadIdx.x) * g.chunk;
      const int found = __syncthreads_count(at < N && key[at] == id);
      n += found;
      if (found < EM_THREADS) break;
    }
    float sum[W];
#pragma unroll
    for (int k = 0; k < W; ++k) sum[k] = 0.f;
    for (int j0 = slice; in && j0 <= n; j0 += GR_JOIN_AHEAD * SLICES) {
      float v[GR_JOIN_AHEAD][W];
#pragma unroll
      for (int a = 0; a < GR_JOIN_AHEAD; ++a) {
        const int j = j0 + a * SLICES;
        if (j <= n)
          load_w<W, float>(
              partial + (((size_t)(chunk + j) * 2 + (j == 0 ? 1 : 0)) * g.units + u) * W, v[a]);
      }
#pragma unroll
      for (int a = 0; a < GR_JOIN_AHEAD; ++a) {
        if (j0 + a * SLICES > n) break;
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += v[a][k];
      }
    }
#pragma unroll
    for (int k = 0; k < W; ++k) sh[slice][k * GR_JOIN_UNITS + lane] = sum[k];
    __syncthreads();
    if (slice == 0 && in) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        for (int o = 1; o < SLICES; ++o) sum[k] += sh[o][k * GR_JOIN_UNITS + lane];
        sum[k] *= scale;
      }
      store_w<W, TW>(dweight + ((size_t)id * g.units + u) * W, sum);
    }
    __syncthreads();
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_embedding(const char* what, int wdtype, int odtype, int64_t N, int64_t V, int64_t D) {
  if (N < 0 || N > EM_MAX_N || V <= 0 || V >= INT32_MAX || D <= 0 || D > INT32_MAX / 8) {
    set_error("%s: unsupported sizes N=%lld V=%lld D=%lld", what, (long long)N, (long long)V,
              (long long)D);
    return DABSN_ERR_SHAPE;
  }
  for (int d : {wdtype, odtype})
    if (d != DABSN_F32 && d != DABSN_BF16) {
      set_error("%s: tables and outputs must be FP32 or BF16", what);
      return DABSN_ERR_DTYPE;
    }
  return DABSN_OK;
}

template <typename TW, typename TO>
int launch_lookup(int64_t N, int64_t V, int64_t D, const int64_t* tokens, const void* weight,
                  int64_t ldw, float scale, void* out, cudaStream_t st) {
  const bool vec = D % 8 == 0 && ldw % 8 == 0 && aligned16(weight) && aligned16(out);
  const int units = (int)(vec ? D / 8 : D);
  // eight units a thread where that still fills the SMs, else one
  const bool fills = N * units >= (int64_t)148 * 8 * 8 * EM_THREADS;
  const int group = fills ? std::max(1, 8 * EM_THREADS / units)
                          : std::max(1, EM_THREADS / units);
  const unsigned grid = (unsigned)((N + group - 1) / group);
  if (vec)
    embedding_fwd_kernel<TW, TO, 8><<<grid, EM_THREADS, 0, st>>>(
        N, (int)V, units, group, tokens, (const TW*)weight, ldw, scale, (TO*)out,
        device_status());
  else
    embedding_fwd_kernel<TW, TO, 1><<<grid, EM_THREADS, 0, st>>>(
        N, (int)V, units, group, tokens, (const TW*)weight, ldw, scale, (TO*)out,
        device_status());
  return launch_status("embedding_fwd");
}

// Bytes of the sort's arrays, rounded up so that the partial sums behind them
// are aligned; of the partial sums.
size_t sort_bytes(int64_t N, int64_t V) {
  const size_t n = ((size_t)4 * N + (size_t)sort_plan(N, V).blocks * RS_DIGITS) * sizeof(int);
  return (n + 15) / 16 * 16;
}
size_t partial_bytes(int64_t N, int64_t D) {
  const size_t chunks = (size_t)grad_plan(N, 1, 1).chunks;
  return chunks * 2 * (size_t)D * sizeof(float);
}

template <typename TG, typename TW, int W>
int launch_grad_w(int64_t N, int64_t V, int units, const int* key, const int* pos,
                  const void* dout, float scale, void* dweight, float* partial,
                  cudaStream_t st) {
  const GradPlan g = grad_plan(N, V, units);
  embedding_grad_kernel<TG, TW, W><<<dim3(g.blocks + g.zero_blocks, g.tiles), EM_THREADS, 0, st>>>(
      (int)N, (int)V, g, key, pos, (const TG*)dout, scale, (TW*)dweight, partial);
  if (g.chunks > 2)  // a run covers a chunk whole and goes on on both sides
    embedding_join_kernel<TW, W>
        <<<dim3((g.chunks + GR_JOIN_CHUNKS - 1) / GR_JOIN_CHUNKS,
                (units + GR_JOIN_UNITS - 1) / GR_JOIN_UNITS),
           EM_THREADS, 0, st>>>((int)N, (int)V, g, key, partial, scale, (TW*)dweight);
  return launch_status("embedding_bwd");
}

template <typename TG, typename TW>
int launch_grad(int64_t N, int64_t V, int64_t D, const int* key, const int* pos,
                const void* dout, float scale, void* dweight, float* partial, cudaStream_t st) {
  constexpr int W = 16 / sizeof(TG);
  const bool vec = D % W == 0 && aligned16(dout) && aligned16(dweight) && aligned16(partial);
  return vec ? launch_grad_w<TG, TW, W>(N, V, (int)(D / W), key, pos, dout, scale, dweight,
                                        partial, st)
             : launch_grad_w<TG, TW, 1>(N, V, (int)D, key, pos, dout, scale, dweight, partial,
                                        st);
}

}  // namespace
}  // namespace dabsn

using namespace dabsn;

extern "C" int dabsn_embedding_fwd(int weight_dtype, int out_dtype, int64_t N, int64_t V,
                                   int64_t D, const int64_t* tokens, const void* weight,
                                   int64_t ldw, float scale, void* out, void* stream) {
  int bad = check_embedding("embedding_fwd", weight_dtype, out_dtype, N, V, D);
  if (bad) return bad;
  if (ldw < D) {
    set_error("embedding_fwd: row stride %lld below the width %lld", (long long)ldw,
              (long long)D);
    return DABSN_ERR_SHAPE;
  }
  if (N == 0) return DABSN_OK;
  bad = check_pointers("embedding_fwd", {tokens, weight, out});
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  if (weight_dtype == DABSN_BF16)
    return out_dtype == DABSN_BF16
               ? launch_lookup<bf16, bf16>(N, V, D, tokens, weight, ldw, scale, out, st)
               : launch_lookup<bf16, float>(N, V, D, tokens, weight, ldw, scale, out, st);
  return out_dtype == DABSN_BF16
             ? launch_lookup<float, bf16>(N, V, D, tokens, weight, ldw, scale, out, st)
             : launch_lookup<float, float>(N, V, D, tokens, weight, ldw, scale, out, st);
}

extern "C" size_t dabsn_embedding_bwd_workspace(int64_t N, int64_t V, int64_t D) {
  if (N < 0 || N > EM_MAX_N || V <= 0 || V >= INT32_MAX || D <= 0) return 0;
  return sort_bytes(N, V) + partial_bytes(N, D);
}

extern "C" int dabsn_embedding_bwd(int out_dtype, int weight_dtype, int64_t N, int64_t V,
                                   int64_t D, const int64_t* tokens, int64_t padding_idx,
                                   const void* dout, float scale, void* dweight, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int bad = check_embedding("embedding_bwd", weight_dtype, out_dtype, N, V, D);
  if (bad) return bad;
  if (workspace_bytes < dabsn_embedding_bwd_workspace(N, V, D)) {
    set_error("embedding_bwd: workspace of %zu bytes is too small", workspace_bytes);
    return DABSN_ERR_UNSUPPORTED;
  }
  bad = check_pointers("embedding_bwd", {dweight, workspace});
  if (!bad && N > 0) bad = check_pointers("embedding_bwd", {tokens, dout});
  if (bad) return bad;
  cudaStream_t st = (cudaStream_t)stream;
  const SortPlan plan = sort_plan(N, V);
  const SortSpace s = sort_space(workspace, N);
  const int mask = (1 << plan.bits) - 1;
  const int n = (int)N, v = (int)V, out = (plan.passes - 1) & 1;
  const bool small = N <= RS_SMALL;
  if (small && N > 0) {
    if (!kernel_prepared((const void*)sort_small_kernel, RS_SMALL_SMEM)) return DABSN_ERR_LAUNCH;
    sort_small_kernel<<<1, RS_SMALL_THREADS, RS_SMALL_SMEM, st>>>(
        n, v, padding_idx, plan.passes, plan.bits, tokens, s.key[out], s.pos[out]);
  }
  for (int pass = 0; pass < plan.passes && !small; ++pass) {
    const int shift = pass * plan.bits, to = pass & 1, from = to ^ 1;
    if (pass == 0) {
      sort_count_kernel<true><<<plan.blocks, EM_THREADS, 0, st>>>(
          n, v, padding_idx, plan.tile, shift, mask, tokens, nullptr, s.hist);
      sort_place_kernel<true><<<plan.blocks, EM_THREADS, 0, st>>>(
          n, v, padding_idx, plan.tile, shift, plan.bits, tokens, nullptr, nullptr, s.hist,
          s.key[to], s.pos[to]);
    } else {
      sort_count_kernel<false><<<plan.blocks, EM_THREADS, 0, st>>>(
          n, v, padding_idx, plan.tile, shift, mask, nullptr, s.key[from], s.hist);
      sort_place_kernel<false><<<plan.blocks, EM_THREADS, 0, st>>>(
          n, v, padding_idx, plan.tile, shift, plan.bits, nullptr, s.key[from], s.pos[from],
          s.hist, s.key[to], s.pos[to]);
    }
  }
  const int* key = s.key[out];
  const int* pos = s.pos[out];
  float* partial = (float*)((char*)workspace + sort_bytes(N, V));
  if (out_dtype == DABSN_BF16)
    return weight_dtype == DABSN_BF16
               ? launch_grad<bf16, bf16>(N, V, D, key, pos, dout, scale, dweight, partial, st)
               : launch_grad<bf16, float>(N, V, D, key, pos, dout, scale, dweight, partial, st);
  return weight_dtype == DABSN_BF16
             ? launch_grad<float, bf16>(N, V, D, key, pos, dout, scale, dweight, partial, st)
             : launch_grad<float, float>(N, V, D, key, pos, dout, scale, dweight, partial, st);
}
