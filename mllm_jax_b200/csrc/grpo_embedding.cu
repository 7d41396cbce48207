// Embedding table: scaled lookup, and its gradient by sorted tokens.
//
//   out[n, :] = scale * W[id_n, :]            dW[v, :] = scale * sum_{n: id_n = v} dout[n, :]
//
// Lookup: N*H elements read and written, bound by memory; one thread moves one vector of a row.
//
// Gradient: the new [V, H] gradient has to be written whole (at V = 151936, H = 3584 that is 2.18 GB of f32 against
// 0.23 GB of token gradients), so the kernel that writes it walks the TABLE's rows and sums a row's tokens on the
// way.  It needs the tokens grouped by id in an order that depends on the ids alone: a stable radix sort of
// (id, token) pairs by ONE cluster of eight CTAs, whose digit counts meet in distributed shared memory, in one
// launch.  A row with very many tokens (padding, a frequent word) would keep one CTA busy long after all others:
// runs of 32 equal ids that start at a multiple of 32 in the sorted order are summed beforehand, and runs of 1024
// from those, so that a row of any length is a few dozen additions.  Every sum is f32 in a fixed order.
#include <cuda_fp16.h>

#include "grpo_cluster.cuh"
#include "grpo_common.cuh"
#include "grpo_launch.h"

namespace grpo {
namespace emb {

constexpr int kThreads = 256;

// n / d for n < 2^32 by a multiplication (d > 0): the quotient of Granlund and Montgomery's method.
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t div) : d(div) {
    uint32_t l = 0;
    while (l < 32 && (uint64_t(1) << l) < div) ++l;
    m = uint32_t((((uint64_t(1) << l) - div) << 32) / div + 1);
    s = l;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    const uint32_t t = __umulhi(m, n);
    return s == 0 ? n : (t + ((n - t) >> 1)) >> (s - 1);
  }
};

template <typename T>
struct Conv;
template <>
struct Conv<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Conv<__half> {
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Conv<float> {
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};

template <typename T, int EV>
struct alignas(sizeof(T) * EV) Vec {
  T v[EV];
};

struct LookupParams {
  int64_t weight_stride, out_stride, vocab_start, vocab, vocab_total;
  uint32_t row_vecs, total;  // vectors of a row, of all rows of this launch
  FastDiv by_row;
  float scale;
  const int32_t* ids;
  const void* weight;
  void* out;
  int32_t* device_status;
};

template <typename T, int EV, int UNROLL>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const LookupParams p) {
  using V = Vec<T, EV>;
  const uint32_t base = blockIdx.x * uint32_t(kThreads * UNROLL) + threadIdx.x;
  V x[UNROLL];
  uint32_t tok[UNROLL], col[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const uint32_t i = base + u * kThreads;
#pragma unroll
    for (int j = 0; j < EV; ++j) x[u].v[j] = Conv<T>::down(0.f);
    if (i >= p.total) continue;
    tok[u] = p.by_row.div(i);
    col[u] = i - tok[u] * p.row_vecs;
    const int64_t id = p.ids[tok[u]];
    const int64_t local = id - p.vocab_start;
    if (local >= 0 && local < p.vocab)
      x[u] = *(reinterpret_cast<const V*>(static_cast<const T*>(p.weight) + local * p.weight_stride) + col[u]);
    else if (col[u] == 0 && (id < 0 || id >= p.vocab_total) && p.device_status)
      atomicOr(p.device_status, MLLM_GRPO_DEV_ID_IGNORED);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (base + u * kThreads >= p.total) continue;
    V y;
#pragma unroll
    for (int j = 0; j < EV; ++j) y.v[j] = Conv<T>::down(Conv<T>::up(x[u].v[j]) * p.scale);
    *(reinterpret_cast<V*>(static_cast<T*>(p.out) + int64_t(tok[u]) * p.out_stride) + col[u]) = y;
  }
}

// ---------------------------------------------------------------------------------------------
// Stable radix sort of (id, token) by one cluster of eight CTAs, 9 bits a pass.  CTA r owns the r-th eighth of
// the pairs.  A pass: digit counts of the eighth; all eight counts through distributed shared memory give every
// digit its first place; then tiles of 4096 pairs, 128 consecutive ones per warp, get their places by the warp's
// match of equal digits (stable: lower lanes first) and the running counts of the warps before it.
// ---------------------------------------------------------------------------------------------
constexpr int kSortCtas = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kRounds = 4;
constexpr int kTile = kSortThreads * kRounds;
constexpr int kBits = 9;
constexpr int kBins = 1 << kBits;

struct SortParams {
  int64_t vocab_start, vocab, vocab_total;
  uint32_t n;
  int passes;
  const int32_t* ids;
  uint32_t* key[2];  // ping-pong; the result is in key[(passes - 1) & 1]
  uint32_t* idx[2];
  int32_t* device_status;
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t first[kBins];
  __shared__ uint16_t count[kSortWarps][kBins];
  __shared__ uint32_t scan[kBins / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cl::cluster_rank();
  const uint32_t per = (p.n + kSortCtas - 1) / kSortCtas;
  const uint32_t lo = min(p.n, rank * per), hi = min(p.n, lo + per);
  const uint32_t lower = (1u << lane) - 1u;

  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * kBits;
    auto key_of = [&](uint32_t i) -> uint32_t {
      if (pass) return __ldcg(p.key[(pass - 1) & 1] + i);
      const int64_t id = p.ids[i], local = id - p.vocab_start;
      if (local >= 0 && local < p.vocab) return uint32_t(local);
      return uint32_t(p.vocab);  // no row of this table: sorted behind all others
    };
    for (int b = tid; b < kBins; b += kSortThreads) hist[b] = 0;
    __syncthreads();
    for (uint32_t i0 = lo; i0 < hi; i0 += kSortThreads) {
      const uint32_t i = i0 + tid;
      const bool ok = i < hi;
      const uint32_t k = ok ? key_of(i) : 0u;
      if (pass == 0 && ok && p.device_status) {
        const int64_t id = p.ids[i];
        if (id < 0 || id >= p.vocab_total) atomicOr(p.device_status, MLLM_GRPO_DEV_ID_IGNORED);
      }
      const uint32_t d = ok ? (k >> shift) & (kBins - 1) : uint32_t(kBins);
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (ok && (same & lower) == 0) atomicAdd(&hist[d], __popc(same));
    }
    cl::cluster_sync_all();
    uint32_t total = 0, before = 0;
    if (tid < kBins) {
      const uint32_t mine = cl::smem_u32(&hist[tid]);
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) {
        const uint32_t h = ld_cluster_u32(cl::map_to_cta(mine, c));
        total += h;
        if (c < int(rank)) before += h;
      }
    }
    // exclusive scan of the totals over the digits (16 warps of 32)
    uint32_t incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (tid < kBins && lane == 31) scan[warp] = incl;
    __syncthreads();
    if (tid < kBins) {
      uint32_t base = incl - total + before;
      for (int w = 0; w < warp; ++w) base += scan[w];
      first[tid] = base;
    }
    uint32_t* key_out = p.key[pass & 1];
    uint32_t* idx_out = p.idx[pass & 1];
    for (uint32_t t0 = lo; t0 < hi; t0 += kTile) {
      uint4* z = reinterpret_cast<uint4*>(&count[0][0]);
      for (int i = tid; i < int(sizeof(count) / 16); i += kSortThreads) z[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      uint32_t k[kRounds], n[kRounds], place[kRounds];
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const uint32_t i = t0 + uint32_t(warp * (32 * kRounds) + r * 32 + lane);
        const bool ok = i < hi;
        k[r] = ok ? key_of(i) : 0u;
        n[r] = ok ? (pass ? __ldcg(p.idx[(pass - 1) & 1] + i) : i) : 0xffffffffu;
      }
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const bool ok = n[r] != 0xffffffffu;
        const uint32_t d = ok ? (k[r] >> shift) & (kBins - 1) : uint32_t(kBins);
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        place[r] = ok ? count[warp][d] + __popc(same & lower) : 0u;
        __syncwarp();
        if (ok && (same & lower) == 0) count[warp][d] = uint16_t(count[warp][d] + __popc(same));
        __syncwarp();
      }
      __syncthreads();
      uint32_t tile_total = 0;
      if (tid < kBins) {
#pragma unroll 8
        for (int w = 0; w < kSortWarps; ++w) {
          const uint32_t c = count[w][tid];
          count[w][tid] = uint16_t(tile_total);
          tile_total += c;
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        if (n[r] == 0xffffffffu) continue;
        const uint32_t d = (k[r] >> shift) & (kBins - 1);
        const uint32_t to = first[d] + count[warp][d] + place[r];
        key_out[to] = k[r];
        idx_out[to] = n[r];
      }
      __syncthreads();
      if (tid < kBins) first[tid] += tile_total;
    }
    cl::cluster_sync_all();  // the pass's pairs are visible to the cluster, and nobody reads `hist` any more
  }
}

// ---------------------------------------------------------------------------------------------
// Sums
// ---------------------------------------------------------------------------------------------
constexpr int kRun = 32, kSuper = 1024;

struct GradParams {
  int64_t vocab, grad_stride, weight_stride;
  uint32_t n, hidden, row_vecs, rows_per_cta;
  FastDiv by_row;
  float scale;
  const uint32_t* key;
  const uint32_t* idx;
  const void* grad;
  void* dweight;
  float* run;    // [n / 32, hidden]
  float* super;  // [n / 1024, hidden]
};

template <typename T, int EV>
__device__ __forceinline__ void add_token(const GradParams& p, float (&acc)[EV], uint32_t token, uint32_t col) {
  const Vec<T, EV> x = *(reinterpret_cast<const Vec<T, EV>*>(static_cast<const T*>(p.grad) + int64_t(token) * p.grad_stride) + col);
#pragma unroll
  for (int j = 0; j < EV; ++j) acc[j] += Conv<T>::up(x.v[j]);
}
template <int EV>
__device__ __forceinline__ void add_sum(const GradParams& p, float (&acc)[EV], const float* sums, uint32_t row, uint32_t col) {
  const float* s = sums + int64_t(row) * p.hidden + int64_t(col) * EV;
#pragma unroll
  for (int j = 0; j < EV; ++j) acc[j] += s[j];
}

// Runs of 32 equal ids.  blockIdx.x = run, blockIdx.y = part of the columns.
template <typename T, int EV>
__global__ void __launch_bounds__(kThreads) run_kernel(const GradParams p) {
  const uint32_t i0 = blockIdx.x * kRun;
  const uint32_t k = p.key[i0];
  if (k != p.key[i0 + kRun - 1] || k >= p.vocab) return;
  for (uint32_t c = blockIdx.y * kThreads + threadIdx.x; c < p.row_vecs; c += gridDim.y * kThreads) {
    float acc[EV] = {};
#pragma unroll 8
    for (int i = 0; i < kRun; ++i) add_token<T, EV>(p, acc, p.idx[i0 + i], c);
    float* out = p.run + int64_t(blockIdx.x) * p.hidden + int64_t(c) * EV;
#pragma unroll
    for (int j = 0; j < EV; ++j) out[j] = acc[j];
  }
}
template <int EV>
__global__ void __launch_bounds__(kThreads) super_kernel(const GradParams p) {
  const uint32_t i0 = blockIdx.x * kSuper;
  const uint32_t k = p.key[i0];
  if (k != p.key[i0 + kSuper - 1] || k >= p.vocab) return;
  for (uint32_t c = blockIdx.y * kThreads + threadIdx.x; c < p.row_vecs; c += gridDim.y * kThreads) {
    float acc[EV] = {};
#pragma unroll 8
    for (int i = 0; i < kSuper / kRun; ++i) add_sum<EV>(p, acc, p.run, blockIdx.x * (kSuper / kRun) + i, c);
    float* out = p.super + int64_t(blockIdx.x) * p.hidden + int64_t(c) * EV;
#pragma unroll
    for (int j = 0; j < EV; ++j) out[j] = acc[j];
  }
}

// Sum of the tokens at sorted places [s, e) in one vector of columns.
template <typename T, int EV>
__device__ __forceinline__ void segment_sum(const GradParams& p, float (&acc)[EV], uint32_t s, uint32_t e, uint32_t col) {
  uint32_t i = s;
  while (i < e) {
    if ((i & (kSuper - 1)) == 0 && i + kSuper <= e) {
      const uint32_t n = (e - i) / kSuper;
#pragma unroll 4
      for (uint32_t q = 0; q < n; ++q) add_sum<EV>(p, acc, p.super, i / kSuper + q, col);
      i += n * kSuper;
    } else if ((i & (kRun - 1)) == 0 && i + kRun <= e) {
      // up to the next multiple of 1024 (or the end)
      const uint32_t stop = min(e, (i & ~uint32_t(kSuper - 1)) + kSuper);
      const uint32_t n = (stop - i) / kRun;
#pragma unroll 4
      for (uint32_t q = 0; q < n; ++q) add_sum<EV>(p, acc, p.run, i / kRun + q, col);
      i += n * kRun;
    } else {
      const uint32_t stop = min(e, (i & ~uint32_t(kRun - 1)) + kRun);
#pragma unroll 4
      for (; i < stop; ++i) add_token<T, EV>(p, acc, p.idx[i], col);
    }
  }
}

// First place in [lo, hi) whose key is >= v, found by a whole warp (32 probes a step).
__device__ __forceinline__ uint32_t warp_lower_bound(const uint32_t* key, uint32_t lo, uint32_t hi, uint64_t v) {
  const uint32_t lane = threadIdx.x & 31;
  while (lo < hi) {
    const uint32_t step = (hi - lo + 31) / 32;
    const uint64_t at = uint64_t(lo) + uint64_t(lane) * step;
    const bool less = at < hi && key[at] < v;
    const uint32_t c = __popc(__ballot_sync(0xffffffffu, less));
    if (c == 0) return lo;
    // probe c-1 is below v, probe c (if there is one) is not
    const uint64_t up = uint64_t(lo) + uint64_t(c) * step;
    hi = up < hi ? uint32_t(up) : hi;
    lo += (c - 1) * step + 1;
  }
  return lo;
}

template <typename O, int EV>
__device__ __forceinline__ void store_row(O* to, const float (&acc)[EV], float scale) {
  Vec<O, EV> y;
#pragma unroll
  for (int j = 0; j < EV; ++j) y.v[j] = Conv<O>::down(acc[j] * scale);
  *reinterpret_cast<Vec<O, EV>*>(to) = y;
}

constexpr int kMostRows = kThreads;

// Writes rows_per_cta consecutive rows of the table's gradient: zeros, or the sum of the row's tokens.
template <typename T, typename O, int EV>
__global__ void __launch_bounds__(kThreads) dense_grad_kernel(const GradParams p) {
  __shared__ uint32_t bound[2];
  __shared__ uint32_t at[kMostRows + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t v0 = int64_t(blockIdx.x) * p.rows_per_cta;
  const uint32_t rows = uint32_t(p.vocab - v0 < p.rows_per_cta ? p.vocab - v0 : p.rows_per_cta);
  if (warp < 2) {
    const uint32_t b = warp_lower_bound(p.key, 0, p.n, uint64_t(v0) + (warp ? rows : 0));
    if (lane == 0) bound[warp] = b;
  }
  __syncthreads();
  const uint32_t s = bound[0], e = bound[1];
  for (uint32_t r = tid; r <= rows; r += kThreads) {
    uint32_t lo = s, hi = e;
    const uint32_t v = uint32_t(v0) + r;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (p.key[mid] < v)
        lo = mid + 1;
      else
        hi = mid;
    }
    at[r] = lo;
  }
  __syncthreads();
  O* out = static_cast<O*>(p.dweight) + v0 * p.weight_stride;
  const uint32_t items = rows * p.row_vecs;
  for (uint32_t i = tid; i < items; i += kThreads) {
    const uint32_t r = p.by_row.div(i), c = i - r * p.row_vecs;
    float acc[EV] = {};
    const uint32_t a = at[r], b = at[r + 1];
    if (a != b) segment_sum<T, EV>(p, acc, a, b, c);
    store_row<O, EV>(out + int64_t(r) * p.weight_stride + int64_t(c) * EV, acc, p.scale);
  }
}

// Adds to the rows that have tokens.  One CTA per sorted place; the first of an id does the row.
template <typename T, int EV>
__global__ void __launch_bounds__(kThreads) accumulate_grad_kernel(const GradParams p) {
  const uint32_t s = blockIdx.x;
  const uint32_t k = p.key[s];
  if (k >= p.vocab || (s > 0 && p.key[s - 1] == k)) return;
  const uint32_t e = s + 1 < p.n && p.key[s + 1] == k ? warp_lower_bound(p.key, s + 1, p.n, uint64_t(k) + 1) : s + 1;
  float* out = static_cast<float*>(p.dweight) + int64_t(k) * p.weight_stride;
  for (uint32_t c = threadIdx.x; c < p.row_vecs; c += kThreads) {
    float acc[EV] = {};
    segment_sum<T, EV>(p, acc, s, e, c);
    Vec<float, EV>* to = reinterpret_cast<Vec<float, EV>*>(out) + c;
    Vec<float, EV> y = *to;
#pragma unroll
    for (int j = 0; j < EV; ++j) y.v[j] += acc[j] * p.scale;
    *to = y;
  }
}

static cudaError_t done() {
  count_launch();
  return cudaGetLastError();
}

static int64_t elem(int dtype) { return dtype == MLLM_GRPO_F32 ? 4 : 2; }
static bool aligned(const void* q, int64_t a) { return (reinterpret_cast<uintptr_t>(q) & uintptr_t(a - 1)) == 0; }

// Widest vector (in elements, a power of two up to `most`) that rows of `hidden` elements at this base and stride allow.
static int vec_of(int64_t hidden, int most, const void* a, int64_t sa, int64_t ea, const void* b, int64_t sb, int64_t eb) {
  int ev = most;
  while (ev > 1 && (hidden % ev || (sa * ea) % (ev * ea) || (sb * eb) % (ev * eb) || !aligned(a, ev * ea) || !aligned(b, ev * eb)))
    ev >>= 1;
  return ev;
}

template <typename T, int EV>
static cudaError_t launch_lookup(const LookupParams& p, cudaStream_t s) {
  // one vector per thread until every SM has work, four (in flight together) beyond that
  if (p.total <= 148u * kThreads * 4u) {
    lookup_kernel<T, EV, 1><<<(p.total + kThreads - 1) / kThreads, kThreads, 0, s>>>(p);
  } else {
    lookup_kernel<T, EV, 4><<<(p.total + kThreads * 4 - 1) / (kThreads * 4), kThreads, 0, s>>>(p);
  }
  return done();
}

template <typename T>
static cudaError_t launch_lookup_t(const mllm_grpo_embedding_args* a, LookupParams p, cudaStream_t s) {
  constexpr int kMost = 16 / int(sizeof(T));
  const int ev = vec_of(a->hidden, kMost, a->weight, a->weight_stride, sizeof(T), a->out, a->token_stride, sizeof(T));
  const int64_t row_vecs = a->hidden / ev;
  // vectors are counted in 32 bits: very large batches go in several launches
  const int64_t tokens_per = (int64_t(1) << 31) / row_vecs;
  p.row_vecs = uint32_t(row_vecs);
  p.by_row = FastDiv(uint32_t(row_vecs));
  for (int64_t t0 = 0; t0 < a->n_tokens; t0 += tokens_per) {
    const int64_t n = a->n_tokens - t0 < tokens_per ? a->n_tokens - t0 : tokens_per;
    p.total = uint32_t(n * row_vecs);
    p.ids = a->ids + t0;
    p.out = static_cast<T*>(a->out) + t0 * a->token_stride;
    cudaError_t e;
    if (ev == kMost)
      e = launch_lookup<T, kMost>(p, s);
    else if (ev == 4)
      e = launch_lookup<T, 4>(p, s);
    else if (ev == 2)
      e = launch_lookup<T, 2>(p, s);
    else
      e = launch_lookup<T, 1>(p, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, int EV>
static cudaError_t launch_runs(const GradParams& p, cudaStream_t s) {
  const unsigned ny = (p.row_vecs + kThreads - 1) / kThreads;
  if (p.n >= kRun) {
    run_kernel<T, EV><<<dim3(p.n / kRun, ny), kThreads, 0, s>>>(p);
    const cudaError_t e = done();
    if (e != cudaSuccess) return e;
  }
  if (p.n >= kSuper) {
    super_kernel<EV><<<dim3(p.n / kSuper, ny), kThreads, 0, s>>>(p);
    const cudaError_t e = done();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, typename O, int EV>
static cudaError_t launch_dense(GradParams p, cudaStream_t s) {
  // about 64 KB of gradient per CTA: enough to cover the search for the CTA's tokens
  int64_t rows = 65536 / (int64_t(p.hidden) * int64_t(sizeof(O)));
  rows = rows < 1 ? 1 : (rows > kMostRows ? kMostRows : rows);
  p.rows_per_cta = uint32_t(rows);
  dense_grad_kernel<T, O, EV><<<unsigned((p.vocab + rows - 1) / rows), kThreads, 0, s>>>(p);
  return done();
}

template <typename T, int EV>
static cudaError_t launch_grad_ev(const mllm_grpo_embedding_args* a, const GradParams& p, cudaStream_t s) {
  cudaError_t e = launch_runs<T, EV>(p, s);
  if (e != cudaSuccess) return e;
  if (a->accumulate) {
    if (p.n == 0) return cudaSuccess;
    accumulate_grad_kernel<T, EV><<<p.n, kThreads, 0, s>>>(p);
    return done();
  }
  if (a->out_dtype == MLLM_GRPO_F32) return launch_dense<T, float, EV>(p, s);
  if (a->out_dtype == MLLM_GRPO_F16) return launch_dense<T, __half, EV>(p, s);
  return launch_dense<T, __nv_bfloat16, EV>(p, s);
}

template <typename T>
static cudaError_t launch_grad_t(const mllm_grpo_embedding_args* a, GradParams p, cudaStream_t s) {
  // four elements a vector: f32 rows are stored 16 bytes a thread
  const int ev = vec_of(a->hidden, 4, a->grad_out, a->token_stride, sizeof(T), a->dweight, a->weight_stride, elem(a->out_dtype));
  p.row_vecs = uint32_t(a->hidden / (ev == 4 ? 4 : 1));
  p.by_row = FastDiv(p.row_vecs);
  return ev == 4 ? launch_grad_ev<T, 4>(a, p, s) : launch_grad_ev<T, 1>(a, p, s);
}

static int64_t round16(int64_t b) { return (b + 15) & ~int64_t(15); }

static int check(const mllm_grpo_embedding_args* a) {
  if (a == nullptr) return MLLM_GRPO_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(mllm_grpo_embedding_args)) return MLLM_GRPO_ERR_STRUCT_SIZE;
  if (a->n_tokens < 0 || a->vocab <= 0 || a->hidden <= 0 || a->weight_stride < a->hidden || a->token_stride < a->hidden ||
      a->vocab_start < 0)
    return MLLM_GRPO_ERR_BAD_SHAPE;
  constexpr int64_t kMost = (int64_t(1) << 31) - 1;
  if (a->vocab >= kMost || a->hidden > (int64_t(1) << 20) || a->n_tokens > kMost || a->vocab_start > kMost)
    return MLLM_GRPO_ERR_TOO_LARGE;
  if (a->vocab_total != 0 && a->vocab_total < a->vocab_start + a->vocab) return MLLM_GRPO_ERR_BAD_SHAPE;
  if (a->dtype < 0 || a->dtype > MLLM_GRPO_F32 || a->scale != a->scale) return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (!aligned(a->ids, 4) || !aligned(a->device_status, 4)) return MLLM_GRPO_ERR_ALIGNMENT;
  return MLLM_GRPO_OK;
}

}  // namespace emb
}  // namespace grpo

using namespace grpo;

extern "C" {

int mllm_grpo_embedding_lookup(const mllm_grpo_embedding_args* a, void* stream) {
  const int st = emb::check(a);
  if (st) return st;
  if (a->n_tokens == 0) return MLLM_GRPO_OK;
  if (!a->ids || !a->weight || !a->out) return MLLM_GRPO_ERR_NULL_POINTER;
  const int64_t es = emb::elem(a->dtype);
  if (!emb::aligned(a->weight, es) || !emb::aligned(a->out, es)) return MLLM_GRPO_ERR_ALIGNMENT;
  emb::LookupParams p{a->weight_stride, a->token_stride, a->vocab_start, a->vocab,
                      a->vocab_total ? a->vocab_total : a->vocab_start + a->vocab, 0, 0, emb::FastDiv(1), a->scale,
                      a->ids, a->weight, a->out, a->device_status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == MLLM_GRPO_BF16)
    e = emb::launch_lookup_t<__nv_bfloat16>(a, p, s);
  else if (a->dtype == MLLM_GRPO_F16)
    e = emb::launch_lookup_t<__half>(a, p, s);
  else
    e = emb::launch_lookup_t<float>(a, p, s);
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

int64_t mllm_grpo_embedding_workspace_bytes(int64_t n_tokens, int64_t hidden) {
  if (n_tokens < 0 || hidden <= 0 || n_tokens >= (int64_t(1) << 31) || hidden > (int64_t(1) << 20)) return 0;
  return 16 + 4 * emb::round16(n_tokens * 4) + (n_tokens / emb::kRun + n_tokens / emb::kSuper) * hidden * 4;
}

int mllm_grpo_embedding_grad(const mllm_grpo_embedding_args* a, void* stream) {
  const int st = emb::check(a);
  if (st) return st;
  if (a->out_dtype < 0 || a->out_dtype > MLLM_GRPO_F32 || (a->accumulate && a->out_dtype != MLLM_GRPO_F32))
    return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (!a->dweight || !a->workspace || (a->n_tokens > 0 && (!a->ids || !a->grad_out))) return MLLM_GRPO_ERR_NULL_POINTER;
  if (!emb::aligned(a->grad_out, emb::elem(a->dtype)) || !emb::aligned(a->dweight, emb::elem(a->out_dtype)) ||
      !emb::aligned(a->workspace, 16))
    return MLLM_GRPO_ERR_ALIGNMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t n = uint32_t(a->n_tokens);
  char* w = static_cast<char*>(a->workspace);
  const int64_t list = emb::round16(int64_t(n) * 4);
  emb::SortParams q;
  q.vocab_start = a->vocab_start;
  q.vocab = a->vocab;
  q.vocab_total = a->vocab_total ? a->vocab_total : a->vocab_start + a->vocab;
  q.n = n;
  int bits = 1;
  while ((int64_t(1) << bits) <= a->vocab) ++bits;  // ids up to and including `vocab`, the mark of no row
  q.passes = (bits + emb::kBits - 1) / emb::kBits;
  q.ids = a->ids;
  for (int i = 0; i < 2; ++i) {
    q.key[i] = reinterpret_cast<uint32_t*>(w + (2 * i) * list);
    q.idx[i] = reinterpret_cast<uint32_t*>(w + (2 * i + 1) * list);
  }
  q.device_status = a->device_status;
  cudaError_t e = cudaSuccess;
  if (n) {
    emb::sort_kernel<<<emb::kSortCtas, emb::kSortThreads, 0, s>>>(q);
    e = emb::done();
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  const int last = (q.passes - 1) & 1;
  float* run = reinterpret_cast<float*>(w + 4 * list);
  emb::GradParams p{a->vocab, a->token_stride, a->weight_stride, n, uint32_t(a->hidden), 0, 0, emb::FastDiv(1), a->scale,
                    q.key[last], q.idx[last], a->grad_out, a->dweight, run, run + int64_t(n / emb::kRun) * a->hidden};
  if (a->dtype == MLLM_GRPO_BF16)
    e = emb::launch_grad_t<__nv_bfloat16>(a, p, s);
  else if (a->dtype == MLLM_GRPO_F16)
    e = emb::launch_grad_t<__half>(a, p, s);
  else
    e = emb::launch_grad_t<float>(a, p, s);
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

}  // extern "C"
