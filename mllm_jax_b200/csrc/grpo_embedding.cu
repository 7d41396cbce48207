// Embedding table: scaled lookup, and its gradient by sorted tokens.
//
//   out[n, :] = scale * W[id_n, :]            dW[v, :] = scale * sum_{n: id_n = v} dout[n, :]
//
// Lookup: N*H elements read and written, bound by memory; one thread moves one vector of a row.
//
// Gradient: the new [V, H] gradient has to be written whole (at V = 151936, H = 3584 that is 2.18 GB of f32 against
// 0.23 GB of token gradients), nearly all of it zeros.  Its sums need the tokens grouped by id in an order that depends
// on the ids alone: a stable radix sort of (id, token) pairs by ONE cluster of CTAs, whose digit counts meet in
// distributed shared memory.  It leaves nearly all SMs idle, so zeros are written beside it: their launch does not wait
// for the sort's (programmatic launch), only CTAs late in it do, which then list the rows that have tokens.  A last launch
// sums and writes those, after the zeros.  Where the rows with tokens are so many that writing them twice costs more than
// the sort (rows_beside), only the first part of the table gets its zeros early, and the last launch fills the rest where
// there are no tokens: a few resident CTAs sum rows from the list and short CTAs fill, 32 KB each in the order of the
// addresses.  (CTAs that stay resident and walk the table fill it at 6.1 TB/s, short ones in order at 7.5.  A loop over
// the table's rows that sums where there are tokens holds the fill up: a load waits several microseconds behind the
// stores.)
// A row with very many tokens (padding, a frequent word) would keep one CTA busy long after all others: runs of 32
// equal ids that start at a multiple of 32 in the sorted order are summed beforehand, and eight warps share what is left
// of such a row.  Every sum is f32 in a fixed order.
#include <cuda_fp16.h>

#include <cstring>
#include <mutex>
#include <type_traits>

#include "grpo_cluster.cuh"
#include "grpo_common.cuh"
#include "grpo_launch.h"

namespace grpo {
namespace emb {

constexpr int kThreads = 256;

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
// Stable radix sort of (id, token) by one cluster of eight CTAs (one CTA for up to 4096 pairs, 16 beyond 32768), 9 bits a
// pass.  CTA r owns the r-th eighth (sixteenth) of the pairs, in tiles of 4096, 128 consecutive pairs per warp.  Inside a tile a pair's place among
// its digit is found by the warp's match of equal digits (stable: lower lanes first) and the running counts of the warps
// before it; all eight CTAs' digit counts through distributed shared memory give every digit its first place.  Two
// passes: 14 us for up to 4096 pairs, 25 us for 32768.
// ---------------------------------------------------------------------------------------------
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
  uint4* busy;       // 16 rows' marks a word, to be zeroed by the CTAs behind the sort's (none for an accumulated gradient)
  uint32_t* counts;  // [2] to be zeroed
  int32_t* device_status;
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int CTAS>
__device__ __forceinline__ void sort_sync() {
  if (CTAS == 1)
    __syncthreads();
  else
    cl::cluster_sync_all();
}

template <int CTAS>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t first[kBins];
  __shared__ alignas(16) uint16_t count[kSortWarps][kBins];
  __shared__ uint32_t scan[kBins / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // zeros, if they come next, need not wait
  if (blockIdx.x >= CTAS) {  // whole clusters
    const int64_t words = (p.vocab + 15) / 16, step = int64_t(gridDim.x - CTAS) * kSortThreads;
    for (int64_t i = int64_t(blockIdx.x - CTAS) * kSortThreads + tid; i < words; i += step) p.busy[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const uint32_t rank = CTAS == 1 ? 0u : cl::cluster_rank();
  const uint32_t per = (p.n + CTAS - 1) / CTAS;
  const uint32_t lo = min(p.n, rank * per), hi = min(p.n, lo + per);
  const uint32_t lower = (1u << lane) - 1u;
  const bool one_tile = CTAS == 1 || per <= uint32_t(kTile);  // then the tile's counts are the eighth's
  if (rank == 0 && tid < 2) p.counts[tid] = 0u;

  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * kBits;
    const bool odd = pass & 1;
    const uint32_t* key_in = odd ? p.key[0] : p.key[1];
    const uint32_t* idx_in = odd ? p.idx[0] : p.idx[1];
    uint32_t* key_out = odd ? p.key[1] : p.key[0];
    uint32_t* idx_out = odd ? p.idx[1] : p.idx[0];
    auto key_of = [&](uint32_t i) -> uint32_t {
      if (pass) return __ldcg(key_in + i);
      const int64_t id = p.ids[i], local = id - p.vocab_start;
      if (local >= 0 && local < p.vocab) return uint32_t(local);
      if ((id < 0 || id >= p.vocab_total) && p.device_status) atomicOr(p.device_status, MLLM_GRPO_DEV_ID_IGNORED);
      return uint32_t(p.vocab);  // no row of this table: sorted behind all others
    };
    // one tile: keys, tokens, and the places among their digits; leaves the digits' totals of a thread's bin
    uint32_t k[kRounds], n[kRounds], place[kRounds];
    auto rank_tile = [&](uint32_t t0) -> uint32_t {
      uint4* z = reinterpret_cast<uint4*>(&count[0][0]);
      for (int i = tid; i < int(sizeof(count) / 16); i += kSortThreads) z[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const uint32_t i = t0 + uint32_t(warp * (32 * kRounds) + r * 32 + lane);
        const bool ok = i < hi;
        k[r] = ok ? key_of(i) : 0u;
        n[r] = ok ? (pass ? __ldcg(idx_in + i) : i) : 0xffffffffu;
      }
      __syncthreads();
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
      uint32_t total = 0;
      if (tid < kBins) {
#pragma unroll 8
        for (int w = 0; w < kSortWarps; ++w) {
          const uint32_t c = count[w][tid];
          count[w][tid] = uint16_t(total);
          total += c;
        }
      }
      return total;
    };
    auto scatter_tile = [&] {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        if (n[r] == 0xffffffffu) continue;
        const uint32_t d = (k[r] >> shift) & (kBins - 1);
        const uint32_t to = first[d] + count[warp][d] + place[r];
        key_out[to] = k[r];
        idx_out[to] = n[r];
      }
    };

    uint32_t tile_total = 0;
    if (one_tile) {
      tile_total = rank_tile(lo);
      if (tid < kBins) hist[tid] = tile_total;
    } else {
      for (int b = tid; b < kBins; b += kSortThreads) hist[b] = 0;
      __syncthreads();
      for (uint32_t i0 = lo; i0 < hi; i0 += kSortThreads) {
        const uint32_t i = i0 + tid;
        const bool ok = i < hi;
        const uint32_t d = ok ? (key_of(i) >> shift) & (kBins - 1) : uint32_t(kBins);
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (ok && (same & lower) == 0) atomicAdd(&hist[d], __popc(same));
      }
    }
    sort_sync<CTAS>();
    uint32_t total = 0, before = 0;
    if (CTAS == 1) {
      total = tile_total;
    } else if (tid < kBins) {
      const uint32_t mine = cl::smem_u32(&hist[tid]);
#pragma unroll
      for (int c = 0; c < CTAS; ++c) {
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
    __syncthreads();
    if (one_tile) {
      scatter_tile();
    } else {
      for (uint32_t t0 = lo; t0 < hi; t0 += kTile) {
        tile_total = rank_tile(t0);
        __syncthreads();
        scatter_tile();
        __syncthreads();
        if (tid < kBins) first[tid] += tile_total;
      }
    }
    sort_sync<CTAS>();  // the pass's pairs are visible to the cluster, and nobody reads `hist` any more
  }
}

// Zeros in the rows without tokens, kVecs words W a thread in the order of their addresses.
constexpr int kVecs = 8;
struct FillParams {
  int64_t stride;  // of a row, in words
  uint32_t total;  // words of this launch's rows
  uint32_t row_words;
  FastDiv by_row;
  const uint8_t* busy;  // of this launch's rows; null: no row has tokens
  void* out;
  uint16_t* end;  // 2-byte pieces behind the last whole word (fewer than 8)
  uint32_t pieces;
};
template <typename W>
__device__ __forceinline__ void fill(const FillParams& p, uint32_t block) {
  const uint32_t base = block * uint32_t(kThreads * kVecs) + threadIdx.x;
  if (block == 0 && threadIdx.x < p.pieces) p.end[threadIdx.x] = 0;
  uint32_t skip = 0;
  if (p.busy) {
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const uint32_t i = base + u * kThreads;
      if (i < p.total && p.busy[p.by_row.div(i)]) skip |= 1u << u;
    }
  }
  W zero;
  memset(&zero, 0, sizeof(W));
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const uint32_t i = base + u * kThreads;
    if (i >= p.total || (skip >> u & 1u)) continue;
    const uint32_t r = p.by_row.div(i);
    static_cast<W*>(p.out)[r * p.stride + (i - r * p.row_words)] = zero;
  }
}
template <typename W>
__global__ void __launch_bounds__(kThreads, 8) fill_kernel(const FillParams p) {
  fill<W>(p, blockIdx.x);
}

// ---------------------------------------------------------------------------------------------
// Sums
// ---------------------------------------------------------------------------------------------
constexpr uint32_t kRun = 32;
constexpr int kSumWarps = kThreads / 32;
constexpr int kCols = 4;  // vectors of a light row that a thread has on the way

// The rows that have tokens, in no particular order (each is summed by itself): light ones with up to kLight tokens,
// whose records say all that is needed to start, and heavy ones by the place of their first token.
constexpr uint32_t kLight = 16;
static_assert(kLight <= kRun, "");
struct alignas(16) Light {
  uint32_t row, first, count, pad;  // row of the table, sorted place of its first token, how many
};
struct Lists {
  uint32_t* counts;  // [0] light rows, [1] heavy rows
  Light* light;      // [n]
  uint32_t* heavy;   // [n / (kLight + 1)]
};

struct GradParams {
  int64_t grad_stride, weight_stride;
  uint32_t n, hidden, vocab, row_vecs, accumulate;
  uint32_t filled;  // rows below this one have their zeros already (all of them where the gradient is accumulated)
  uint32_t group;  // threads that share a light row: 32, 64, 128 or 256
  uint32_t parts;  // parts of 32 vectors of a row
  uint32_t row_ctas;
  FastDiv by_part;
  float scale;
  const uint32_t* key;
  const uint32_t* idx;
  uint8_t* busy;  // [vocab] 1 where a row has tokens
  Lists lists;
  const void* grad;
  void* dweight;
  float* run;  // [n / 32, hidden]
};

template <typename T, int EV>
__device__ __forceinline__ Vec<T, EV> token_vec(const GradParams& p, uint32_t token, uint32_t col) {
  return *(reinterpret_cast<const Vec<T, EV>*>(static_cast<const T*>(p.grad) + int64_t(token) * p.grad_stride) + col);
}
template <typename T, int EV>
__device__ __forceinline__ void add_vec(float (&acc)[EV], const Vec<T, EV>& x) {
#pragma unroll
  for (int j = 0; j < EV; ++j) acc[j] += Conv<T>::up(x.v[j]);
}
// f32 sums are kept in rows of `hidden`, read and written four at a time where the width allows it (EV >= 4 does).
template <int EV>
__device__ __forceinline__ void add_sum(const GradParams& p, float (&acc)[EV], const float* sums, uint32_t row, uint32_t col) {
  const float* s = sums + int64_t(row) * p.hidden + int64_t(col) * EV;
  if constexpr (EV >= 4) {
#pragma unroll
    for (int j = 0; j < EV; j += 4) {
      const float4 v = *reinterpret_cast<const float4*>(s + j);
      acc[j] += v.x;
      acc[j + 1] += v.y;
      acc[j + 2] += v.z;
      acc[j + 3] += v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < EV; ++j) acc[j] += s[j];
  }
}
template <typename O, int EV>
__device__ __forceinline__ void store_vec(O* to, const float (&acc)[EV], float scale) {
  constexpr int kPart = EV * int(sizeof(O)) > 16 ? 16 / int(sizeof(O)) : EV;
#pragma unroll
  for (int i = 0; i < EV; i += kPart) {
    Vec<O, kPart> y;
#pragma unroll
    for (int j = 0; j < kPart; ++j) y.v[j] = Conv<O>::down(acc[i + j] * scale);
    *reinterpret_cast<Vec<O, kPart>*>(to + i) = y;
  }
}

// Lists and marks the rows that have tokens: one warp per 32 sorted places.
__device__ __forceinline__ void list_rows(const GradParams& p, uint32_t block) {
  const uint32_t lane = threadIdx.x & 31, i = block * kRun + lane;
  const uint32_t mine = i < p.n ? p.key[i] : 0xffffffffu;
  const uint32_t before = i > 0 && i < p.n ? p.key[i - 1] : 0xffffffffu;
  const uint32_t after = i + kRun < p.n ? p.key[i + kRun] : 0xffffffffu;  // the next 32 places
  const bool head = mine < p.vocab && (i == 0 || before != mine);
  // how many tokens the row has (up to 64 are seen from here): equal keys are neighbours
  const uint32_t last = __shfl_sync(0xffffffffu, mine, 31);
  const uint32_t over = __popc(__ballot_sync(0xffffffffu, after == last));
  const uint32_t count = __popc(__match_any_sync(0xffffffffu, mine)) + (mine == last ? over : 0u);
  const bool heavy = head && count > kLight;
  const uint32_t lower = (1u << lane) - 1u;
  const uint32_t hs = __ballot_sync(0xffffffffu, heavy), ls = __ballot_sync(0xffffffffu, head && !heavy);
  uint32_t at = 0;
  if (lane == 0 && ls) at = atomicAdd(p.lists.counts, uint32_t(__popc(ls)));
  if (lane == 1 && hs) at = atomicAdd(p.lists.counts + 1, uint32_t(__popc(hs)));
  const uint32_t lb = __shfl_sync(0xffffffffu, at, 0), hb = __shfl_sync(0xffffffffu, at, 1);
  if (heavy)
    p.lists.heavy[hb + __popc(hs & lower)] = i;
  else if (head)
    p.lists.light[lb + __popc(ls & lower)] = Light{mine, i, count, 0u};
  if (head && mine >= p.filled) p.busy[mine] = 1;
}

// Sums 32 places whose ids are all equal, EV columns a thread (c is this thread's vector of them), 8 token rows of 16
// bytes a thread (16 of 8 or fewer) on the way at a time.
template <typename T, int EV>
__device__ __forceinline__ void sum_run(const GradParams& p, uint32_t block, uint32_t c, uint32_t row_vecs) {
  constexpr uint32_t B = EV * sizeof(T) == 16 ? 8 : 16;
  const uint32_t i = block * kRun + (threadIdx.x & 31);
  const uint32_t mine = i < p.n ? p.key[i] : 0xffffffffu;
  const uint32_t tokens = i < p.n ? p.idx[i] : 0u;
  const uint32_t k = __shfl_sync(0xffffffffu, mine, 0);
  if (__shfl_sync(0xffffffffu, mine, 31) != k || k >= p.vocab) return;
  const bool ok = c < row_vecs;
  float acc[EV] = {};
#pragma unroll
  for (uint32_t q = 0; q < kRun; q += B) {
    Vec<T, EV> x[B];
#pragma unroll
    for (uint32_t j = 0; j < B; ++j) {
      const uint32_t token = __shfl_sync(0xffffffffu, tokens, q + j);
      if (ok) x[j] = token_vec<T, EV>(p, token, c);
    }
#pragma unroll
    for (uint32_t j = 0; j < B; ++j)
      if (ok) add_vec<T, EV>(acc, x[j]);
  }
  if (ok) store_vec<float, EV>(p.run + int64_t(block) * p.hidden + int64_t(c) * EV, acc, 1.0f);
}

// blockIdx.x = 32 sorted places, blockIdx.y = part of the columns, the last one the list.
template <typename T, int EV>
__global__ void __launch_bounds__(128) run_kernel(const GradParams p, const uint32_t row_vecs) {
  if (blockIdx.y == gridDim.y - 1) {
    if (threadIdx.x < 32) list_rows(p, blockIdx.x);
    return;
  }
  sum_run<T, EV>(p, blockIdx.x, blockIdx.y * blockDim.x + threadIdx.x, row_vecs);
}

// The same beside the zeros: CTAs [first, first + list_ctas + sum_ctas) wait for the sort to be complete, then list rows
// and sum runs, the others fill.
struct Beside {
  uint32_t row_vecs, parts;  // vectors of a row; warps that share one run
  uint32_t first, list_ctas, sum_ctas;
};
template <typename T, int EV, typename W>
__global__ void __launch_bounds__(kThreads, 3) fill_runs_kernel(const GradParams p, const FillParams f, const Beside b) {
  if (blockIdx.x < b.first) {
    fill<W>(f, blockIdx.x);
    return;
  }
  const uint32_t at = blockIdx.x - b.first, warps = kThreads / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (at >= b.list_ctas + b.sum_ctas) {
    fill<W>(f, blockIdx.x - b.list_ctas - b.sum_ctas);
    return;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t runs = (p.n + kRun - 1) / kRun;
  if (at < b.list_ctas) {
    if (at * warps + warp < runs) list_rows(p, at * warps + warp);
    return;
  }
  const uint32_t item = (at - b.list_ctas) * warps + warp, run = item / b.parts;
  if (run < runs) sum_run<T, EV>(p, run, (item - run * b.parts) * 32 + lane, b.row_vecs);
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
__device__ __forceinline__ void finish_row(const GradParams& p, const float (&acc)[EV], uint32_t row, uint32_t col) {
  O* to = static_cast<O*>(p.dweight) + int64_t(row) * p.weight_stride + int64_t(col) * EV;
  if (p.accumulate) {
#pragma unroll
    for (int j = 0; j < EV; ++j) to[j] = Conv<O>::down(Conv<O>::up(to[j]) + acc[j] * p.scale);
  } else {
    store_vec<O, EV>(to, acc, p.scale);
  }
}

// Rows with more than kLight tokens, 32 vectors of one per CTA and step: its single tokens and its runs go round the
// eight warps, which meet in shared memory.
template <typename T, typename O, int EV>
__device__ __forceinline__ void heavy_rows(const GradParams& p, float (&meet)[kSumWarps][32][EV]) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t items = p.lists.counts[1] * p.parts;
  for (uint32_t item = p.row_ctas - 1 - blockIdx.x; item < items; item += p.row_ctas) {  // the last CTAs have the fewest light rows
    const uint32_t r = p.by_part.div(item), c = (item - r * p.parts) * 32 + lane;
    const bool ok = c < p.row_vecs;
    const uint32_t s = p.lists.heavy[r], k = p.key[s];
    const uint32_t e = warp_lower_bound(p.key, s + kLight, p.n, uint64_t(k) + 1);
    // single tokens up to a multiple of 32, whole runs, the tokens behind the last of them
    const uint32_t a0 = min(e, (s + kRun - 1) / kRun * kRun), a1 = max(a0, e / kRun * kRun);
    float acc[EV] = {};
    if (ok) {
#pragma unroll 4
      for (uint32_t i = s + warp; i < a0; i += kSumWarps) add_vec<T, EV>(acc, token_vec<T, EV>(p, p.idx[i], c));
#pragma unroll 4
      for (uint32_t q = a0 / kRun + warp; q < a1 / kRun; q += kSumWarps) add_sum<EV>(p, acc, p.run, q, c);
#pragma unroll 4
      for (uint32_t i = a1 + warp; i < e; i += kSumWarps) add_vec<T, EV>(acc, token_vec<T, EV>(p, p.idx[i], c));
    }
#pragma unroll
    for (int j = 0; j < EV; ++j) meet[warp][lane][j] = acc[j];
    __syncthreads();
    if (warp == 0 && ok) {
#pragma unroll
      for (int w = 1; w < kSumWarps; ++w)
#pragma unroll
        for (int j = 0; j < EV; ++j) acc[j] += meet[w][lane][j];
      finish_row<O, EV>(p, acc, k, c);
    }
    __syncthreads();
  }
}

// Rows with up to kLight tokens, p.group threads each, kCols vectors a thread.  While one is summed, the next one's
// tokens and the record of the one after that are on their way.
template <typename T, typename O, int EV>
__device__ __forceinline__ void light_rows(const GradParams& p) {
  const uint32_t lane = threadIdx.x & 31, groups = kThreads / p.group, mine = threadIdx.x / p.group, at = threadIdx.x % p.group;
  const uint32_t rows = p.lists.counts[0], step = p.row_ctas * groups;
  const Light none{0, 0, 0, 0};
  auto record = [&](uint32_t r) { return r < rows ? p.lists.light[r] : none; };
  auto tokens_of = [&](const Light& l) { return lane < l.count ? p.idx[l.first + lane] : 0u; };
  uint32_t r = blockIdx.x * groups + mine;
  Light now = record(r), next = record(r + step);
  uint32_t tokens = tokens_of(now);
  for (; r < rows; r += step) {
    const Light after = record(r + 2 * step);
    const uint32_t next_tokens = tokens_of(next);
    for (uint32_t c0 = at; c0 < p.row_vecs + at; c0 += p.group * kCols) {  // whole warps: the tokens come from its lanes
      float acc[kCols][EV] = {};
      for (uint32_t i = 0; i < now.count; i += 2) {
        Vec<T, EV> x[2][kCols];
        const uint32_t first = __shfl_sync(0xffffffffu, tokens, i & 31), second = __shfl_sync(0xffffffffu, tokens, (i + 1) & 31);
        const bool two = i + 1 < now.count;
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
          const uint32_t c = c0 + u * p.group;
          if (c < p.row_vecs) x[0][u] = token_vec<T, EV>(p, first, c);
          if (two && c < p.row_vecs) x[1][u] = token_vec<T, EV>(p, second, c);
        }
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
          const uint32_t c = c0 + u * p.group;
          if (c < p.row_vecs) add_vec<T, EV>(acc[u], x[0][u]);
          if (two && c < p.row_vecs) add_vec<T, EV>(acc[u], x[1][u]);
        }
      }
#pragma unroll
      for (int u = 0; u < kCols; ++u)
        if (c0 + u * p.group < p.row_vecs) finish_row<O, EV>(p, acc[u], now.row, c0 + u * p.group);
    }
    now = next;
    next = after;
    tokens = next_tokens;
  }
}

// CTAs [0, p.row_ctas) sum the rows that have tokens; the others fill.
template <typename T, typename O, int EV, typename W>
__global__ void __launch_bounds__(kThreads, 4) grad_rows_kernel(const GradParams p, const FillParams f) {
  __shared__ float meet[kSumWarps][32][EV];
  if (blockIdx.x >= p.row_ctas) {
    fill<W>(f, blockIdx.x - p.row_ctas);
    return;
  }
  heavy_rows<T, O, EV>(p, meet);
  light_rows<T, O, EV>(p);
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

constexpr int64_t kMostWords = int64_t(1) << 31;  // words are counted in 32 bits

// The rows [r0, r0 + rows) of the gradient in words of W.
template <typename W>
static FillParams fill_params(const mllm_grpo_embedding_args* a, const uint8_t* busy, int64_t r0, int64_t rows) {
  const int64_t eo = elem(a->out_dtype), row_words = a->hidden * eo / int64_t(sizeof(W));
  FillParams f{a->weight_stride * eo / int64_t(sizeof(W)), uint32_t(rows * row_words), uint32_t(row_words),
               FastDiv(uint32_t(row_words)), busy ? busy + r0 : nullptr, nullptr, nullptr, 0};
  f.out = static_cast<W*>(a->dweight) + r0 * f.stride;
  return f;
}
// A whole table whose rows follow one another, as one row of 16-byte words, whatever its width (odd widths an element at
// a time: 3.3 TB/s).
static bool flat_table(const mllm_grpo_embedding_args* a) {
  return a->weight_stride == a->hidden && aligned(a->dweight, 16) && a->vocab * a->hidden * elem(a->out_dtype) / 16 <= kMostWords;
}
static FillParams flat_params(const mllm_grpo_embedding_args* a) {
  const int64_t bytes = a->vocab * a->hidden * elem(a->out_dtype), words = bytes / 16;
  return FillParams{0, uint32_t(words), uint32_t(words), FastDiv(words ? uint32_t(words) : 1u), nullptr, a->dweight,
                    reinterpret_cast<uint16_t*>(static_cast<char*>(a->dweight) + words * 16), uint32_t(bytes % 16 / 2)};
}
static unsigned fill_ctas(const FillParams& f) { return f.total / (kThreads * kVecs) + 1; }

template <typename W>
static int64_t rows_per_fill(const mllm_grpo_embedding_args* a) { return kMostWords / (a->hidden * elem(a->out_dtype) / int64_t(sizeof(W))); }

template <typename W>
static cudaError_t launch_fill(const mllm_grpo_embedding_args* a, const uint8_t* busy, int64_t from, int64_t to, cudaStream_t s) {
  const int64_t rows_per = rows_per_fill<W>(a);
  for (int64_t r0 = from; r0 < to; r0 += rows_per) {
    const FillParams f = fill_params<W>(a, busy, r0, to - r0 < rows_per ? to - r0 : rows_per);
    fill_kernel<W><<<fill_ctas(f), kThreads, 0, s>>>(f);
    const cudaError_t e = done();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Bytes of zeros that take as long as the sort (14 us, 25 us for 32768 tokens), and somewhat more: 18 us and 36.
static int64_t sort_bytes(int64_t n_tokens) { return (int64_t(128) << 20) + n_tokens * 4096; }

// Beside the sort: the zeros of the first p.filled rows, the list and the sums of runs.
template <typename T, int EV, typename W>
static cudaError_t launch_fill_runs(const mllm_grpo_embedding_args* a, const GradParams& p, uint32_t row_vecs, cudaStream_t s) {
  const bool flat = sizeof(W) == 16 && p.filled == p.vocab && flat_table(a);
  const int64_t rows_per = flat ? p.vocab : rows_per_fill<W>(a), rows = p.filled < rows_per ? p.filled : rows_per;
  const FillParams f = flat ? flat_params(a) : fill_params<W>(a, nullptr, 0, rows);
  const uint32_t warps = kThreads / 32, runs = (p.n + kRun - 1) / kRun, fills = fill_ctas(f);
  Beside b;
  b.row_vecs = row_vecs;
  b.parts = (row_vecs + 31) / 32;
  b.list_ctas = (runs + warps - 1) / warps;
  b.sum_ctas = uint32_t((int64_t(runs) * b.parts + warps - 1) / warps);
  // late enough for the sort to be done
  const int64_t late = sort_bytes(p.n) / (kThreads * kVecs * int64_t(sizeof(W)));
  b.first = uint32_t(fills < late ? fills : late);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(fills + b.list_ctas + b.sum_ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fill_runs_kernel<T, EV, W>, p, f, b);
  count_launch();
  return e == cudaSuccess && rows < p.filled ? launch_fill<W>(a, nullptr, rows, p.filled, s) : e;
}

template <typename T, typename O, int EV, typename W>
static cudaError_t launch_rows_w(const mllm_grpo_embedding_args* a, GradParams p, cudaStream_t s) {
  // four CTAs are resident per SM: with many rows they are all busy with rows at first
  const int64_t most = 148 * 4, items = (int64_t(p.n) * p.group + kThreads - 1) / kThreads;
  p.row_ctas = uint32_t(items < most ? items : most);
  if (p.filled == p.vocab) {
    grad_rows_kernel<T, O, EV, W><<<p.row_ctas, kThreads, 0, s>>>(p, FillParams{0, 0, 1, FastDiv(1), nullptr, nullptr, nullptr, 0});
    return done();
  }
  const int64_t left = a->vocab - p.filled, rows = left < rows_per_fill<W>(a) ? left : rows_per_fill<W>(a);
  const FillParams f = fill_params<W>(a, p.busy, p.filled, rows);
  grad_rows_kernel<T, O, EV, W><<<p.row_ctas + fill_ctas(f), kThreads, 0, s>>>(p, f);
  const cudaError_t e = done();
  return e == cudaSuccess ? launch_fill<W>(a, p.busy, p.filled + rows, p.vocab, s) : e;
}

// Zeros are written in the widest words that every row allows: 16 bytes, or an element.
static bool wide_rows(const mllm_grpo_embedding_args* a) {
  const int64_t eo = elem(a->out_dtype);
  return ((a->hidden * eo | a->weight_stride * eo | int64_t(reinterpret_cast<uintptr_t>(a->dweight) & 15)) & 15) == 0;
}

// The whole gradient's zeros.
static cudaError_t launch_zeros(const mllm_grpo_embedding_args* a, cudaStream_t s) {
  if (flat_table(a)) {
    const FillParams f = flat_params(a);
    fill_kernel<uint4><<<fill_ctas(f), kThreads, 0, s>>>(f);
    return done();
  }
  if (wide_rows(a)) return launch_fill<uint4>(a, nullptr, 0, a->vocab, s);
  return a->out_dtype == MLLM_GRPO_F32 ? launch_fill<uint32_t>(a, nullptr, 0, a->vocab, s) : launch_fill<uint16_t>(a, nullptr, 0, a->vocab, s);
}

// Rows whose zeros are written beside the sort.  Those of them that have tokens are written twice.  All rows where that
// costs little, because few or narrow rows can have tokens: 151936 f32 rows, this way / all zeros in the last launch,
// 2048 tokens of width 896 81 / 94 us, 32768 of them 124 / 135, 4096 of width 3584 317 / 328.  (But 16384 of width 3584
// 390 / 366.)  Otherwise as many as fill the time until the rows with tokens are known: 8192 of width 3584 322, 16384
// 352 (three times as many: 357, six times: 364).
static int64_t rows_beside(const mllm_grpo_embedding_args* a) {
  const int64_t row = a->hidden * elem(a->out_dtype);
  if (a->accumulate || row <= 4096 || a->n_tokens * row <= int64_t(64) << 20) return a->vocab;
  const int64_t rows = sort_bytes(a->n_tokens) / row + 1;
  return rows < a->vocab ? rows : a->vocab;
}

template <typename T, int EV>
static cudaError_t launch_runs(const mllm_grpo_embedding_args* a, const GradParams& p, cudaStream_t s) {
  const auto go = [&](auto wide, uint32_t row_vecs) {
    constexpr int V = decltype(wide)::value;
    if (!p.accumulate) {
      if (wide_rows(a) || (p.filled == p.vocab && flat_table(a))) return launch_fill_runs<T, V, uint4>(a, p, row_vecs, s);
      return a->out_dtype == MLLM_GRPO_F32 ? launch_fill_runs<T, V, uint32_t>(a, p, row_vecs, s)
                                           : launch_fill_runs<T, V, uint16_t>(a, p, row_vecs, s);
    }
    const uint32_t runs = (p.n + kRun - 1) / kRun, threads = row_vecs <= 32 ? 32 : (row_vecs <= 64 ? 64 : 128);
    run_kernel<T, V><<<dim3(runs, (row_vecs + threads - 1) / threads + 1), threads, 0, s>>>(p, row_vecs);
    return done();
  };
  constexpr int kWide = 16 / int(sizeof(T));
  if (vec_of(p.hidden, kWide, p.grad, p.grad_stride, sizeof(T), p.run, p.hidden, 2) == kWide)
    return go(std::integral_constant<int, kWide>(), p.hidden / kWide);
  return go(std::integral_constant<int, EV>(), p.row_vecs);
}

template <typename T, typename O, int EV>
static cudaError_t launch_rows(const mllm_grpo_embedding_args* a, const GradParams& p, cudaStream_t s) {
  if (wide_rows(a)) return launch_rows_w<T, O, EV, uint4>(a, p, s);
  return launch_rows_w<T, O, EV, O>(a, p, s);
}

template <typename T, int EV>
static cudaError_t launch_grad_ev(const mllm_grpo_embedding_args* a, const GradParams& p, cudaStream_t s) {
  const cudaError_t e = launch_runs<T, EV>(a, p, s);
  if (e != cudaSuccess) return e;
  if (a->out_dtype == MLLM_GRPO_F32) return launch_rows<T, float, EV>(a, p, s);
  if (a->out_dtype == MLLM_GRPO_F16) return launch_rows<T, __half, EV>(a, p, s);
  return launch_rows<T, __nv_bfloat16, EV>(a, p, s);
}

template <typename T>
static cudaError_t launch_grad_t(const mllm_grpo_embedding_args* a, GradParams p, cudaStream_t s) {
  // four elements a vector (16 bytes of f32 sums and gradients), or one
  const int ev = vec_of(a->hidden, 4, a->grad_out, a->token_stride, sizeof(T), a->dweight, a->weight_stride, elem(a->out_dtype));
  p.row_vecs = uint32_t(a->hidden / (ev == 4 ? 4 : 1));
  p.group = 32;
  while (p.group * kCols < p.row_vecs && p.group < uint32_t(kThreads)) p.group *= 2;
  p.parts = (p.row_vecs + 31) / 32;
  p.by_part = FastDiv(p.parts);
  return ev == 4 ? launch_grad_ev<T, 4>(a, p, s) : launch_grad_ev<T, 1>(a, p, s);
}

static cudaError_t launch_sort(const SortParams& q, bool zero_rows, cudaStream_t s) {
  const int ctas = q.n <= uint32_t(kTile) ? 1 : (q.n <= uint32_t(8 * kTile) ? 8 : 16);
  // 16 rows' marks a thread, in whole clusters
  int64_t more = zero_rows ? (q.vocab + kSortThreads * 16 - 1) / (kSortThreads * 16) : 0;
  more = more > 128 ? 128 : more;
  more = (more + ctas - 1) / ctas * ctas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas + more));
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(ctas);
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  if (ctas == 16) {
    static std::once_flag once[64];
    static cudaError_t err[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::call_once(once[dev], [&] {
      err[dev] = cudaFuncSetAttribute(sort_kernel<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (err[dev] != cudaSuccess) return err[dev];
  }
  const cudaError_t e = ctas == 1 ? cudaLaunchKernelEx(&cfg, sort_kernel<1>, q)
                                  : (ctas == 8 ? cudaLaunchKernelEx(&cfg, sort_kernel<8>, q) : cudaLaunchKernelEx(&cfg, sort_kernel<16>, q));
  count_launch();
  return e;
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
                      a->vocab_total ? a->vocab_total : a->vocab_start + a->vocab, 0, 0, FastDiv(1), a->scale,
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

int64_t mllm_grpo_embedding_workspace_bytes(int64_t n_tokens, int64_t hidden, int64_t vocab) {
  if (n_tokens < 0 || hidden <= 0 || vocab <= 0 || n_tokens >= (int64_t(1) << 31) || hidden > (int64_t(1) << 20) ||
      vocab >= (int64_t(1) << 31) - 1)
    return 0;
  // marks of the rows, two ping-pong pairs of lists, the lists of rows that have tokens, the sums of runs
  return emb::round16(vocab) + 5 * emb::round16(n_tokens * 4) + 16 + n_tokens * int64_t(sizeof(emb::Light)) +
         n_tokens / emb::kRun * hidden * 4;
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
  if (n == 0 && a->accumulate) return MLLM_GRPO_OK;
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
  q.busy = reinterpret_cast<uint4*>(w);
  w += emb::round16(a->vocab);
  for (int i = 0; i < 2; ++i) {
    q.key[i] = reinterpret_cast<uint32_t*>(w + (2 * i) * list);
    q.idx[i] = reinterpret_cast<uint32_t*>(w + (2 * i + 1) * list);
  }
  w += 4 * list;
  emb::Lists lists;
  lists.heavy = reinterpret_cast<uint32_t*>(w);
  lists.counts = reinterpret_cast<uint32_t*>(w + list);
  lists.light = reinterpret_cast<emb::Light*>(w + list + 16);
  q.counts = lists.counts;
  q.device_status = a->device_status;
  const int last = (q.passes - 1) & 1;
  cudaError_t e = cudaSuccess;
  if (n) {
    const int64_t filled = emb::rows_beside(a);
    e = emb::launch_sort(q, filled < a->vocab, s);
    if (e != cudaSuccess) return record_cuda_error(e);
    emb::GradParams p{a->token_stride, a->weight_stride, n, uint32_t(a->hidden), uint32_t(a->vocab), 0, a->accumulate ? 1u : 0u,
                      uint32_t(filled), 0, 0, 0, FastDiv(1), a->scale, q.key[last], q.idx[last], reinterpret_cast<uint8_t*>(q.busy), lists,
                      a->grad_out, a->dweight,
                      reinterpret_cast<float*>(w + list + 16 + int64_t(n) * int64_t(sizeof(emb::Light)))};
    if (a->dtype == MLLM_GRPO_BF16)
      e = emb::launch_grad_t<__nv_bfloat16>(a, p, s);
    else if (a->dtype == MLLM_GRPO_F16)
      e = emb::launch_grad_t<__half>(a, p, s);
    else
      e = emb::launch_grad_t<float>(a, p, s);
  }
  if (n == 0) e = emb::launch_zeros(a, s);  // the accumulated form has returned
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

}  // extern "C"
