// Preference loss over paired log ratios, forward and backward, from logits or from per-token log-probs.
//
//   lp_st = y_c - log sum_j e^(y_j)     lp_s = sum_t m_st lp_st (/ sum_t m_st)     d_s = lp_s - ref_s
//   h_p = d_p - d_(P+p)     loss = sum_p w_p l(h_p) / total
//   d loss / d x_stj = c_s m_st (onehot_j - softmax_j),   c_p = w_p l'(h_p) / total (/ sum m),  c_(P+p) likewise, negated
//
// Three launches from logits: pref_stats_kernel reads every row whose mask is not 0 once, pref_pairs_kernel adds
// the tokens up and finds c_s, pref_dlogits_kernel reads those rows again and writes the gradient.  A pair's
// coefficient depends on all of its rows, and a pair (hundreds of MB at a large vocabulary) does not stay on chip,
// so the second read cannot be saved as in the token loss.
//
// A sequence sum of a thousand log-probs is compared with another one nearly as large: what would be harmless in
// one log-prob adds up.  So the row maximum is carried as the exponent offset mk = m*log2(e) that the exponentials
// really use (e^(y-m) as 2^(y*log2e - mk) is off by the rounding of mk, the same way for every row with this
// maximum), and log-sum-exp, differences and sums are double precision, a few operations per token.
#include "grpo_common.cuh"
#include "grpo_launch.h"
#include "grpo_rowpass.cuh"

namespace grpo {
namespace pref {

constexpr int kMaxSplits = 32;
constexpr int64_t kTargetCtas = 4736;   // 32 per SM, about half of which have a masked row and leave
constexpr int64_t kWarpCols = 2048;
constexpr int64_t kMinSplitCols = 8192; // 16 KB of a row per CTA at least
// Threads per pair, for answers of more than kShortTokens and for short ones (8192 pairs of single tokens: 62 us with
// 512, 17 with 128; 8 pairs of 1024: 6.1 and 8.1; one pair of 16384: 25 and 82).
constexpr int kPairThreads = 512, kPairThreadsShort = 128;
constexpr int64_t kShortTokens = 128;

struct Params {
  int64_t n_pairs, seq_rows, scored_rows, vocab, row_stride;
  int kind, average, splits, ref_per_sequence;
  int64_t split_cols;  // columns per split, a multiple of 8
  float beta, smooth, softcap, grad_scale, total;
  const uint16_t* logits;
  const int32_t* ids;
  const float* logps;
  const void* mask;
  int64_t ids_stride, mask_stride;
  int mask_int;
  const float* ref;
  const float* weights;
  const float* total_dev;
  const float* grad_scale_dev;
  float* loss;
  float* rewards;
  float* seq_logps;
  float* dlogps;
  uint16_t* dlogits;
  // workspace
  double* terms;        // [P]
  float* coef;          // [2P]
  unsigned int* ticket; // [0] pairs done, [1] MLLM_GRPO_DEV_* bits of this call
  float* lse;           // [N]
  float* chosen;        // [N]
  float2* stats;        // [N, splits] (mk, S)
  int32_t* device_status;
  int32_t* call_status;
};

__host__ __device__ inline int64_t round16(int64_t b) { return (b + 15) & ~int64_t(15); }

// Splits of a row over CTAs: only as many as it takes to give every SM a few CTAs.
static int64_t max_splits(int64_t n_tokens) {
  const int64_t s = (kTargetCtas + n_tokens - 1) / n_tokens;
  return s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : s);
}

__device__ __forceinline__ bool live_token(const Params& p, int64_t s, int64_t t, float* m) {
  *m = 1.0f;
  if (p.mask) {
    const int64_t at = s * p.mask_stride + t;
    *m = p.mask_int ? float(static_cast<const int32_t*>(p.mask)[at]) : static_cast<const float*>(p.mask)[at];
  }
  return *m != 0.f;
}

// Running (m, S) of a thread; mk = fl(m * log2e) is the offset every exponential of the thread uses.
struct Acc {
  float m, mk, s;
  __device__ __forceinline__ void init() {
    m = kNegInit;
    mk = kNegInit * kLog2e;
    s = 0.f;
  }
  __device__ __forceinline__ void raise(float to) {
    const float k = to * kLog2e;
    s *= ex2f(mk - k);
    m = to;
    mk = k;
  }
};

template <bool CAP, int NV>
__device__ __forceinline__ void fold(Acc& a, const uint4 (&v)[NV], const SoftCap& sc) {
  uint32_t mx2 = v[0].x;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i) mx2 = bf16x2_max(mx2, v[i].x);
    mx2 = bf16x2_max(mx2, v[i].y);
    mx2 = bf16x2_max(mx2, v[i].z);
    mx2 = bf16x2_max(mx2, v[i].w);
  }
  float mx = fmaxf(bf16lo(mx2), bf16hi(mx2));
  if (CAP) mx = sc.y(mx);
  if (mx > a.m) a.raise(mx);
  const float mk = a.mk;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = bf16lo(w[j]), y = bf16hi(w[j]);
      if (CAP) {
        x = sc.y(x);
        y = sc.y(y);
      }
      s0 += ex2f(fmaf(x, kLog2e, -mk));
      s1 += ex2f(fmaf(y, kLog2e, -mk));
    }
  }
  a.s += s0 + s1;
}

template <bool CAP>
__device__ __forceinline__ void fold_one(Acc& a, uint16_t raw, const SoftCap& sc) {
  const float x = __uint_as_float(uint32_t(raw) << 16);
  const float y = CAP ? sc.y(x) : x;
  if (y > a.m) a.raise(y);
  a.s += ex2f(fmaf(y, kLog2e, -a.mk));
}

// THREADS threads per row (threadIdx.x), ROWS rows per CTA (threadIdx.y): one, or kRowsPerCta of a warp each.
constexpr int kRowsPerCta = 8;

// One CTA (warp) per (scored row, split).  Bound by reading the unmasked rows once.
template <int THREADS, int ROWS, int UNROLL, bool CAP>
__global__ void __launch_bounds__(THREADS * ROWS, ROWS > 1 ? 5 : 0) pref_stats_kernel(const Params p) {
  constexpr int NW = THREADS / 32;
  __shared__ float red[2][NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blockIdx.x == 0 && (ROWS == 1 || threadIdx.y == 0) && tid < 2) p.ticket[tid] = 0u;
  const unsigned item = ROWS > 1 ? blockIdx.x * ROWS + threadIdx.y : blockIdx.x;
  if (ROWS > 1 && item >= unsigned(2 * p.n_pairs * p.scored_rows)) return;
  const int64_t n = item / unsigned(p.splits);
  const int k = int(item - n * p.splits);
  float mask;
  const int64_t b = n / p.scored_rows, t = n - b * p.scored_rows;
  if (!live_token(p, b, t, &mask)) return;
  const uint16_t* row = p.logits + (b * p.seq_rows + t) * p.row_stride;
  const int64_t c0 = int64_t(k) * p.split_cols;
  const int64_t V = p.vocab - c0 < p.split_cols ? p.vocab - c0 : p.split_cols;  // > 0 by the choice of splits
  const SoftCap sc(CAP ? p.softcap : 1.0f);
  Acc a;
  a.init();
  const uint16_t* row16 = row + c0;
  const RowSplit sp(row16, V);
  if (tid < sp.head) fold_one<CAP>(a, row16[tid], sc);
  if (tid < sp.tail) fold_one<CAP>(a, row16[sp.head + (sp.nvec << 3) + tid], sc);
  const uint4* vec = reinterpret_cast<const uint4*>(row16 + sp.head);
  int64_t i = tid;
  constexpr int64_t kStep = int64_t(UNROLL) * THREADS;
  for (; i + kStep - THREADS < sp.nvec; i += kStep) {
    uint4 v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) v[u] = ldg_stream(vec + i + int64_t(u) * THREADS);
    fold<CAP, UNROLL>(a, v, sc);
  }
  if (i < sp.nvec) {
    uint4 v[UNROLL - 1];
#pragma unroll
    for (int u = 0; u < UNROLL - 1; ++u)
      if (i + int64_t(u) * THREADS < sp.nvec) v[u] = ldg_stream(vec + i + int64_t(u) * THREADS);
#pragma unroll
    for (int u = 0; u < UNROLL - 1; ++u) {
      if (i + int64_t(u) * THREADS < sp.nvec) {
        const uint4 one[1] = {v[u]};
        fold<CAP, 1>(a, one, sc);
      }
    }
  }
  const float Mw = warp_max(a.mk);
  const float Sw = warp_sum(a.s * ex2f(a.mk - Mw));
  if (NW > 1) {
    if (lane == 0) {
      red[0][warp] = Mw;
      red[1][warp] = Sw;
    }
    __syncthreads();
  }
  if (warp == 0) {
    float M = Mw, S = Sw;
    if (NW > 1) {
      const float m_in = lane < NW ? red[0][lane] : kNegInit * kLog2e;
      M = warp_max(m_in);
      S = warp_sum(lane < NW ? red[1][lane] * ex2f(m_in - M) : 0.f);
    }
    if (lane == 0) {
      p.stats[n * p.splits + k] = make_float2(M, S);
      int64_t c = p.ids[b * p.ids_stride + t];
      c = c < 0 ? 0 : (c >= p.vocab ? p.vocab - 1 : c);  // the launch that follows reports it
      if (c >= c0 && c < c0 + V) {
        const float x = __uint_as_float(uint32_t(row[c]) << 16);
        p.chosen[n] = CAP ? sc.y(x) : x;
      }
    }
  }
}

// Log-prob of token (s, t) in double precision; from logits, its log-sum-exp is kept for the backward sweep.
template <bool LOGPS>
__device__ __forceinline__ double token_logp(const Params& p, int64_t s, int64_t t) {
  const int64_t n = s * p.scored_rows + t;
  if (LOGPS) return double(p.logps[n]);
  const int64_t c = p.ids[s * p.ids_stride + t];
  if (c < 0 || c >= p.vocab) {
    atomicOr(p.ticket + 1, unsigned(MLLM_GRPO_DEV_ID_CLAMPED));
    if (p.device_status) atomicOr(p.device_status, MLLM_GRPO_DEV_ID_CLAMPED);
  }
  const float2* st = p.stats + n * p.splits;
  float M = st[0].x;
  for (int k = 1; k < p.splits; ++k) M = fmaxf(M, st[k].x);
  double S = 0.0;
  for (int k = 0; k < p.splits; ++k) S += double(st[k].y) * double(exp2f(st[k].x - M));
  // the sums are powers of two with the f32 constant kLog2e in the exponent: dividing by the same constant
  // cancels its rounding to first order
  const double lse = (double(M) + log2(S)) / double(kLog2e);
  p.lse[n] = float(lse);
  return double(p.chosen[n]) - lse;
}

struct SeqSums {
  double diff, lp, count;
};

// This thread's share (tid of nt) of sequence s.
template <bool LOGPS>
__device__ __forceinline__ SeqSums sequence_sums(const Params& p, int64_t s, int tid, int nt) {
  SeqSums a{0.0, 0.0, 0.0};
  const bool per_token = p.ref != nullptr && !p.ref_per_sequence;
#pragma unroll 2
  for (int64_t t = tid; t < p.scored_rows; t += nt) {
    float m;
    if (!live_token(p, s, t, &m)) continue;
    const double lp = token_logp<LOGPS>(p, s, t);
    a.lp += double(m) * lp;
    a.diff += double(m) * (per_token ? lp - double(p.ref[s * p.scored_rows + t]) : lp);
    a.count += double(m);
  }
  return a;
}

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ SeqSums warp_add(SeqSums a) { return SeqSums{warp_add(a.diff), warp_add(a.lp), warp_add(a.count)}; }

// log(1 + e^z) without overflow
__device__ __forceinline__ double softplus(double z) { return z > 0.0 ? z + log1p(exp(-z)) : log1p(exp(z)); }

// Everything of pair `pair` once its six sums are known; returns the two coefficients.
__device__ __forceinline__ float2 finish_pair(const Params& p, int64_t pair, SeqSums c, SeqSums r) {
  const int64_t P = p.n_pairs;
  double inv_c = 1.0, inv_r = 1.0;
  if (p.average) {
    inv_c = c.count != 0.0 ? 1.0 / c.count : 0.0;
    inv_r = r.count != 0.0 ? 1.0 / r.count : 0.0;
  }
  // sums of an empty (or cancelling) mask stay 0 instead of 0 * inf
  double dc = c.diff * inv_c, dr = r.diff * inv_r;
  if (p.ref != nullptr && p.ref_per_sequence) {
    dc -= double(p.ref[pair]);
    dr -= double(p.ref[P + pair]);
  }
  const double h = dc - dr, beta = double(p.beta), e = double(p.smooth), z = beta * h;
  double term, dh;
  if (p.kind == MLLM_GRPO_PREFERENCE_SIGMOID) {
    term = (1.0 - e) * softplus(-z);
    dh = -beta * (1.0 - e) / (1.0 + exp(z));
    if (e != 0.0) {
      term += e * softplus(z);
      dh += beta * e / (1.0 + exp(-z));
    }
  } else if (p.kind == MLLM_GRPO_PREFERENCE_HINGE) {
    term = z < 1.0 ? 1.0 - z : (z == z ? 0.0 : z);
    dh = z < 1.0 ? -beta : (z == z ? 0.0 : z);
  } else {
    const double off = h - 0.5 / beta;
    term = off * off;
    dh = 2.0 * off;
  }
  const float w = p.weights ? p.weights[pair] : 1.0f;
  const double total = double(p.total_dev ? *p.total_dev : p.total);
  // a pair of weight 0 is padding: whatever its sums are, it adds nothing
  const double scale = w != 0.f ? double(w) / total : 0.0;
  p.terms[pair] = w != 0.f ? double(w) * term : 0.0;
  p.rewards[pair] = float(beta * dc);
  p.rewards[P + pair] = float(beta * dr);
  if (p.seq_logps) {
    p.seq_logps[pair] = float(c.lp * inv_c);
    p.seq_logps[P + pair] = float(r.lp * inv_r);
  }
  const float2 k = scale != 0.0 ? make_float2(float(dh * scale * inv_c), float(-dh * scale * inv_r)) : make_float2(0.f, 0.f);
  p.coef[pair] = k.x;
  p.coef[P + pair] = k.y;
  return k;
}

__device__ __forceinline__ void write_dlogps(const Params& p, int64_t s, float coef, int tid, int nt) {
  const float gs = p.grad_scale_dev ? *p.grad_scale_dev : p.grad_scale;
  for (int64_t t = tid; t < p.scored_rows; t += nt) {
    float m;
    p.dlogps[s * p.scored_rows + t] = live_token(p, s, t, &m) ? coef * m * gs : 0.f;
  }
}

__device__ __forceinline__ double block_sum(double v, double* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = warp_add(v);
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  double tot = 0.0;
  for (int w = 0; w < nw; ++w) tot += red[w];
  return tot;
}

__device__ __forceinline__ void reduce_loss(const Params& p, double* red) {
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < p.n_pairs; i += blockDim.x) a += __ldcg(p.terms + i);
  a = block_sum(a, red);
  if (threadIdx.x == 0) *p.loss = float(a / double(p.total_dev ? *p.total_dev : p.total));
}

// One CTA per pair, half of it per answer.  From logits the CTA that finishes last adds the pairs up (the ticket was
// zeroed by the stats launch before this one); from log-probs the sum has a launch of its own, since nothing ran before
// to zero it (5 us for both, up to a few hundred pairs; one CTA that does everything took 8.6 us for 8 pairs of 255
// tokens and 49 for 256 pairs of one).
template <bool LOGPS, int THREADS>
__global__ void __launch_bounds__(THREADS) pref_pairs_kernel(const Params p) {
  constexpr int kHalf = THREADS / 2, kHalfWarps = kHalf / 32;
  __shared__ double red[32];
  __shared__ SeqSums sums[2 * kHalfWarps];
  __shared__ float2 k_shared;
  __shared__ bool last;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int side = threadIdx.x / kHalf, tid = threadIdx.x % kHalf;
  const int64_t pair = blockIdx.x, s = side * p.n_pairs + pair;
  const SeqSums mine = warp_add(sequence_sums<LOGPS>(p, s, tid, kHalf));
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    SeqSums a[2];
    for (int k = 0; k < 2; ++k) {
      a[k] = sums[k * kHalfWarps];
      for (int w = 1; w < kHalfWarps; ++w) {
        a[k].diff += sums[k * kHalfWarps + w].diff;
        a[k].lp += sums[k * kHalfWarps + w].lp;
        a[k].count += sums[k * kHalfWarps + w].count;
      }
    }
    k_shared = finish_pair(p, pair, a[0], a[1]);
    if (!LOGPS) {
      __threadfence();
      last = atomicAdd(p.ticket, 1u) == unsigned(p.n_pairs - 1);
      __threadfence();
    }
  }
  __syncthreads();
  if (LOGPS) {
    if (p.dlogps) write_dlogps(p, s, side ? k_shared.y : k_shared.x, tid, kHalf);
  } else if (last) {
    reduce_loss(p, red);
    if (threadIdx.x == 0 && p.call_status) *p.call_status = int32_t(atomicOr(p.ticket + 1, 0u));
  }
}

__global__ void __launch_bounds__(kPairThreads) pref_loss_kernel(const Params p) {
  __shared__ double red[32];
  reduce_loss(p, red);
  if (threadIdx.x == 0 && p.call_status) *p.call_status = 0;  // no ids, nothing to raise
}

// Gradient of one row (or its split); rows without a coefficient are written as zeros and not read.  Taking the rows in
// the opposite order of the forward sweep, with or without L2 policies that keep its last 32 MB, changed nothing
// measurable (229 us against 228 for 4 x 256 pairs at 151936 columns).
template <int THREADS, int ROWS, int UNROLL, bool CAP, bool SCALAR>
__global__ void __launch_bounds__(THREADS * ROWS, ROWS > 1 ? 5 : 0) pref_dlogits_kernel(const Params p) {
  const unsigned item = ROWS > 1 ? blockIdx.x * ROWS + threadIdx.y : blockIdx.x;
  if (ROWS > 1 && item >= unsigned(2 * p.n_pairs * p.seq_rows)) return;
  const int64_t r = item / unsigned(p.splits);
  const int k = int(item - r * p.splits);
  const int64_t b = r / p.seq_rows, t = r - b * p.seq_rows;
  const int64_t c0 = int64_t(k) * p.split_cols;
  const int64_t V = p.vocab - c0 < p.split_cols ? p.vocab - c0 : p.split_cols;
  const uint16_t* x16 = p.logits + r * p.row_stride + c0;
  uint16_t* d16 = p.dlogits + r * p.row_stride + c0;
  float g = 0.f, lse = 0.f;
  int64_t cl = -1;
  float m = 0.f;
  const bool live = t < p.scored_rows && live_token(p, b, t, &m);
  // beside pref_pairs_kernel: zeros need nothing of it; some CTA has to end after it in any case
  if (live || blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (live) {
    const float gs = p.grad_scale_dev ? *p.grad_scale_dev : p.grad_scale;
    g = -p.coef[b] * m * gs;
    lse = p.lse[b * p.scored_rows + t];
    int64_t c = p.ids[b * p.ids_stride + t];
    c = c < 0 ? 0 : (c >= p.vocab ? p.vocab - 1 : c);
    cl = c - c0;
  }
  const SoftCap sc(CAP ? p.softcap : 1.0f);
  if (!SCALAR) {
    row_pass2<THREADS, UNROLL, CAP, 1>(x16, d16, V, g, lse, cl, sc, 0);
  } else {
    // logits and dlogits rows that do not share their offset from a 16-byte boundary
    for (int64_t j = threadIdx.x; j < V; j += THREADS) {
      float d = 0.f;
      if (g != 0.f) {
        const float x = __uint_as_float(uint32_t(x16[j]) << 16);
        const float y = CAP ? sc.y(x) : x;
        d = g * ex2f((y - lse) * kLog2e);
        if (j == cl) d -= g;
        if (CAP) d *= sc.dydx(y);
      }
      d16[j] = __bfloat16_as_ushort(__float2bfloat16_rn(d));
    }
  }
}

static cudaError_t done() {
  count_launch();
  return cudaGetLastError();
}

template <bool LOGPS>
static cudaError_t launch_pairs(const Params& p, cudaStream_t s) {
  if (p.scored_rows <= kShortTokens)
    pref_pairs_kernel<LOGPS, kPairThreadsShort><<<unsigned(p.n_pairs), kPairThreadsShort, 0, s>>>(p);
  else
    pref_pairs_kernel<LOGPS, kPairThreads><<<unsigned(p.n_pairs), kPairThreads, 0, s>>>(p);
  return done();
}

// Short rows are a warp's each: 26 x 773 rows of 231 columns 30 us, with a CTA each 50; 32 x 512 of 2048 39 and 47, of
// 4096 67 and 63.
static bool warp_rows(const Params& p) { return p.splits == 1 && p.vocab <= kWarpCols; }

static cudaError_t launch_forward(const Params& p, cudaStream_t s) {
  const unsigned grid = unsigned(2 * p.n_pairs * p.scored_rows * p.splits);
  const bool cap = p.softcap > 0.f, small = p.split_cols <= 16384;
  if (warp_rows(p)) {
    const unsigned ctas = (grid + kRowsPerCta - 1) / kRowsPerCta;
    if (cap)
      pref_stats_kernel<32, kRowsPerCta, 4, true><<<ctas, dim3(32, kRowsPerCta), 0, s>>>(p);
    else
      pref_stats_kernel<32, kRowsPerCta, 4, false><<<ctas, dim3(32, kRowsPerCta), 0, s>>>(p);
  } else if (small) {
    if (cap)
      pref_stats_kernel<128, 1, 4, true><<<grid, 128, 0, s>>>(p);
    else
      pref_stats_kernel<128, 1, 4, false><<<grid, 128, 0, s>>>(p);
  } else if (cap) {
    pref_stats_kernel<512, 1, 4, true><<<grid, 512, 0, s>>>(p);
  } else {
    pref_stats_kernel<512, 1, 4, false><<<grid, 512, 0, s>>>(p);
  }
  cudaError_t e = done();
  if (e != cudaSuccess) return e;
  return launch_pairs<false>(p, s);
}

template <typename K>
static cudaError_t launch_rows(K* kernel, const Params& p, unsigned grid, dim3 threads, bool beside, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = threads;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = beside ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  count_launch();
  return e;
}

template <bool CAP>
static cudaError_t launch_backward_t(const Params& p, unsigned grid, bool same_phase, bool beside, cudaStream_t s) {
  if (!same_phase) return launch_rows(pref_dlogits_kernel<256, 1, 4, CAP, true>, p, grid, 256, beside, s);
  if (warp_rows(p)) {
    const unsigned ctas = (grid + kRowsPerCta - 1) / kRowsPerCta;
    return launch_rows(pref_dlogits_kernel<32, kRowsPerCta, 4, CAP, false>, p, ctas, dim3(32, kRowsPerCta), beside, s);
  }
  if (p.split_cols <= 16384) return launch_rows(pref_dlogits_kernel<128, 1, 4, CAP, false>, p, grid, 128, beside, s);
  return launch_rows(pref_dlogits_kernel<512, 1, 4, CAP, false>, p, grid, 512, beside, s);
}

// beside: right behind launch_forward, whose last launch it need not wait for as a whole.
static cudaError_t launch_backward(const Params& p, bool beside, cudaStream_t s) {
  const unsigned grid = unsigned(2 * p.n_pairs * p.seq_rows * p.splits);
  const bool same_phase = ((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.dlogits)) & 15) == 0;
  return p.softcap > 0.f ? launch_backward_t<true>(p, grid, same_phase, beside, s)
                         : launch_backward_t<false>(p, grid, same_phase, beside, s);
}

static bool aligned(const void* q, size_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) == 0; }

enum Need : unsigned { kLogits = 1, kForward = 2, kBackward = 4, kLogps = 8 };

static int bind(const mllm_grpo_preference_args* a, unsigned need, Params* p) {
  if (a == nullptr) return MLLM_GRPO_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(mllm_grpo_preference_args)) return MLLM_GRPO_ERR_STRUCT_SIZE;
  if (a->n_pairs <= 0 || a->scored_rows <= 0) return MLLM_GRPO_ERR_BAD_SHAPE;
  constexpr int64_t kMost = (int64_t(1) << 31) - 1;
  if (a->n_pairs > kMost / 2 || a->scored_rows > kMost / (2 * a->n_pairs)) return MLLM_GRPO_ERR_TOO_LARGE;
  const int64_t N = 2 * a->n_pairs * a->scored_rows;
  p->splits = 1;
  p->split_cols = 0;
  if (need & kLogits) {
    if (a->seq_rows < a->scored_rows || a->vocab <= 0 || a->row_stride < a->vocab) return MLLM_GRPO_ERR_BAD_SHAPE;
    if (a->seq_rows > kMost / (2 * a->n_pairs)) return MLLM_GRPO_ERR_TOO_LARGE;
    int64_t splits = (a->vocab + kMinSplitCols - 1) / kMinSplitCols;
    const int64_t most = max_splits(N);
    if (splits > most) splits = most;
    p->split_cols = ((a->vocab + splits - 1) / splits + 7) & ~int64_t(7);
    p->splits = int((a->vocab + p->split_cols - 1) / p->split_cols);  // none of them empty
    if (2 * a->n_pairs * a->seq_rows > kMost / p->splits) return MLLM_GRPO_ERR_TOO_LARGE;
  }
  if ((a->ids_stride != 0 && a->ids_stride < a->scored_rows) || (a->mask_stride != 0 && a->mask_stride < a->scored_rows))
    return MLLM_GRPO_ERR_BAD_SHAPE;
  if (a->kind < 0 || a->kind > MLLM_GRPO_PREFERENCE_IPO || !(a->beta > 0.f) || !(a->softcap >= 0.f) ||
      !(a->label_smoothing >= 0.f && a->label_smoothing <= 0.5f) ||
      (a->label_smoothing != 0.f && a->kind != MLLM_GRPO_PREFERENCE_SIGMOID))
    return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (!a->total_pairs_dev && !(a->total_pairs > 0.f)) return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (!a->workspace) return MLLM_GRPO_ERR_NULL_POINTER;
  if ((need & kLogits) && (!a->logits || !a->chosen_ids)) return MLLM_GRPO_ERR_NULL_POINTER;
  if ((need & kForward) && (!a->loss || !a->rewards)) return MLLM_GRPO_ERR_NULL_POINTER;
  if ((need & kLogps) && !a->token_logps) return MLLM_GRPO_ERR_NULL_POINTER;
  if ((need & kBackward) && !a->dlogits) return MLLM_GRPO_ERR_NULL_POINTER;
  const void* words[] = {a->chosen_ids, a->token_logps, a->mask, a->ref_logps, a->pair_weights, a->total_pairs_dev,
                         a->grad_scale_dev, a->loss, a->rewards, a->sequence_logps, a->dtoken_logps, a->device_status,
                         a->call_status};
  for (const void* q : words)
    if (!aligned(q, 4)) return MLLM_GRPO_ERR_ALIGNMENT;
  if (!aligned(a->logits, 2) || !aligned(a->dlogits, 2) || !aligned(a->workspace, 16)) return MLLM_GRPO_ERR_ALIGNMENT;

  p->n_pairs = a->n_pairs;
  p->seq_rows = a->seq_rows;
  p->scored_rows = a->scored_rows;
  p->vocab = a->vocab;
  p->row_stride = a->row_stride;
  p->kind = a->kind;
  p->average = a->average;
  p->ref_per_sequence = a->ref_per_sequence;
  p->beta = a->beta;
  p->smooth = a->label_smoothing;
  p->softcap = a->softcap;
  p->grad_scale = a->grad_scale;
  p->total = a->total_pairs;
  p->logits = static_cast<const uint16_t*>(a->logits);
  p->ids = a->chosen_ids;
  p->logps = a->token_logps;
  p->mask = a->mask;
  p->mask_int = a->mask_int;
  p->ids_stride = a->ids_stride ? a->ids_stride : a->scored_rows;
  p->mask_stride = a->mask_stride ? a->mask_stride : a->scored_rows;
  p->ref = a->ref_logps;
  p->weights = a->pair_weights;
  p->total_dev = a->total_pairs_dev;
  p->grad_scale_dev = a->grad_scale_dev;
  p->loss = a->loss;
  p->rewards = a->rewards;
  p->seq_logps = a->sequence_logps;
  p->dlogps = a->dtoken_logps;
  p->dlogits = static_cast<uint16_t*>(a->dlogits);
  p->device_status = a->device_status;
  p->call_status = a->call_status;
  char* w = static_cast<char*>(a->workspace);
  p->ticket = reinterpret_cast<unsigned int*>(w);
  w += 16;
  p->terms = reinterpret_cast<double*>(w);
  w += round16(a->n_pairs * 8);
  p->coef = reinterpret_cast<float*>(w);
  w += round16(a->n_pairs * 8);
  p->lse = reinterpret_cast<float*>(w);
  w += round16(N * 4);
  p->chosen = reinterpret_cast<float*>(w);
  w += round16(N * 4);
  p->stats = reinterpret_cast<float2*>(w);
  return MLLM_GRPO_OK;
}

}  // namespace pref
}  // namespace grpo

using namespace grpo;

extern "C" {

int64_t mllm_grpo_preference_workspace_bytes(int64_t n_pairs, int64_t scored_rows) {
  constexpr int64_t kMost = (int64_t(1) << 31) - 1;
  if (n_pairs <= 0 || scored_rows <= 0 || n_pairs > kMost / 2 || scored_rows > kMost / (2 * n_pairs)) return 0;
  const int64_t N = 2 * n_pairs * scored_rows;
  return 16 + 2 * pref::round16(n_pairs * 8) + 2 * pref::round16(N * 4) + N * pref::max_splits(N) * 8;
}

int mllm_grpo_preference_fwd(const mllm_grpo_preference_args* args, void* stream) {
  pref::Params p;
  const int st = pref::bind(args, pref::kLogits | pref::kForward, &p);
  if (st) return st;
  const cudaError_t e = pref::launch_forward(p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

int mllm_grpo_preference_bwd(const mllm_grpo_preference_args* args, void* stream) {
  pref::Params p;
  const int st = pref::bind(args, pref::kLogits | pref::kBackward, &p);
  if (st) return st;
  const cudaError_t e = pref::launch_backward(p, false, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

int mllm_grpo_preference_fwd_bwd(const mllm_grpo_preference_args* args, void* stream) {
  pref::Params p;
  const int st = pref::bind(args, pref::kLogits | pref::kForward | pref::kBackward, &p);
  if (st) return st;
  cudaError_t e = pref::launch_forward(p, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = pref::launch_backward(p, true, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

int mllm_grpo_preference_logps(const mllm_grpo_preference_args* args, void* stream) {
  pref::Params p;
  const int st = pref::bind(args, pref::kLogps | pref::kForward, &p);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = pref::launch_pairs<true>(p, s);
  if (e == cudaSuccess) {
    pref::pref_loss_kernel<<<1, pref::kPairThreads, 0, s>>>(p);
    e = pref::done();
  }
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

}  // extern "C"
