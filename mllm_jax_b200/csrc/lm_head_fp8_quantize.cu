// Quantising to e4m3 with a scale for each block of 128: rows of activations (1 x 128) or tiles of a weight
// (128 x 128).
//
//   top = max(max |x|, 448 * 2^-126)     scale = top / 448     q = e4m3(448 x / top)
//
// Bound by memory: every element is read once and kept in registers between the maximum and the conversion.
//
// The quotient: inputs of few bits often make 448 x / top EXACTLY the middle between two e4m3 values, where rounding
// to even decides; x * fl(448 / top) is off by up to 2 ulp and would fall to either side.  A true quotient of two
// 11-bit numbers that is not such a middle is at least 2^-17 (relative) away from it, so the product is rounded to 19
// bits first, which restores the middles and crosses none.  (For f32 inputs a quotient within 2^-19 of a middle
// counts as the middle.)  A division per element would cost more than the memory traffic allows.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "grpo_common.cuh"
#include "grpo_launch.h"

namespace grpo {
namespace fp8q {

constexpr int kThreads = 256;
constexpr float kMost = 448.0f;
constexpr float kLeast = 448.0f * 1.17549435e-38f;

struct Params {
  int64_t rows, cols, x_stride, q_stride, blocks;  // blocks along a row
  const void* x;
  uint8_t* q;
  float* scales;
};

__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(float v) { return v; }

template <typename T, int EV>
struct alignas(sizeof(T) * EV) Vec {
  T v[EV];
};
template <int EV>
struct alignas(EV) Bytes {
  uint8_t v[EV];
};

// y rounded to 19 bits: (33 y) - (33 y - y) keeps the upper part.
__device__ __forceinline__ float snap(float y) {
  const float c = __fmul_rn(y, 33.0f);
  return __fsub_rn(c, __fsub_rn(c, y));
}

// Two f32 -> two e4m3 bytes (first in the low byte), to nearest even; a NaN becomes the e4m3 NaN.
__device__ __forceinline__ uint16_t to_e4m3x2(float a, float b) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(b), "f"(a));
  return d;
}

// Scale of a block and the factor that brings it to [-448, 448].
__device__ __forceinline__ float factor(float amax, float* scale) {
  const float top = fmaxf(amax, kLeast);
  *scale = __fdiv_rn(top, kMost);
  return __fdiv_rn(kMost, top);
}

template <int EV, typename F>
__device__ __forceinline__ Bytes<EV> convert(const F& value, float r) {
  Bytes<EV> b;
  if (EV == 1) {
    b.v[0] = uint8_t(to_e4m3x2(snap(value(0) * r), 0.f));
  } else {
#pragma unroll
    for (int j = 0; j < EV; j += 2) {
      const uint16_t w = to_e4m3x2(snap(value(j) * r), snap(value(j + 1) * r));
      b.v[j] = uint8_t(w);
      b.v[j + 1] = uint8_t(w >> 8);
    }
  }
  return b;
}

// 1 x 128: 128 / EV consecutive threads hold a block (EV elements each; with one element a thread, 32 threads hold
// four each, 32 apart).
template <typename T, int EV>
__global__ void __launch_bounds__(kThreads) row_blocks_kernel(const Params p) {
  constexpr int G = EV == 1 ? 32 : (128 / EV > 32 ? 32 : 128 / EV);  // threads per block
  constexpr int U = 128 / (G * EV);                                   // vectors per thread
  const int64_t g = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / G;  // block of the whole matrix
  const int l = threadIdx.x % G;
  const int64_t row = g / p.blocks, b = g - row * p.blocks;
  const bool in = row < p.rows;
  const int64_t c0 = b * 128;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + c0;
  Vec<T, EV> v[U];
  float amax = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (u * G + l) * EV;
#pragma unroll
    for (int j = 0; j < EV; ++j) v[u].v[j] = T(0.f);
    if (in && c0 + c < p.cols) v[u] = *reinterpret_cast<const Vec<T, EV>*>(x + c);
#pragma unroll
    for (int j = 0; j < EV; ++j) amax = fmaxf(amax, fabsf(up(v[u].v[j])));
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float scale;
  const float r = factor(amax, &scale);
  if (!in) return;
  if (l == 0) p.scales[g] = scale;
  uint8_t* q = p.q + row * p.q_stride + c0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (u * G + l) * EV;
    if (c0 + c < p.cols)
      *reinterpret_cast<Bytes<EV>*>(q + c) = convert<EV>([&](int j) { return up(v[u].v[j]); }, r);
  }
}

// 128 x 128: one CTA per tile, the tile in registers.
template <typename T, int EV>
__global__ void __launch_bounds__(kThreads) tile_blocks_kernel(const Params p) {
  constexpr int PER_ROW = 128 / EV;                    // vectors of a tile row
  constexpr int U = 128 * PER_ROW / kThreads;          // vectors per thread
  __shared__ float red[kThreads / 32];
  const int64_t tr = blockIdx.x / p.blocks, tb = blockIdx.x - tr * p.blocks;
  const int64_t r0 = tr * 128, c0 = tb * 128;
  const T* x = static_cast<const T*>(p.x) + r0 * p.x_stride + c0;
  Vec<T, EV> v[U];
  float amax = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * kThreads + threadIdx.x, rr = i / PER_ROW, cc = (i % PER_ROW) * EV;
#pragma unroll
    for (int j = 0; j < EV; ++j) v[u].v[j] = T(0.f);
    if (r0 + rr < p.rows && c0 + cc < p.cols) v[u] = *reinterpret_cast<const Vec<T, EV>*>(x + rr * p.x_stride + cc);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < EV; ++j) amax = fmaxf(amax, fabsf(up(v[u].v[j])));
  amax = warp_max(amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, red[w]);
  float scale;
  const float r = factor(amax, &scale);
  if (threadIdx.x == 0) p.scales[blockIdx.x] = scale;
  uint8_t* q = p.q + r0 * p.q_stride + c0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * kThreads + threadIdx.x, rr = i / PER_ROW, cc = (i % PER_ROW) * EV;
    if (r0 + rr < p.rows && c0 + cc < p.cols)
      *reinterpret_cast<Bytes<EV>*>(q + rr * p.q_stride + cc) = convert<EV>([&](int j) { return up(v[u].v[j]); }, r);
  }
}

template <typename T, int EV>
static cudaError_t launch(const Params& p, int block_rows, cudaStream_t s) {
  if (block_rows == 1) {
    constexpr int G = EV == 1 ? 32 : (128 / EV > 32 ? 32 : 128 / EV);
    const int64_t groups = p.rows * p.blocks;
    row_blocks_kernel<T, EV><<<unsigned((groups + kThreads / G - 1) / (kThreads / G)), kThreads, 0, s>>>(p);
  } else {
    tile_blocks_kernel<T, EV><<<unsigned((p.rows + 127) / 128 * p.blocks), kThreads, 0, s>>>(p);
  }
  count_launch();
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_t(const Params& p, int block_rows, cudaStream_t s) {
  // widest vector (16 bytes of x at most) that every row of x and q allows
  int ev = 16 / int(sizeof(T));
  const uintptr_t x = reinterpret_cast<uintptr_t>(p.x), q = reinterpret_cast<uintptr_t>(p.q);
  while (ev > 1 && (p.cols % ev || p.x_stride % ev || p.q_stride % ev || x % (ev * sizeof(T)) || q % ev)) ev >>= 1;
  if (ev == 8) return launch<T, sizeof(T) == 2 ? 8 : 4>(p, block_rows, s);
  if (ev == 4) return launch<T, 4>(p, block_rows, s);
  if (ev == 2) return launch<T, 2>(p, block_rows, s);
  return launch<T, 1>(p, block_rows, s);
}

}  // namespace fp8q
}  // namespace grpo

using namespace grpo;

extern "C" int mllm_lm_head_fp8_quantize(const mllm_lm_head_fp8_quantize_args* a, void* stream) {
  if (a == nullptr) return MLLM_GRPO_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(mllm_lm_head_fp8_quantize_args)) return MLLM_GRPO_ERR_STRUCT_SIZE;
  if (a->rows < 0 || a->cols <= 0 || a->x_stride < a->cols || a->q_stride < a->cols) return MLLM_GRPO_ERR_BAD_SHAPE;
  if ((a->block_rows != 1 && a->block_rows != 128) || a->dtype < 0 || a->dtype > MLLM_GRPO_F32)
    return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  const int64_t blocks = (a->cols - 1) / 128 + 1;
  if (a->rows > (int64_t(1) << 32) || blocks > (int64_t(1) << 24)) return MLLM_GRPO_ERR_TOO_LARGE;
  // one CTA holds at least 8 row blocks, or one tile
  if ((a->block_rows == 1 ? a->rows / 8 + 1 : a->rows / 128 + 1) * blocks > (int64_t(1) << 31) - 1) return MLLM_GRPO_ERR_TOO_LARGE;
  if (a->rows == 0) return MLLM_GRPO_OK;
  if (!a->x || !a->q || !a->scales) return MLLM_GRPO_ERR_NULL_POINTER;
  const uintptr_t es = a->dtype == MLLM_GRPO_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->x) % es || reinterpret_cast<uintptr_t>(a->scales) % 4) return MLLM_GRPO_ERR_ALIGNMENT;
  const fp8q::Params p{a->rows, a->cols, a->x_stride, a->q_stride, blocks, a->x, static_cast<uint8_t*>(a->q), a->scales};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == MLLM_GRPO_BF16)
    e = fp8q::launch_t<__nv_bfloat16>(p, a->block_rows, s);
  else if (a->dtype == MLLM_GRPO_F16)
    e = fp8q::launch_t<__half>(p, a->block_rows, s);
  else
    e = fp8q::launch_t<float>(p, a->block_rows, s);
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}
