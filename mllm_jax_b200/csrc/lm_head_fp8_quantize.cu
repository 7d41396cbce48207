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

#include "grpo_common.cuh"
#include "grpo_launch.h"
#include "grpo_rowpass.cuh"

namespace grpo {
namespace fp8q {

constexpr int kThreads = 256;
constexpr float kMost = 448.0f;
constexpr float kLeast = 448.0f * 1.17549435e-38f;

template <typename T>
struct IsBf16 {
  static constexpr bool value = false;
};
template <>
struct IsBf16<__nv_bfloat16> {
  static constexpr bool value = true;
};

struct Params {
  int64_t rows, cols, x_stride, q_stride, blocks;  // blocks along a row
  FastDiv by_row;
  const void* x;
  uint8_t* q;
  float* scales;
};

// EV elements of x as raw 32-bit words: kept as they were read (two to a word for the 16-bit types) between the
// maximum and the conversion, and the maximum is taken on pairs.  (Holding f32 values instead took 224 registers in
// the 128 x 128 kernel, one CTA per SM: 815 us for a 151936 x 3584 weight.)
template <typename T, int EV>
struct Raw {
  static constexpr int kBytes = int(sizeof(T)) * EV;
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const T* at) {
    if constexpr (kBytes == 16) {
      const uint4 v = ldg_stream(reinterpret_cast<const uint4*>(at));
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
      w[0] = v.x;
      w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = __ldg(reinterpret_cast<const unsigned int*>(at));
    } else {
      w[0] = __ldg(reinterpret_cast<const unsigned short*>(at));
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else {
      const uint16_t h = uint16_t(w[j / 2] >> (16 * (j & 1)));
      if constexpr (IsBf16<T>::value)
        return __uint_as_float(uint32_t(h) << 16);
      else
        return __half2float(__ushort_as_half(h));
    }
  }
};

// Running maximum of magnitudes that leaves NaNs out.
template <typename T>
struct AbsMax {
  uint32_t m = 0u;  // f32 bits, or two 16-bit maxima
  template <int EV>
  __device__ __forceinline__ void add(const Raw<T, EV>& x) {
#pragma unroll
    for (int i = 0; i < Raw<T, EV>::kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        m = __float_as_uint(fmaxf(__uint_as_float(m), fabsf(__uint_as_float(x.w[i]))));
      } else if constexpr (IsBf16<T>::value) {
        m = bf16x2_max(m, x.w[i] & 0x7fff7fffu);
      } else {
        asm("max.f16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(x.w[i] & 0x7fff7fffu));
      }
    }
  }
  __device__ __forceinline__ float value() const {
    Raw<T, sizeof(T) == 4 ? 1 : 2> r;
    r.w[0] = m;
    if constexpr (sizeof(T) == 4)
      return r.get(0);
    else
      return fmaxf(r.get(0), r.get(1));
  }
};

// EV e4m3 bytes as one word.
template <int EV>
struct Word;
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<4> {
  using type = uint32_t;
};
template <>
struct Word<2> {
  using type = uint16_t;
};

// Two elements times r, rounded to 19 bits: with y = x r, (33 y) - (33 y - y) keeps the upper part.
__device__ __forceinline__ void scaled(float& a, float& b, float r) {
  const f32x2 y = mul2(pack2(a, b), pack2(r, r)), c = mul2(y, pack2(33.0f, 33.0f)), minus = pack2(-1.0f, -1.0f);
  unpack2(fma2(fma2(y, minus, c), minus, c), a, b);
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

__device__ __forceinline__ uint32_t pair(float a, float b, float r) {
  scaled(a, b, r);
  return to_e4m3x2(a, b);
}
template <typename T, int EV>
__device__ __forceinline__ typename Word<EV>::type convert(const Raw<T, EV>& x, float r) {
  if constexpr (EV == 8) {
    return make_uint2(pair(x.get(0), x.get(1), r) | (pair(x.get(2), x.get(3), r) << 16),
                      pair(x.get(4), x.get(5), r) | (pair(x.get(6), x.get(7), r) << 16));
  } else if constexpr (EV == 4) {
    return pair(x.get(0), x.get(1), r) | (pair(x.get(2), x.get(3), r) << 16);
  } else {
    return uint16_t(pair(x.get(0), x.get(1), r));
  }
}

// 1 x 128: 128 / EV consecutive threads hold a block (EV elements each; with fewer elements a thread, 32 threads hold
// several vectors each).
template <typename T, int EV>
struct RowGroup {
  static constexpr int kThreadsPerBlock = 128 / EV > 32 ? 32 : 128 / EV;
  static constexpr int kVecs = 128 / (kThreadsPerBlock * EV);
  static constexpr int kAtOnce = 4;
};
// A group of threads takes four blocks, all of them on their way before the first is looked at; their maxima are found
// together, and each of the two divisions of a scale is done by one lane for its block while others do theirs.  65536 x
// 3584 bf16 in 121 us, 141965 x 477 in 73 (one block at a time, every lane dividing, its place from a 64-bit division:
// 181 and 131 us).
template <typename T, int EV>
__global__ void __launch_bounds__(kThreads, 5) row_blocks_kernel(const Params p) {
  constexpr int G = RowGroup<T, EV>::kThreadsPerBlock;
  constexpr int U = RowGroup<T, EV>::kVecs;
  constexpr int R = RowGroup<T, EV>::kAtOnce;
  constexpr int GROUPS = kThreads / G;
  const int l = threadIdx.x % G;
  const uint32_t first = blockIdx.x * uint32_t(GROUPS * R) + threadIdx.x / G;  // block of this launch's rows
  const uint32_t rows = uint32_t(p.rows), blocks = uint32_t(p.blocks);
  Raw<T, EV> v[R][U];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = p.by_row.div(first + r * GROUPS), c0 = (first + r * GROUPS - row * blocks) * 128;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride + c0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = (u * G + l) * EV;
      v[r][u].zero();
      if (row < rows && c0 + c < uint32_t(p.cols)) v[r][u].load(x + c);
    }
  }
  // maxima of all R blocks at once: the first two steps leave lane l with block l % 4
  static_assert(R == 4, "");
  float m[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    AbsMax<T> top;
#pragma unroll
    for (int u = 0; u < U; ++u) top.add(v[r][u]);
    m[r] = top.value();
  }
  const bool odd = l & 1, upper = l & 2;
  const float m0 = fmaxf(odd ? m[1] : m[0], __shfl_xor_sync(0xffffffffu, odd ? m[0] : m[1], 1));
  const float m1 = fmaxf(odd ? m[3] : m[2], __shfl_xor_sync(0xffffffffu, odd ? m[2] : m[3], 1));
  float amax = fmaxf(upper ? m1 : m0, __shfl_xor_sync(0xffffffffu, upper ? m0 : m1, 2));
#pragma unroll
  for (int o = 4; o < G; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float my_scale;
  const float mine = factor(amax, &my_scale);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float f = __shfl_sync(0xffffffffu, mine, r, G), scale = __shfl_sync(0xffffffffu, my_scale, r, G);
    const uint32_t row = p.by_row.div(first + r * GROUPS), c0 = (first + r * GROUPS - row * blocks) * 128;
    if (row >= rows) continue;
    if (l == 0) p.scales[first + r * GROUPS] = scale;
    uint8_t* q = p.q + row * p.q_stride + c0;
#pragma unroll
    for (int u = 0; u < U; u += EV == 1 ? 2 : 1) {
      const int c = (u * G + l) * EV;
      if constexpr (EV == 1) {  // two single elements are converted together
        const uint32_t two = pair(v[r][u].get(0), v[r][u + 1].get(0), f);
        if (c0 + c < uint32_t(p.cols)) q[c] = uint8_t(two);
        if (c0 + c + G < uint32_t(p.cols)) q[c + G] = uint8_t(two >> 8);
      } else {
        if (c0 + c < uint32_t(p.cols)) *reinterpret_cast<typename Word<EV>::type*>(q + c) = convert<T, EV>(v[r][u], f);
      }
    }
  }
}

// 128 x 128: one CTA per tile, the tile in registers.
template <typename T, int EV>
__global__ void __launch_bounds__(kThreads, 16 * EV >= 64 && sizeof(T) == 2 ? 4 : 2) tile_blocks_kernel(const Params p) {
  constexpr int PER_ROW = 128 / EV;            // vectors of a tile row
  constexpr int U = 128 * PER_ROW / kThreads;  // vectors per thread
  constexpr int STEP = kThreads / PER_ROW;     // rows between a thread's vectors
  __shared__ float red[kThreads / 32];
  const int64_t tr = blockIdx.x / p.blocks, tb = blockIdx.x - tr * p.blocks;
  const int rr = threadIdx.x / PER_ROW, cc = (threadIdx.x % PER_ROW) * EV;
  const int64_t r0 = tr * 128 + rr, c0 = tb * 128 + cc;
  // vectors of this thread that are inside: its column is, and the first `mine` of its rows
  const int64_t left = p.rows - r0;
  const int mine = c0 < p.cols ? int(left <= 0 ? 0 : (left + STEP - 1) / STEP < U ? (left + STEP - 1) / STEP : U) : 0;
  const T* x = static_cast<const T*>(p.x) + r0 * p.x_stride + c0;
  Raw<T, EV> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    v[u].zero();
    if (u < mine) v[u].load(x + u * (STEP * p.x_stride));
  }
  AbsMax<T> top;
#pragma unroll
  for (int u = 0; u < U; ++u) top.add(v[u]);
  float amax = warp_max(top.value());
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, red[w]);
  float scale;
  const float r = factor(amax, &scale);
  if (threadIdx.x == 0) p.scales[blockIdx.x] = scale;
  uint8_t* q = p.q + r0 * p.q_stride + c0;
#pragma unroll
  for (int u = 0; u < U; u += EV == 1 ? 2 : 1) {
    if constexpr (EV == 1) {
      const uint32_t two = pair(v[u].get(0), v[u + 1].get(0), r);
      if (u < mine) q[u * (STEP * p.q_stride)] = uint8_t(two);
      if (u + 1 < mine) q[(u + 1) * (STEP * p.q_stride)] = uint8_t(two >> 8);
    } else {
      if (u < mine) *reinterpret_cast<typename Word<EV>::type*>(q + u * (STEP * p.q_stride)) = convert<T, EV>(v[u], r);
    }
  }
}

template <typename T, int EV>
static cudaError_t launch(const Params& p, int block_rows, cudaStream_t s) {
  if (block_rows == 1) {
    constexpr int64_t kPer = kThreads / RowGroup<T, EV>::kThreadsPerBlock * RowGroup<T, EV>::kAtOnce;
    // blocks are counted in 32 bits: more than 2^31 of them go in several launches
    const int64_t rows_per = (int64_t(1) << 31) / p.blocks;
    for (int64_t r0 = 0; r0 < p.rows; r0 += rows_per) {
      Params part = p;
      part.rows = p.rows - r0 < rows_per ? p.rows - r0 : rows_per;
      part.x = static_cast<const T*>(p.x) + r0 * p.x_stride;
      part.q = p.q + r0 * p.q_stride;
      part.scales = p.scales + r0 * p.blocks;
      row_blocks_kernel<T, EV><<<unsigned((part.rows * part.blocks + kPer - 1) / kPer), kThreads, 0, s>>>(part);
      count_launch();
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  }
  tile_blocks_kernel<T, EV><<<unsigned((p.rows + 127) / 128 * p.blocks), kThreads, 0, s>>>(p);
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
  if (a->block_rows != 1 && (a->rows / 128 + 1) * blocks > (int64_t(1) << 31) - 1) return MLLM_GRPO_ERR_TOO_LARGE;
  if (a->rows == 0) return MLLM_GRPO_OK;
  if (!a->x || !a->q || !a->scales) return MLLM_GRPO_ERR_NULL_POINTER;
  const uintptr_t es = a->dtype == MLLM_GRPO_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->x) % es || reinterpret_cast<uintptr_t>(a->scales) % 4) return MLLM_GRPO_ERR_ALIGNMENT;
  const fp8q::Params p{a->rows, a->cols, a->x_stride, a->q_stride, blocks, FastDiv(uint32_t(blocks)), a->x, static_cast<uint8_t*>(a->q), a->scales};
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
