// Block-scaled 8-bit product for a few rows of x (logits of single tokens): bound by reading the weight once.
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
//
// The weight goes straight from memory into the fragments of mma.sync (m16n8k32, e4m3): 16 weight rows are the A
// operand, 8 tokens the B operand, so a tensor-core tile of 128 rows is not filled with zeros and no shared-
// memory stage or barrier stands between a load and its use.  The order of k inside a block is free as long as both
// operands use the same one: lane t of a quad takes bytes [32 t, 32 t + 32) of a block, one load where the rows start on
// 32-byte boundaries, and a quad reads the 128 contiguous bytes of a row's block.  A warp sums its blocks in f32 registers; the KS warps
// that share 16 rows split K and meet in shared memory in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/mllm_grpo.h"
#include "grpo_common.cuh"
#include "grpo_launch.h"
#include "grpo_rowpass.cuh"
#include "lm_head_fp8.h"

namespace grpo {
namespace fp8 {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kWarps = kRowsThreads / 32;

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void put(float* to, float v) { *to = v; }
__device__ __forceinline__ void put(__nv_bfloat16* to, float v) { *to = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* to, float v) { *to = __float2half_rn(v); }

// 32 bytes at p + k, of which `n` (0, 16 or 32) are inside the row.
template <bool WIDE>
__device__ __forceinline__ void load32(uint32_t (&v)[8], const uint8_t* p, int k, int n) {
  if (WIDE && n >= 32) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p + k));
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 x = n >= 16 * (h + 1) ? ldg_stream(reinterpret_cast<const uint4*>(p + k + 16 * h)) : make_uint4(0, 0, 0, 0);
    v[4 * h] = x.x;
    v[4 * h + 1] = x.y;
    v[4 * h + 2] = x.z;
    v[4 * h + 3] = x.w;
  }
}

// KS: warps that split K.  WIDE: weight rows start on 32-byte boundaries.
template <int KS, bool WIDE, typename O>
__global__ void __launch_bounds__(kRowsThreads, 3) few_rows_kernel(const Params p) {
  constexpr int GROUPS = kWarps / KS;  // groups of 16 weight rows per CTA
  constexpr int DEPTH = 2;             // blocks on their way per warp
  __shared__ float red[KS][GROUPS][8][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int group = warp % GROUPS, part = warp / GROUPS;
  const int64_t n0 = (int64_t(blockIdx.x) * GROUPS + group) * 16;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (n0 < p.vocab) {
    // rows past the vocabulary and tokens past the batch read the last one: their sums are not written
    auto row = [&](int r) { return n0 + r < p.vocab ? n0 + r : p.vocab - 1; };
    auto token = [&](int m) { return m < p.n_rows ? int64_t(m) : p.n_rows - 1; };
    const uint8_t* wa = p.w + row(g) * p.weight_stride + t * 32;
    const uint8_t* wb = p.w + row(g + 8) * p.weight_stride + t * 32;
    const uint8_t* xr = p.x + token(g) * p.hidden_stride + t * 32;
    const float* sx0 = p.x_scales + token(2 * t) * p.k_blocks;
    const float* sx1 = p.x_scales + token(2 * t + 1) * p.k_blocks;
    const float* sw = p.w_scales + n0 / 128 * p.k_blocks;
    const int left = int(p.hidden) - t * 32;  // bytes of a row from this lane's first on (a multiple of 16)
    // one block per warp and step, the next DEPTH of them on their way
    uint32_t a[DEPTH][8], b[DEPTH][8];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = (part + d * KS) * 128;
      load32<WIDE>(a[d], wa, k, left - k);
      load32<WIDE>(b[d], wb, k, left - k);
    }
    for (int kb0 = part; kb0 < p.k_blocks; kb0 += KS * DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int kb = kb0 + d * KS;
        if (kb >= p.k_blocks) break;
        const int k = kb * 128, next = k + DEPTH * KS * 128;
        const float s = __ldg(sw + kb);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 x = left - k >= 16 * (h + 1) ? __ldg(reinterpret_cast<const uint4*>(xr + k + 16 * h)) : make_uint4(0, 0, 0, 0);
          mma_e4m3(c, a[d][4 * h], b[d][4 * h], a[d][4 * h + 1], b[d][4 * h + 1], x.x, x.y);
          mma_e4m3(c, a[d][4 * h + 2], b[d][4 * h + 2], a[d][4 * h + 3], b[d][4 * h + 3], x.z, x.w);
        }
        const float f0 = s * __ldg(sx0 + kb), f1 = s * __ldg(sx1 + kb);
        acc[0] = fmaf(c[0], f0, acc[0]);
        acc[1] = fmaf(c[1], f1, acc[1]);
        acc[2] = fmaf(c[2], f0, acc[2]);
        acc[3] = fmaf(c[3], f1, acc[3]);
        load32<WIDE>(a[d], wa, next, left - next);
        load32<WIDE>(b[d], wb, next, left - next);
      }
    }
  }
  red[part][group][2 * t][g] = acc[0];
  red[part][group][2 * t + 1][g] = acc[1];
  red[part][group][2 * t][g + 8] = acc[2];
  red[part][group][2 * t + 1][g + 8] = acc[3];
  __syncthreads();
  O* out = static_cast<O*>(p.out);
  for (int i = threadIdx.x; i < GROUPS * 16 * 8; i += kRowsThreads) {
    const int m = i / (GROUPS * 16), r = i % (GROUPS * 16);
    const int64_t n = int64_t(blockIdx.x) * GROUPS * 16 + r;
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) y += red[k][r / 16][m][r % 16];
    if (m < p.n_rows && n < p.vocab) put(out + int64_t(m) * p.out_stride + n, y);
  }
}

template <int KS, bool WIDE, typename O>
cudaError_t launch_rows(const Params& p, cudaStream_t s) {
  constexpr int64_t kPer = kWarps / KS * 16;
  few_rows_kernel<KS, WIDE, O><<<unsigned((p.vocab + kPer - 1) / kPer), kRowsThreads, 0, s>>>(p);
  count_launch();
  return cudaGetLastError();
}

template <bool WIDE, typename O>
cudaError_t launch_w(const Params& p, cudaStream_t s) {
  // K over four warps; over eight where that leaves less than a CTA per SM (4096 x 4096: 4.4 us, 5.7 with four); over one
  // or two where a warp of four would have few blocks and there are CTAs enough (142803 x 288: 11.8 us, 16.7 with four;
  // 151936 x 1536: 43 with two, 47 with four)
  if (p.vocab <= int64_t(148) * 32) return launch_rows<8, WIDE, O>(p, s);
  if (p.vocab > int64_t(2) * 148 * 128 && p.k_blocks <= 8) return launch_rows<1, WIDE, O>(p, s);
  if (p.vocab > int64_t(2) * 148 * 128 && p.k_blocks <= 14) return launch_rows<2, WIDE, O>(p, s);
  return launch_rows<4, WIDE, O>(p, s);
}

template <typename O>
cudaError_t launch_o(const Params& p, cudaStream_t s) {
  const bool wide = ((reinterpret_cast<uintptr_t>(p.w) | uintptr_t(p.weight_stride)) & 31) == 0;
  return wide ? launch_w<true, O>(p, s) : launch_w<false, O>(p, s);
}

}  // namespace

cudaError_t launch_few_rows(const Params& p, int out_dtype, cudaStream_t s) {
  if (out_dtype == MLLM_GRPO_F32) return launch_o<float>(p, s);
  if (out_dtype == MLLM_GRPO_F16) return launch_o<__half>(p, s);
  return launch_o<__nv_bfloat16>(p, s);
}

}  // namespace fp8
}  // namespace grpo
