// What the kernels of the block-scaled 8-bit product share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace grpo {
namespace fp8 {

struct Params {
  int64_t n_rows, vocab, hidden, hidden_stride, weight_stride, out_stride, vocab_start, vocab_total;
  int m_tiles, n_tiles, k_blocks, tiles_per_split, splits;
  int out_aligned;  // rows of out start on 16-byte boundaries
  int stop_after;   // tiles of a CTA (pair) that are multiplied: all, unless a test makes the waits run out
  float softcap;
  const uint8_t* x;
  const uint8_t* w;
  const float* x_scales;
  const float* w_scales;
  void* out;
  const int32_t* chosen_ids;
  float4* partials;  // [1 + ranges, n_rows]: the merged entry, then one entry per column range
  float inv_temperature;
  float* logps;
  float* entropy;
  float* lse;
  int32_t* device_status;
};

// The product for at most kFewRows rows of x (lm_head_fp8_rows.cu).  One tile of 8 tokens: 151936 x 3584 in 90 us for
// any of them (tensor-memory tiles: 105-131 us for 9 to 128 rows, from run to run); a second tile of 8 took 126 us, no less.
constexpr int64_t kFewRows = 8;
cudaError_t launch_few_rows(const Params& p, int out_dtype, cudaStream_t s);

}  // namespace fp8
}  // namespace grpo
