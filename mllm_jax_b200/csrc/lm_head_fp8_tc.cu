// lm_head product in 8-bit floating point with a scale for each block of 128, on the tensor cores.
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] p_b[m, n],   p_b[m, n] = sum_{k in block b} x[m, k] w[n, k]
//
// Either the [M, N] product is written (logits of a few prompts, of one token), or its tiles are folded into the
// softmax statistics of the loss as lm_head_tc.cu does it for bf16 (log-probs of a frozen reference model).
//
// One 128-byte row of the swizzled tiles holds exactly one block of 128 along K, so a pipeline stage is a block, and
// its p_b (four tcgen05.mma of kind::f8f6f4, K = 32) is complete in tensor memory when the stage is read.  The scales
// change from block to block and row to row, so the sum over blocks is formed in f32 registers: eight epilogue warps
// fetch p_b with tcgen05.ld and add sx * sw * p_b, while the MMA warp fills the next accumulator.  384 threads:
//   warp 0      TMA producer (x[128 x 128], w[BN x 128] per stage)
//   warp 1      allocates tensor memory (512 columns = 512 / BN accumulators) and issues the MMAs from one thread
//   warps 2, 3  idle (register budgets are set for whole warpgroups)
//   warps 4-11  epilogue: warp -> (quarter of the 128 rows, half of the BN columns), thread = one row
// An epilogue thread holds BN / 2 sums and 64 values on their way from tensor memory, more than the 168 registers that
// 384 threads leave each: the first warpgroup gives registers up (setmaxnreg).
#include "grpo_launch.h"
#include "grpo_tc.cuh"
#include "lm_head_fp8.h"

namespace grpo {
namespace fp8 {

using namespace tc;

constexpr int kBM = 128;
constexpr int kBK = 128;
constexpr int kStages = 4;
constexpr int kThreads = 384;
// Registers per thread: at launch, then of the first warpgroup and of the two epilogue warpgroups.
constexpr int kRegsLaunch = 168, kRegsFirst = 40, kRegsEpilogue = 224;
static_assert(kRegsFirst * 128 + kRegsEpilogue * 256 <= kRegsLaunch * kThreads, "setmaxnreg.inc would wait forever");
constexpr int kTmemCols = 512;
constexpr int kABytes = kBM * kBK;

template <int BN>
struct Tile {
  static constexpr int kStageBytes = kABytes + BN * kBK;
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + 1024 /* alignment slack */ + 256 /* barriers */;
};

__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: D f32 (bit 4), A and B e4m3 (0), both K-major, N/8 at bits 17-22, M/16 at bits 24-28.
__host__ __device__ constexpr uint32_t instr_desc(int M, int N) {
  return (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
template <int REGS>
__device__ __forceinline__ void regs_give() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void regs_take() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}

// Store 8 f32 as consecutive elements of the output type.
template <typename O>
__device__ __forceinline__ void store8(O* to, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* to, const float (&v)[8]) {
  *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* to, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                             pack_bf16x2(v[6], v[7]));
}
template <>
__device__ __forceinline__ void store8<__half>(__half* to, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = make_uint4(cl::pack_f16x2(v[0], v[1]), cl::pack_f16x2(v[2], v[3]),
                                             cl::pack_f16x2(v[4], v[5]), cl::pack_f16x2(v[6], v[7]));
}
template <typename O>
__device__ __forceinline__ O down(float v);
template <>
__device__ __forceinline__ float down<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half down<__half>(float v) {
  return __float2half_rn(v);
}

// STATS: fold the tiles into (max, sumexp, sum e*y, chosen) instead of writing them as O.
template <int BN, bool STATS, typename O>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Params p) {
  constexpr int kBufs = kTmemCols / BN;
  constexpr int CW = BN / 2;  // columns of an epilogue warp
  constexpr int kStageBytes = Tile<BN>::kStageBytes;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = cl::smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const uint32_t bars = tiles + uint32_t(kStages) * kStageBytes;
  auto full_bar = [&](int s) { return bars + 8u * uint32_t(s); };
  auto empty_bar = [&](int s) { return bars + 8u * uint32_t(kStages + s); };
  auto acc_full = [&](int a) { return bars + 8u * uint32_t(2 * kStages + a); };
  auto acc_empty = [&](int a) { return bars + 8u * uint32_t(2 * kStages + kBufs + a); };
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // Work of this CTA: `n_mine` tiles.  Tiles (or, folded, runs of tiles of one row tile) are numbered so that the
  // CTAs that run together take up to 16 row tiles of the same weight tile, which L2 then serves to all of them.
  const int units = STATS ? p.splits : p.n_tiles;
  auto place = [&](int unit_id, int* m_tile, int* unit) {
    const int per_group = 16 * units;
    const int group = unit_id / per_group, within = unit_id - group * per_group;
    const int rows_in_group = min(16, p.m_tiles - group * 16);
    *m_tile = group * 16 + within % rows_in_group;
    *unit = within / rows_in_group;
  };
  int m_fixed = 0, split = 0, n_mine;
  if (STATS) {
    place(blockIdx.x, &m_fixed, &split);
    n_mine = max(0, min(p.tiles_per_split, p.n_tiles - split * p.tiles_per_split));
  } else {
    n_mine = (p.m_tiles * p.n_tiles - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x);
  }
  auto tile_at = [&](int i, int* m_tile, int* n_tile) {
    if (STATS) {
      *m_tile = m_fixed;
      *n_tile = split * p.tiles_per_split + i;
    } else {
      place(int(blockIdx.x) + i * int(gridDim.x), m_tile, n_tile);
    }
  };

  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      cl::mbar_init(full_bar(s), 1);
      cl::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < kBufs; ++a) {
      cl::mbar_init(acc_full(a), 1);
      cl::mbar_init(acc_empty(a), 8);  // one arrival per epilogue warp
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&map_x);
    prefetch_tmap(&map_w);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(cl::smem_u32(&tmem_base_slot)),
                 "r"(uint32_t(kTmemCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;

  if (warp < 4) {
    regs_give<kRegsFirst>();
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer ----------------
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = 0; t < n_mine && ok; ++t) {
        int m_tile, n_tile;
        tile_at(t, &m_tile, &n_tile);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          ok = wait_or_abort(empty_bar(stage), phase ^ 1u, &abort_flag, p.device_status);
          if (!ok) break;
          const uint32_t a_dst = tiles + uint32_t(stage) * kStageBytes;
          cl::mbar_expect_tx(full_bar(stage), uint32_t(kStageBytes));
          tma_load_2d(a_dst, &map_x, kb * kBK, m_tile * kBM, full_bar(stage));
          tma_load_2d(a_dst + kABytes, &map_w, kb * kBK, n_tile * BN, full_bar(stage));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc = instr_desc(kBM, BN);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      for (int t = 0; t < n_mine && ok; ++t) {
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          ok = wait_or_abort(acc_empty(buf), buf_phase ^ 1u, &abort_flag, p.device_status) &&
               wait_or_abort(full_bar(stage), phase, &abort_flag, p.device_status);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_src = tiles + uint32_t(stage) * kStageBytes;
          const uint64_t adesc = smem_desc(a_src), bdesc = smem_desc(a_src + kABytes);
          const uint32_t d_addr = tmem_base + uint32_t(buf * BN);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)  // 32 bytes further along K inside the swizzled row: +2 in the address field
            mma_f8(d_addr, adesc + uint64_t(2 * k), bdesc + uint64_t(2 * k), idesc, k != 0 ? 1u : 0u);
          mma_commit(empty_bar(stage));
          mma_commit(acc_full(buf));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++buf == kBufs) {
            buf = 0;
            buf_phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue ----------------
    regs_take<kRegsEpilogue>();
    const int quarter = warp & 3;  // the TMEM lanes a warp may read: 32*(warp id mod 4) ...
    const int half = (warp - 4) >> 2;
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    // folded form: running statistics of this thread's row over the tiles
    int64_t c = -1;
    float m = kNegInit, s = 0.f, u = 0.f, yc = 0.f;
    const bool cap = STATS && p.softcap > 0.f;
    const SoftCap sc(cap ? p.softcap : 1.0f);
    if (STATS) {
      const int64_t row = int64_t(m_fixed) * kBM + quarter * 32 + lane;
      c = row < p.n_rows ? p.chosen_ids[row] : 0;
      if (row < p.n_rows && (c < 0 || c >= p.vocab_total)) {
        c = c < 0 ? 0 : p.vocab_total - 1;
        if (p.device_status) atomicOr(p.device_status, MLLM_GRPO_DEV_ID_CLAMPED);
      }
      c -= p.vocab_start;
      if (c < 0 || c >= p.vocab) c = -1;
    }
    for (int t = 0; t < n_mine && ok; ++t) {
      int m_tile, n_tile;
      tile_at(t, &m_tile, &n_tile);
      const int64_t row = int64_t(m_tile) * kBM + quarter * 32 + lane;
      const int64_t n0 = int64_t(n_tile) * BN + half * CW;
      // scales of this thread's row and of this warp's columns (one block of 128 weight rows or part of it)
      const float* sx = p.x_scales + (row < p.n_rows ? row : p.n_rows - 1) * p.k_blocks;
      const float* sw = p.w_scales + (n0 < p.vocab ? n0 / 128 : 0) * p.k_blocks;
      f32x2 acc[CW / 2];
#pragma unroll
      for (int j = 0; j < CW / 2; ++j) acc[j] = 0ull;
      float f_next = sx[0] * sw[0];
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        const f32x2 f = pack2(f_next, f_next);
        if (kb + 1 < p.k_blocks) f_next = sx[kb + 1] * sw[kb + 1];
        ok = wait_or_abort(acc_full(buf), buf_phase, &abort_flag, p.device_status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_addr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(buf * BN + half * CW);
        uint32_t v[2][32];
        tmem_ld32(t_addr, v[0]);
#pragma unroll
        for (int ch = 0; ch < CW / 32; ++ch) {
          tmem_ld_wait();
          if (ch + 1 < CW / 32) tmem_ld32(t_addr + uint32_t((ch + 1) * 32), v[(ch + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[ch * 16 + j] = fma2(pack2(__uint_as_float(v[ch & 1][2 * j]), __uint_as_float(v[ch & 1][2 * j + 1])), f,
                                    acc[ch * 16 + j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) cl::mbar_arrive(acc_empty(buf));
        if (++buf == kBufs) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      if (!ok) break;
      const int valid = int(p.vocab - n0 < CW ? (p.vocab - n0 > 0 ? p.vocab - n0 : 0) : CW);
      if (!STATS) {
        if (row < p.n_rows) {
          O* out = static_cast<O*>(p.out) + row * p.out_stride + n0;
#pragma unroll
          for (int j = 0; j < CW / 8; ++j) {
            float y[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) unpack2(acc[j * 4 + q], y[2 * q], y[2 * q + 1]);
            if (p.out_aligned && j * 8 + 8 <= valid) {
              store8<O>(out + j * 8, y);
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (j * 8 + q < valid) out[j * 8 + q] = down<O>(y[q]);
            }
          }
        }
      } else if (valid > 0) {
        const int64_t c_local = c >= 0 ? c - n0 : -1;
        float y[CW];
        float cm = kNegInit;
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) {
          unpack2(acc[j], y[2 * j], y[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          if (cap) y[j] = sc.y(y[j]);
          if (j == c_local) yc = y[j];
          y[j] = j < valid ? y[j] : kNegInit;
          cm = fmaxf(cm, y[j]);
        }
        if (cm > m) {
          const float r = ex2f((m - cm) * kLog2e);
          s *= r;
          u *= r;
          m = cm;
        }
        const float mk = m * kLog2e;
        float s0 = 0.f, s1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll
        for (int j = 0; j < CW; j += 2) {
          const float e0 = ex2f(fmaf(y[j], kLog2e, -mk)), e1 = ex2f(fmaf(y[j + 1], kLog2e, -mk));
          s0 += e0;
          s1 += e1;
          u0 = fmaf(e0, y[j], u0);
          u1 = fmaf(e1, y[j + 1], u1);
        }
        s += s0 + s1;
        u += u0 + u1;
      }
    }
    if (STATS) {
      const int64_t row = int64_t(m_fixed) * kBM + quarter * 32 + lane;
      if (row < p.n_rows)
        p.partials[(int64_t(split) * 2 + half + 1) * p.n_rows + row] =
            ok ? make_float4(m, s, u, yc) : make_float4(kNegInit, 0.f, 0.f, 0.f);
    }
  }

  // ---------------- teardown: every role arrives here, also after an abort ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (abort_flag) {
      for (int i = 0; i < 4; ++i) __nanosleep(500000);  // copies or MMAs may still be in flight: bounded time for them
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(kTmemCols)) : "memory");
  }
}

// Partials of all column ranges of a row -> one (entry 0 of the buffer): 32 rows per CTA, eight threads per row.
__global__ void __launch_bounds__(256) merge_kernel(float4* partials, int64_t n_rows, int entries) {
  __shared__ float4 part[8][32];
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t row = int64_t(blockIdx.x) * 32 + r;
  float m = kNegInit, s = 0.f, u = 0.f, yc = 0.f;
  auto add = [&](float4 q) {
    if (q.x > m) {
      const float f = ex2f((m - q.x) * kLog2e);
      s *= f;
      u *= f;
      m = q.x;
    }
    const float f = ex2f((q.x - m) * kLog2e);
    s = fmaf(q.y, f, s);
    u = fmaf(q.z, f, u);
    yc += q.w;
  };
  if (row < n_rows) {
    for (int e = g; e < entries; e += 8) add(partials[int64_t(e + 1) * n_rows + row]);
  }
  part[g][r] = make_float4(m, s, u, yc);
  __syncthreads();
  if (g == 0 && row < n_rows) {
    for (int i = 1; i < 8; ++i) add(part[i][r]);
    partials[row] = make_float4(m, s, u, yc);
  }
}

// e4m3 [rows, cols] with `ld` bytes between rows -> boxes of box_rows x 128 bytes, 128-byte swizzle, zeros outside.
static bool make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(ld)};
  const cuuint32_t box[2] = {cuuint32_t(kBK), cuuint32_t(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSms = 148;

// Column ranges of the folded form: as many whole tiles per CTA as balance the SMs best (each CTA costs about a
// third of a tile to start and end).
static int fold_tiles_per_split(int64_t m_tiles, int64_t n_tiles) {
  double best = 1e300;
  int64_t pick = 1;
  for (int64_t per = 1; per <= n_tiles && per <= 64; ++per) {
    const int64_t ctas = m_tiles * ((n_tiles + per - 1) / per);
    const double cost = double((ctas + kSms - 1) / kSms) * (double(per) + 0.33);
    if (cost < best * 0.999) {
      best = cost;
      pick = per;
    }
  }
  return int(pick);
}

constexpr int kFoldBN = 256;

static void fold_plan(int64_t n_rows, int64_t vocab, int* tiles_per_split, int* splits) {
  const int64_t m_tiles = (n_rows + kBM - 1) / kBM, n_tiles = (vocab + kFoldBN - 1) / kFoldBN;
  *tiles_per_split = fold_tiles_per_split(m_tiles, n_tiles);
  *splits = int((n_tiles + *tiles_per_split - 1) / *tiles_per_split);
}

template <int BN, bool STATS, typename O>
static int launch_t(const Params& p, unsigned grid, const CUtensorMap& mx, const CUtensorMap& mw, cudaStream_t s) {
  static std::once_flag attr_once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MLLM_GRPO_ERR_NO_DEVICE;
  std::call_once(attr_once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(product_kernel<BN, STATS, O>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         int(Tile<BN>::kSmemBytes));
    cudaFuncAttributes fa;
    if (attr_err[dev] == cudaSuccess) attr_err[dev] = cudaFuncGetAttributes(&fa, product_kernel<BN, STATS, O>);
    // the epilogue takes registers that the launch must have brought along
    if (attr_err[dev] == cudaSuccess && fa.numRegs < kRegsLaunch) attr_err[dev] = cudaErrorInvalidConfiguration;
  });
  if (attr_err[dev] != cudaSuccess) return record_cuda_error(attr_err[dev]);
  product_kernel<BN, STATS, O><<<grid, kThreads, Tile<BN>::kSmemBytes, s>>>(mx, mw, p);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

template <int BN, bool STATS, typename O>
static int launch(Params p, const mllm_lm_head_fp8_args* a, cudaStream_t s) {
  p.m_tiles = int((p.n_rows + kBM - 1) / kBM);
  p.n_tiles = int((p.vocab + BN - 1) / BN);
  CUtensorMap mx, mw;
  if (!make_map(&mx, a->hidden, a->n_rows, a->hidden_dim, a->hidden_stride, kBM) ||
      !make_map(&mw, a->weight, a->vocab, a->hidden_dim, a->weight_stride, BN))
    return MLLM_GRPO_ERR_NO_DEVICE;
  int64_t grid;
  if (STATS) {
    fold_plan(p.n_rows, p.vocab, &p.tiles_per_split, &p.splits);
    grid = int64_t(p.m_tiles) * p.splits;
  } else {
    grid = int64_t(p.m_tiles) * p.n_tiles;
    if (grid >= (int64_t(1) << 30)) return MLLM_GRPO_ERR_TOO_LARGE;
    if (grid > kSms) grid = kSms;
  }
  if (grid >= (int64_t(1) << 30)) return MLLM_GRPO_ERR_TOO_LARGE;
  return launch_t<BN, STATS, O>(p, unsigned(grid), mx, mw, s);
}

template <typename O>
static int launch_product(const Params& p, const mllm_lm_head_fp8_args* a, cudaStream_t s) {
  // tiles of 256 columns read the least per product; with fewer of them than SMs, twice as many of 128
  const int64_t tiles = ((p.n_rows + kBM - 1) / kBM) * ((p.vocab + 255) / 256);
  return tiles <= kSms ? launch<128, false, O>(p, a, s) : launch<256, false, O>(p, a, s);
}

static bool aligned(const void* q, uintptr_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) == 0; }

static int check(const mllm_lm_head_fp8_args* a, Params* p) {
  if (a == nullptr) return MLLM_GRPO_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(mllm_lm_head_fp8_args)) return MLLM_GRPO_ERR_STRUCT_SIZE;
  if (a->n_rows < 0 || a->vocab <= 0 || a->hidden_dim <= 0 || a->hidden_stride < a->hidden_dim ||
      a->weight_stride < a->hidden_dim)
    return MLLM_GRPO_ERR_BAD_SHAPE;
  constexpr int64_t kMost = (int64_t(1) << 31) - 1024;
  if (a->n_rows > kMost || a->vocab > kMost || a->hidden_dim > kMost) return MLLM_GRPO_ERR_TOO_LARGE;
  if ((a->hidden_dim % 16) || (a->hidden_stride % 16) || (a->weight_stride % 16)) return MLLM_GRPO_ERR_UNSUPPORTED;
  if (a->n_rows > 0 && (!a->hidden || !a->hidden_scales)) return MLLM_GRPO_ERR_NULL_POINTER;
  if (!a->weight || !a->weight_scales) return MLLM_GRPO_ERR_NULL_POINTER;
  if (!aligned(a->hidden, 16) || !aligned(a->weight, 16) || !aligned(a->hidden_scales, 4) ||
      !aligned(a->weight_scales, 4) || !aligned(a->device_status, 4))
    return MLLM_GRPO_ERR_ALIGNMENT;
  *p = Params{};
  p->n_rows = a->n_rows;
  p->vocab = a->vocab;
  p->hidden = a->hidden_dim;
  p->hidden_stride = a->hidden_stride;
  p->weight_stride = a->weight_stride;
  p->out_stride = a->out_stride;
  p->k_blocks = int((a->hidden_dim + kBK - 1) / kBK);
  p->x = static_cast<const uint8_t*>(a->hidden);
  p->w = static_cast<const uint8_t*>(a->weight);
  p->x_scales = a->hidden_scales;
  p->w_scales = a->weight_scales;
  p->out = a->out;
  p->chosen_ids = a->chosen_ids;
  p->partials = static_cast<float4*>(a->partials);
  p->softcap = a->softcap;
  p->device_status = a->device_status;
  return MLLM_GRPO_OK;
}

}  // namespace fp8
}  // namespace grpo

using namespace grpo;

extern "C" {

int mllm_lm_head_fp8_matmul(const mllm_lm_head_fp8_args* a, void* stream) {
  fp8::Params p;
  const int st = fp8::check(a, &p);
  if (st) return st;
  if (a->out_stride < a->vocab) return MLLM_GRPO_ERR_BAD_SHAPE;
  if (a->out_dtype < 0 || a->out_dtype > MLLM_GRPO_F32) return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (a->n_rows == 0) return MLLM_GRPO_OK;
  if (!a->out) return MLLM_GRPO_ERR_NULL_POINTER;
  const int64_t es = a->out_dtype == MLLM_GRPO_F32 ? 4 : 2;
  if (!fp8::aligned(a->out, es)) return MLLM_GRPO_ERR_ALIGNMENT;
  p.out_aligned = fp8::aligned(a->out, 16) && (a->out_stride * es) % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->out_dtype == MLLM_GRPO_F32) return fp8::launch_product<float>(p, a, s);
  if (a->out_dtype == MLLM_GRPO_F16) return fp8::launch_product<__half>(p, a, s);
  return fp8::launch_product<__nv_bfloat16>(p, a, s);
}

int64_t mllm_lm_head_fp8_partials_bytes(int64_t n_rows, int64_t vocab) {
  if (n_rows <= 0 || vocab <= 0) return 0;
  int per, splits;
  fp8::fold_plan(n_rows, vocab, &per, &splits);
  return (int64_t(splits) * 2 + 1) * n_rows * 16;
}

int mllm_lm_head_fp8_partials(const mllm_lm_head_fp8_args* a, void* stream) {
  fp8::Params p;
  int st = fp8::check(a, &p);
  if (st) return st;
  if (a->n_rows == 0) return MLLM_GRPO_ERR_BAD_SHAPE;
  if (!a->chosen_ids || !a->partials) return MLLM_GRPO_ERR_NULL_POINTER;
  if (a->vocab_start < 0 || (a->vocab_total > 0 && a->vocab_start + a->vocab > a->vocab_total)) return MLLM_GRPO_ERR_BAD_SHAPE;
  if (!(a->softcap >= 0.f)) return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (!fp8::aligned(a->partials, 16) || !fp8::aligned(a->chosen_ids, 4)) return MLLM_GRPO_ERR_ALIGNMENT;
  p.vocab_start = a->vocab_start;
  p.vocab_total = a->vocab_total > 0 ? a->vocab_total : a->vocab_start + a->vocab;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = fp8::launch<fp8::kFoldBN, true, float>(p, a, s);
  if (st) return st;
  int per, splits;
  fp8::fold_plan(a->n_rows, a->vocab, &per, &splits);
  fp8::merge_kernel<<<unsigned((a->n_rows + 31) / 32), 256, 0, s>>>(p.partials, a->n_rows, splits * 2);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

}  // extern "C"
