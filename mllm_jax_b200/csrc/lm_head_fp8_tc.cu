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
//   warps 2, 3  scales: sx * sw of the coming block for every row, through shared memory (a row's scales are contiguous
//               along K: reading them in the epilogue touched 32 lines a load)
//   warps 4-11  two epilogue warpgroups: warp -> a quarter of the 128 rows, thread = one row
// An epilogue thread holds up to 128 sums and 64 values on their way from tensor memory, more than the 168 registers
// that 384 threads leave each: the first warpgroup gives registers up (setmaxnreg).
//
// With BN = 256 there are two accumulators, and what bounds the kernel is the way from a commit through the epilogue
// back to the MMA warp: the epilogue releases an accumulator as soon as its last values are in registers, before it
// adds them.  (Four accumulators of 128 columns, multiplied separately, would leave more time, but a pair's MMA of 128
// columns takes as long as one of 256.)  BN = 128 serves problems with fewer tiles than SMs.
//
// CTAS = 1: a CTA computes its tile by itself.  CTAS = 2: two CTAs of a cluster on neighbouring SMs compute 256 x 256
// together (tcgen05 cta_group::2): each loads its own 128 rows of x and HALF of the weight tile, the tensor cores read
// both halves.  With one CTA per 128 x 256 tile an SM asks L2 for 48 KB per block of 512 MMA cycles, more than L2
// delivers (measured without any epilogue work: 914 cycles per block); the pair asks for 32 KB each.
//
// The finished tile goes through shared memory and leaves by TMA while the next one is accumulated (threads writing
// their own rows: 4096 cycles per tile; coalesced stores from shared memory: 3300).
//
// Every wait is bounded.  When one runs out, the epilogue writes NaN to the elements of its tiles that it has not
// reached, so that a product nobody checked the status of cannot be taken for one.
#include <atomic>
#include <type_traits>

#include "grpo_launch.h"
#include "grpo_tc.cuh"
#include "lm_head_fp8.h"

namespace grpo {
namespace fp8 {

using namespace tc;

constexpr int kBM = 128;
constexpr int kBK = 128;
constexpr int kThreads = 384;
// Registers per thread: at launch, then of the first warpgroup and of the two epilogue warpgroups.
constexpr int kRegsLaunch = 168, kRegsFirst = 40, kRegsEpilogue = 224;
static_assert(kRegsFirst * 128 + kRegsEpilogue * 256 <= kRegsLaunch * kThreads, "setmaxnreg.inc would wait forever");
constexpr int kTmemCols = 512;
constexpr int kABytes = kBM * kBK;

constexpr int kBarBytes = 256;

template <int BN, int CTAS>
struct Tile {
  static constexpr int kBufs = kTmemCols / BN;  // accumulators
  static constexpr int kBRows = BN / CTAS;      // weight rows that one CTA loads
  static constexpr int kStageBytes = kABytes + kBRows * kBK;
  static constexpr int kStages = kStageBytes > 32768 ? 3 : 4;
  static constexpr int CW = BN / 2;             // columns of an epilogue warp
  static constexpr int kHalves = BN / 128;      // blocks of weight rows in a tile
  static constexpr int kScaleBytes = kBufs * kHalves * kBM * 4;
  static constexpr int kStoreBytes = 32 * CW * 2;  // per epilogue warp: 32 rows of bf16 on their way out
  static constexpr size_t kSmemBytes = 1024 /* alignment slack */ + size_t(kStages) * kStageBytes + 8 * kStoreBytes + kBarBytes +
                                       kScaleBytes;
  static_assert(kSmemBytes <= 227 * 1024, "");
  // barriers: full[kStages], empty[kStages], then per accumulator: full, empty (the MMA warp's), slot_empty (the scale
  // warps')
  static_assert((2 * kStages + 3 * kBufs) * 8 <= kBarBytes, "");
};

template <int CTAS>
__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives at the barrier (of both CTAs of a pair) when the MMAs issued so far are done.
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CTAS == 1)
    mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(uint16_t(3))
        : "memory");
}
// Tile load into this CTA's shared memory; for a pair the barrier is the leader's.
template <int CTAS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (CTAS == 1)
    tma_load_2d(dst, map, c0, c1, bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
// Arrival at a barrier of the pair's leader.  What it releases are tensor-memory reads, which tcgen05.wait and the
// fence before it have ordered: the default scope (the CTA) does.  A release at cluster scope waits for every store
// of the thread as well and doubled the kernel's time.
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cl::map_to_cta(bar, 0)) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
  if constexpr (CTAS == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(uint32_t(kTmemCols)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(uint32_t(kTmemCols)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t base) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(uint32_t(kTmemCols)) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(uint32_t(kTmemCols)) : "memory");
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

// 16 bytes of output from the f32 pairs that hold them.
template <typename O>
struct Out;
template <>
struct Out<float> {
  static constexpr int kPerVec = 4;
  static __device__ __forceinline__ uint4 pack(const f32x2* v) {
    uint4 o;
    float a, b;
    unpack2(v[0], a, b);
    o.x = __float_as_uint(a);
    o.y = __float_as_uint(b);
    unpack2(v[1], a, b);
    o.z = __float_as_uint(a);
    o.w = __float_as_uint(b);
    return o;
  }
};
template <>
struct Out<__nv_bfloat16> {
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ uint32_t two(f32x2 v) {
    float a, b;
    unpack2(v, a, b);
    return pack_bf16x2(a, b);
  }
  static __device__ __forceinline__ uint4 pack(const f32x2* v) { return make_uint4(two(v[0]), two(v[1]), two(v[2]), two(v[3])); }
};
template <>
struct Out<__half> {
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ uint32_t two(f32x2 v) {
    float a, b;
    unpack2(v, a, b);
    return cl::pack_f16x2(a, b);
  }
  static __device__ __forceinline__ uint4 pack(const f32x2* v) { return make_uint4(two(v[0]), two(v[1]), two(v[2]), two(v[3])); }
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <typename O>
__device__ __forceinline__ void put_element(char* to, uint32_t from) {
  if constexpr (sizeof(O) == 4) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
    *reinterpret_cast<uint32_t*>(to) = v;
  } else {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
    *reinterpret_cast<uint16_t*>(to) = v;
  }
}

// 16 bytes of a followed by b, from byte 16 - s on (s in [0, 16), even).
__device__ __forceinline__ uint4 joined(const uint4& a, const uint4& b, int s) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const int from = 16 - s;
  uint32_t x[6], y[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) x[i] = from & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) y[i] = from & 4 ? x[i + 1] : x[i];
  uint4 v;
  v.x = s ? __funnelshift_r(y[0], y[1], (from & 3) * 8) : b.x;
  v.y = s ? __funnelshift_r(y[1], y[2], (from & 3) * 8) : b.y;
  v.z = s ? __funnelshift_r(y[2], y[3], (from & 3) * 8) : b.z;
  v.w = s ? __funnelshift_r(y[3], y[4], (from & 3) * 8) : b.w;
  return v;
}

// Rows of a warp's staged boxes to global memory where TMA cannot write them: 32 rows of NC chunks of 16 bytes, of which
// the first `bytes` are written.  A row starts s bytes behind a 16-byte boundary.  A lane writes the aligned 16 bytes that
// end inside its own chunk, the first s of them from its neighbour's.  What lies before a row's first boundary and behind
// its last are 16 bytes together, too; a lane per row writes them in pieces of 8, 4 and 2 bytes from its first and last
// chunk in registers, or, where the tile ends inside the row, element by element.  (All elements by consecutive lanes:
// 2267 x 65697 x 688 in 341 us, now 218; with rows on 16-byte boundaries, by TMA, 157.)
template <typename O, int NC>
__device__ __forceinline__ void store_shifted(char* out, int64_t pitch, int rows, int bytes, const uint4& first,
                                              const uint4& last, uint32_t buf, int lane) {
  constexpr int kRowsAtOnce = 32 / NC;
  const auto chunk = [&](int r, int j) { return buf + uint32_t((j >> 3) * (32 * 128) + r * 128 + (((j & 7) ^ (r & 7)) << 4)); };
  const int j = lane % NC;
#pragma unroll 2
  for (int r0 = 0; r0 < 32; r0 += kRowsAtOnce) {
    const int r = r0 + lane / NC;
    char* const row = out + r * pitch;
    const int s = int(reinterpret_cast<uintptr_t>(row) & 15), at = 16 * j - s;
    uint4 own, left;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(own.x), "=r"(own.y), "=r"(own.z), "=r"(own.w) : "r"(chunk(r, j)) : "memory");
    left.x = __shfl_up_sync(0xffffffffu, own.x, 1, NC);
    left.y = __shfl_up_sync(0xffffffffu, own.y, 1, NC);
    left.z = __shfl_up_sync(0xffffffffu, own.z, 1, NC);
    left.w = __shfl_up_sync(0xffffffffu, own.w, 1, NC);
    const uint4 v = joined(left, own, s);
    if (r < rows && at >= 0 && at + 16 <= bytes) *reinterpret_cast<uint4*>(row + at) = v;
  }
  if (lane >= rows) return;
  char* const row = out + lane * pitch;
  const int s = int(reinterpret_cast<uintptr_t>(row) & 15);
  if (bytes == 16 * NC) {
    const uint4 v = joined(last, first, s);  // the last s bytes of the row, its first 16 - s
    char* const head = row - s;
    char* const tail = head + 16 * NC;
    const int up = (s + 3) & ~3;
    if (s & 8) *reinterpret_cast<uint2*>(tail) = make_uint2(v.x, v.y);
    if (s & 4) *reinterpret_cast<uint32_t*>(tail + (s & 8)) = s & 8 ? v.z : v.x;
    if (s > 0 && up <= 8) *reinterpret_cast<uint2*>(head + 8) = make_uint2(v.z, v.w);
    if (up & 4) *reinterpret_cast<uint32_t*>(head + up) = up & 8 ? v.w : v.y;
    if (s & 2) {
      const uint32_t w = s & 8 ? (s & 4 ? v.w : v.z) : (s & 4 ? v.y : v.x);
      *reinterpret_cast<uint16_t*>(tail + (s & 12)) = uint16_t(w);
      *reinterpret_cast<uint16_t*>(head + s) = uint16_t(w >> 16);
    }
  } else {
    constexpr int E = int(sizeof(O));
    const int head = s ? (16 - s < bytes ? 16 - s : bytes) : 0;
    const int tail = ((bytes + s) & ~15) - s > head ? ((bytes + s) & ~15) - s : head;
    for (int e = 0; e < 16; e += E) {
      const int at = tail + e;
      if (e < head) put_element<O>(row + e, chunk(lane, 0) + uint32_t(e));
      if (at < bytes) put_element<O>(row + at, chunk(lane, at >> 4) + uint32_t(at & 15));
    }
  }
}

// Writes a warp's 32 rows x CW columns, each thread holding a row.  Boxes of 32 rows x 128 bytes in shared memory, laid
// out as TMA's 128-byte swizzle has them (16-byte chunk c of row r at c ^ (r mod 8): no bank conflicts), go out
// asynchronously; columns and rows past the output are cut off by the tensor map, columns in steps of 16 bytes.  Rows
// that do not start on 16-byte boundaries, and a last tile that ends inside 16 bytes (the cut would write the rest of
// them), are written from there by the threads.
template <typename O, int CW, int BYTES>
__device__ __forceinline__ void store_rows(const Params& p, const CUtensorMap* map, const f32x2 (&acc)[CW / 2], int64_t row0,
                                           int64_t n0, int valid, uint32_t buf, int lane) {
  constexpr int PV = Out<O>::kPerVec;       // elements of a 16-byte chunk
  constexpr int BOX = 8 * PV;               // columns of a box
  constexpr int ROOM = BYTES / (32 * 128);  // boxes that fit the warp's buffer
  if (valid <= 0 || row0 >= p.n_rows) return;
#pragma unroll
  for (int c0 = 0; c0 < CW; c0 += BOX) {
    if (c0 >= valid) break;  // uniform over the warp
    constexpr int LAST = CW / BOX - 1;
    const int at = (c0 / BOX) % ROOM;
    if (at == 0) {
      // the stores that last used this buffer have been read
      if (lane == 0) cl::bulk_wait_read();
      __syncwarp();
    }
    const uint32_t box = buf + uint32_t(at) * (32 * 128);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      cl::sts128(box + uint32_t(lane * 128 + ((k ^ (lane & 7)) << 4)), Out<O>::pack(&acc[(c0 + k * PV) / 2]));
    // the boxes that fit the buffer go out together
    if (at != ROOM - 1 && c0 / BOX != LAST && c0 + BOX < valid) continue;
    if (p.out_aligned && (valid == CW || valid % PV == 0)) {
      cl::fence_async_smem();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < ROOM; ++i)
          if (i <= at) tma_store_2d(map, int(n0) + c0 - (at - i) * BOX, int(row0), buf + uint32_t(i) * (32 * 128));
      }
    } else {
      __syncwarp();
      const int first = c0 - at * BOX, cols = valid < c0 + BOX ? valid - first : c0 + BOX - first;
      store_shifted<O, 8 * ROOM>(reinterpret_cast<char*>(static_cast<O*>(p.out) + row0 * p.out_stride + n0 + first),
                                 p.out_stride * int64_t(sizeof(O)), int(p.n_rows - row0 < 32 ? p.n_rows - row0 : 32),
                                 cols * int(sizeof(O)), Out<O>::pack(&acc[(c0 - at * BOX) / 2]), Out<O>::pack(&acc[(c0 + BOX - PV) / 2]), buf, lane);
      __syncwarp();
    }
  }
}

// NaN in a warp's 32 rows x valid columns of a tile that will not be computed.
template <typename O>
__device__ __forceinline__ void void_rows(const Params& p, int64_t row0, int64_t n0, int valid, int lane) {
  using Bits = typename std::conditional<sizeof(O) == 4, uint32_t, uint16_t>::type;
  for (int64_t row = row0; row < row0 + 32 && row < p.n_rows; ++row) {
    Bits* const to = static_cast<Bits*>(p.out) + row * p.out_stride + n0;
    for (int c = lane; c < valid; c += 32) to[c] = Bits(~Bits(0)) >> 1;
  }
}

// STATS: fold the tiles into (max, sumexp, sum e*y, chosen) instead of writing them as O.
template <int BN, int CTAS, bool STATS, typename O>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ CUtensorMap map_out, const Params p) {
  using T = Tile<BN, CTAS>;
  constexpr int kHalves = T::kHalves, kBufs = T::kBufs, kStages = T::kStages, kStageBytes = T::kStageBytes;
  constexpr int CW = T::CW;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = cl::smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const uint32_t store_buf = tiles + uint32_t(kStages) * kStageBytes;
  const uint32_t bars = store_buf + 8u * T::kStoreBytes;
  auto full_bar = [&](int s) { return bars + 8u * uint32_t(s); };
  auto empty_bar = [&](int s) { return bars + 8u * uint32_t(kStages + s); };
  auto acc_full = [&](int a) { return bars + 8u * uint32_t(2 * kStages + a); };
  auto acc_empty = [&](int a) { return bars + 8u * uint32_t(2 * kStages + kBufs + a); };
  auto slot_empty = [&](int a) { return bars + 8u * uint32_t(2 * kStages + 2 * kBufs + a); };
  float* const scales = reinterpret_cast<float*>(smem_raw + (bars - raw) + kBarBytes);  // [accumulator][half][row]
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CTAS == 1 ? 0 : int(cl::cluster_rank());
  const int team = int(blockIdx.x) / CTAS, teams = int(gridDim.x) / CTAS;

  // Work of this CTA (pair): `n_mine` tiles.  Tiles (or, folded, runs of tiles of the same rows) are numbered so that
  // the CTAs that run together take up to 2048 rows of the same weight tile, which L2 then serves to all of them.
  constexpr int kGroup = 16 / CTAS;
  const int units = STATS ? p.splits : p.n_tiles;
  const int m_teams = (p.m_tiles + CTAS - 1) / CTAS;
  auto place = [&](int unit_id, int* m_tile, int* unit) {
    const int per_group = kGroup * units;
    const int group = unit_id / per_group, within = unit_id - group * per_group;
    const int rows_in_group = min(kGroup, m_teams - group * kGroup);
    *m_tile = (group * kGroup + within % rows_in_group) * CTAS + rank;
    *unit = within / rows_in_group;
  };
  int m_fixed = 0, split = 0, n_mine;
  if (STATS) {
    place(team, &m_fixed, &split);
    n_mine = max(0, min(p.tiles_per_split, p.n_tiles - split * p.tiles_per_split));
  } else {
    n_mine = (m_teams * p.n_tiles - team + teams - 1) / teams;
  }
  auto tile_at = [&](int i, int* m_tile, int* n_tile) {
    if (STATS) {
      *m_tile = m_fixed;
      *n_tile = split * p.tiles_per_split + i;
    } else {
      place(team + i * teams, m_tile, n_tile);
    }
  };

  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      cl::mbar_init(full_bar(s), 1);
      cl::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < kBufs; ++a) {
      cl::mbar_init(acc_full(a), 3);          // the MMAs' commit and both scale warps
      cl::mbar_init(acc_empty(a), 8 * CTAS);  // one arrival per epilogue warp (of both CTAs, in the leader)
      cl::mbar_init(slot_empty(a), 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&map_x);
    prefetch_tmap(&map_w);
  }
  if (warp == 1) tmem_alloc<CTAS>(cl::smem_u32(&tmem_base_slot));
  tc_fence_before();
  if (CTAS == 1)
    __syncthreads();
  else
    cl::cluster_sync_all();
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
          // the bytes of both CTAs are counted at the leader's barrier
          if (rank == 0) cl::mbar_expect_tx(full_bar(stage), uint32_t(CTAS * kStageBytes));
          const uint32_t bar = CTAS == 1 ? full_bar(stage) : cl::map_to_cta(full_bar(stage), 0);
          load_tile<CTAS>(a_dst, &map_x, kb * kBK, m_tile * kBM, bar);
          load_tile<CTAS>(a_dst + kABytes, &map_w, kb * kBK, n_tile * BN + rank * T::kBRows, bar);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // the stages' last releases come from the leader's tensor core: none may be on its way when this CTA leaves
      for (int i = 0; i < kStages && ok; ++i) {
        ok = wait_or_abort(empty_bar(stage), phase ^ 1u, &abort_flag, p.device_status);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------- MMA issuer (the leader's) ----------------
      constexpr uint32_t idesc = instr_desc(kBM * CTAS, BN);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      const int n_tiles = min(n_mine, p.stop_after);
      for (int t = 0; t < n_tiles && ok; ++t) {
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          // the tiles are there long before the accumulator is free: that wait comes last, with everything prepared
          ok = wait_or_abort(full_bar(stage), phase, &abort_flag, p.device_status);
          if (!ok) break;
          const uint32_t a_src = tiles + uint32_t(stage) * kStageBytes;
          const uint64_t adesc = smem_desc(a_src), bdesc = smem_desc(a_src + kABytes);
          const uint32_t d_addr = tmem_base + uint32_t(buf * BN);
          ok = wait_or_abort(acc_empty(buf), buf_phase ^ 1u, &abort_flag, p.device_status);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)  // 32 bytes further along K inside the swizzled row: +2 in the address field
            mma_f8<CTAS>(d_addr, adesc + uint64_t(2 * k), bdesc + uint64_t(2 * k), idesc, k != 0 ? 1u : 0u);
          commit<CTAS>(acc_full(buf));
          commit<CTAS>(empty_bar(stage));
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
    } else if (warp >= 2) {
      // ---------------- scales ----------------
      int buf = 0;
      uint32_t buf_phase = 0;
      bool ok = true;
      for (int t = 0; t < n_mine && ok; ++t) {
        int m_tile, n_tile;
        tile_at(t, &m_tile, &n_tile);
        const int r0 = (warp - 2) * 64 + lane;
        const int64_t row = int64_t(m_tile) * kBM + r0, n0 = int64_t(n_tile) * BN;
        const float* sx0 = p.x_scales + (row < p.n_rows ? row : p.n_rows - 1) * p.k_blocks;
        const float* sx1 = p.x_scales + (row + 32 < p.n_rows ? row + 32 : p.n_rows - 1) * p.k_blocks;
        const float* sw[kHalves];
        float w[kHalves];
#pragma unroll
        for (int g = 0; g < kHalves; ++g) {
          // columns past the vocabulary have no scales: whatever they get is cut off
          sw[g] = p.w_scales + (n0 + g * 128 < p.vocab ? n0 + g * 128 : n0) / 128 * p.k_blocks;
          w[g] = sw[g][0];
        }
        float x0 = sx0[0], x1 = sx1[0];
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          float a0[kHalves], a1[kHalves];
#pragma unroll
          for (int g = 0; g < kHalves; ++g) {
            a0[g] = x0 * w[g];
            a1[g] = x1 * w[g];
          }
          if (kb + 1 < p.k_blocks) {
            x0 = sx0[kb + 1];
            x1 = sx1[kb + 1];
#pragma unroll
            for (int g = 0; g < kHalves; ++g) w[g] = sw[g][kb + 1];
          }
          ok = wait_or_abort(slot_empty(buf), buf_phase ^ 1u, &abort_flag, p.device_status);
          if (!ok) break;
#pragma unroll
          for (int g = 0; g < kHalves; ++g) {
            scales[(buf * kHalves + g) * kBM + r0] = a0[g];
            scales[(buf * kHalves + g) * kBM + r0 + 32] = a1[g];
          }
          __syncwarp();
          if (lane == 0) cl::mbar_arrive(acc_full(buf));
          if (++buf == kBufs) {
            buf = 0;
            buf_phase ^= 1u;
          }
        }
      }
    }
  } else {
    // ---------------- epilogue ----------------
    regs_take<kRegsEpilogue>();
    const int quarter = warp & 3;  // the TMEM lanes a warp may read: 32*(warp id mod 4) ...
    const int half = (warp - 4) >> 2;
    const uint32_t my_store = store_buf + uint32_t(warp - 4) * T::kStoreBytes;
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
    int t = 0;
    for (; t < n_mine; ++t) {
      int m_tile, n_tile;
      tile_at(t, &m_tile, &n_tile);
      const int64_t n0 = int64_t(n_tile) * BN + half * CW;
      f32x2 acc[CW / 2];
#pragma unroll
      for (int j = 0; j < CW / 2; ++j) acc[j] = 0ull;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        ok = wait_or_abort(acc_full(buf), buf_phase, &abort_flag, p.device_status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_addr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(buf * BN + half * CW);
        uint32_t v[2][32];
        tmem_ld32(t_addr, v[0]);
        tmem_ld32(t_addr + 32u, v[1]);
        const float scale = scales[(buf * kHalves + half % kHalves) * kBM + quarter * 32 + lane];
        const f32x2 f = pack2(scale, scale);
#pragma unroll
        for (int ch = 0; ch < CW / 32; ++ch) {
          if ((ch & 1) == 0) {
            tmem_ld_wait();  // two chunks of 32 columns per wait
            if (ch + 2 >= CW / 32) {
              // everything of this accumulator is in registers: hand it back
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if (CTAS == 1)
                  cl::mbar_arrive(acc_empty(buf));
                else
                  arrive_leader(acc_empty(buf));
                cl::mbar_arrive(slot_empty(buf));
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[ch * 16 + j] = fma2(pack2(__uint_as_float(v[ch & 1][2 * j]), __uint_as_float(v[ch & 1][2 * j + 1])), f,
                                    acc[ch * 16 + j]);
          if (ch + 2 < CW / 32) tmem_ld32(t_addr + uint32_t((ch + 2) * 32), v[ch & 1]);
        }
        if (++buf == kBufs) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      if (!ok) break;
      const int valid = int(p.vocab - n0 < CW ? (p.vocab - n0 > 0 ? p.vocab - n0 : 0) : CW);
      if (!STATS) {
        store_rows<O, CW, T::kStoreBytes>(p, &map_out, acc, int64_t(m_tile) * kBM + quarter * 32, n0, valid, my_store, lane);
      } else if (valid > 0) {
        float y[CW];
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) unpack2(acc[j], y[2 * j], y[2 * j + 1]);
        if (cap) {
#pragma unroll
          for (int j = 0; j < CW; ++j) y[j] = sc.y(y[j]);
        }
        // a chosen column is in few tiles, the end of the vocabulary in one: whole warps skip looking for them
        const int64_t c_local = c >= 0 ? c - n0 : -1;
        if (__any_sync(0xffffffffu, c_local >= 0 && c_local < CW)) {
#pragma unroll
          for (int j = 0; j < CW; ++j)
            if (j == c_local) yc = y[j];
        }
        if (valid < CW) {
#pragma unroll
          for (int j = 0; j < CW; ++j) y[j] = j < valid ? y[j] : kNegInit;
        }
        float cm = y[0];
#pragma unroll
        for (int j = 1; j < CW; ++j) cm = fmaxf(cm, y[j]);
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
    } else {
      for (; t < n_mine; ++t) {  // a wait has run out in tile t
        int m_tile, n_tile;
        tile_at(t, &m_tile, &n_tile);
        const int64_t n0 = int64_t(n_tile) * BN + half * CW;
        void_rows<O>(p, int64_t(m_tile) * kBM + quarter * 32, n0, int(p.vocab - n0 < CW ? p.vocab - n0 : CW), lane);
      }
      if (lane == 0) cl::bulk_wait_all();  // the buffers are read and written out before this CTA's shared memory goes
    }
  }

  // ---------------- teardown: every role arrives here, also after an abort ----------------
  __syncwarp();
  if (abort_flag && warp == 1) {
    for (int i = 0; i < 4; ++i) __nanosleep(500000);  // copies or MMAs may still be in flight: bounded time for them
  }
  tc_fence_before();
  if (CTAS == 1)
    __syncthreads();
  else
    cl::cluster_sync_all();  // neither CTA leaves while the other may signal its barriers or read its tiles
  if (warp == 1) {
    tc_fence_after();
    tmem_free<CTAS>(tmem_base);
  }
}

// Partials of all column ranges of a row -> one (entry 0 of the buffer) and what follows from it: 32 rows per CTA, eight
// threads per row.
__global__ void __launch_bounds__(256) merge_kernel(const Params p, int entries, int32_t* status) {
  if (status && blockIdx.x == 0 && threadIdx.x == 0 && *p.device_status) atomicOr(status, *p.device_status);
  float4* const partials = p.partials;
  const int64_t n_rows = p.n_rows;
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
    const float lse = m + logf(s);
    if (p.logps) p.logps[row] = (yc - lse) * p.inv_temperature;
    if (p.entropy) p.entropy[row] = lse - u / s;
    if (p.lse) p.lse[row] = lse;
  }
}

// [rows, cols] of `elem` bytes with `ld` bytes between rows -> boxes of box_rows x 128 bytes, 128-byte swizzle, zeros
// outside.
static bool make_map(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, int64_t rows, int64_t cols,
                     int64_t ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(ld)};
  const cuuint32_t box[2] = {cuuint32_t(128 / elem), cuuint32_t(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSms = 148;
constexpr int kFoldBN = 256;

// Pairs of CTAs from two row tiles on: half of a pair would idle with one.
static int ctas_for(int64_t m_tiles) { return m_tiles >= 2 ? 2 : 1; }

// Column ranges of the folded form: as many whole tiles per CTA (pair) as balance the SMs best; each costs about a
// third of a tile to start and end.
static void fold_plan(int64_t n_rows, int64_t vocab, int* tiles_per_split, int* splits) {
  const int64_t m_tiles = (n_rows + kBM - 1) / kBM, n_tiles = (vocab + kFoldBN - 1) / kFoldBN;
  const int ctas = ctas_for(m_tiles);
  const int64_t m_teams = (m_tiles + ctas - 1) / ctas, slots = kSms / ctas;
  double best = 1e300;
  int64_t pick = 1;
  for (int64_t per = 1; per <= n_tiles && per <= 64; ++per) {
    const int64_t teams = m_teams * ((n_tiles + per - 1) / per);
    const double cost = double((teams + slots - 1) / slots) * (double(per) + 0.33);
    if (cost < best * 0.999) {
      best = cost;
      pick = per;
    }
  }
  *tiles_per_split = int(pick);
  *splits = int((n_tiles + pick - 1) / pick);
}

template <int BN, int CTAS, bool STATS, typename O>
static int launch_t(const Params& p, unsigned grid, const CUtensorMap& mx, const CUtensorMap& mw,
                    const CUtensorMap& mo, cudaStream_t s) {
  using T = Tile<BN, CTAS>;
  auto* kernel = product_kernel<BN, CTAS, STATS, O>;
  static std::once_flag attr_once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MLLM_GRPO_ERR_NO_DEVICE;
  std::call_once(attr_once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(T::kSmemBytes));
    cudaFuncAttributes fa;
    if (attr_err[dev] == cudaSuccess) attr_err[dev] = cudaFuncGetAttributes(&fa, kernel);
    // the epilogue takes registers that the launch must have brought along
    if (attr_err[dev] == cudaSuccess && fa.numRegs < kRegsLaunch) attr_err[dev] = cudaErrorInvalidConfiguration;
  });
  if (attr_err[dev] != cudaSuccess) return record_cuda_error(attr_err[dev]);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = T::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CTAS;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CTAS > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mx, mw, mo, p);
  count_launch();
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

template <int BN, int CTAS, bool STATS, typename O>
static int launch(Params p, const mllm_lm_head_fp8_args* a, cudaStream_t s) {
  p.m_tiles = int((p.n_rows + kBM - 1) / kBM);
  p.n_tiles = int((p.vocab + BN - 1) / BN);
  CUtensorMap mx, mw, mo;
  if (!make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->hidden, a->n_rows, a->hidden_dim, a->hidden_stride, kBM) ||
      !make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->weight, a->vocab, a->hidden_dim, a->weight_stride, Tile<BN, CTAS>::kBRows))
    return MLLM_GRPO_ERR_NO_DEVICE;
  mo = mx;  // not read unless the output goes out by TMA
  if (!STATS && p.out_aligned) {
    const CUtensorMapDataType type = sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    if (!make_map(&mo, type, int(sizeof(O)), p.out, p.n_rows, p.vocab, p.out_stride * int64_t(sizeof(O)), 32))
      return MLLM_GRPO_ERR_NO_DEVICE;
  }
  const int64_t m_teams = (p.m_tiles + CTAS - 1) / CTAS;
  int64_t teams;
  if (STATS) {
    fold_plan(p.n_rows, p.vocab, &p.tiles_per_split, &p.splits);
    teams = m_teams * p.splits;
  } else {
    teams = m_teams * p.n_tiles;
  }
  if (teams >= (int64_t(1) << 29)) return MLLM_GRPO_ERR_TOO_LARGE;
  if (!STATS && teams > kSms / CTAS) teams = kSms / CTAS;
  return launch_t<BN, CTAS, STATS, O>(p, unsigned(teams * CTAS), mx, mw, mo, s);
}

template <typename O>
static int launch_product(const Params& p, const mllm_lm_head_fp8_args* a, cudaStream_t s) {
  // tiles of 256 columns read the least per product; with fewer of them than SMs, twice as many of 128
  const int64_t m_tiles = (p.n_rows + kBM - 1) / kBM, tiles = m_tiles * ((p.vocab + 255) / 256);
  if (tiles <= kSms) return launch<128, 1, false, O>(p, a, s);
  return ctas_for(m_tiles) == 2 ? launch<256, 2, false, O>(p, a, s) : launch<256, 1, false, O>(p, a, s);
}

static std::atomic<int> stop_after{-1};  // test hook

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
  const int stop = stop_after.load(std::memory_order_relaxed);
  p->stop_after = stop < 0 ? INT32_MAX : stop;
  return MLLM_GRPO_OK;
}

}  // namespace fp8
}  // namespace grpo

using namespace grpo;

extern "C" {

void mllm_lm_head_fp8_stop_after(int32_t tiles) { fp8::stop_after.store(tiles, std::memory_order_relaxed); }

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
  if (a->n_rows <= fp8::kFewRows && a->hidden_dim < (int64_t(1) << 30)) {  // it counts bytes of a row in 32 bits
    const cudaError_t e = fp8::launch_few_rows(p, a->out_dtype, s);
    return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
  }
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
  if (!(a->softcap >= 0.f) || !(a->temperature >= 0.f)) return MLLM_GRPO_ERR_BAD_ATTRIBUTE;
  if (!fp8::aligned(a->partials, 16) || !fp8::aligned(a->chosen_ids, 4) || !fp8::aligned(a->per_token_logps, 4) ||
      !fp8::aligned(a->token_entropy, 4) || !fp8::aligned(a->lse, 4) || !fp8::aligned(a->call_status, 4))
    return MLLM_GRPO_ERR_ALIGNMENT;
  // one word is reported into: the call's own, added to the caller's by the last launch
  if (a->call_status) p.device_status = a->call_status;
  const float temperature = a->temperature > 0.f ? a->temperature : 1.0f;
  if (a->token_entropy && temperature != 1.0f) return MLLM_GRPO_ERR_UNSUPPORTED;
  // a shard of the vocabulary does not know a row's log-sum-exp
  if ((a->per_token_logps || a->token_entropy || a->lse) &&
      (a->vocab_start != 0 || (a->vocab_total > 0 && a->vocab_total != a->vocab)))
    return MLLM_GRPO_ERR_UNSUPPORTED;
  p.inv_temperature = 1.0f / temperature;
  p.logps = a->per_token_logps;
  p.entropy = a->token_entropy;
  p.lse = a->lse;
  p.vocab_start = a->vocab_start;
  p.vocab_total = a->vocab_total > 0 ? a->vocab_total : a->vocab_start + a->vocab;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->call_status) {
    const cudaError_t e = cudaMemsetAsync(a->call_status, 0, sizeof(int32_t), s);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  st = fp8::ctas_for((a->n_rows + fp8::kBM - 1) / fp8::kBM) == 2 ? fp8::launch<fp8::kFoldBN, 2, true, float>(p, a, s)
                                                                  : fp8::launch<fp8::kFoldBN, 1, true, float>(p, a, s);
  if (st) return st;
  int per, splits;
  fp8::fold_plan(a->n_rows, a->vocab, &per, &splits);
  fp8::merge_kernel<<<unsigned((a->n_rows + 31) / 32), 256, 0, s>>>(p, splits * 2, a->call_status ? a->device_status : nullptr);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MLLM_GRPO_OK : record_cuda_error(e);
}

}  // extern "C"
