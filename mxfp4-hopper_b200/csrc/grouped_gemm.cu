// The experts' MXFP4 products with a fused epilogue (sm_100a): for the rows r of
// expert e, z[r] = A[r] . B_e^T + bias_e, c[r] = act(z[r]) + residual[r].
//
// Rows are sorted by expert and the split is ragged and only known on the
// device: every CTA builds the running sums of m_splits in shared memory and
// walks tiles of (expert, row block, column block).  A's rows start anywhere, so
// its E8M0 bytes are read from the row-major layout that the quantizer and the
// permute write, and put into the order of the tcgen05 block-scale layout on the
// way to tensor memory; a tile's rows past its group's end are computed and not
// written.
//
// Two kernels, chosen by grouped_plan() below:
//   wide    256 rows x 256 or 128 weight rows a tile: the rows are the M side of
//           MMAs that two CTAs share.
//   narrow  16 or 64 rows x 128 (gated: 256) weight rows a tile: the weights are
//           the M side, so that a few rows do not pay for 128.  A cluster of up
//           to 8 CTAs splits K; the partial accumulators meet in distributed
//           shared memory, always summed in the same order.
#include <cuda_bf16.h>

#include <algorithm>

#include "capi_util.h"
#include "common.cuh"
#include "epilogue.cuh"
#include "groups.cuh"
#include "host_util.h"
#include "qrow.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace mxb {
namespace {

constexpr int kStepK = 256;  // elements of K per pipeline stage: 128 code bytes, 8 scales a row

struct GroupedArgs {
  const uint8_t* a_scales;
  int64_t a_spitch;
  const uint8_t* b_scales;
  const int32_t* m_splits;
  int64_t M;
  int E, width, K;  // width: columns of the result (N, gated N / 2)
  int act, bias_f32;
  const void* bias;
  const uint8_t* residual;
  int64_t residual_ld;
  uint8_t *pre, *c;
  int64_t pre_ld, c_ld;
  uint8_t *c_codes, *c_scales;
  int a_scales_tma;  // A's scales have a tensor map
};

// E8M0 bytes b0 .. b0 + 31 (four K steps) of a warp's 32 rows -> dst[32][32] in
// shared memory; zero past a row's S bytes and past the `rows` there are.  Whole
// aligned words where the rows have them (4 rows an instruction), else a byte a
// lane and a row an instruction: neighbouring lanes read neighbouring bytes either way.
__device__ __forceinline__ void gather_scales(uint8_t* dst, const uint8_t* src, int64_t pitch,
                                              int rows, int b0, int S, bool words) {
  const int lane = threadIdx.x & 31;
  if (words) {
    const int at = b0 + 4 * (lane & 7);
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3);
      v[i] = r < rows && at < S ? __ldg(reinterpret_cast<const uint32_t*>(src + r * pitch + at)) : 0u;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<uint32_t*>(dst + (4 * i + (lane >> 3)) * 32 + 4 * (lane & 7)) = v[i];
  } else {
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 16) {
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = r0 + i < rows && b0 + lane < S ? __ldg(src + (r0 + i) * pitch + b0 + lane) : 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) dst[(r0 + i) * 32 + lane] = (uint8_t)v[i];
    }
  }
}
// Whether every row's scale bytes are whole aligned words.
__device__ __forceinline__ bool scale_words(const GroupedArgs& p) {
  return ((reinterpret_cast<uintptr_t>(p.a_scales) | (uintptr_t)p.a_spitch |
           (uintptr_t)(p.K / 32)) & 3) == 0;
}

// 16 bytes from byte `at` (0 .. 15) of two neighbouring lines on.
__device__ __forceinline__ uint4 bytes_from(const uint4& x, const uint4& y, uint32_t at) {
  const bool two = at & 8, one = at & 4;
  const uint32_t d0 = two ? x.z : x.x, d1 = two ? x.w : x.y, d2 = two ? y.x : x.z,
                 d3 = two ? y.y : x.w, d4 = two ? y.z : y.x, d5 = two ? y.w : y.y;
  const uint32_t e0 = one ? d1 : d0, e1 = one ? d2 : d1, e2 = one ? d3 : d2, e3 = one ? d4 : d3,
                 e4 = one ? d5 : d4, sh = at % 4 * 8;
  return make_uint4(__funnelshift_r(e0, e1, sh), __funnelshift_r(e1, e2, sh),
                    __funnelshift_r(e2, e3, sh), __funnelshift_r(e3, e4, sh));
}

// 32 BF16 columns of a row: in 32-byte sectors where base and pitch allow it, else in
// 16-byte pieces; columns past the `cols` there are (a multiple of 8) are left alone.
__device__ __forceinline__ bool sectors(const void* base, int64_t ld) {
  return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(ld * 2)) & 31) == 0;
}
__device__ __forceinline__ void store_cols(uint8_t* out, int cols, bool whole, const uint32_t (&w)[16]) {
  if (whole && cols >= 32) {
#pragma unroll
    for (int k = 0; k < 2; ++k) st_v8(out + 32 * k, w + 8 * k);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (8 * k < cols)
        *reinterpret_cast<uint4*>(out + 16 * k) =
            make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  }
}
__device__ __forceinline__ void load_cols(const uint8_t* src, int cols, bool whole, uint32_t (&w)[16]) {
  if (whole && cols >= 32) {
#pragma unroll
    for (int k = 0; k < 2; ++k) ld_v8(src + 32 * k, w + 8 * k);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (8 * k < cols) x = __ldg(reinterpret_cast<const uint4*>(src + 16 * k));
      w[4 * k] = x.x; w[4 * k + 1] = x.y; w[4 * k + 2] = x.z; w[4 * k + 3] = x.w;
    }
  }
}
__device__ __forceinline__ void pack32(const float* v, uint32_t (&w)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = cvt_bf16x2(v[2 * j], v[2 * j + 1]);
}

__device__ __forceinline__ float load_bias(const GroupedArgs& p, int64_t i) {
  return p.bias_f32 ? static_cast<const float*>(p.bias)[i]
                    : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[i]);
}

// ---------------------------------------------------------------- wide
// A persistent pair of CTAs (cta_group::2) per two SMs; a tile has 256 rows, 128
// in each CTA, and kN weight rows, of which each CTA holds half: columns n0 ..
// n0 + kN - 1 of the result, or (gated) the gate and the up rows of columns n0 ..
// n0 + kN / 2 - 1.  kN is 256, where each operand byte crosses L2 -> shared memory
// once per 256 x 256 tile instead of once per 128 x 256, or 128, where twice the
// tiles fill the GPU better.
//   warp 0       TMA of this CTA's half of A's and B's codes, completing on CTA
//                0's barrier
//   warp 1       (CTA 0) MMA issue: four M = 256, N = kN, K = 64 a step
//   warp 2       scales of four K steps at a time: a TMA box of 32 bytes of each
//                of A's rows, bulk copies of B's atoms (both halves)
//   warp 3       (kLines) A's scale rows that TMA cannot take, their base or pitch
//                not being a multiple of 16: the three 16-byte lines that hold a
//                row's 32 bytes, by cp.async, whose completion counts on warp 2's
//                barrier.  Byte loads by the scale warps took 186 instead of 166 us
//                (16384 rows over 32 experts, gated 2 x 2880 x 2880) and 51.5
//                instead of 40.9 (4096 x 4096 x 4160); with both kinds of row in one
//                kernel those of TMA became 4 % slower
//   warps 4-7    scales: each warp gathers its lane quadrant's words of a step
//                from shared memory and writes them to the step's tensor memory
//                columns with tcgen05.st, so that the tensor pipe carries MMAs
//                only, and arrives on the barrier that the codes complete on:
//                one wait a step
//   warps 8-15   epilogue: two groups of four warps, each with half the columns.
//                The accumulator is read into registers at once and given back,
//                so that the next tile's products run under the epilogue.  A
//                thread has a row and writes it in whole 32-byte sectors
constexpr int kWideThreads = 512;
constexpr int kWideStages = 6;
constexpr uint32_t kBoxBytes = 128 * 128;  // 128 rows of 128 code bytes
constexpr uint32_t kAtoms = 2 * 512;       // scale atoms of 128 rows and one K step
constexpr uint32_t kWideStage = 2 * kBoxBytes;
constexpr int kSbStages = 2;               // shared-memory scales of four steps each:
constexpr uint32_t kLineRow = 48;          // A's 128 rows of 32 bytes, or of three lines,
constexpr uint32_t kSbA = 128 * kLineRow;
constexpr uint32_t kSbB = 4 * kAtoms;      // 8 atoms of each of B's halves
constexpr uint32_t kSbStage = kSbA + 2 * kSbB;
constexpr uint32_t kScaleCol = 256;        // tensor memory: accumulator, then scales
constexpr uint32_t kTmemCols = 512;
constexpr size_t kWideSmem = 1024 + kWideStages * kWideStage + kSbStages * kSbStage + 256 * 4 +
                             kGroupTableInts * 4 + 512;
static_assert(kWideSmem <= 227 * 1024, "one CTA per SM");
static_assert(kScaleCol + 24 * kWideStages <= kTmemCols, "scales fit beside the accumulator");
static_assert(kWideStage % 1024 == 0, "swizzled boxes start on 1024 bytes");
// Registers: 512 threads x 128 at launch = 128 x 64 + 128 x 96 + 256 x 176.  (A scale
// warp should not spill: a spilled load is waited for where it is issued.  The compiler
// reports 64 spilled bytes for the kernels of 256 weight rows, 20 where gated, and up to
// 4 (stored; 32 reloaded) for those of 128, 20 (140) where gated with TMA's scale rows.)
constexpr int kWideCopyRegs = 64, kWideScaleRegs = 96, kWideEpilogueRegs = 176;

template <int kAct, int kN, bool kLines>
__global__ void __launch_bounds__(kWideThreads, 1) grouped_wide_kernel(
    const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
    const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ GroupedArgs p) {
  constexpr bool kGlu = kAct == MXB_ACT_SWIGLU;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* scales = smem + kWideStages * kWideStage;
  float* bias_s = reinterpret_cast<float*>(scales + kSbStages * kSbStage);
  // CTA 0's: a step's codes of both CTAs have landed and its scales are in tensor memory
  uint64_t* full = reinterpret_cast<uint64_t*>(bias_s + 256);
  uint64_t* empty = full + kWideStages;
  uint64_t* sb_full = empty + kWideStages;   // four steps' scales in shared memory
  uint64_t* sb_empty = sb_full + kSbStages;
  uint64_t* acc_full = sb_empty + kSbStages;
  uint64_t* acc_empty = acc_full + 1;  // CTA 0's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 1);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  GroupTable g;
  g.off = failed + 1;
  g.tile = g.off + p.E + 1;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int rank = (int)cluster_rank();
  constexpr int kTileN = kGlu ? kN / 2 : kN;
  constexpr uint32_t kBBox = kN / 2 * 128;  // this CTA's weight rows of a stage
  // 128-row scale blocks a tile reads: two, but one for 128 columns of a plain result
  constexpr bool kTwoBlocks = kGlu || kN == 256;
  const int ntn = (p.width + kTileN - 1) / kTileN;
  const int ksteps = (p.K + kStepK - 1) / kStepK;
  const int S = p.K / 32, S4 = (S + 3) / 4;

  if (warp == 0) {
    wait_for_previous_kernel();
    build_groups(g, p.m_splits, p.E, p.M, [&](int rows) { return (rows + 255) / 256 * ntn; });
  } else if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
  } else if (t == 64) {
    for (int s = 0; s < kWideStages; ++s) {
      mbar_init(&full[s], 1 + 8);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kSbStages; ++s) {
      mbar_init(&sb_full[s], kLines ? 1 + 32 : 1);
      mbar_init(&sb_empty[s], 4);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 16);
    fence_mbar_init();
    *failed = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_sync();
  allow_next_kernel();  // every CTA of this one has its tensor memory
  wait_for_previous_kernel();
  const uint32_t tmem = *tmem_slot;
  const int tiles = g.tile[p.E];
  const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  const int my_tiles = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0;

  struct Tile {
    int e, m0, n0;  // m0: this CTA's first row
  };
  auto tile_at = [&](int i) {
    const int id = pair + i * pairs;
    Tile r;
    r.e = find_group(g.tile, p.E, id);
    const int local = id - g.tile[r.e];
    r.m0 = g.off[r.e] + local / ntn * 256 + rank * 128;
    r.n0 = local % ntn * kTileN;
    return r;
  };

  // columns 128 .. 255 of a plain tile may all lie past the result: then their scales
  // and CTA 1's weight rows are not loaded, and what is stale there makes columns that
  // are not written
  auto has_second = [&](const Tile& tl) { return kGlu || kN == 128 || tl.n0 + 128 < p.width; };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideCopyRegs));
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------ TMA producer
      const uint32_t full0 = peer_addr(smem_addr(full), 0);
      int gs = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile tl = tile_at(i);
        const int row = kGlu ? (2 * tl.e + rank) * p.width + tl.n0
                             : tl.e * p.width + tl.n0 + kN / 2 * rank;
        const bool second = has_second(tl);
        for (int ks = 0; ks < ksteps; ++ks, ++gs) {
          const int s = gs % kWideStages;
          if (gs >= kWideStages && !mbar_wait_suspend(&empty[s], (uint32_t)((gs / kWideStages - 1) & 1))) {
            atomicExch(failed, 1);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kWideStage;
          if (rank == 0)
            mbar_arrive_expect_tx(&full[s], 2 * kBoxBytes + (second ? 2 : 1) * kBBox);
          const int kx = ks * (kStepK / 2);
          tma_load_2d_pair(st, &map_a, kx, tl.m0, full0 + 8 * s);
          if (rank == 0 || second) tma_load_2d_pair(st + kBoxBytes, &map_b, kx, row, full0 + 8 * s);
        }
      }
      // do not leave while copies are still landing (CTA 0 waits for both CTAs' codes)
      for (int q = gs > kWideStages ? gs - kWideStages : 0; rank == 0 && q < gs; ++q)
        mbar_wait_suspend(&full[q % kWideStages], (uint32_t)((q / kWideStages) & 1));
    } else if (warp == 2 && lane == 0) {
      // ------------------------------------------------ scales, four steps a time
      const int nbp = (p.width + 127) / 128;  // 128-row scale blocks of a weight part
      int gq = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile tl = tile_at(i);
        const int block = (kGlu ? 2 : 1) * tl.e * nbp + tl.n0 / 128;
        const uint8_t* src0 = p.b_scales + (int64_t)block * S4 * 512;
        const uint8_t* src1 = src0 + (int64_t)(kGlu ? nbp : 1) * S4 * 512;
        const bool second = has_second(tl);
        for (int k4 = 0; k4 < S4; k4 += 8, ++gq) {
          const int s = gq % kSbStages;
          if (gq >= kSbStages && !mbar_wait_suspend(&sb_empty[s], (uint32_t)((gq / kSbStages - 1) & 1))) {
            atomicExch(failed, 1);
            ok = false;
            break;
          }
          uint8_t* sb = scales + s * kSbStage;
          const uint32_t atoms = (uint32_t)min(8, S4 - k4) * 512;
          const bool two = kTwoBlocks && second;
          mbar_arrive_expect_tx(&sb_full[s], (kLines ? 0 : 128 * 32) + (two ? 2 : 1) * atoms);
          if (!kLines) tma_load_2d(sb, &map_sa, 4 * k4, tl.m0, &sb_full[s]);
          bulk_load_1d(sb + kSbA, src0 + k4 * 512, atoms, &sb_full[s]);
          if (two) bulk_load_1d(sb + kSbA + kSbB, src1 + k4 * 512, atoms, &sb_full[s]);
        }
      }
      for (int q = gq > kSbStages ? gq - kSbStages : 0; q < gq; ++q)
        mbar_wait_suspend(&sb_full[q % kSbStages], (uint32_t)((q / kSbStages) & 1));
    } else if (kLines && warp == 3) {
      // ------------------------------------------------ A's scale rows, four steps a time
      int gq = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile tl = tile_at(i);
        const uint8_t* const row0 = p.a_scales + ((int64_t)tl.m0 + lane) * p.a_spitch;
        const int rows = (int)min((int64_t)128, p.M - tl.m0);
        for (int b0 = 0; b0 < S; b0 += 32, ++gq) {
          const int s = gq % kSbStages;
          const bool free = gq < kSbStages ||
                            mbar_wait_suspend(&sb_empty[s], (uint32_t)((gq / kSbStages - 1) & 1));
          if (!__all_sync(0xffffffffu, free)) {
            atomicExch(failed, 1);
            ok = false;
            break;
          }
          const uint32_t sb = smem_addr(scales + s * kSbStage) + lane * kLineRow;
          const uint8_t* from = row0 + b0;
#pragma unroll
          for (int k = 0; k < 4; ++k, from += 32 * p.a_spitch) {
            // the row's 32 bytes, or what is left of it; the rest becomes zero.  What the
            // first line holds before them is read and not used (an allocation starts on
            // a line, so a line with a byte of it lies in it).
            const bool there = 32 * k + lane < rows;
            const uint8_t* line = there ? from : p.a_scales;
            const int before = (int)(reinterpret_cast<uintptr_t>(line) & 15u);
            line -= before;
            const int end = there ? before + min(32, S - b0) : 0;
#pragma unroll
            for (int c = 0; c < 3; ++c)
              cp_async16_zfill(sb + k * 32 * kLineRow + 16 * c, line + (end > 16 * c ? 16 * c : 0),
                               (uint32_t)max(0, min(16, end - 16 * c)));
          }
          cp_async_arrive(&sb_full[s]);
        }
      }
      cp_async_wait_all();
    } else if (warp == 1 && rank == 0) {
      // ------------------------------------------------ MMA issuer
      const bool one = elect_one();
      bool ok = true, ready = false;
      int gs = 0;
      for (int i = 0; ok && i < my_tiles; ++i) {
        if (i > 0 && !mbar_wait_suspend(acc_empty, (uint32_t)((i - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int ks = 0; ks < ksteps; ++ks, ++gs) {
          const int s = gs % kWideStages;
          if (!ready && !mbar_wait_suspend(&full[s], (uint32_t)((gs / kWideStages) & 1))) {
            ok = false;
            break;
          }
          // whether the next step is ready as well: known by the time it is needed
          ready = mbar_peek(&full[(gs + 1) % kWideStages], (uint32_t)(((gs + 1) / kWideStages) & 1));
          tc_fence_after();
          __syncwarp();
          const uint8_t* st = smem + s * kWideStage;
          const uint32_t sfc = tmem + kScaleCol + (uint32_t)(s * 24);
          const int left = p.K - ks * kStepK;  // elements of K from this step on
          const uint64_t da = smem_desc_sw128(st);
          const uint64_t db = smem_desc_sw128(st + kBoxBytes);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (64 * j >= left) break;
            const uint32_t sf_id = (uint32_t)(j & 1) * 2u;
            tc_mma_pair(tmem, da + (uint64_t)(2 * j), db + (uint64_t)(2 * j),
                        mxf4_idesc(256, kN, sf_id), (sfc + 4 * (j >> 1)) | (sf_id << 30),
                        (sfc + 8 + kN / 32 * (j >> 1)) | (sf_id << 30),
                        (ks > 0 || j > 0) ? 1u : 0u, one);
          }
          tc_commit_pair(&empty[s], one);
        }
        __syncwarp();
        tc_commit_pair(acc_full, one);
      }
      if (!ok) atomicExch(failed, 1);
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideScaleRegs));
    // ------------------------------------------------ scales
    const int q = warp - 4;
    const uint32_t full0 = peer_addr(smem_addr(full), 0);
    const uint32_t col0 = tmem + ((uint32_t)(q * 32) << 16) + kScaleCol;
    int gs = 0, gq = 0;
    bool ok = true;
    for (int i = 0; ok && i < my_tiles; ++i) {
      const Tile tl = tile_at(i);
      // where the 32 bytes of row 32 c + lane start
      uint32_t at[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        at[c] = kLines ? (uint32_t)(32 * c + lane) * kLineRow +
                             (((uint32_t)reinterpret_cast<uintptr_t>(p.a_scales) +
                               (uint32_t)(tl.m0 + 32 * c + lane) * (uint32_t)p.a_spitch) & 15u)
                       : (uint32_t)(32 * c + lane) * 32;
      for (int ks0 = 0; ok && ks0 < ksteps; ks0 += 4, ++gq) {
        const int sq = gq % kSbStages;
        uint8_t* sb = scales + sq * kSbStage;
        bool up = mbar_wait_suspend(&sb_full[sq], (uint32_t)((gq / kSbStages) & 1));
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const int two = min(2, ksteps - ks0 - j);
          if (two <= 0) break;
          // a row's 16 bytes are two steps of two atoms; the four rows of a lane fill
          // the atoms' four columns
          uint4 ra[4];
          if constexpr (!kLines) {
#pragma unroll
            for (int c = 0; c < 4; ++c) ra[c] = *reinterpret_cast<const uint4*>(sb + at[c] + j * 8);
          } else {
            // two whole lines of each row, shifted down
            uint4 x[4], y[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint4* const l = reinterpret_cast<const uint4*>(sb + (at[c] & ~15u)) + j / 2;
              x[c] = l[0];
              y[c] = l[1];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) ra[c] = bytes_from(x[c], y[c], at[c] & 15u);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h >= two) break;
            const uint32_t a[8] = {h ? ra[0].z : ra[0].x, h ? ra[1].z : ra[1].x,
                                   h ? ra[2].z : ra[2].x, h ? ra[3].z : ra[3].x,
                                   h ? ra[0].w : ra[0].y, h ? ra[1].w : ra[1].y,
                                   h ? ra[2].w : ra[2].y, h ? ra[3].w : ra[3].y};
            // a column of B's scales is 32 of its kN rows; the columns of one K atom are
            // neighbours: 4 + 4 of two blocks, 4 of one, or (gated, kN = 128) the two
            // halves' 2 + 2 columns from where n0 lies in their blocks
            uint32_t b[kN / 16];
            const uint8_t* sbb = sb + kSbA + 2 * (j + h) * 512 + lane * 16;
            if constexpr (kN == 256) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint4 w = *reinterpret_cast<const uint4*>(sbb + (k & 1) * kSbB + (k >> 1) * 512);
                b[4 * k] = w.x; b[4 * k + 1] = w.y; b[4 * k + 2] = w.z; b[4 * k + 3] = w.w;
              }
            } else if constexpr (kGlu) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint2 w = *reinterpret_cast<const uint2*>(
                    sbb + (k & 1) * kSbB + (k >> 1) * 512 + (tl.n0 & 64) / 8);
                b[2 * k] = w.x; b[2 * k + 1] = w.y;
              }
            } else {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const uint4 w = *reinterpret_cast<const uint4*>(sbb + k * 512);
                b[4 * k] = w.x; b[4 * k + 1] = w.y; b[4 * k + 2] = w.z; b[4 * k + 3] = w.w;
              }
            }
            const int s = gs % kWideStages;
            up = up && (gs < kWideStages ||
                        mbar_wait_suspend(&empty[s], (uint32_t)((gs / kWideStages - 1) & 1)));
            tc_fence_after();
            __syncwarp();
            tmem_st8(col0 + (uint32_t)(s * 24), a);
            if constexpr (kN == 256) tmem_st16(col0 + (uint32_t)(s * 24 + 8), b);
            else tmem_st8(col0 + (uint32_t)(s * 24 + 8), b);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) peer_signal(full0 + 8 * s);
            ++gs;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sb_empty[sq]);
        if (!__all_sync(0xffffffffu, up)) {
          atomicExch(failed, 1);
          ok = false;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideEpilogueRegs));
    // ------------------------------------------------ epilogue
    const int half = (warp - 8) >> 2, quad = warp & 3;
    const int r = quad * 32 + lane, ht = t & 127;
    float* bias_h = bias_s + half * 128;
    constexpr int kHalfN = kTileN / 2;  // result columns of this group
    constexpr int kAcc = kN / 2;        // its accumulator columns: of z, or gate then up
    constexpr int kUp = kAcc / 2;       // where up starts among them
    const uint32_t acc_empty0 = peer_addr(smem_addr(acc_empty), 0);
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const bool c32 = sectors(p.c, p.c_ld), pre32 = sectors(p.pre, p.pre_ld) && p.width % 16 == 0;
    const bool res32 = sectors(p.residual, p.residual_ld);
    for (int i = 0; i < my_tiles; ++i) {
      const Tile tl = tile_at(i);
      const int rows = min(128, g.off[tl.e + 1] - tl.m0);  // none or fewer: CTA 1's share
      const int nh = tl.n0 + half * kHalfN;                // first result column of this group
      const bool mine = r < rows;
      float bias = 0.0f;
      if (p.bias && ht < kAcc) {
        const int col = nh + (kGlu ? ht % kUp : ht);
        const int64_t at = kGlu ? (int64_t)tl.e * 2 * p.width + (ht < kUp ? 0 : p.width) + col
                                : (int64_t)tl.e * p.width + col;
        if (col < p.width) bias = load_bias(p, at);
      }
      named_sync(1 + half, 128);  // the tile before has read its bias
      bias_h[ht] = bias;
      const int64_t row = (int64_t)tl.m0 + r;
      // this row's residual of one chunk of 32 columns, read a chunk ahead
      uint32_t res[16];
      auto load_residual = [&](int n) {
        if (p.residual && mine && n < p.width)
          load_cols(p.residual + (row * p.residual_ld + n) * 2, p.width - n, res32, res);
      };
      load_residual(nh);
      const bool ok = mbar_wait_suspend(acc_full, (uint32_t)(i & 1));
      tc_fence_after();
      const bool live = ok && !*((volatile int*)failed);
      if (named_sync_or(1 + half, 128, !live)) break;  // the four warps leave together
      uint32_t acc[kAcc];
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kAcc; k += 32)
        tmem_ld32(lane_base + (uint32_t)(kGlu ? k / kUp * (kN / 2) + half * kUp + k % kUp
                                              : half * kAcc + k),
                  acc + k);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) peer_signal(acc_empty0);
      if (!mine) continue;
      // One copy of the code for all chunks of 32 columns: the registers move down.
#pragma unroll 1
      for (int ch = 0; ch < kHalfN / 32; ++ch) {
        const int n = nh + 32 * ch, cols = p.width - n;
        if (cols <= 0) break;
        float v[32], u[kGlu ? 32 : 1];
        auto add_bias = [&](const uint32_t* a, const float* b, float* z) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 w = *reinterpret_cast<const float4*>(b + j);
            add2(F2(__uint_as_float(a[j]), __uint_as_float(a[j + 1])), F2(w.x, w.y)).get(z[j], z[j + 1]);
            add2(F2(__uint_as_float(a[j + 2]), __uint_as_float(a[j + 3])), F2(w.z, w.w)).get(z[j + 2], z[j + 3]);
          }
        };
        add_bias(acc, bias_h + 32 * ch, v);
        if constexpr (kGlu) {
          add_bias(acc + kUp, bias_h + kUp + 32 * ch, u);
#pragma unroll
          for (int j = 0; j + 32 < kUp; ++j) {
            acc[j] = acc[32 + j];
            acc[kUp + j] = acc[kUp + 32 + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j + 32 < kAcc; ++j) acc[j] = acc[32 + j];
        }
        uint32_t w[16];
        if (p.pre) {
          uint8_t* out = p.pre + (row * p.pre_ld + n) * 2;
          pack32(v, w);
          store_cols(out, cols, pre32, w);
          if constexpr (kGlu) {
            pack32(u, w);
            store_cols(out + (int64_t)p.width * 2, cols, pre32, w);
          }
        }
        if constexpr (kGlu) {
          act_each<MXB_ACT_SILU>(v);
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            mul2(F2(v[j], v[j + 1]), F2(u[j], u[j + 1])).get(v[j], v[j + 1]);
        } else {
          act_each<kAct>(v);
        }
        if (p.residual) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            v[2 * j] += bf16lo_to_f(res[j]);
            v[2 * j + 1] += bf16hi_to_f(res[j]);
          }
          if (ch + 1 < kHalfN / 32) load_residual(n + 32);
        }
        pack32(v, w);
        if (p.c) store_cols(p.c + (row * p.c_ld + n) * 2, cols, c32, w);
        if (p.c_codes) {
          uint32_t q[4], byte;
          quant_block32<true>(w, QuantParams{1e-10f, -6.0f, 6.0f}, q, byte);
          *reinterpret_cast<uint4*>(p.c_codes + (row * p.width + n) / 2) =
              make_uint4(q[0], q[1], q[2], q[3]);
          p.c_scales[(row * p.width + n) / 32] = (uint8_t)byte;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' products and copies have completed
  if (warp == 1) tmem_dealloc_pair(tmem, kTmemCols);
  __syncwarp();
  cluster_sync();
}

// ---------------------------------------------------------------- narrow
// The weights are the MMA's M side (kBlocks 128-row boxes: one, or gate and up)
// and the kT rows its N side.  The CTAs of a cluster take consecutive ranges of
// K; CTA r of the cluster owns the result columns n0 + r * 128 / size ...: every
// CTA writes its partial accumulators into the owners' shared memory, and each
// owner sums its columns over the ranks in order and runs the epilogue on them.
//   warp 0       TMA of the weights' and rows' codes, the weights' scale atoms
//   warp 1       MMA issue into one of two accumulators
//   warps 2-5    accumulator -> owners, then sum + epilogue of the own columns
//   warps 6, 7   the rows' scale bytes
constexpr int kNarrowThreads = 256;

template <bool kGlu, int kT>
struct Narrow {
  static constexpr int kBlocks = kGlu ? 2 : 1;
  static constexpr uint32_t kStage =
      kBlocks * (kBoxBytes + kAtoms) + (uint32_t)kT * 128 + kAtoms;
  static constexpr uint32_t kPart = kBlocks * kT * 128 * 4;  // partial sums, all ranks
  static constexpr size_t kFixed = 1024 + kPart + 2 * 1024 + kGroupTableInts * 4 + 512;
  static constexpr int kMost = (int)((227 * 1024 - kFixed) / kStage);
  // Four stages: 128 rows over 32 experts of 4096 x 7168 take 77 us with 3 or 4, 81
  // with the 5 that fit, and one row of 7168 x 2048 8.5 us with 4, 8.8 with 9.
  static constexpr int kStages = kMost > 4 ? 4 : kMost;
  // More than half of an SM's shared memory: two CTAs that own tensor memory never share
  // an SM.  (The second would wait in its allocation, and two clusters that each got one
  // of two SMs' tensor memory would wait for each other.)
  static constexpr size_t kNeeded = kFixed + kStages * kStage;
  static constexpr size_t kSmem = kNeeded < 116 * 1024 ? 116 * 1024 : kNeeded;
  static constexpr uint32_t kScaleCols = kBlocks * 8 + 8;
  static_assert(kStages >= 3 && 2 * kBlocks * kT <= 256 && 256 + kStages * kScaleCols <= kTmemCols,
                "the ring and tensor memory fit");
};

template <bool kGlu, int kT>
__global__ void __launch_bounds__(kNarrowThreads, 1) grouped_narrow_kernel(
    const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
    const __grid_constant__ GroupedArgs p) {
  using L = Narrow<kGlu, kT>;
  constexpr int kBlocks = L::kBlocks, kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  float* part = reinterpret_cast<float*>(smem + kStages * L::kStage);
  uint8_t* row_bytes = reinterpret_cast<uint8_t*>(part + L::kPart / 4);  // 1 KB a scale warp
  uint64_t* full = reinterpret_cast<uint64_t*>(row_bytes + 2 * 1024);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;    // [2]
  uint64_t* part_full = acc_empty + 2;
  uint64_t* part_empty = part_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_empty + 1);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  GroupTable g;
  g.off = failed + 1;
  g.tile = g.off + p.E + 1;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int ntn = (p.width + 127) / 128;
  const int ksteps = (p.K + kStepK - 1) / kStepK;
  const int k_begin = (int)((int64_t)ksteps * rank / ranks);
  const int k_end = (int)((int64_t)ksteps * (rank + 1) / ranks);
  const int S = p.K / 32, S4 = (S + 3) / 4;

  if (warp == 0) {
    wait_for_previous_kernel();
    build_groups(g, p.m_splits, p.E, p.M, [&](int rows) { return (rows + kT - 1) / kT * ntn; });
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  } else if (t == 64) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1 + (kT + 31) / 32);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    mbar_init(part_full, ranks);
    mbar_init(part_empty, ranks);
    fence_mbar_init();
    *failed = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_sync();  // every CTA's barriers are ready for its peers
  allow_next_kernel();  // every CTA of this one has its tensor memory
  wait_for_previous_kernel();
  const uint32_t tmem = *tmem_slot;
  const int tiles = g.tile[p.E];
  const int cluster = (int)(blockIdx.x / ranks), clusters = (int)(gridDim.x / ranks);
  const int my_tiles = cluster < tiles ? (tiles - 1 - cluster) / clusters + 1 : 0;

  struct Tile {
    int e, m0, n0;
  };
  // row blocks fastest: the tiles that read the same weights run side by side
  auto tile_at = [&](int i) {
    const int id = cluster + i * clusters;
    Tile r;
    r.e = find_group(g.tile, p.E, id);
    const int local = id - g.tile[r.e];
    const int ntm = (g.tile[r.e + 1] - g.tile[r.e]) / ntn;
    r.m0 = g.off[r.e] + local % ntm * kT;
    r.n0 = local / ntm * 128;
    return r;
  };

  if (warp == 0) {
    // ------------------------------------------------ TMA producer
    if (lane == 0) {
      int issued = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile tl = tile_at(i);
        for (int ks = k_begin; ks < k_end; ++ks) {
          const int gs = issued, s = gs % kStages;
          if (gs >= kStages && !mbar_wait_suspend(&empty[s], (uint32_t)((gs / kStages - 1) & 1))) {
            atomicExch(failed, 1);
            ok = false;
            break;
          }
          uint8_t* st = smem + s * L::kStage;
          uint8_t* sf = st + kBlocks * kBoxBytes + kT * 128;
          const uint32_t atoms = (uint32_t)min(2, S4 - 2 * ks) * 512;
          mbar_arrive_expect_tx(&full[s], kBlocks * (kBoxBytes + atoms) + kT * 128);
          const int kx = ks * (kStepK / 2);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            tma_load_2d(st + b * kBoxBytes, &map_b, kx, (kBlocks * tl.e + b) * p.width + tl.n0,
                        &full[s]);
            bulk_load_1d(sf + b * kAtoms,
                         p.b_scales +
                             ((int64_t)((kBlocks * tl.e + b) * ntn + tl.n0 / 128) * S4 + 2 * ks) * 512,
                         atoms, &full[s]);
          }
          tma_load_2d(st + kBlocks * kBoxBytes, &map_a, kx, tl.m0, &full[s]);
          issued = gs + 1;
        }
      }
      // do not leave while copies of this CTA are still landing
      for (int gs = issued > kStages ? issued - kStages : 0; gs < issued; ++gs)
        mbar_wait_suspend(&full[gs % kStages], (uint32_t)((gs / kStages) & 1));
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer
    {
      const bool one = elect_one();
      bool ok = true;
      int gs = 0;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int buf = i & 1;
        if (i > 1 && !mbar_wait_suspend(&acc_empty[buf], (uint32_t)((i / 2 - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int ks = k_begin; ks < k_end; ++ks, ++gs) {
          const int s = gs % kStages;
          if (!mbar_wait_suspend(&full[s], (uint32_t)((gs / kStages) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          __syncwarp();
          const uint8_t* st = smem + s * L::kStage;
          const uint8_t* sf = st + kBlocks * kBoxBytes + kT * 128;
          const uint32_t sfw = tmem + kScaleCol + (uint32_t)s * L::kScaleCols;
          const uint32_t sfr = sfw + kBlocks * 8;
          const int left = p.K - ks * kStepK;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            if (128 * a >= left) break;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
              tc_copy_sf(sfw + 8 * b + 4 * a, smem_desc_sf(sf + b * kAtoms + a * 512), one);
            tc_copy_sf(sfr + 4 * a, smem_desc_sf(sf + kBlocks * kAtoms + a * 512), one);
          }
          const uint64_t dr = smem_desc_sw128(st + kBlocks * kBoxBytes);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (64 * j >= left) break;
            const uint32_t sf_id = (uint32_t)(j & 1) * 2u;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
              tc_mma(tmem + (uint32_t)((buf * kBlocks + b) * kT),
                     smem_desc_sw128(st + b * kBoxBytes) + (uint64_t)(2 * j),
                     dr + (uint64_t)(2 * j), mxf4_idesc(128, kT, sf_id),
                     (sfw + 8 * b + 4 * (j >> 1)) | (sf_id << 30),
                     (sfr + 4 * (j >> 1)) | (sf_id << 30), (ks > k_begin || j > 0) ? 1u : 0u, one);
          }
          tc_commit(&empty[s], one);
        }
        __syncwarp();
        tc_commit(&acc_full[buf], one);
      }
      if (!ok) atomicExch(failed, 1);
    }
  } else if (warp < 6) {
    // ------------------------------------------------ exchange and epilogue
    const int quad = warp & 3, et = t - 64;
    const int cols = 128 / (int)ranks;  // result columns of an owner
    const int n_acc = quad * 32 + lane;
    const uint32_t to = peer_addr(smem_addr(part), (uint32_t)(n_acc / cols)) +
                        (uint32_t)(((int)rank * kBlocks * kT * cols + n_acc % cols) * 4);
    for (int i = 0; i < my_tiles; ++i) {
      const Tile tl = tile_at(i);
      const int rows = min(kT, g.off[tl.e + 1] - tl.m0);
      const int buf = i & 1;
      bool ok = mbar_wait_suspend(&acc_full[buf], (uint32_t)((i / 2) & 1));
      // every owner has summed tile i - 1 (alone, this CTA's barrier below says so)
      if (i > 0 && ranks > 1) ok = mbar_wait_cluster(part_empty, (uint32_t)((i - 1) & 1)) && ok;
      tc_fence_after();
      if (!ok) atomicExch(failed, 1);
      __syncwarp();
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int c = 0; c < kT; c += 16) {
          uint32_t acc[16];
          tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)((buf * kBlocks + b) * kT + c),
                    acc);
          tmem_ld_wait();
          if (ranks == 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              part[(b * kT + c + j) * 128 + n_acc] = __uint_as_float(acc[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              peer_store(to + (uint32_t)((b * kT + c + j) * cols * 4), __uint_as_float(acc[j]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
      if (ranks > 1) {
        named_sync(1, 128);
        if (et < (int)ranks) {
          fence_cluster();
          peer_arrive(peer_addr(smem_addr(part_full), (uint32_t)et));
        }
        __syncwarp();
        ok = mbar_wait_cluster(part_full, (uint32_t)(i & 1));
        if (!ok) atomicExch(failed, 1);
      }
      // a wait that gave up ends the tiles of this CTA; its peers give up in turn
      if (named_sync_or(1, 128, !ok || *((volatile int*)failed))) break;
      {
        const int per_row = cols / 8;
        for (int x = et; x < kT * per_row; x += 128) {
          const int tr = x / per_row, c8 = x % per_row * 8;
          const int n = tl.n0 + (int)rank * cols + c8;
          float v[8], u[kGlu ? 8 : 1];
          const bool in = tr < rows && n < p.width;
          if (in) {
            auto sum = [&](int b, float* z) {
              const float* src = part + (b * kT + tr) * cols + c8;
#pragma unroll
              for (int k = 0; k < 8; ++k) z[k] = 0.0f;
              for (int q = 0; q < (int)ranks; ++q, src += kBlocks * kT * cols) {
                const float4 lo = *reinterpret_cast<const float4*>(src);
                const float4 hi = *reinterpret_cast<const float4*>(src + 4);
                z[0] += lo.x; z[1] += lo.y; z[2] += lo.z; z[3] += lo.w;
                z[4] += hi.x; z[5] += hi.y; z[6] += hi.z; z[7] += hi.w;
              }
              if (p.bias) {
                const int64_t at = (int64_t)(kBlocks * tl.e + b) * p.width + n;
#pragma unroll
                for (int k = 0; k < 8; ++k) z[k] += load_bias(p, at + k);
              }
            };
            const int64_t row = (int64_t)tl.m0 + tr;
            sum(0, v);
            if (p.pre)
              *reinterpret_cast<uint4*>(p.pre + (row * p.pre_ld + n) * 2) = pack8_bf16(v);
            if constexpr (kGlu) {
              sum(1, u);
              if (p.pre)
                *reinterpret_cast<uint4*>(p.pre + (row * p.pre_ld + p.width + n) * 2) =
                    pack8_bf16(u);
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = act_value<MXB_ACT_SILU>(v[k]) * u[k];
            } else {
              act_apply(p.act, v);
            }
            if (p.residual)
              add8_bf16(v, *reinterpret_cast<const uint4*>(p.residual + (row * p.residual_ld + n) * 2));
            if (p.c) *reinterpret_cast<uint4*>(p.c + (row * p.c_ld + n) * 2) = pack8_bf16(v);
          }
          if (p.c_codes)
            quant_quad(p.c_codes, p.c_scales, v, in, ((int64_t)tl.m0 + tr) * p.width + n);
        }
      }
      // the partial sums have been read
      named_sync(1, 128);
      if (ranks > 1 && et < (int)ranks) {
        fence_cluster();
        peer_arrive(peer_addr(smem_addr(part_empty), (uint32_t)et));
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------ the rows' scale bytes
    if ((warp - 6) * 32 < kT) {
      // The bytes of four steps are gathered through a scratch of this warp into
      // registers, a row a thread.
      const bool words = scale_words(p);
      uint8_t* scratch = row_bytes + (warp - 6) * 1024;
      uint4 next[2];
      auto fetch = [&](const Tile& tl, int ks) {
        const int64_t row0 = (int64_t)tl.m0 + (warp - 6) * 32;
        __syncwarp();
        gather_scales(scratch, p.a_scales + row0 * p.a_spitch, p.a_spitch,
                      (int)max((int64_t)0, min((int64_t)min(32, kT - (warp - 6) * 32), p.M - row0)),
                      ks * 8, S, words);
        __syncwarp();
        next[0] = *reinterpret_cast<const uint4*>(scratch + lane * 32);
        next[1] = *reinterpret_cast<const uint4*>(scratch + lane * 32 + 16);
      };
      int gs = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile tl = tile_at(i);
        for (int ks0 = k_begin; ok && ks0 < k_end; ks0 += 4) {
          fetch(tl, ks0);
          const uint32_t now[8] = {next[0].x, next[0].y, next[0].z, next[0].w,
                                   next[1].x, next[1].y, next[1].z, next[1].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (ks0 + j >= k_end) break;
            const int s = gs % kStages;
            if (gs >= kStages && !mbar_wait_suspend(&empty[s], (uint32_t)((gs / kStages - 1) & 1))) {
              atomicExch(failed, 1);
              ok = false;
              break;
            }
            uint8_t* sf = smem + s * L::kStage + kBlocks * (kBoxBytes + kAtoms) + kT * 128 +
                          lane * 16 + (warp - 6) * 4;
            *reinterpret_cast<uint32_t*>(sf) = now[2 * j];
            *reinterpret_cast<uint32_t*>(sf + 512) = now[2 * j + 1];
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[s]);
            ++gs;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
  __syncwarp();
  cluster_sync();  // no peer still writes to, or arrives in, this CTA's shared memory
}

// ---------------------------------------------------------------- scales
// One thread per 4-byte word (4 scales of a row) of the tiled layout.
__global__ void __launch_bounds__(256) swizzle_grouped_kernel(const uint8_t* __restrict__ scales,
                                                              int64_t ranges, int64_t rows, int S,
                                                              uint32_t* __restrict__ out) {
  const int64_t rb = (rows + 127) / 128, S4 = (S + 3) / 4;
  const int64_t words = ranges * rb * 128 * S4;
  for (int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x; w < words;
       w += (int64_t)gridDim.x * 256) {
    // word w of the output: atom (range, row block, column of atoms), lane row, quarter
    const int in_atom = (int)(w & 127);
    const int64_t atom = w >> 7, c4 = atom % S4, block = atom / S4;
    const int64_t range = block / rb, r = block % rb * 128 + (in_atom & 3) * 32 + (in_atom >> 2);
    uint32_t v = 0;
    if (r < rows) {
      const uint8_t* src = scales + (range * rows + r) * S + c4 * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c4 * 4 + i < S) v |= (uint32_t)src[i] << (8 * i);
    }
    out[w] = v;
  }
}

// ---------------------------------------------------------------- host side
// Which kernel, and how.  rows: row-tile height (256 = wide); ranks: CTAs that
// split K.
struct Plan {
  int rows, ranks;
  int64_t tiles;  // upper bound over all splits
  int n = 0;      // wide: weight rows of a tile
};

int64_t most_tiles(int64_t M, int64_t E, int rows, int64_t ntn) {
  const int64_t groups = std::min(E, M);  // groups with a row
  return (groups + (M - groups) / rows) * ntn;
}

// Few rows an expert (the weights' bytes are the time): narrow.  Else the least of three
// estimates in tenths of a microsecond, each a start with the last tile's epilogue, so
// much a K step, and a further round of tiles at the longer of its steps and an
// epilogue; at least the weights' bytes at the rate each reaches.  They order the variants
// and are no prediction: epilogue operands and rows that start inside a sector are not in
// them (3001 rows over 16 experts of 1416 x 2080 with bias and gelu_tanh: 16.3 against 24.2
// us measured).  The coefficients were read off products without epilogue operands of 40 to
// 8192 rows, e.g. (us, narrow / 128 / 256 weight rows a tile): 200 x 1024 x 256 7.9 / 6.3 / 8.5; 300 x 3600 x 4096 13.3 / 9.6 / 13.1;
// 130 x 512 x 7168, where narrow splits K eight ways, 8.8 / 11.2 / 16.0;
// 1500 x 2048 x 2048 19.4 / 10.5 / 12.0; 2000 x 4096 x 4096 43.9 / 23.9 / 21.5;
// 1500 rows over 32 experts of 4096 x 7168 96 / 132 / 103.
Plan grouped_plan(const GroupedArgs& p, bool glu) {
  const int sms = sm_count(), pairs = std::max(1, sms / 2);
  const int64_t ksteps = cdiv(p.K, kStepK), cols = (int64_t)p.width * (glu ? 2 : 1);
  const int64_t groups = std::min<int64_t>(p.E, p.M);  // experts with rows, at most
  // row blocks of an even split
  auto blocks = [&](int rows) {
    return p.E == 1 ? cdiv(p.M, rows) : std::max(groups, p.M / rows + cdiv(groups, 2));
  };
  Plan r{p.M <= 8 * (int64_t)p.E ? 16 : 64, 1, 0};
  r.tiles = most_tiles(p.M, p.E, r.rows, cdiv(p.width, 128));
  const int most = p.c_codes ? 4 : 8;  // a quantized block of 32 columns has one owner
  while (r.ranks < most && r.tiles * r.ranks * 2 <= sms && ksteps >= r.ranks * 4) r.ranks *= 2;
  if (p.M <= 32 * (int64_t)p.E) {
    // long tiles in a few rounds: half tiles fill the last round better (128 rows over
    // 32 experts of 4096 x 7168: 82 -> 77 us)
    if (r.ranks == 1 && ksteps >= 16 && r.tiles <= 8 * sms) r.ranks = 2;
    return r;
  }
  // start, rounds, a step's cost in hundredths, a round's least
  auto estimate = [&](int64_t start, int64_t rounds, int64_t steps, int64_t step, int64_t least) {
    const int64_t tile = steps * step / 10;
    return start + tile + (rounds - 1) * std::max(least, tile + 5);
  };
  const int64_t weights = groups * cols * p.K * 17 / 32;
  const int64_t narrow =
      std::max(estimate(r.ranks > 1 ? 85 : 70, cdiv(blocks(64) * cdiv(p.width, 128) * r.ranks, sms),
                        cdiv(ksteps, r.ranks), glu ? 56 : 35, 35),
               weights / 580000);
  // rows of scales that TMA cannot take cost a little more a step
  const int64_t wide128 = std::max(estimate(60, cdiv(blocks(256) * cdiv(cols, 128), pairs), ksteps,
                                            p.a_scales_tma ? 21 : 26, 22),
                                   weights / 490000);
  const int64_t wide256 = std::max(estimate(85, cdiv(blocks(256) * cdiv(cols, 256), pairs), ksteps,
                                            p.a_scales_tma ? 31 : 35, 47),
                                   weights / 490000);
  if (narrow <= std::min(wide128, wide256)) return r;
  const int n = wide128 < wide256 ? 128 : 256;
  return Plan{256, 1, most_tiles(p.M, p.E, 256, cdiv(cols, n)), n};
}

// Persistent clusters, which share the tiles: pairs of CTAs (wide), or those that split K.
int64_t clusters_of(const Plan& plan) {
  return std::min<int64_t>(plan.tiles, std::max(1, sm_count() / (plan.n ? 2 : plan.ranks)));
}

template <int kAct, int kN, bool kLines>
mxb_status launch_wide_n(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ts,
                         const GroupedArgs& p, const Plan& plan, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  const auto kernel = grouped_wide_kernel<kAct, kN, kLines>;
  MXB_REQUIRE(grant_smem((const void*)kernel, kWideSmem, done), MXB_ERR_CUDA,
              "grouped_gemm_mxfp4: cannot reserve shared memory");
  return launch_cluster("grouped_gemm_mxfp4", kernel,
                        (unsigned)clusters_of(plan), 2, kWideThreads, kWideSmem, s, ta, tb, ts, p);
}
template <int kAct>
mxb_status launch_wide(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ts,
                       const GroupedArgs& p, const Plan& plan, cudaStream_t s) {
  if (p.a_scales_tma)
    return plan.n == 128 ? launch_wide_n<kAct, 128, false>(ta, tb, ts, p, plan, s)
                         : launch_wide_n<kAct, 256, false>(ta, tb, ts, p, plan, s);
  return plan.n == 128 ? launch_wide_n<kAct, 128, true>(ta, tb, ts, p, plan, s)
                       : launch_wide_n<kAct, 256, true>(ta, tb, ts, p, plan, s);
}

template <bool kGlu, int kT>
mxb_status launch_narrow(const CUtensorMap& ta, const CUtensorMap& tb, const GroupedArgs& p,
                         const Plan& plan, cudaStream_t s) {
  using L = Narrow<kGlu, kT>;
  static std::atomic<uint64_t> done{0};
  MXB_REQUIRE(grant_smem((const void*)grouped_narrow_kernel<kGlu, kT>, L::kSmem, done),
              MXB_ERR_CUDA, "grouped_gemm_mxfp4: cannot reserve shared memory");
  return launch_cluster("grouped_gemm_mxfp4", grouped_narrow_kernel<kGlu, kT>,
                        (unsigned)clusters_of(plan), (unsigned)plan.ranks, kNarrowThreads, L::kSmem,
                        s, ta, tb, p);
}

}  // namespace
}  // namespace mxb

using namespace mxb;

extern "C" mxb_status mxb_swizzle_scales_grouped(const void* scales, int64_t E, int64_t N,
                                                 int64_t S, int32_t parts, void* out,
                                                 mxb_stream_t stream) {
  MXB_REQUIRE(E >= 0 && N >= 0 && S >= 0 && S <= INT32_MAX && (parts == 1 || parts == 2) &&
                  N % parts == 0,
              MXB_ERR_INVALID_ARGUMENT,
              "swizzle_scales_grouped: need parts 1 or 2 and N %% parts == 0 (N=%lld parts=%d)",
              (long long)N, parts);
  if (E == 0 || N == 0 || S == 0) return MXB_OK;
  MXB_REQUIRE(scales && out, MXB_ERR_INVALID_ARGUMENT, "swizzle_scales_grouped: null pointer");
  MXB_REQUIRE(aligned(out, 16), MXB_ERR_MISALIGNED,
              "swizzle_scales_grouped: out must be 16-byte aligned");
  const int64_t words = E * parts * cdiv(N / parts, 128) * 128 * cdiv(S, 4);
  swizzle_grouped_kernel<<<(unsigned)std::min<int64_t>(cdiv(words, 256), 16 * kSMs), 256, 0,
                           to_cuda(stream)>>>((const uint8_t*)scales, E * parts, N / parts, (int)S,
                                              (uint32_t*)out);
  return launch_status("swizzle_scales_grouped");
}

extern "C" mxb_status mxb_grouped_gemm_plan(int64_t M, int32_t E, int64_t N, int64_t K,
                                            int32_t activation, int32_t quantized,
                                            int32_t scale_rows_aligned, int64_t plan[5]) {
  const bool glu = activation == MXB_ACT_SWIGLU;
  MXB_REQUIRE(plan && M >= 1 && M <= INT32_MAX - 512 && E >= 1 && E <= MXB_MAX_EXPERTS && N >= 1 &&
                  N % (glu ? 16 : 8) == 0 && (int64_t)E * N <= INT32_MAX - 512 && K >= 32 &&
                  K % 32 == 0 && K <= (1 << 24) && activation >= MXB_ACT_NONE &&
                  activation <= MXB_ACT_SWIGLU,
              MXB_ERR_INVALID_ARGUMENT,
              "grouped_gemm_plan: need a plan and a call's sizes (M=%lld E=%d N=%lld K=%lld)",
              (long long)M, E, (long long)N, (long long)K);
  GroupedArgs p = {};
  p.M = M;
  p.E = E;
  p.width = (int)(N / (glu ? 2 : 1));
  p.K = (int)K;
  uint8_t some = 0;
  p.c_codes = quantized ? &some : nullptr;
  p.a_scales_tma = scale_rows_aligned != 0;
  const Plan r = grouped_plan(p, glu);
  const int64_t values[5] = {r.rows, r.n ? r.n : glu ? 256 : 128, r.ranks, r.tiles, clusters_of(r)};
  std::copy(values, values + 5, plan);
  return MXB_OK;
}

extern "C" mxb_status mxb_grouped_gemm_mxfp4(const void* a_codes, int64_t a_codes_pitch,
                                             const void* a_scales, int64_t a_scales_pitch,
                                             int64_t M, const int32_t* m_splits, int32_t E,
                                             const void* b_codes, const void* b_scales, int64_t N,
                                             int64_t K, const mxb_epilogue* ep, void* c,
                                             mxb_stream_t stream) {
  const char* const what = "grouped_gemm_mxfp4";
  MXB_REQUIRE(ep, MXB_ERR_INVALID_ARGUMENT, "%s: null epilogue", what);
  MXB_REQUIRE(ep->activation >= MXB_ACT_NONE && ep->activation <= MXB_ACT_SWIGLU,
              MXB_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, ep->activation);
  const bool glu = ep->activation == MXB_ACT_SWIGLU;
  const int64_t parts = glu ? 2 : 1;
  MXB_REQUIRE(M >= 0 && M <= INT32_MAX - 512 && E >= 1 && E <= MXB_MAX_EXPERTS, MXB_ERR_INVALID_ARGUMENT,
              "%s: need 0 <= M < 2^31 and 1 <= E <= %d (M=%lld E=%d)", what, MXB_MAX_EXPERTS,
              (long long)M, E);
  MXB_REQUIRE(N >= 0 && N % (8 * parts) == 0 && K >= 32 && K % 32 == 0 && K <= (1 << 24),
              MXB_ERR_INVALID_ARGUMENT,
              "%s: need N %% %d == 0, K %% 32 == 0 and 32 <= K <= 2^24 (N=%lld K=%lld)", what,
              (int)(8 * parts), (long long)N, (long long)K);
  MXB_REQUIRE((int64_t)E * N <= INT32_MAX - 512, MXB_ERR_INVALID_ARGUMENT,
              "%s: need E * N < 2^31 (E=%d N=%lld)", what, E, (long long)N);
  if (M == 0 || N == 0) return MXB_OK;
  const int64_t W = N / parts;
  MXB_REQUIRE(a_codes && a_scales && b_codes && b_scales && (m_splits || E == 1),
              MXB_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  MXB_REQUIRE(c || ep->pre || ep->c_codes, MXB_ERR_INVALID_ARGUMENT, "%s: no output", what);
  MXB_REQUIRE(!ep->c_codes == !ep->c_scales && (!ep->c_codes || W % 32 == 0),
              MXB_ERR_INVALID_ARGUMENT,
              "%s: a quantized result needs both c_codes and c_scales and a width %% 32 == 0", what);
  MXB_REQUIRE(a_codes_pitch >= K / 2 && a_scales_pitch >= K / 32 && (!c || ep->c_ld >= W) &&
                  (!ep->pre || ep->pre_ld >= N) && (!ep->residual || ep->residual_ld >= W),
              MXB_ERR_INVALID_ARGUMENT, "%s: a pitch does not cover its row", what);
  MXB_REQUIRE(aligned(a_codes, 16) && a_codes_pitch % 16 == 0 && aligned(b_codes, 16) &&
                  aligned(b_scales, 16) && aligned(c, 16) && aligned(ep->pre, 16) &&
                  aligned(ep->residual, 16) && aligned(ep->c_codes, 16),
              MXB_ERR_MISALIGNED, "%s: operands must be 16-byte aligned", what);
  MXB_REQUIRE((!c || ep->c_ld % 8 == 0) && (!ep->pre || ep->pre_ld % 8 == 0) &&
                  (!ep->residual || ep->residual_ld % 8 == 0),
              MXB_ERR_MISALIGNED, "%s: pitches of c, pre and residual must be multiples of 8", what);
  MXB_REQUIRE(!ep->bias || aligned(ep->bias, ep->bias_f32 ? 4 : 2), MXB_ERR_MISALIGNED,
              "%s: bias is not aligned to its elements", what);

  GroupedArgs p;
  p.a_scales = (const uint8_t*)a_scales;
  p.a_spitch = a_scales_pitch;
  p.b_scales = (const uint8_t*)b_scales;
  p.m_splits = m_splits;
  p.M = M;
  p.E = E;
  p.width = (int)W;
  p.K = (int)K;
  p.act = ep->activation;
  p.bias = ep->bias;
  p.bias_f32 = ep->bias_f32;
  p.residual = (const uint8_t*)ep->residual;
  p.residual_ld = ep->residual_ld;
  p.pre = (uint8_t*)ep->pre;
  p.pre_ld = ep->pre_ld;
  p.c = (uint8_t*)c;
  p.c_ld = ep->c_ld;
  p.c_codes = (uint8_t*)ep->c_codes;
  p.c_scales = (uint8_t*)ep->c_scales;
  p.a_scales_tma = aligned(a_scales, 16) && a_scales_pitch % 16 == 0;
  const Plan plan = grouped_plan(p, glu);
  MXB_REQUIRE(plan.tiles <= INT32_MAX, MXB_ERR_INVALID_ARGUMENT, "%s: too many tiles", what);

  const cudaStream_t s = to_cuda(stream);
  CUtensorMap ta, tb;
  if (!make_tensor_map_2d(&ta, a_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, M, K / 2, a_codes_pitch,
                          128, (uint32_t)std::min(plan.rows, 128), CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&tb, b_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (int64_t)E * N, K / 2,
                          K / 2, 128, plan.n == 128 ? 64 : 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return MXB_ERR_CUDA;
  if (plan.rows == 16)
    return glu ? launch_narrow<true, 16>(ta, tb, p, plan, s)
               : launch_narrow<false, 16>(ta, tb, p, plan, s);
  if (plan.rows == 64)
    return glu ? launch_narrow<true, 64>(ta, tb, p, plan, s)
               : launch_narrow<false, 64>(ta, tb, p, plan, s);
  CUtensorMap ts = ta;
  if (p.a_scales_tma && !make_tensor_map_2d(&ts, a_scales, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, M,
                                            K / 32, a_scales_pitch, 32, 128))
    return MXB_ERR_CUDA;
  switch (p.act) {
    case MXB_ACT_RELU: return launch_wide<MXB_ACT_RELU>(ta, tb, ts, p, plan, s);
    case MXB_ACT_RELU2: return launch_wide<MXB_ACT_RELU2>(ta, tb, ts, p, plan, s);
    case MXB_ACT_SILU: return launch_wide<MXB_ACT_SILU>(ta, tb, ts, p, plan, s);
    case MXB_ACT_GELU: return launch_wide<MXB_ACT_GELU>(ta, tb, ts, p, plan, s);
    case MXB_ACT_GELU_TANH: return launch_wide<MXB_ACT_GELU_TANH>(ta, tb, ts, p, plan, s);
    case MXB_ACT_SWIGLU: return launch_wide<MXB_ACT_SWIGLU>(ta, tb, ts, p, plan, s);
    default: return launch_wide<MXB_ACT_NONE>(ta, tb, ts, p, plan, s);
  }
}
