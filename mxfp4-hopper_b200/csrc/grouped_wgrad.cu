// The experts' weight gradients (sm_100a): dw[e][n, k] = sum over the rows r of
// expert e of dy[r, n] * x[r, k], dy in BF16 as autograd hands it over, x the
// MXFP4 rows saved by the forward pass.
//
// The contraction runs over rows, the outer dimension of both operands, so both
// are MN-major for the tensor core and neither is transposed in memory.  An
// E2M1 value times 2^(e - 127) is exact in BF16: eight warps expand x's codes
// into a BF16 tile in shared memory while the tensor core works on the tiles
// before, and the product is kind::f16 (BF16 x BF16 -> f32).  Two CTAs share a
// tile (cta_group::2) of 256 columns of dy, the M side, 128 loaded by each, by 256
// columns of x, 128 expanded by each, 64 rows a step: every byte of dy and x
// crosses L2 -> shared memory once per 256 columns of the other.  A warp of the
// epilogue then has 32 rows of dw and writes (or adds) them 128 bytes of a row at a
// time by TMA from a staging box of its own: whole lines, clipped to the expert.
// (With rows as columns of the accumulator a BF16 dw left in 64-byte pieces: 1650 us
// instead of 490 for 32 experts of 4096 x 7168 with 4096 rows.)
//
// Ragged groups: a step's rows past its expert's end are expanded as zeros, and
// the same rows of dy (the next expert's, whatever they hold) are overwritten
// with zeros in shared memory, so that an infinity or NaN there cannot reach
// this expert's sums.
#include <cuda_bf16.h>

#include <algorithm>

#include "capi_util.h"
#include "common.cuh"
#include "groups.cuh"
#include "host_util.h"
#include "tma.cuh"
#include "umma.cuh"

namespace mxb {
namespace {

constexpr int kWgThreads = 448;  // TMA, MMA, 4 epilogue warps, 8 expanding warps
constexpr int kWgStages = 5;
constexpr int kWgRows = 64;                 // rows per step
constexpr int kTileX = 256, kTileY = 256;   // columns of x and of dy, half in each CTA
constexpr uint32_t kWgBox = kWgRows * 128;  // 64 rows x 64 bf16 columns
constexpr uint32_t kWgX = 2 * kWgBox, kWgStage = 2 * kWgX;
constexpr uint32_t kWgOut = 2 * 32 * 128;   // two boxes of an epilogue warp: 32 rows of 128 bytes
constexpr size_t kWgSmem = 1024 + kWgStages * kWgStage + 4 * kWgOut + kGroupTableInts * 4 + 256;
static_assert(kWgSmem <= 227 * 1024, "one CTA per SM");

struct WgradArgs {
  const uint8_t* x_codes;
  int64_t x_pitch;
  const uint8_t* x_scales;
  int64_t s_pitch;
  const int32_t* m_splits;
  int64_t M;
  int E, N, K;
  int accumulate;
};

// 32 codes (16 bytes) and their E8M0 byte -> 32 BF16 values in element order.
// The eight magnitudes times 2^(e - 127) are made first and split into tables of low
// and high bytes, which prmt looks up for four codes at a time.  The factor's BF16
// pattern is e << 7, for e = 0 the subnormal 0x40 (BF16 multiplies take subnormals): the
// products are exact, past BF16's range infinite.  e = 255 is the E8M0 NaN.
__device__ __forceinline__ void expand32(uint4 codes, uint32_t e, uint32_t (&out)[16]) {
  const uint32_t f = (e == 255u ? 0x7FFFu : max(e << 7, 0x40u)) * 0x10001u;
  uint32_t m[4] = {0x3F000000u, 0x3FC03F80u, 0x40404000u, 0x40C04080u};  // 0 .5 | 1 1.5 | 2 3 | 4 6
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = mul_bf16x2(m[i], f);
  const uint32_t lo0 = prmt(m[0], m[1], 0x6420u), lo1 = prmt(m[2], m[3], 0x6420u);
  const uint32_t hi0 = prmt(m[0], m[1], 0x7531u), hi1 = prmt(m[2], m[3], 0x7531u);
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t mag = w[i] & 0x77777777u, neg = (w[i] >> 3) & 0x11111111u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = prmt(lo0, lo1, mag >> (16 * h));
      const uint32_t hi = prmt(hi0, hi1, mag >> (16 * h)) | prmt(0x00008000u, 0u, neg >> (16 * h));
      out[4 * i + 2 * h] = prmt(lo, hi, 0x5140u);
      out[4 * i + 2 * h + 1] = prmt(lo, hi, 0x7362u);
    }
  }
}

template <bool kF32>
__global__ void __launch_bounds__(kWgThreads, 1) grouped_wgrad_kernel(
    const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_dw,
    const __grid_constant__ WgradArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* staging = smem + kWgStages * kWgStage;
  uint64_t* dy_full = reinterpret_cast<uint64_t*>(staging + 4 * kWgOut);
  uint64_t* full = dy_full + kWgStages;  // CTA 0's: both CTAs' halves are in place
  uint64_t* empty = full + kWgStages;
  uint64_t* acc_full = empty + kWgStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2], CTA 0's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  GroupTable g;
  g.off = failed + 1;
  g.tile = g.off + p.E + 1;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int nty = (p.N + kTileY - 1) / kTileY, ntx = (p.K + kTileX - 1) / kTileX;
  const int per_expert = nty * ntx;
  const int rank = (int)cluster_rank();

  if (warp == 0) {
    wait_for_previous_kernel();
    build_groups(g, p.m_splits, p.E, p.M, [&](int) { return 0; });
  } else if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
  } else if (t == 64) {
    for (int s = 0; s < kWgStages; ++s) {
      mbar_init(&dy_full[s], 1);
      mbar_init(&full[s], 4);  // a pair of warps in each CTA
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
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
  const int tiles = p.E * per_expert;
  const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  const int my_tiles = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0;

  struct Tile {
    int e, x0, y0, row0, rows, steps;  // x0, y0: the pair's first columns of x and dy
  };
  auto tile_at = [&](int i) {
    const int id = pair + i * pairs;
    Tile r;
    r.e = id / per_expert;
    const int local = id % per_expert;
    r.x0 = local / nty * kTileX;
    r.y0 = local % nty * kTileY;
    r.row0 = g.off[r.e];
    r.rows = g.off[r.e + 1] - r.row0;
    r.steps = (r.rows + kWgRows - 1) / kWgRows;
    return r;
  };

  if (warp == 0) {
    // ------------------------------------------------ TMA producer
    if (lane == 0) {
      int gs = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const Tile tl = tile_at(i);
        for (int st = 0; st < tl.steps; ++st) {
          const int s = gs % kWgStages;
          if (gs >= kWgStages && !mbar_wait_suspend(&empty[s], (uint32_t)((gs / kWgStages - 1) & 1))) {
            atomicExch(failed, 1);
            ok = false;
            break;
          }
          // both boxes, also past dy's last column (zeros): the wait has one form
          mbar_arrive_expect_tx(&dy_full[s], 2 * kWgBox);
#pragma unroll
          for (int b = 0; b < 2; ++b)
            tma_load_2d(smem + s * kWgStage + kWgX + b * kWgBox, &map_dy,
                        tl.y0 + rank * (kTileY / 2) + 64 * b, tl.row0 + st * kWgRows, &dy_full[s]);
          ++gs;
        }
      }
      // do not leave while copies of this CTA are still landing
      for (int q = gs > kWgStages ? gs - kWgStages : 0; q < gs; ++q)
        mbar_wait_suspend(&dy_full[q % kWgStages], (uint32_t)((q / kWgStages) & 1));
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer
    if (rank == 0) {
      const bool one = elect_one();
      bool ok = true, ready = false;
      int gs = 0;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int buf = i & 1, steps = tile_at(i).steps;
        if (i > 1 && !mbar_wait_suspend(&acc_empty[buf], (uint32_t)((i / 2 - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int st = 0; st < steps; ++st, ++gs) {
          const int s = gs % kWgStages;
          if (!ready && !mbar_wait_suspend(&full[s], (uint32_t)((gs / kWgStages) & 1))) {
            ok = false;
            break;
          }
          // whether the next step is ready as well: known by the time it is needed
          ready = mbar_peek(&full[(gs + 1) % kWgStages], (uint32_t)(((gs + 1) / kWgStages) & 1));
          tc_fence_after();
          __syncwarp();
          const uint64_t dx = smem_desc_mn_sw128(smem + s * kWgStage, kWgBox);
          const uint64_t dyd = smem_desc_mn_sw128(smem + s * kWgStage + kWgX, kWgBox);
#pragma unroll
          for (int j = 0; j < kWgRows / 16; ++j)  // 16 rows of 128 bytes further each
            tc_mma_bf16_pair(tmem + (uint32_t)(buf * kTileX), dyd + (uint64_t)(128 * j),
                             dx + (uint64_t)(128 * j), bf16_mn_idesc(kTileY, kTileX),
                             (st > 0 || j > 0) ? 1u : 0u, one);
          tc_commit_pair(&empty[s], one);
        }
        __syncwarp();
        tc_commit_pair(&acc_full[buf], one);
      }
      if (!ok) atomicExch(failed, 1);
    }
  } else if (warp < 6) {
    // ------------------------------------------------ epilogue: lane = column of dy
    const int quad = warp & 3;
    const uint32_t acc_empty0 = peer_addr(smem_addr(acc_empty), 0);
    uint8_t* boxes = staging + quad * kWgOut;
    int turn = 0;
    constexpr int kCols = kF32 ? 32 : 64;  // 128 bytes of a row
    for (int i = 0; i < my_tiles; ++i) {
      const Tile tl = tile_at(i);
      const int buf = i & 1;
      const bool ok = mbar_wait_suspend(&acc_full[buf], (uint32_t)((i / 2) & 1));
      tc_fence_after();
      if (named_sync_or(1, 128, !ok || *((volatile int*)failed))) break;
      const int n0 = tl.y0 + rank * (kTileY / 2) + quad * 32;  // this warp's first row of dw
      const bool store = n0 < p.N && (tl.steps > 0 || !p.accumulate);
#pragma unroll 1
      for (int c = 0; store && c < kTileX && tl.x0 + c < p.K; c += kCols) {
        uint32_t w[32];
        __syncwarp();
        if constexpr (kF32) {
          tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * kTileX + c), w);
          tmem_ld_wait();
        } else {
          uint32_t acc[64];
          tmem_ld64(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * kTileX + c), acc);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            w[j] = cvt_bf16x2(__uint_as_float(acc[2 * j]), __uint_as_float(acc[2 * j + 1]));
        }
        if (tl.steps == 0) {
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = 0u;
        }
        bulk_wait_read_1();  // the store before the last, of this box, has read it
        __syncwarp();
        uint8_t* box = boxes + turn * (kWgOut / 2);
        turn ^= 1;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
              make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (kF32 && p.accumulate)
          tma_store_3d<true>(&map_dw, tl.x0 + c, n0, tl.e, box, lane == 0);
        else
          tma_store_3d<false>(&map_dw, tl.x0 + c, n0, tl.e, box, lane == 0);
        bulk_commit();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) peer_signal(acc_empty0 + 8 * buf);
    }
    bulk_wait_all();
  } else {
    // ------------------------------------------------ x: MXFP4 -> BF16 tile
    // Four pairs of warps take every fourth step each: expanding one is a chain of
    // about a thousand cycles (wait, decode, shared memory, proxy fence, signal), which
    // bound the kernel when all eight warps worked on the same step.  Warp w of a pair
    // has rows 32w .. 32w + 31; lane (b, r) the block of 32 columns b of rows r, r + 8,
    // ...: 64 contiguous code bytes a row, and eight lanes of a 16-byte store phase in
    // eight different rows, whose swizzled chunks are distinct.  The codes of the
    // pair's next step are in flight in registers.
    const int first = (warp - 6) >> 1, b = lane >> 3;
    const int r0 = ((warp - 6) & 1) * 32 + (lane & 7);
    const uint32_t full0 = peer_addr(smem_addr(full), 0);
    const int64_t c8 = 8 * p.x_pitch, s8 = 8 * p.s_pitch;
    int i = -1, left = 0;  // tile; its rows from this pair's step on
    const uint8_t *cp = nullptr, *sp = nullptr;  // this lane's codes and scale in row r0 of the step
    bool in_k = false;
    // moves n steps on; false when there are no more
    auto move = [&](int n) {
      left -= n * kWgRows;
      if (left > 0) {
        cp += n * 8 * c8;
        sp += n * 8 * s8;
        return true;
      }
      // steps past this tile's last one are the next tiles' first ones
      int over = -left / kWgRows;
      Tile tl;
      for (;;) {
        if (++i >= my_tiles) return false;
        tl = tile_at(i);
        if (over < tl.steps) break;
        over -= tl.steps;
      }
      left = tl.rows - over * kWgRows;
      const int64_t row = (int64_t)tl.row0 + over * kWgRows + r0;
      const int k = tl.x0 + rank * (kTileX / 2) + 32 * b;
      in_k = k < p.K;
      cp = p.x_codes + row * p.x_pitch + k / 2;
      sp = p.x_scales + row * p.s_pitch + k / 32;
      return true;
    };
    uint4 codes[4];
    uint32_t scale[4];
    auto load = [&] {
      if (left >= kWgRows && in_k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          codes[j] = __ldg(reinterpret_cast<const uint4*>(cp + j * c8));
          scale[j] = __ldg(sp + j * s8);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          codes[j] = make_uint4(0u, 0u, 0u, 0u);
          scale[j] = 127u;
          if (r0 + 8 * j < left && in_k) {
            codes[j] = __ldg(reinterpret_cast<const uint4*>(cp + j * c8));
            scale[j] = __ldg(sp + j * s8);
          }
        }
      }
    };
    // where this lane's 16-byte chunks go: its rows are the same modulo 8
    uint32_t chunk[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      chunk[q] = (uint32_t)((b >> 1) * kWgBox + r0 * 128 + ((((b & 1) * 4 + q) ^ (r0 & 7)) << 4));
    bool more = move(first);
    if (more) load();
    for (int gs = first; more; gs += 4) {
      const int s = gs % kWgStages;
      uint8_t* stage = smem + s * kWgStage;
      const int here = left;  // rows of the expert from this step on
      if (gs >= kWgStages && !mbar_wait_suspend(&empty[s], (uint32_t)((gs / kWgStages - 1) & 1))) {
        atomicExch(failed, 1);
        break;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t v[16];
        expand32(codes[j], scale[j], v);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(stage + chunk[q] + j * 1024) =
              make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      }
      more = move(4);
      if (more) load();
      if (!mbar_wait_suspend(&dy_full[s], (uint32_t)((gs / kWgStages) & 1))) {
        atomicExch(failed, 1);
        break;
      }
      if (here < kWgRows) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = r0 + 8 * j;
          if (r >= here) {  // past the expert's last row: its four lanes clear dy's four half rows
            uint8_t* dyr = stage + kWgX + (b >> 1) * kWgBox + r * 128 + (b & 1) * 64;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(dyr + 16 * q) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) peer_signal(full0 + 8 * s);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' products and copies have completed
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
  __syncwarp();
  cluster_sync();
}

template <bool kF32>
mxb_status launch_wgrad(const CUtensorMap& map_dy, const CUtensorMap& map_dw, const WgradArgs& p,
                        cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  MXB_REQUIRE(grant_smem((const void*)grouped_wgrad_kernel<kF32>, kWgSmem, done), MXB_ERR_CUDA,
              "grouped_wgrad_mxfp4: cannot reserve shared memory");
  const int64_t tiles = (int64_t)p.E * cdiv(p.N, kTileY) * cdiv(p.K, kTileX);
  MXB_REQUIRE(tiles <= INT32_MAX, MXB_ERR_INVALID_ARGUMENT, "grouped_wgrad_mxfp4: too many tiles");
  return launch_cluster("grouped_wgrad_mxfp4", grouped_wgrad_kernel<kF32>,
                        (unsigned)std::min<int64_t>(tiles, std::max(1, sm_count() / 2)), 2,
                        kWgThreads, kWgSmem, s, map_dy, map_dw, p);
}

}  // namespace
}  // namespace mxb

using namespace mxb;

extern "C" mxb_status mxb_grouped_wgrad_mxfp4(const void* dy, int64_t dy_ld, const void* x_codes,
                                              int64_t x_codes_pitch, const void* x_scales,
                                              int64_t x_scales_pitch, int64_t M,
                                              const int32_t* m_splits, int32_t E, int64_t N,
                                              int64_t K, void* dw, int32_t dw_f32,
                                              int32_t accumulate, mxb_stream_t stream) {
  const char* const what = "grouped_wgrad_mxfp4";
  MXB_REQUIRE(M >= 0 && M <= INT32_MAX - 512 && E >= 1 && E <= MXB_MAX_EXPERTS, MXB_ERR_INVALID_ARGUMENT,
              "%s: need 0 <= M < 2^31 and 1 <= E <= %d (M=%lld E=%d)", what, MXB_MAX_EXPERTS,
              (long long)M, E);
  MXB_REQUIRE(N >= 0 && N <= INT32_MAX - 512 && N % 8 == 0 && K >= 0 && K <= INT32_MAX - 512 &&
                  K % 32 == 0,
              MXB_ERR_INVALID_ARGUMENT, "%s: need N %% 8 == 0 and K %% 32 == 0 (N=%lld K=%lld)",
              what, (long long)N, (long long)K);
  MXB_REQUIRE(!accumulate || dw_f32, MXB_ERR_UNSUPPORTED, "%s: only a float dw accumulates", what);
  if (N == 0 || K == 0) return MXB_OK;
  MXB_REQUIRE(dw && (m_splits || E == 1), MXB_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  MXB_REQUIRE(aligned(dw, 16), MXB_ERR_MISALIGNED, "%s: operands must be 16-byte aligned", what);
  if (M == 0) {  // no expert has rows
    if (!accumulate &&
        cudaMemsetAsync(dw, 0, (size_t)E * N * K * (dw_f32 ? 4 : 2), to_cuda(stream)) != cudaSuccess)
      return launch_status(what);
    return MXB_OK;
  }
  MXB_REQUIRE(dy && x_codes && x_scales, MXB_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  MXB_REQUIRE(dy_ld >= N && x_codes_pitch >= K / 2 && x_scales_pitch >= K / 32,
              MXB_ERR_INVALID_ARGUMENT, "%s: a pitch does not cover its row", what);
  MXB_REQUIRE(aligned(dy, 16) && dy_ld % 8 == 0 && aligned(x_codes, 16) && x_codes_pitch % 16 == 0,
              MXB_ERR_MISALIGNED, "%s: operands must be 16-byte aligned", what);
  CUtensorMap map, map_dw;
  if (!make_tensor_map_2d(&map, dy, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, M, N, dy_ld, 64, kWgRows,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_3d(&map_dw, dw,
                          dw_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          dw_f32 ? 4 : 2, E, N, K, dw_f32 ? 32 : 64, 32, CU_TENSOR_MAP_SWIZZLE_128B))
    return MXB_ERR_CUDA;
  WgradArgs p;
  p.x_codes = (const uint8_t*)x_codes;
  p.x_pitch = x_codes_pitch;
  p.x_scales = (const uint8_t*)x_scales;
  p.s_pitch = x_scales_pitch;
  p.m_splits = m_splits;
  p.M = M;
  p.E = E;
  p.N = (int)N;
  p.K = (int)K;
  p.accumulate = accumulate;
  return dw_f32 ? launch_wgrad<true>(map, map_dw, p, to_cuda(stream))
                : launch_wgrad<false>(map, map_dw, p, to_cuda(stream));
}
