// The streaming operators around the experts' products (sm_100a):
//   * bias_act_grad: dz = dy * act'(pre), the rowwise MXFP4 of dz for the input
//     gradient's product, and the bias gradient, in one pass over dy and pre;
//   * moe_unpermute: the weighted sum of each token's expert rows;
//   * moe_unpermute_grad: its gradient towards the rows and the weights.
// All are bound by HBM: every operand is read once in 16-byte pieces, with
// several rows' loads in flight per thread.
#include <cuda_bf16.h>

#include <algorithm>

#include "capi_util.h"
#include "common.cuh"
#include "epilogue.cuh"
#include "groups.cuh"
#include "host_util.h"
#include "umma.cuh"

namespace mxb {
namespace {

// ---------------------------------------------------------------- bias_act_grad
// A CTA takes up to 128 rows of one expert by 256 columns of dy: a warp a row, a
// lane eight columns.  Column sums stay in registers over a
// warp's rows, meet in shared memory in warp order, and leave as one partial sum
// per CTA; a second kernel adds an expert's partials in row order, so the bias
// gradient does not depend on scheduling.  Up to 512 rows one kernel does it: a cluster
// of up to eight CTAs has an expert's rows, 64 each, and CTA 0 adds the CTAs' sums in
// order (333 x 1024: 10.5 us with two kernels and 128 rows a CTA, 6.0 with 32, 5.8
// with one; a launch and a workspace less on the host, 10.4 -> 5.8 us a call).
constexpr int kGradThreads = 256, kGradWarps = 8, kGradCols = 256;
constexpr int kGradClusterRows = 64, kGradMaxCluster = 8;

// CTAs of a cluster that has all rows of an expert; 0: too many rows for one.
int grad_cluster(int64_t M) {
  if (M > kGradClusterRows * kGradMaxCluster) return 0;
  int n = 1;
  while (n * kGradClusterRows < M) n *= 2;
  return n;
}
// Rows of a CTA without clusters: fewer where 128 would leave SMs without work.
int grad_rows(int64_t M, int64_t N) {
  return (M / 128) * cdiv(N, kGradCols) >= 2 * kSMs ? 128 : 32;
}
__device__ __forceinline__ int grad_chunks(int rows, int per) {
  return rows > per ? (rows + per - 1) / per : 1;
}
int64_t most_grad_chunks(int64_t M, int64_t E, int per) { return M / per + E; }

struct ActGradArgs {
  const uint8_t *dy, *pre;
  const int32_t* m_splits;
  int64_t M;
  int E, N, width, per, cluster;  // per: rows of a CTA; cluster: CTAs of one, or 0
  uint8_t *dz, *codes, *scales;
  float* sums;  // [chunks, N] partials, or (clusters) dbias; NULL: no bias gradient
};

// Bytes in flight come from many warps with few rows each: swiglu 16384 x 8192 took
// 148 us with four rows a thread and one CTA per SM, 128 with two and two, 119 with
// one row and four CTAs; gelu of the same size 253, 167 and (two rows, four CTAs) 143.
template <int kAct, bool kQuant>
__global__ void __launch_bounds__(kGradThreads, kQuant ? 2 : 4)
    act_grad_kernel(const ActGradArgs p, int slabs) {
  constexpr bool kGlu = kAct == MXB_ACT_SWIGLU;
  constexpr int kParts = kGlu ? 2 : 1;
  __shared__ int32_t table[kGroupTableInts];
  __shared__ float red[kParts][kGradWarps][kGradCols];
  extern __shared__ float all[];  // clusters, CTA 0's: every CTA's sums [cluster][kParts][kGradCols]
  const GroupTable g{table, table + p.E + 1};
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  wait_for_previous_kernel();
  if (warp == 0)
    build_groups(g, p.m_splits, p.E, p.M, [&](int rows) { return grad_chunks(rows, p.per); });
  __syncthreads();
  int e, slab, r0, rank = 0;
  int64_t out_row;
  if (p.cluster) {
    cluster_sync();  // CTA 0's shared memory can be written
    const int id = (int)(blockIdx.x / p.cluster);
    rank = (int)(blockIdx.x % p.cluster);
    e = id / slabs;
    slab = id % slabs;
    r0 = g.off[e] + rank * p.per;
    out_row = e;
  } else {
    const int chunk = (int)(blockIdx.x / slabs);
    if (chunk >= g.tile[p.E]) return;
    slab = (int)(blockIdx.x % slabs);
    e = find_group(g.tile, p.E, chunk);
    r0 = g.off[e] + (chunk - g.tile[e]) * p.per;
    out_row = chunk;
  }
  const int r1 = min(r0 + p.per, g.off[e + 1]);
  const int n = slab * kGradCols + lane * 8;
  const bool in = n < p.width;
  float sum[kParts][8] = {};
  constexpr int kRows = kGlu ? 1 : 2;
  for (int r = r0 + warp; r < r1; r += kGradWarps * kRows) {
    uint4 d[kRows], z[kParts][kRows];
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int64_t row = r + q * kGradWarps;
      if (in && row < r1) {
        d[q] = ld_stream_v4(p.dy + (row * p.width + n) * 2);
        if (kAct != MXB_ACT_NONE) {
#pragma unroll
          for (int h = 0; h < kParts; ++h)
            z[h][q] = ld_stream_v4(p.pre + (row * p.N + h * p.width + n) * 2);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int64_t row = r + q * kGradWarps;
      if (row >= r1) break;  // the same for the whole warp
      float dv[8], o[kParts][8];
      if (in) {
        unpack8_bf16(d[q], dv);
        if constexpr (kGlu) {
          float a[8], b[8];
          unpack8_bf16(z[0][q], a);
          unpack8_bf16(z[1][q], b);
          F2 g[4], s[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) g[k] = F2(a[2 * k], a[2 * k + 1]);
          logistic_pairs<4>(g, s);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const F2 d2(dv[2 * k], dv[2 * k + 1]), gs = mul2(g[k], s[k]);
            const F2 slope = fma2(gs, fma2(s[k], both(-1.0f), both(1.0f)), s[k]);
            mul2(mul2(d2, F2(b[2 * k], b[2 * k + 1])), slope).get(o[0][2 * k], o[0][2 * k + 1]);
            mul2(d2, gs).get(o[1][2 * k], o[1][2 * k + 1]);
          }
        } else {
          float a[8] = {}, s[8];
          if (kAct != MXB_ACT_NONE) unpack8_bf16(z[0][q], a);
          slope8<kAct>(a, s);
#pragma unroll
          for (int k = 0; k < 8; ++k) o[0][k] = dv[k] * s[k];
        }
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
#pragma unroll
          for (int k = 0; k < 8; ++k) sum[h][k] += o[h][k];
          if (p.dz)
            *reinterpret_cast<uint4*>(p.dz + (row * p.N + h * p.width + n) * 2) = pack8_bf16(o[h]);
        }
      }
      if constexpr (kQuant) {
#pragma unroll
        for (int h = 0; h < kParts; ++h)
          quant_quad(p.codes, p.scales, o[h], in, row * p.N + h * p.width + n);
      }
    }
  }
  if (!p.sums) return;
#pragma unroll
  for (int h = 0; h < kParts; ++h)
#pragma unroll
    for (int k = 0; k < 8; ++k) red[h][warp][lane * 8 + k] = sum[h][k];
  __syncthreads();
  const int col = slab * kGradCols + t;
  float total[kParts];
#pragma unroll
  for (int h = 0; h < kParts; ++h) {
    total[h] = 0.0f;
#pragma unroll
    for (int w = 0; w < kGradWarps; ++w) total[h] += red[h][w][t];
  }
  if (p.cluster > 1) {
#pragma unroll
    for (int h = 0; h < kParts; ++h)
      peer_store(peer_addr(smem_addr(&all[(rank * kParts + h) * kGradCols + t]), 0), total[h]);
    cluster_sync();
    if (rank > 0) return;
#pragma unroll
    for (int h = 0; h < kParts; ++h) {
      total[h] = 0.0f;
      for (int q = 0; q < p.cluster; ++q) total[h] += all[(q * kParts + h) * kGradCols + t];
    }
  }
  if (col < p.width) {
#pragma unroll
    for (int h = 0; h < kParts; ++h) p.sums[out_row * p.N + h * p.width + col] = total[h];
  }
}

// dbias[e][n] = the sum of expert e's partials: 32 columns a CTA, eight warps
// taking every eighth partial, added in warp order.
__global__ void __launch_bounds__(kGradThreads) bias_sum_kernel(const float* __restrict__ partial,
                                                                const int32_t* m_splits, int64_t M,
                                                                int E, int N, int per,
                                                                float* __restrict__ dbias) {
  __shared__ int32_t table[kGroupTableInts];
  __shared__ float red[kGradWarps][32];
  const GroupTable g{table, table + E + 1};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) build_groups(g, m_splits, E, M, [&](int rows) { return grad_chunks(rows, per); });
  __syncthreads();
  const int e = blockIdx.y, n = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (n < N) {
    const int end = g.tile[e + 1];
#pragma unroll 4
    for (int c = g.tile[e] + warp; c < end; c += kGradWarps) s += partial[(int64_t)c * N + n];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && n < N) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kGradWarps; ++w) total += red[w][lane];
    dbias[(int64_t)e * N + n] = total;
  }
}

template <int kAct>
mxb_status launch_act_grad(const ActGradArgs& p, int64_t blocks, int slabs, cudaStream_t s) {
  const auto kernel = p.codes ? act_grad_kernel<kAct, true> : act_grad_kernel<kAct, false>;
  if (p.cluster)
    return launch_cluster("bias_act_grad", kernel, (unsigned)blocks, (unsigned)p.cluster,
                          kGradThreads,
                          (size_t)p.cluster * (kAct == MXB_ACT_SWIGLU ? 2 : 1) * kGradCols * 4, s, p,
                          slabs);
  kernel<<<(unsigned)blocks, kGradThreads, 0, s>>>(p, slabs);
  return launch_status("bias_act_grad");
}

// ---------------------------------------------------------------- unpermute
// A thread owns eight columns of a token and has its rows' loads, eight at a
// time, in flight together; the sum runs over k in order, in f32.
constexpr int kUnpThreads = 256;
constexpr int kUnpBatch = 8;

struct UnpermuteMap {
  const int32_t* map;
  int64_t pitch;
  const float* weight;
  int topk;
  int64_t R;
  // row of (t, k), or -1
  __device__ __forceinline__ int64_t row(int64_t t, int k) const {
    const int32_t r = map[t * pitch + k];
    return r >= 0 && r < R ? r : -1;
  }
  __device__ __forceinline__ float w(int64_t t, int k) const {
    return weight ? weight[t * topk + k] : 1.0f;
  }
};

__global__ void __launch_bounds__(kUnpThreads, 4) unpermute_kernel(const uint8_t* __restrict__ y,
                                                                const UnpermuteMap m, int64_t T,
                                                                int64_t H,
                                                                uint8_t* __restrict__ out) {
  const int64_t per_row = H / 8, items = T * per_row;
  for (int64_t i = (int64_t)blockIdx.x * kUnpThreads + threadIdx.x; i < items;
       i += (int64_t)gridDim.x * kUnpThreads) {
    const int64_t t = i / per_row, c = i % per_row;
    float acc[8] = {};
    for (int k0 = 0; k0 < m.topk; k0 += kUnpBatch) {
      uint4 v[kUnpBatch];
      float w[kUnpBatch];
      bool there[kUnpBatch];
#pragma unroll
      for (int k = 0; k < kUnpBatch; ++k) {
        const int64_t r = k0 + k < m.topk ? m.row(t, k0 + k) : -1;
        there[k] = r >= 0;
        if (there[k]) {
          v[k] = ld_stream_v4(y + (r * H + c * 8) * 2);
          w[k] = m.w(t, k0 + k);
        }
      }
#pragma unroll
      for (int k = 0; k < kUnpBatch; ++k) {
        if (!there[k]) continue;
        float x[8];
        unpack8_bf16(v[k], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += w[k] * x[j];
      }
    }
    *reinterpret_cast<uint4*>(out + (t * H + c * 8) * 2) = pack8_bf16(acc);
  }
}

// A warp per (token, k): the row's dot product is one sum over the lanes, in a fixed
// order, and the eight warps of a CTA read the same token's dout, mostly from L1.
// (4096 tokens x 8 rows x 7168: 164 us; a CTA per token with eight rows a thread 265.)
template <bool kQuant>
__global__ void __launch_bounds__(kUnpThreads, kQuant ? 2 : 6) unpermute_grad_kernel(
    const uint8_t* __restrict__ dout, const uint8_t* __restrict__ y, const UnpermuteMap m,
    int64_t T, int64_t H, uint8_t* __restrict__ dy, uint8_t* __restrict__ codes,
    uint8_t* __restrict__ scales, float* __restrict__ dweight) {
  constexpr int kUnroll = 2;
  const int lane = threadIdx.x & 31;
  const int64_t per_row = H / 8, items = T * m.topk;
  for (int64_t i = (int64_t)blockIdx.x * (kUnpThreads / 32) + (threadIdx.x >> 5); i < items;
       i += (int64_t)gridDim.x * (kUnpThreads / 32)) {
    const int64_t t = i / m.topk;
    const int k = (int)(i % m.topk);
    const int64_t row = m.row(t, k);
    if (row < 0) {
      if (dweight && lane == 0) dweight[i] = 0.0f;
      continue;
    }
    const float w = m.w(t, k);
    const uint8_t* dt = dout + t * H * 2;
    float dot = 0.0f;
    for (int64_t c0 = 0; c0 < per_row; c0 += 32 * kUnroll) {
      uint4 d[kUnroll], v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t c = c0 + 32 * u + lane;
        if (c < per_row) {
          d[u] = __ldg(reinterpret_cast<const uint4*>(dt + c * 16));
          if (dweight) v[u] = ld_stream_v4(y + (row * H + c * 8) * 2);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (c0 + 32 * u >= per_row) break;  // the same for the whole warp
        const int64_t c = c0 + 32 * u + lane;
        const bool in = c < per_row;
        float dv[8] = {};
        if (in) unpack8_bf16(d[u], dv);
        if (dweight && in) {
          float x[8];
          unpack8_bf16(v[u], x);
#pragma unroll
          for (int j = 0; j < 8; ++j) dot += dv[j] * x[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) dv[j] *= w;
        if (dy && in) *reinterpret_cast<uint4*>(dy + (row * H + c * 8) * 2) = pack8_bf16(dv);
        if constexpr (kQuant) quant_quad(codes, scales, dv, in, row * H + c * 8);
      }
    }
    if (dweight) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
      if (lane == 0) dweight[i] = dot;
    }
  }
}

mxb_status check_unpermute(const char* what, int64_t R, int64_t H, int64_t map_pitch, int32_t topk,
                           int64_t T) {
  MXB_REQUIRE(T >= 0 && R >= 0 && R <= INT32_MAX && H >= 0 && H % 8 == 0, MXB_ERR_INVALID_ARGUMENT,
              "%s: need T >= 0, 0 <= R < 2^31 and H %% 8 == 0 (T=%lld R=%lld H=%lld)", what,
              (long long)T, (long long)R, (long long)H);
  MXB_REQUIRE(topk >= 1 && topk <= 1024 && map_pitch >= topk, MXB_ERR_INVALID_ARGUMENT,
              "%s: need 1 <= topk <= 1024 and map_pitch >= topk (topk=%d map_pitch=%lld)", what,
              topk, (long long)map_pitch);
  return MXB_OK;
}

}  // namespace
}  // namespace mxb

using namespace mxb;

extern "C" int64_t mxb_bias_act_grad_workspace(int64_t M, int32_t E, int64_t N) {
  if (grad_cluster(M) || E < 1 || N < 1) return 0;
  return most_grad_chunks(M, E, grad_rows(M, N)) * N * 4;
}

extern "C" mxb_status mxb_bias_act_grad(const void* dy, const void* pre, int64_t M,
                                        const int32_t* m_splits, int32_t E, int64_t N,
                                        int32_t activation, void* dz, void* dz_codes,
                                        void* dz_scales, float* dbias, void* workspace,
                                        int64_t workspace_bytes, mxb_stream_t stream) {
  const char* const what = "bias_act_grad";
  MXB_REQUIRE(activation >= MXB_ACT_NONE && activation <= MXB_ACT_SWIGLU, MXB_ERR_INVALID_ARGUMENT,
              "%s: unknown activation %d", what, activation);
  const int parts = activation == MXB_ACT_SWIGLU ? 2 : 1;
  MXB_REQUIRE(M >= 0 && M <= INT32_MAX - 512 && E >= 1 && E <= MXB_MAX_EXPERTS, MXB_ERR_INVALID_ARGUMENT,
              "%s: need 0 <= M < 2^31 and 1 <= E <= %d (M=%lld E=%d)", what, MXB_MAX_EXPERTS,
              (long long)M, E);
  MXB_REQUIRE(N >= 0 && N <= INT32_MAX - 512 && N % (8 * parts) == 0, MXB_ERR_INVALID_ARGUMENT,
              "%s: need N %% %d == 0 (N=%lld)", what, 8 * parts, (long long)N);
  MXB_REQUIRE(!dz_codes == !dz_scales && (!dz_codes || N % (32 * parts) == 0),
              MXB_ERR_INVALID_ARGUMENT,
              "%s: a quantized dz needs both dz_codes and dz_scales and N %% %d == 0", what,
              32 * parts);
  if (N == 0) return MXB_OK;
  MXB_REQUIRE(m_splits || E == 1, MXB_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  MXB_REQUIRE(dz || dz_codes || dbias, MXB_ERR_INVALID_ARGUMENT, "%s: no output", what);
  const cudaStream_t s = to_cuda(stream);
  if (M == 0) {
    if (dbias && cudaMemsetAsync(dbias, 0, (size_t)E * N * 4, s) != cudaSuccess)
      return launch_status(what);
    return MXB_OK;
  }
  MXB_REQUIRE(dy && (pre || activation == MXB_ACT_NONE), MXB_ERR_INVALID_ARGUMENT,
              "%s: null pointer", what);
  MXB_REQUIRE(aligned(dy, 16) && aligned(pre, 16) && aligned(dz, 16) && aligned(dz_codes, 16) &&
                  aligned(dbias, 4) && aligned(workspace, 16),
              MXB_ERR_MISALIGNED, "%s: operands must be 16-byte aligned", what);
  const int64_t need = dbias ? mxb_bias_act_grad_workspace(M, E, N) : 0;
  MXB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MXB_ERR_INVALID_ARGUMENT,
              "%s: workspace of %lld bytes needed, %lld given", what, (long long)need,
              (long long)workspace_bytes);
  ActGradArgs p;
  p.dy = (const uint8_t*)dy;
  p.pre = (const uint8_t*)pre;
  p.m_splits = m_splits;
  p.M = M;
  p.E = E;
  p.N = (int)N;
  p.width = (int)(N / parts);
  p.cluster = grad_cluster(M);
  p.per = p.cluster ? kGradClusterRows : grad_rows(M, N);
  p.dz = (uint8_t*)dz;
  p.codes = (uint8_t*)dz_codes;
  p.scales = (uint8_t*)dz_scales;
  p.sums = !dbias ? nullptr : need ? (float*)workspace : dbias;
  const int slabs = (int)cdiv(p.width, kGradCols);
  const int64_t blocks = (p.cluster ? (int64_t)E : most_grad_chunks(M, E, p.per)) * slabs;
  MXB_REQUIRE(blocks * kGradMaxCluster <= INT32_MAX, MXB_ERR_INVALID_ARGUMENT,
              "%s: too many blocks", what);
  mxb_status st;
  switch (activation) {
    case MXB_ACT_NONE: st = launch_act_grad<MXB_ACT_NONE>(p, blocks, slabs, s); break;
    case MXB_ACT_RELU: st = launch_act_grad<MXB_ACT_RELU>(p, blocks, slabs, s); break;
    case MXB_ACT_RELU2: st = launch_act_grad<MXB_ACT_RELU2>(p, blocks, slabs, s); break;
    case MXB_ACT_SILU: st = launch_act_grad<MXB_ACT_SILU>(p, blocks, slabs, s); break;
    case MXB_ACT_GELU: st = launch_act_grad<MXB_ACT_GELU>(p, blocks, slabs, s); break;
    case MXB_ACT_GELU_TANH: st = launch_act_grad<MXB_ACT_GELU_TANH>(p, blocks, slabs, s); break;
    default: st = launch_act_grad<MXB_ACT_SWIGLU>(p, blocks, slabs, s); break;
  }
  if (st != MXB_OK || !need) return st;
  bias_sum_kernel<<<dim3((unsigned)cdiv(N, 32), (unsigned)E), kGradThreads, 0, s>>>(
      (const float*)workspace, m_splits, M, E, (int)N, p.per, dbias);
  return launch_status(what);
}

extern "C" mxb_status mxb_moe_unpermute(const void* y, int64_t R, int64_t H, const int32_t* map,
                                        int64_t map_pitch, int32_t topk, const float* weight,
                                        int64_t T, void* out, mxb_stream_t stream) {
  const char* const what = "moe_unpermute";
  const mxb_status st = check_unpermute(what, R, H, map_pitch, topk, T);
  if (st != MXB_OK) return st;
  if (T == 0 || H == 0) return MXB_OK;
  MXB_REQUIRE((y || R == 0) && map && out, MXB_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  MXB_REQUIRE(aligned(y, 16) && aligned(out, 16) && aligned(map, 4) && aligned(weight, 4),
              MXB_ERR_MISALIGNED, "%s: y and out must be 16-byte aligned", what);
  const UnpermuteMap m{map, map_pitch, weight, topk, R};
  const int64_t blocks = std::min<int64_t>(cdiv(T * (H / 8), kUnpThreads), INT32_MAX);
  unpermute_kernel<<<(unsigned)blocks, kUnpThreads, 0, to_cuda(stream)>>>((const uint8_t*)y, m, T,
                                                                          H, (uint8_t*)out);
  return launch_status(what);
}

extern "C" mxb_status mxb_moe_unpermute_grad(const void* dout, const void* y, int64_t R, int64_t H,
                                             const int32_t* map, int64_t map_pitch, int32_t topk,
                                             const float* weight, int64_t T, void* dy,
                                             void* dy_codes, void* dy_scales, float* dweight,
                                             mxb_stream_t stream) {
  const char* const what = "moe_unpermute_grad";
  const mxb_status st = check_unpermute(what, R, H, map_pitch, topk, T);
  if (st != MXB_OK) return st;
  MXB_REQUIRE(!dy_codes == !dy_scales && (!dy_codes || H % 32 == 0), MXB_ERR_INVALID_ARGUMENT,
              "%s: a quantized dy needs both dy_codes and dy_scales and H %% 32 == 0", what);
  MXB_REQUIRE(dy || dy_codes || dweight, MXB_ERR_INVALID_ARGUMENT, "%s: no output", what);
  if (T == 0) return MXB_OK;
  MXB_REQUIRE((dout || H == 0) && map && (y || !dweight || R == 0 || H == 0),
              MXB_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  MXB_REQUIRE(aligned(dout, 16) && aligned(y, 16) && aligned(dy, 16) && aligned(dy_codes, 16) &&
                  aligned(map, 4) && aligned(weight, 4) && aligned(dweight, 4),
              MXB_ERR_MISALIGNED, "%s: operands must be 16-byte aligned", what);
  const UnpermuteMap m{map, map_pitch, weight, topk, R};
  const auto kernel = dy_codes ? unpermute_grad_kernel<true> : unpermute_grad_kernel<false>;
  kernel<<<(unsigned)std::min<int64_t>(cdiv(T * topk, kUnpThreads / 32), INT32_MAX), kUnpThreads, 0,
           to_cuda(stream)>>>((const uint8_t*)dout, (const uint8_t*)y, m, T, H, (uint8_t*)dy,
                              (uint8_t*)dy_codes, (uint8_t*)dy_scales, dweight);
  return launch_status(what);
}
