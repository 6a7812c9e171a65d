// Epilogue arithmetic of the MXFP4 matrix products: the activations, their
// derivatives and packing helpers.  Everything is evaluated in f32 on the f32
// accumulator; the only rounding is the one to BF16 when a result is written.
//
//   relu       max(z, 0)                       relu2      max(z, 0)^2
//   silu       z * s(z), s(z) = 1 / (1 + e^-z)
//   gelu       z * (1 + erf(z / sqrt 2)) / 2
//   gelu_tanh  z * s(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3): the tanh form
//              written with the logistic function, (1 + tanh u) / 2 = s(2 u)
//   swiglu     silu(gate) * up, gate and up from two halves of the columns
//
// The logistic function uses the hardware exponential and reciprocal (about
// 2^-22 relative), which a BF16 result cannot tell from exact.
#pragma once
#include <cstdint>

#include "common.cuh"
#include "mxfp4_b200.h"
#include "qrow.cuh"

namespace mxb {

__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float logistic(float z) { return rcp_approx(1.0f + __expf(-z)); }

constexpr float kSqrt2OverPi = 0.7978845608028654f;
constexpr float kGeluCubic = 0.044715f;
constexpr float kInvSqrt2 = 0.7071067811865476f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

template <int kAct>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (kAct == MXB_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if constexpr (kAct == MXB_ACT_RELU2) return z > 0.0f ? z * z : (z != z ? z : 0.0f);
  if constexpr (kAct == MXB_ACT_SILU) return z * logistic(z);
  if constexpr (kAct == MXB_ACT_GELU) return 0.5f * z * (1.0f + erff(z * kInvSqrt2));
  if constexpr (kAct == MXB_ACT_GELU_TANH)
    return z * logistic(2.0f * kSqrt2OverPi * (z + kGeluCubic * z * z * z));
  return z;
}

// d act / d z
template <int kAct>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (kAct == MXB_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if constexpr (kAct == MXB_ACT_RELU2) return z > 0.0f ? 2.0f * z : 0.0f;
  if constexpr (kAct == MXB_ACT_SILU) {
    const float s = logistic(z);
    return s * (1.0f + z * (1.0f - s));
  }
  if constexpr (kAct == MXB_ACT_GELU)
    return 0.5f * (1.0f + erff(z * kInvSqrt2)) + z * kInvSqrt2Pi * __expf(-0.5f * z * z);
  if constexpr (kAct == MXB_ACT_GELU_TANH) {
    const float s = logistic(2.0f * kSqrt2OverPi * (z + kGeluCubic * z * z * z));
    return s + z * s * (1.0f - s) * 2.0f * kSqrt2OverPi * (1.0f + 3.0f * kGeluCubic * z * z);
  }
  return 1.0f;
}

// One activation over n values held in registers; the branch is uniform.
template <int kAct, int n>
__device__ __forceinline__ void act_each(float (&v)[n]) {
#pragma unroll
  for (int i = 0; i < n; ++i) v[i] = act_value<kAct>(v[i]);
}
template <int n>
__device__ __forceinline__ void act_apply(int act, float (&v)[n]) {
  switch (act) {
    case MXB_ACT_RELU: act_each<MXB_ACT_RELU>(v); break;
    case MXB_ACT_RELU2: act_each<MXB_ACT_RELU2>(v); break;
    case MXB_ACT_SILU: act_each<MXB_ACT_SILU>(v); break;
    case MXB_ACT_GELU: act_each<MXB_ACT_GELU>(v); break;
    case MXB_ACT_GELU_TANH: act_each<MXB_ACT_GELU_TANH>(v); break;
    default: break;
  }
}

__device__ __forceinline__ uint4 pack8_bf16(const float* v) {
  return make_uint4(cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3]), cvt_bf16x2(v[4], v[5]),
                    cvt_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void add8_bf16(float* v, uint4 r) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] += bf16lo_to_f(w[i]);
    v[2 * i + 1] += bf16hi_to_f(w[i]);
  }
}
__device__ __forceinline__ void unpack8_bf16(uint4 r, float* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16lo_to_f(w[i]);
    v[2 * i + 1] = bf16hi_to_f(w[i]);
  }
}

// The rowwise MXFP4 of 32 columns held by four neighbouring lanes, eight
// each (a lane without a row takes part in the shuffles only).
__device__ __forceinline__ void quant_quad(uint8_t* codes, uint8_t* scales, const float* v, bool in,
                                           int64_t at) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if (in) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = cvt_bf16x2(v[2 * k], v[2 * k + 1]);
  }
  uint32_t all[16];
  const int quad0 = (threadIdx.x & 31) & ~3;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) all[4 * q + k] = __shfl_sync(0xffffffffu, w[k], quad0 + q);
  if (!in) return;
  uint32_t out[4], byte;
  quant_block32<true>(all, QuantParams{1e-10f, -6.0f, 6.0f}, out, byte);
  const int q = threadIdx.x & 3;
  *reinterpret_cast<uint32_t*>(codes + at / 2) = q == 0 ? out[0] : q == 1 ? out[1] : q == 2 ? out[2] : out[3];
  if (q == 0) scales[at / 32] = (uint8_t)byte;
}

}  // namespace mxb
