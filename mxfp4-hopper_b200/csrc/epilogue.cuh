// Epilogue arithmetic of the MXFP4 matrix products: the activations, their
// derivatives and packing helpers.  Everything is evaluated in f32 on the f32
// accumulator; the only rounding is the one to BF16 when a result is written.
//
//   relu       max(z, 0)                       relu2      max(z, 0)^2
//   silu       z * s(z), s(z) = 1 / (1 + e^-z)
//   gelu       z * (1 + erf(z / sqrt 2)) / 2 = z (1 - q(z)) for z > 0, else z q(z),
//              q(z) = erfc(|z| / sqrt 2) / 2: no cancellation in the negative tail
//   gelu_tanh  z * s(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3): the tanh form
//              written with the logistic function, (1 + tanh u) / 2 = s(2 u)
//   swiglu     silu(gate) * up, gate and up from two halves of the columns
//
// The logistic function uses the hardware exponential and reciprocal: about 2^-22
// relative, and |z| 2^-23 more for the rounded exponent, which a BF16 result cannot tell
// from exact.  Below 2^-126 it is 0: silu is -0 for z < -87.3, where it should be
// at most 1.03e-36 in size.  q(z) is taken as t P(t) exp(-z^2 / 2) with t = 1 / (1 + 0.3 |z|)
// and P a polynomial of degree 7 fitted here to erfc in relative error (least squares on
// Chebyshev nodes of t, reweighted towards the minimax: 1.7e-7 for |z| <= 14 with the
// coefficients in f32; the exponent's rounding adds z^2 2^-24).  From |z| = 13.2 on
// the exponential is 0, and with it z q, which is below 2^-126 there.
// With erff, whose two ranges a warp both runs, the epilogue of an 8192^2 x 7168
// product took 14.7 thousand cycles a tile for the activation alone, longer than the
// tile's products.
#pragma once
#include <cstdint>

#include "common.cuh"
#include "mxfp4_b200.h"
#include "qrow.cuh"

namespace mxb {

__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float logistic(float z) {
  return rcp_approx(1.0f + ex2_approx(-kLog2e * z));
}

constexpr float kSqrt2OverPi = 0.7978845608028654f;
constexpr float kGeluCubic = 0.044715f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

// P of q(z), lowest coefficient first.
__host__ __device__ constexpr float tail_coeff(int c) {
  return c == 0   ? 0.11962930113077164f
         : c == 1 ? 0.12075395882129669f
         : c == 2 ? 0.09991348534822464f
         : c == 3 ? 0.12856164574623108f
         : c == 4 ? -0.05368367210030556f
         : c == 5 ? 0.20635353028774261f
         : c == 6 ? -0.15720310807228088f
                  : 0.03567477688193321f;
}

// One value of the activations that need no more than a few instructions.
template <int kAct>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (kAct == MXB_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if constexpr (kAct == MXB_ACT_RELU2) return z > 0.0f ? z * z : (z != z ? z : 0.0f);
  if constexpr (kAct == MXB_ACT_SILU) return z * logistic(z);
  return z;
}

// Two floats in a register pair, for the packed f32 instructions.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  }
  __device__ __forceinline__ void get(float& a, float& b) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  }
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 both(float x) { return F2(x, x); }

// logistic() of kP pairs.
template <int kP>
__device__ __forceinline__ void logistic_pairs(const F2 (&z)[kP], F2 (&s)[kP]) {
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    float a, b;
    mul2(z[i], both(-kLog2e)).get(a, b);
    s[i] = add2(F2(ex2_approx(a), ex2_approx(b)), both(1.0f));
  }
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    float a, b;
    s[i].get(a, b);
    s[i] = F2(rcp_approx(a), rcp_approx(b));
  }
}

// The factor of gelu for kP pairs: 1 - q(z) where z > 0, else q(z); and exp(-z^2 / 2).
template <int kP>
__device__ __forceinline__ void normal_cdf_pairs(const float* v, const F2 (&z)[kP], F2 (&cdf)[kP],
                                                 F2 (&gauss)[kP]) {
  F2 t[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    float a, b;
    fma2(F2(fabsf(v[2 * i]), fabsf(v[2 * i + 1])), both(0.3f), both(1.0f)).get(a, b);
    t[i] = F2(rcp_approx(a), rcp_approx(b));
  }
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    float a, b;
    mul2(mul2(z[i], z[i]), both(-0.5f * kLog2e)).get(a, b);
    gauss[i] = F2(ex2_approx(a), ex2_approx(b));
  }
#pragma unroll
  for (int i = 0; i < kP; ++i) cdf[i] = fma2(both(tail_coeff(7)), t[i], both(tail_coeff(6)));
#pragma unroll
  for (int c = 5; c >= 0; --c)
#pragma unroll
    for (int i = 0; i < kP; ++i) cdf[i] = fma2(cdf[i], t[i], both(tail_coeff(c)));
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const F2 q = mul2(mul2(cdf[i], t[i]), gauss[i]);
    float q0, q1, r0, r1;
    q.get(q0, q1);
    fma2(q, both(-1.0f), both(1.0f)).get(r0, r1);
    cdf[i] = F2(v[2 * i] > 0.0f ? r0 : q0, v[2 * i + 1] > 0.0f ? r1 : q1);
  }
}
// 2 u of gelu_tanh: 2 sqrt(2 / pi) (z + 0.044715 z^3).
__device__ __forceinline__ F2 tanh_arg(F2 z) {
  return mul2(fma2(mul2(z, both(kGeluCubic)), mul2(z, z), z), both(2.0f * kSqrt2OverPi));
}

// Eight values at a time, step by step and in pairs: a value alone is a chain of
// dependent instructions (about 110 cycles for gelu), and the epilogue has two
// warps a scheduler to hide it with; in packed f32 instructions (gelu: 12 a value
// instead of 23).
template <int kAct>
__device__ __forceinline__ void act8(float* v) {
  constexpr int kP = 4;
  if constexpr (kAct == MXB_ACT_SILU || kAct == MXB_ACT_GELU || kAct == MXB_ACT_GELU_TANH) {
    F2 z[kP], s[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) z[i] = F2(v[2 * i], v[2 * i + 1]);
    if constexpr (kAct == MXB_ACT_SILU) {
      logistic_pairs<kP>(z, s);
    } else if constexpr (kAct == MXB_ACT_GELU_TANH) {
      F2 u[kP];
#pragma unroll
      for (int i = 0; i < kP; ++i) u[i] = tanh_arg(z[i]);
      logistic_pairs<kP>(u, s);
    } else {
      F2 gauss[kP];
      normal_cdf_pairs<kP>(v, z, s, gauss);
    }
#pragma unroll
    for (int i = 0; i < kP; ++i) mul2(z[i], s[i]).get(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value<kAct>(v[i]);
  }
}
// The derivatives of eight values, likewise: with s the logistic (or normal)
// factor, silu s + z s (1 - s), gelu_tanh s + z s (1 - s) d(2u)/dz, gelu s + z times
// the normal density.
template <int kAct>
__device__ __forceinline__ void slope8(const float* v, float* out) {
  constexpr int kP = 4;
  if constexpr (kAct == MXB_ACT_SILU || kAct == MXB_ACT_GELU || kAct == MXB_ACT_GELU_TANH) {
    F2 z[kP], s[kP], o[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) z[i] = F2(v[2 * i], v[2 * i + 1]);
    if constexpr (kAct == MXB_ACT_GELU) {
      F2 gauss[kP];
      normal_cdf_pairs<kP>(v, z, s, gauss);
#pragma unroll
      for (int i = 0; i < kP; ++i) o[i] = fma2(mul2(z[i], both(kInvSqrt2Pi)), gauss[i], s[i]);
    } else {
      if constexpr (kAct == MXB_ACT_SILU) {
        logistic_pairs<kP>(z, s);
      } else {
#pragma unroll
        for (int i = 0; i < kP; ++i) o[i] = tanh_arg(z[i]);
        logistic_pairs<kP>(o, s);
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        F2 zs;
        if constexpr (kAct == MXB_ACT_GELU_TANH) {
          // z bounded: past +-32 s is exactly 0 or 1, and z^3 must not become an infinity
          // that meets s (1 - s) = 0 (it does from 1.3e13 on)
          const F2 c(fminf(fmaxf(v[2 * i], -32.0f), 32.0f),
                     fminf(fmaxf(v[2 * i + 1], -32.0f), 32.0f));
          zs = mul2(mul2(c, s[i]), fma2(mul2(c, c), both(6.0f * kSqrt2OverPi * kGeluCubic),
                                        both(2.0f * kSqrt2OverPi)));
        } else {
          zs = mul2(z[i], s[i]);
        }
        o[i] = fma2(zs, fma2(s[i], both(-1.0f), both(1.0f)), s[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kP; ++i) o[i].get(out[2 * i], out[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      out[i] = kAct == MXB_ACT_RELU    ? (v[i] > 0.0f ? 1.0f : 0.0f)
               : kAct == MXB_ACT_RELU2 ? (v[i] > 0.0f ? 2.0f * v[i] : 0.0f)
                                       : 1.0f;
  }
}
template <int kAct, int n>
__device__ __forceinline__ void act_each(float (&v)[n]) {
#pragma unroll
  for (int i = 0; i < n; i += 8) act8<kAct>(v + i);
}
// One activation over n values held in registers; the branch is uniform.
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
