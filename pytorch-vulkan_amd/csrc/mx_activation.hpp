// Activations of the linear layers and their derivatives (FP32), shared by the
// products' epilogues and the backward's elementwise pass.
//
// The library's erff, expf and tanhf make the elementwise pass of a GELU
// compute-bound (dz and its sums for 4096 x 4096: 62 us, 47 so), so the two below
// are built on the hardware's exp2 and reciprocal, which are good to one place.
#pragma once

#include <hip/hip_runtime.h>

#include "mx.h"

namespace mx {

constexpr float kInvSqrt2Pi = 0.39894228040143268f, kLog2E = 1.44269504088896341f;
constexpr float kLog2ELow = 1.92596299e-8f, kLn2 = 0.69314718055994531f;  // kLog2E + kLog2ELow = log2(e) to 48 bits
constexpr float kSqrt2OverPi = 0.79788456080286536f, kTanhCubic = 0.044715f;

// 1 / (1 + e^-v): 0 and 1 at the infinities.  The rounding of log2(e) v and log2(e)'s
// own are up to 2^-24 of it each, so that e^-v alone would be off by 31 u of itself
// at v = -40 (u = 2^-24): what they leave out, r, comes back as the factor 1 + r ln 2.
// Where log2(e) v is infinite so is r, or NaN, and the plain exp2 is the result.
__device__ __forceinline__ float sigmoid(float v) {
  const float t = -kLog2E * v, r = fmaf(-kLog2ELow, v, fmaf(-kLog2E, v, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_amdgcn_rcpf(1.f + (fabsf(t) < 128.f ? fmaf(e, r * kLn2, e) : e));
}

// Normal distribution's integral from -inf to z; density gets e^(-z^2 / 2).
// The tail beyond |z| is density t P(t) with t = 1 / (1 + 0.3 |z| / sqrt 2) and P
// the degree 8 polynomial nearest to erfcx / (2 t) in relative error on |z| < 20
// (least squares reweighted towards the largest error, which is 6.0e-8, at 0); in
// FP32 the whole is within 2.4e-7, and a lower tail within 11 u of itself down to
// z = -3, from where the rounding of z^2 grows on it (32 u at -6; u = 2^-24).
__device__ __forceinline__ float normal_cdf(float z, float& density) {
  density = __builtin_amdgcn_exp2f(-0.5f * kLog2E * z * z);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.21213203435596426f, fabsf(z), 1.f));
  float p = -6.330832094e-02f;
  p = fmaf(p, t, 2.359132469e-01f);
  p = fmaf(p, t, -2.423461378e-01f);
  p = fmaf(p, t, 2.585246563e-01f);
  p = fmaf(p, t, -3.702469915e-02f);
  p = fmaf(p, t, 1.031926274e-01f);
  p = fmaf(p, t, 7.523442060e-02f);
  p = fmaf(p, t, 8.521185815e-02f);
  p = fmaf(p, t, 8.460237831e-02f);
  const float tail = t * p * density;
  return z > 0.f ? 1.f - tail : tail;
}

// 0.5 (1 + tanh u) = sigmoid(2 u).
__device__ __forceinline__ float tanh_gate(float z) { return sigmoid(2.f * kSqrt2OverPi * (z + kTanhCubic * z * z * z)); }

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case MX_ACT_RELU: return z <= 0.f ? 0.f : z;  // NaN stays, as in mx_unary_f32
    case MX_ACT_SILU: return z * sigmoid(z);
    case MX_ACT_GELU: {
      float density;
      return z * normal_cdf(z, density);
    }
    case MX_ACT_GELU_TANH: return z * tanh_gate(z);
    default: return z;
  }
}

__device__ __forceinline__ float activate_slope(int act, float z) {
  switch (act) {
    case MX_ACT_RELU: return z <= 0.f ? 0.f : (z != z ? z : 1.f);
    case MX_ACT_SILU: {
      const float s = sigmoid(z);
      return s * (1.f + z * (1.f - s));
    }
    case MX_ACT_GELU: {
      float density;
      const float cdf = normal_cdf(z, density);
      return cdf + z * (kInvSqrt2Pi * density);
    }
    case MX_ACT_GELU_TANH: {
      const float s = tanh_gate(z);
      return s + 2.f * z * (s * (1.f - s)) * kSqrt2OverPi * (1.f + 3.f * kTanhCubic * z * z);
    }
    default: return 1.f;
  }
}

}  // namespace mx
