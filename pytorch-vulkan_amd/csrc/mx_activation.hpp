// Activations of the linear layers and their derivatives (FP32), shared by the
// products' epilogues and the backward's elementwise pass.
#pragma once

#include <hip/hip_runtime.h>

#include "mx.h"

namespace mx {

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f, kTanhCubic = 0.044715f;

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case MX_ACT_RELU: return z <= 0.f ? 0.f : z;  // NaN stays, as in mx_unary_f32
    case MX_ACT_SILU: return z / (1.f + expf(-z));
    case MX_ACT_GELU: return 0.5f * z * (1.f + erff(z * kSqrtHalf));
    case MX_ACT_GELU_TANH: return 0.5f * z * (1.f + tanhf(kSqrt2OverPi * (z + kTanhCubic * z * z * z)));
    default: return z;
  }
}

__device__ __forceinline__ float activate_slope(int act, float z) {
  switch (act) {
    case MX_ACT_RELU: return z <= 0.f ? 0.f : (z != z ? z : 1.f);
    case MX_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    case MX_ACT_GELU: return 0.5f * (1.f + erff(z * kSqrtHalf)) + z * (kInvSqrt2Pi * expf(-0.5f * z * z));
    case MX_ACT_GELU_TANH: {
      const float t = tanhf(kSqrt2OverPi * (z + kTanhCubic * z * z * z));
      return 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * kSqrt2OverPi * (1.f + 3.f * kTanhCubic * z * z);
    }
    default: return 1.f;
  }
}

}  // namespace mx
