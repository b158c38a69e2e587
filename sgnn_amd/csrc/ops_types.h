// What the typed operators (linear.hip, norm.hip, muon.hip) share: the element types of include/sgnn.h's
// sgnn_dtype, conversions to and from the 32-bit values every sum is held in, and the activations with their
// slopes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sgnn.h"
#include "common.h"
#include "sgnn_internal.h"

namespace sgnn {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T>
SGNN_DEV float to_float(T v) {
  return (float)v;
}
// Round to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32); the only rounding of an output's value.
template <typename T>
SGNN_DEV T from_float(float v) {
  return (T)v;
}

inline size_t dtype_size(int32_t dtype) { return dtype == SGNN_F32 ? 4 : 2; }
inline bool dtype_ok(int32_t dtype) { return dtype == SGNN_F32 || dtype == SGNN_BF16 || dtype == SGNN_F16; }

// Calls f with a null pointer of the element type of `dtype` (checked by the caller).
template <typename F>
int with_type(int32_t dtype, F f) {
  if (dtype == SGNN_F32) return f((float*)nullptr);
  if (dtype == SGNN_BF16) return f((bf16_t*)nullptr);
  return f((f16_t*)nullptr);
}

constexpr float kInvSqrt2 = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;   // 1 / sqrt(2 pi)
constexpr float kSqrt2OverPi = 0.79788456080286536f;  // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

SGNN_DEV float sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }

// act(z).  ReLU keeps a NaN (a comparison, not a maximum).
template <int ACT>
SGNN_DEV float act_value(float z) {
  if constexpr (ACT == SGNN_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == SGNN_ACT_GELU) return 0.5f * z * (1.0f + erff(z * kInvSqrt2));
  // 0.5 (1 + tanh u) = sigmoid(2 u)
  if constexpr (ACT == SGNN_ACT_GELU_TANH) return z * sigmoid(2.0f * kSqrt2OverPi * (z + kGeluCubic * z * z * z));
  if constexpr (ACT == SGNN_ACT_SILU) return z * sigmoid(z);
  return z;
}

// d act / d z.  ReLU's slope at 0 is 0.  Far out, where the smooth ones' second terms are 0 in fp32 but for the
// products of 0 and infinity in them, the first terms alone.
template <int ACT>
SGNN_DEV float act_slope(float z) {
  if constexpr (ACT == SGNN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == SGNN_ACT_GELU) {
    const float phi = 0.5f * (1.0f + erff(z * kInvSqrt2));
    return fabsf(z) > 20.0f ? phi : phi + z * kInvSqrt2Pi * __expf(-0.5f * z * z);
  }
  if constexpr (ACT == SGNN_ACT_GELU_TANH) {
    const float s = sigmoid(2.0f * kSqrt2OverPi * (z + kGeluCubic * z * z * z));
    return fabsf(z) > 20.0f ? s : s + z * s * (1.0f - s) * 2.0f * kSqrt2OverPi * (1.0f + 3.0f * kGeluCubic * z * z);
  }
  if constexpr (ACT == SGNN_ACT_SILU) {
    const float s = sigmoid(z);
    return fabsf(z) > 88.0f ? s : s * (1.0f + z * (1.0f - s));
  }
  return 1.0f;
}

}  // namespace sgnn
