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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any element's alignment (one global_load/store_dwordx4: unaligned access is on for this target)
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// The 16 bytes n (0 .. 16, even) bytes further on; zeros move in.
SGNN_DEV u32x4 move_down(u32x4 v, int n) {
  if (n & 8) v = u32x4{v[2], v[3], 0, 0};
  if (n & 4) v = u32x4{v[1], v[2], v[3], 0};
  if (n & 2)
    v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
  if (n & 16) v = u32x4{0, 0, 0, 0};
  return v;
}

// 16 bytes of T at any alignment <-> floats
template <typename T>
SGNN_DEV void load_vec(const T* p, float* v) {
  constexpr int V = 16 / sizeof(T);
  typedef T TV __attribute__((ext_vector_type(V)));
  const TV t = __builtin_bit_cast(TV, (u32x4)*reinterpret_cast<const u32x4_any*>(p));
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_float(t[i]);
}
template <typename T>
SGNN_DEV void store_vec(T* p, const float* v) {
  constexpr int V = 16 / sizeof(T);
  typedef T TV __attribute__((ext_vector_type(V)));
  TV t;
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = from_float<T>(v[i]);
  *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, t);
}
// 16 bytes of T as they are in memory, the first cnt values there (the others 0), and their floats.
template <typename T>
SGNN_DEV u32x4 load_raw(const T* p, int cnt) {
  constexpr int V = 16 / sizeof(T);
  if (cnt >= V) return *reinterpret_cast<const u32x4_any*>(p);
  typedef T TV __attribute__((ext_vector_type(V)));
  TV t = __builtin_bit_cast(TV, u32x4{0, 0, 0, 0});
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < cnt) t[i] = p[i];
  return __builtin_bit_cast(u32x4, t);
}
template <typename T>
SGNN_DEV void unpack(u32x4 raw, float* v) {
  constexpr int V = 16 / sizeof(T);
  typedef T TV __attribute__((ext_vector_type(V)));
  const TV t = __builtin_bit_cast(TV, raw);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_float(t[i]);
}
// N values of T, the first cnt of them there (the others read as 0, are not written).
template <int N, typename T>
SGNN_DEV void load_some(const T* p, int cnt, float (&v)[N]) {
  constexpr int V = 16 / sizeof(T);
  if (cnt >= N) {
#pragma unroll
    for (int i = 0; i < N; i += V) load_vec(p + i, v + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < cnt ? to_float(p[i]) : 0.0f;
  }
}
template <int N, typename T>
SGNN_DEV void store_some(T* p, int cnt, const float (&v)[N]) {
  constexpr int V = 16 / sizeof(T);
  if (cnt >= N) {
#pragma unroll
    for (int i = 0; i < N; i += V) store_vec(p + i, v + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) p[i] = from_float<T>(v[i]);
  }
}

// v in two values of a 16-bit type, hi + lo 2^-kLoBits, good to 2^-16 (bf16) or 2^-22 (fp16) of it down to 2^-36: lo is
// scaled to hi's size, which keeps it out of fp16's subnormal numbers.  An infinity or a NaN is hi's alone.
template <typename T>
constexpr int kLoBits = std::is_same_v<T, bf16_t> ? 8 : 11;
template <typename T>
SGNN_DEV void split2(float v, T& hi, T& lo) {
  hi = from_float<T>(v);
  const float rest = v - to_float(hi);
  lo = from_float<T>(rest - rest == 0.0f ? rest * (float)(1 << kLoBits<T>) : 0.0f);
}

// Sum over groups of G consecutive lanes (16, 32 or 64), the same in each of them: within 16 lanes by DPP (xor 1, xor
// 2, then the two mirrors), rows of 16 and halves of 32 by the swap instructions -- no LDS.
template <int CTRL>
SGNN_DEV float dpp_mov(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int G>
SGNN_DEV float lanes_sum(float v) {
  v += dpp_mov<0xb1>(v);   // quad_perm 1, 0, 3, 2
  v += dpp_mov<0x4e>(v);   // quad_perm 2, 3, 0, 1
  v += dpp_mov<0x141>(v);  // row_half_mirror
  v += dpp_mov<0x140>(v);  // row_mirror
  if constexpr (G >= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = s[0], b = s[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  if constexpr (G >= 64) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = s[0], b = s[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  return v;
}

// out[c] = sum over the nblk partial rows of `cols` fp32 values, 16 columns per workgroup of 1024 threads: each of 64
// groups of 16 lanes takes every 64th row, then the groups' sums in group order.  Bounded by the latency of its
// nblk / 64 dependent-free loads per lane: a few us up to 2048 rows.  f(c, sum) stores.
constexpr int kSumThreads = 1024, kSumCols = 16;
template <typename F>
SGNN_DEV void sum_partials(const float* partial, int64_t nblk, int64_t cols, F f) {
  __shared__ float part[kSumThreads / kSumCols][kSumCols + 1];
  const int g = threadIdx.x / kSumCols, i = threadIdx.x % kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + i;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int64_t b = g; b < nblk; b += kSumThreads / kSumCols) s += partial[b * cols + c];
  part[g][i] = s;
  __syncthreads();
  if (g != 0 || c >= cols) return;
  s = 0.0f;
#pragma unroll 8
  for (int r = 0; r < kSumThreads / kSumCols; ++r) s += part[r][i];
  f(c, s);
}
inline unsigned sum_grid(int64_t cols) { return (unsigned)((cols + kSumCols - 1) / kSumCols); }

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

// The standard normal distribution function and e = exp(-z^2 / 2), which it shares with its density, by Abramowitz and
// Stegun 7.1.26: 1 - Phi(|z|) = (a1 t + ... + a5 t^5) e / 2, t = 1 / (1 + p |z| / sqrt 2), good to 7.5e-8 (relative:
// 6e-8 at z = -1, 5e-4 at -4, where 1 + erf(z) in fp32 is off by 1e-3) -- for the 16-bit types, whose rounding hides it.
// A third of erff's instructions: 8192 x 2048 -> 8192 in bf16 with gelu and its slopes went from 325 to 296 us.
SGNN_DEV float normal_cdf(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * kInvSqrt2 * fabsf(z));
  e = __expf(-0.5f * z * z);
  const float poly =
      t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  const float tail = 0.5f * poly * e;
  return z < 0.0f ? tail : 1.0f - tail;
}

// act(z) and, where SLOPE, d act / d z, which share their functions; FAST: gelu by normal_cdf.  ReLU keeps a NaN (a comparison, not a maximum);
// its slope at 0 is 0.  Far out, where the smooth ones' second terms are 0 in fp32 but for the products of 0 and
// infinity in them, the slopes are the first terms alone.
template <int ACT, bool SLOPE, bool FAST>
SGNN_DEV void act_both(float z, float& value, float& slope) {
  value = z, slope = 1.0f;
  if constexpr (ACT == SGNN_ACT_RELU) {
    value = z < 0.0f ? 0.0f : z;
    slope = z > 0.0f ? 1.0f : 0.0f;
  }
  if constexpr (ACT == SGNN_ACT_GELU) {
    float phi, e;
    if constexpr (FAST) {
      phi = normal_cdf(z, e);
    } else {
      phi = 0.5f * (1.0f + erff(z * kInvSqrt2));
      e = __expf(-0.5f * z * z);
    }
    value = z * phi;
    if constexpr (SLOPE) slope = fabsf(z) > 20.0f ? phi : phi + z * kInvSqrt2Pi * e;
  }
  if constexpr (ACT == SGNN_ACT_GELU_TANH) {  // 0.5 (1 + tanh u) = sigmoid(2 u)
    const float s = sigmoid(2.0f * kSqrt2OverPi * (z + kGeluCubic * z * z * z));
    value = z * s;
    if constexpr (SLOPE)
      slope = fabsf(z) > 20.0f ? s : s + z * s * (1.0f - s) * 2.0f * kSqrt2OverPi * (1.0f + 3.0f * kGeluCubic * z * z);
  }
  if constexpr (ACT == SGNN_ACT_SILU) {
    const float s = sigmoid(z);
    value = z * s;
    if constexpr (SLOPE) slope = fabsf(z) > 88.0f ? s : s * (1.0f + z * (1.0f - s));
  }
}

}  // namespace sgnn
