// sgnn_norm and its backward pass (include/sgnn.h): LayerNorm over rows, with the reductions of the weight's and
// the bias's gradient in the pass over the rows that forms dx.
#include "ops_types.h"

namespace {
using namespace sgnn;

constexpr int kThreads = 256;
constexpr int kWavesPer = kThreads / 64;

SGNN_DEV float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One wave per row: mean, then the variance of the differences (two passes), then the outputs.
template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void k_norm(const T* x, int64_t ldx, int64_t n, int width, const W* gamma,
                                                   const W* beta, const T* residual, int64_t ldr, float eps, T* y,
                                                   float* mean_out, float* rstd_out) {
  const int l = lane_id();
  const int64_t nw = (int64_t)gridDim.x * kWavesPer;
  for (int64_t r = (int64_t)blockIdx.x * kWavesPer + wave_id(); r < n; r += nw) {
    const T* p = x + r * ldx;
    float s = 0.0f;
    for (int c = l; c < width; c += 64) s += to_float(p[c]);
    const float mean = wave_sum(s) / width;
    float v = 0.0f;
    for (int c = l; c < width; c += 64) {
      const float d = to_float(p[c]) - mean;
      v += d * d;
    }
    const float rstd = 1.0f / sqrtf(wave_sum(v) / width + eps);
    for (int c = l; c < width; c += 64) {
      float o = (to_float(p[c]) - mean) * rstd;
      if (gamma) o *= to_float(gamma[c]);
      if (beta) o += to_float(beta[c]);
      if (residual) o += to_float(residual[r * ldr + c]);
      y[r * width + c] = from_float<T>(o);
    }
    if (l == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void k_norm_dx(const T* dy, int64_t ldd, const T* x, int64_t ldx,
                                                      const float* mean, const float* rstd, const W* gamma, int64_t n,
                                                      int width, T* dx) {
  const int l = lane_id();
  const int64_t nw = (int64_t)gridDim.x * kWavesPer;
  for (int64_t r = (int64_t)blockIdx.x * kWavesPer + wave_id(); r < n; r += nw) {
    const float mu = mean[r], rs = rstd[r];
    float sg = 0.0f, sgh = 0.0f;
    for (int c = l; c < width; c += 64) {
      const float g = to_float(dy[r * ldd + c]) * (gamma ? to_float(gamma[c]) : 1.0f);
      sg += g;
      sgh += g * (to_float(x[r * ldx + c]) - mu) * rs;
    }
    sg = wave_sum(sg) / width;
    sgh = wave_sum(sgh) / width;
    for (int c = l; c < width; c += 64) {
      const float g = to_float(dy[r * ldd + c]) * (gamma ? to_float(gamma[c]) : 1.0f);
      dx[r * width + c] = from_float<T>(rs * (g - sg - (to_float(x[r * ldx + c]) - mu) * rs * sgh));
    }
  }
}

constexpr int kRows = 128;  // rows per partial sum

template <typename T>
__global__ __launch_bounds__(kThreads) void k_norm_partials(const T* dy, int64_t ldd, const T* x, int64_t ldx,
                                                            const float* mean, const float* rstd, int64_t n, int width,
                                                            float* partial) {
  const int c = blockIdx.y * kThreads + threadIdx.x;
  if (c >= width) return;
  const int64_t r0 = (int64_t)blockIdx.x * kRows, r1 = min(r0 + kRows, n);
  float dg = 0.0f, db = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = to_float(dy[r * ldd + c]);
    dg += g * (to_float(x[r * ldx + c]) - mean[r]) * rstd[r];
    db += g;
  }
  partial[(int64_t)blockIdx.x * 2 * width + c] = dg;
  partial[(int64_t)blockIdx.x * 2 * width + width + c] = db;
}

template <typename W>
__global__ __launch_bounds__(kThreads) void k_norm_reduce(const float* partial, int64_t nblk, int width, W* dgamma,
                                                          W* dbeta) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= 2 * width) return;
  float s = 0.0f;
  for (int64_t b = 0; b < nblk; ++b) s += partial[b * 2 * width + c];
  if (c < width) {
    if (dgamma) dgamma[c] = from_float<W>(s);
  } else if (dbeta) {
    dbeta[c - width] = from_float<W>(s);
  }
}

unsigned row_grid(int64_t n) { return (unsigned)std::min<int64_t>((n + kWavesPer - 1) / kWavesPer, 4096); }

template <typename F>
int with_types(int32_t dtype, int32_t wdtype, F f) {
  return with_type(dtype, [&](auto* t) {
    return wdtype == dtype ? f(t, t) : f(t, (float*)nullptr);
  });
}

}  // namespace

extern "C" int sgnn_norm(int32_t dtype, int32_t wdtype, const void* x, int64_t ldx, int64_t n, int32_t width,
                         const void* gamma, const void* beta, const void* residual, int64_t ldr, float eps, void* y,
                         float* mean, float* rstd, void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != SGNN_F32))
    return set_error(SGNN_ERR_INVALID, "norm: unknown dtype, or a weight type that is neither dtype nor fp32");
  if (n < 0 || width < 1 || !(eps >= 0.0f)) return set_error(SGNN_ERR_INVALID, "norm: bad size or eps");
  if (n == 0) return SGNN_OK;
  if (!x || !y || ldx < width || (residual && ldr < width)) return set_error(SGNN_ERR_INVALID, "norm: bad operand");
  with_types(dtype, wdtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    hipLaunchKernelGGL((k_norm<T, W>), dim3(row_grid(n)), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T*>(x), ldx, n, width, static_cast<const W*>(gamma),
                       static_cast<const W*>(beta), static_cast<const T*>(residual), ldr, eps, static_cast<T*>(y),
                       mean, rstd);
    return 0;
  });
  return check_launch("norm");
}

extern "C" size_t sgnn_norm_bwd_workspace_bytes(int64_t n, int32_t width) {
  if (n <= 0 || width <= 0) return 0;
  return sizeof(float) * 2 * (size_t)width * (size_t)((n + kRows - 1) / kRows);
}

extern "C" int sgnn_norm_bwd(int32_t dtype, int32_t wdtype, const void* dy, int64_t ldd, const void* x, int64_t ldx,
                             const float* mean, const float* rstd, const void* gamma, int64_t n, int32_t width,
                             void* dx, void* dgamma, void* dbeta, void* workspace, size_t workspace_bytes,
                             void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != SGNN_F32))
    return set_error(SGNN_ERR_INVALID, "norm_bwd: unknown dtype, or a weight type that is neither dtype nor fp32");
  if (n < 0 || width < 1) return set_error(SGNN_ERR_INVALID, "norm_bwd: bad size");
  if (n > 0 && (!dy || !x || !mean || !rstd || ldd < width || ldx < width))
    return set_error(SGNN_ERR_INVALID, "norm_bwd: bad operand");
  const bool sums = dgamma || dbeta;
  if (sums && n > 0 && (!workspace || workspace_bytes < sgnn_norm_bwd_workspace_bytes(n, width)))
    return set_error(SGNN_ERR_INVALID, "norm_bwd: workspace smaller than sgnn_norm_bwd_workspace_bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t nblk = (n + kRows - 1) / kRows;
  float* part = static_cast<float*>(workspace);
  with_types(dtype, wdtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    const T *up = static_cast<const T*>(dy), *in = static_cast<const T*>(x);
    if (dx && n > 0)
      hipLaunchKernelGGL((k_norm_dx<T, W>), dim3(row_grid(n)), dim3(kThreads), 0, s, up, ldd, in, ldx, mean, rstd,
                         static_cast<const W*>(gamma), n, width, static_cast<T*>(dx));
    if (sums && n > 0)
      hipLaunchKernelGGL(k_norm_partials<T>, dim3((unsigned)nblk, (unsigned)((width + kThreads - 1) / kThreads)),
                         dim3(kThreads), 0, s, up, ldd, in, ldx, mean, rstd, n, width, part);
    if (sums)
      hipLaunchKernelGGL(k_norm_reduce<W>, dim3((unsigned)((2 * (int64_t)width + kThreads - 1) / kThreads)),
                         dim3(kThreads), 0, s, part, nblk, width, static_cast<W*>(dgamma), static_cast<W*>(dbeta));
    return 0;
  });
  return check_launch("norm_bwd");
}
