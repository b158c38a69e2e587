// sgnn_newton_schulz (include/sgnn.h): X = in / (|in|_F + eps), then X <- a X + (b G + c G^2) X, G = X X^T.
#include "gemm.h"
#include "ops_types.h"

namespace {
using namespace sgnn;

constexpr int kThreads = 256;

// One workgroup: out = in / (|in|_F + eps) as dense fp32 [m][n], m <= n (transposed where in is taller).
template <typename T>
__global__ __launch_bounds__(kThreads) void k_ns_begin(const T* in, int64_t ld, int rows, int cols, float eps,
                                                       float* out) {
  __shared__ double part[kThreads / 64];
  const int64_t total = (int64_t)rows * cols;
  double s = 0.0;  // 64 bits: the square of a gradient leaves fp32's range long before the gradient does
  for (int64_t t = threadIdx.x; t < total; t += kThreads) {
    const double v = to_float(in[t / cols * ld + t % cols]);
    s += v * v;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane_id() == 0) part[wave_id()] = s;
  __syncthreads();
  s = part[0] + part[1] + part[2] + part[3];
  const float norm = (float)sqrt(s) + eps;
  for (int64_t t = threadIdx.x; t < total; t += kThreads) {
    const int64_t r = t / cols, c = t % cols;
    out[rows > cols ? c * rows + r : t] = norm == 0.0f ? 0.0f : to_float(in[r * ld + c]) / norm;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_ns_end(const float* x, int rows, int cols, T* out, int64_t ld) {
  const int64_t total = (int64_t)rows * cols;
  for (int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x; t < total; t += (int64_t)gridDim.x * kThreads) {
    const int64_t r = t / cols, c = t % cols;
    out[r * ld + c] = from_float<T>(x[rows > cols ? c * rows + r : t]);
  }
}

size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

Gemm product(int64_t M, int64_t N, int64_t K, bool b_cols) {
  Gemm g;
  g.dtype = SGNN_F32;
  g.M = M, g.N = N, g.K = K, g.b_cols = b_cols;
  return g;
}

struct NsLayout {  // X twice, G and b G + c G^2, the products' own
  size_t x, g, gemm, total;
  NsLayout(int64_t m, int64_t n) {
    x = pad256(sizeof(float) * m * n);
    g = pad256(sizeof(float) * m * m);
    gemm = std::max({gemm_workspace_bytes(product(m, m, n, false)), gemm_workspace_bytes(product(m, m, m, false)),
                     gemm_workspace_bytes(product(m, n, m, true))});
    total = 2 * x + 2 * g + gemm;
  }
};

}  // namespace

extern "C" size_t sgnn_newton_schulz_workspace_bytes(const sgnn_matrix* mats, int32_t count) {
  size_t most = 0;
  for (int32_t i = 0; mats && i < count; ++i) {
    if (mats[i].rows < 1 || mats[i].cols < 1) continue;
    most = std::max(most, NsLayout(std::min(mats[i].rows, mats[i].cols), std::max(mats[i].rows, mats[i].cols)).total);
  }
  return most;
}

extern "C" int sgnn_newton_schulz(int32_t dtype, const sgnn_matrix* mats, int32_t count, int32_t steps, float a,
                                  float b, float c, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype)) return set_error(SGNN_ERR_INVALID, "newton_schulz: unknown dtype");
  if (count < 0 || (count > 0 && !mats) || steps < 0 || !(eps >= 0.0f))
    return set_error(SGNN_ERR_INVALID, "newton_schulz: bad count, steps or eps");
  for (int32_t i = 0; i < count; ++i) {
    const sgnn_matrix& t = mats[i];
    if (t.rows < 0 || t.cols < 0) return set_error(SGNN_ERR_INVALID, "newton_schulz: negative size");
    if (t.rows > 0 && t.cols > 0 && (!t.in || !t.out || t.ld_in < t.cols || t.ld_out < t.cols))
      return set_error(SGNN_ERR_INVALID, "newton_schulz: bad matrix");
  }
  if (workspace_bytes < sgnn_newton_schulz_workspace_bytes(mats, count))
    return set_error(SGNN_ERR_INVALID, "newton_schulz: workspace smaller than sgnn_newton_schulz_workspace_bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int32_t i = 0; i < count; ++i) {
    const sgnn_matrix& t = mats[i];
    if (t.rows == 0 || t.cols == 0) continue;
    const int64_t m = std::min(t.rows, t.cols), n = std::max(t.rows, t.cols);
    const NsLayout at(m, n);
    char* ws = static_cast<char*>(workspace);
    char* gws = ws + 2 * at.x + 2 * at.g;
    float *x = reinterpret_cast<float*>(ws), *next = reinterpret_cast<float*>(ws + at.x);
    float *gram = reinterpret_cast<float*>(ws + 2 * at.x), *poly = reinterpret_cast<float*>(ws + 2 * at.x + at.g);
    with_type(dtype, [&](auto* p) {
      using T = std::remove_pointer_t<decltype(p)>;
      hipLaunchKernelGGL(k_ns_begin<T>, dim3(1), dim3(kThreads), 0, s, static_cast<const T*>(t.in), t.ld_in, t.rows,
                         t.cols, eps, x);
      return 0;
    });
    for (int32_t k = 0; k < steps; ++k) {
      Gemm g = product(m, m, n, false);
      g.A = g.B = x, g.lda = g.ldb = n;
      g.C = gram, g.ldc = m;
      int st = gemm_run(g, gws, at.gemm, stream);
      if (st != SGNN_OK) return st;
      g = product(m, m, m, false);
      g.A = g.B = gram, g.lda = g.ldb = m;   // G is symmetric: its rows are its columns
      g.alpha = c, g.beta = b;
      g.res = gram, g.ldr = m;
      g.C = poly, g.ldc = m;
      if ((st = gemm_run(g, gws, at.gemm, stream)) != SGNN_OK) return st;
      g = product(m, n, m, true);
      g.A = poly, g.lda = m;
      g.B = x, g.ldb = n;
      g.beta = a;
      g.res = x, g.ldr = n;
      g.C = next, g.ldc = n;
      if ((st = gemm_run(g, gws, at.gemm, stream)) != SGNN_OK) return st;
      std::swap(x, next);
    }
    with_type(dtype, [&](auto* p) {
      using T = std::remove_pointer_t<decltype(p)>;
      hipLaunchKernelGGL(k_ns_end<T>, dim3((unsigned)std::min<int64_t>((m * n + kThreads - 1) / kThreads, 2048)),
                         dim3(kThreads), 0, s, x, t.rows, t.cols, static_cast<T*>(t.out), t.ld_out);
      return 0;
    });
    const int st = check_launch("newton_schulz");
    if (st != SGNN_OK) return st;
  }
  return SGNN_OK;
}
