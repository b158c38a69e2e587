// One matrix product for every operand type and storage order (gemm.h): 64 x 64 output tiles, operands staged
// as fp32 through LDS, v_mfma_f32_32x32x2_f32.
#include "gemm.h"

#include "ops_types.h"

namespace {
using namespace sgnn;

constexpr int kTile = 64;    // output tile (M and N) per workgroup
constexpr int kKc = 16;      // K per LDS stage
constexpr int kLdT = kTile + 4;
constexpr int kThreads = 256;

// 64 rows (m or n) x 16 k of an operand into LDS as S[k][row], zero outside the matrix.
template <typename T>
SGNN_DEV void stage(float* S, const T* p, int64_t ld, bool cols, int64_t rows, int64_t K, int64_t r0, int64_t k0) {
  const int t = threadIdx.x;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int r = cols ? (t & 15) * 4 + c : t >> 2, k = cols ? t >> 4 : (t & 3) * 4 + c;
    const int64_t gr = r0 + r, gk = k0 + k;
    S[k * kLdT + r] = gr < rows && gk < K ? to_float(p[cols ? gk * ld + gr : gr * ld + gk]) : 0.0f;
  }
}

template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void k_gemm_typed(Gemm g) {
  __shared__ float As[kKc * kLdT];
  __shared__ float Bs[kKc * kLdT];
  const int l = lane_id(), w = wave_id();
  const int wm = w >> 1, wn = w & 1;
  const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile, b = blockIdx.z;
  const T* A = static_cast<const T*>(g.A) + b * g.batch_a;
  const T* B = static_cast<const T*>(g.B) + b * g.batch_b;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (int64_t k0 = 0; k0 < g.K; k0 += kKc) {
    stage(As, A, g.lda, g.a_cols, g.M, g.K, m0, k0);
    stage(Bs, B, g.ldb, g.b_cols, g.N, g.K, n0, k0);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kKc / 2; ++s) {
      const int k = 2 * s + (l >> 5);
      acc = mfma32(As[k * kLdT + wm * 32 + (l & 31)], Bs[k * kLdT + wn * 32 + (l & 31)], acc);
    }
    __syncthreads();
  }
  const int64_t n = n0 + wn * 32 + (l & 31);
  const T* res = static_cast<const T*>(g.res);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t m = m0 + wm * 32 + crow(r, l >> 5);
    if (m >= g.M || n >= g.N) continue;
    float v = g.alpha * acc[r];
    if (g.bias) v += to_float(static_cast<const T*>(g.bias)[n]);
    if (g.z) static_cast<T*>(g.z)[m * g.N + n] = from_float<T>(v);
    v = act_value<ACT>(v);
    if (res) v += g.beta * to_float(res[b * g.batch_r + m * g.ldr + n]);
    static_cast<T*>(g.C)[b * g.batch_c + m * g.ldc + n] = from_float<T>(v);
  }
}

template <typename T>
void launch(const Gemm& g, hipStream_t s) {
  const dim3 grid((unsigned)((g.M + kTile - 1) / kTile), (unsigned)((g.N + kTile - 1) / kTile), (unsigned)g.batch);
  switch (g.act) {
    case SGNN_ACT_RELU: hipLaunchKernelGGL((k_gemm_typed<T, SGNN_ACT_RELU>), grid, dim3(kThreads), 0, s, g); break;
    case SGNN_ACT_GELU: hipLaunchKernelGGL((k_gemm_typed<T, SGNN_ACT_GELU>), grid, dim3(kThreads), 0, s, g); break;
    case SGNN_ACT_GELU_TANH: hipLaunchKernelGGL((k_gemm_typed<T, SGNN_ACT_GELU_TANH>), grid, dim3(kThreads), 0, s, g); break;
    case SGNN_ACT_SILU: hipLaunchKernelGGL((k_gemm_typed<T, SGNN_ACT_SILU>), grid, dim3(kThreads), 0, s, g); break;
    default: hipLaunchKernelGGL((k_gemm_typed<T, SGNN_ACT_NONE>), grid, dim3(kThreads), 0, s, g);
  }
}

}  // namespace

namespace sgnn {

size_t gemm_workspace_bytes(const Gemm&) { return 0; }

int gemm_run(const Gemm& g, void*, size_t, void* stream) {
  if (g.M == 0 || g.N == 0 || g.batch == 0) return SGNN_OK;
  if ((g.N + kTile - 1) / kTile > 65535 || (g.M + kTile - 1) / kTile > INT32_MAX || g.batch > 65535)
    return set_error(SGNN_ERR_UNSUPPORTED, "gemm: more than 4M columns or 65535 matrices");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(g.dtype, [&](auto* t) {
    launch<std::remove_pointer_t<decltype(t)>>(g, s);
    return 0;
  });
  return check_launch("gemm");
}

}  // namespace sgnn
