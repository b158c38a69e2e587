// sgnn_linear and its backward pass (include/sgnn.h): y = act(x w^T + bias) + residual.
//   dz = dy act'(z)   dx = dz w   dw = dz^T x   db = sum_m dz
// The three products run in gemm.hip; here is the pass over dy that forms dz and the bias gradient's sums.
#include "gemm.h"
#include "ops_types.h"

namespace {
using namespace sgnn;

constexpr int kThreads = 256;
constexpr int kRows = 128;  // rows per partial sum of db

// Workgroup (bx, by): columns [256 bx, +256), rows [128 by, +128): dz = dy act'(z), and those rows' column sums
// in row order.
template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void k_act_bwd(const T* dy, int64_t ldd, const T* z, int64_t M, int64_t N,
                                                      T* dz, float* partial) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= N) return;
  const int64_t r0 = (int64_t)blockIdx.y * kRows, r1 = min(r0 + kRows, M);
  float s = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    float v = to_float(dy[r * ldd + c]);
    if constexpr (ACT != SGNN_ACT_NONE) v *= act_slope<ACT>(to_float(z[r * N + c]));
    if (dz) dz[r * N + c] = from_float<T>(v);
    s += v;
  }
  if (partial) partial[(int64_t)blockIdx.y * N + c] = s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_sum_partials(const float* partial, int64_t nblk, int64_t N, T* out) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= N) return;
  float s = 0.0f;
  for (int64_t b = 0; b < nblk; ++b) s += partial[b * N + c];
  out[c] = from_float<T>(s);
}

template <typename T>
void launch_act_bwd(int32_t act, dim3 grid, hipStream_t s, const T* dy, int64_t ldd, const T* z, int64_t M, int64_t N,
                    T* dz, float* partial) {
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, dy, ldd, z, M, N, dz, partial);
  };
  if (act == SGNN_ACT_RELU) go(k_act_bwd<T, SGNN_ACT_RELU>);
  else if (act == SGNN_ACT_GELU) go(k_act_bwd<T, SGNN_ACT_GELU>);
  else if (act == SGNN_ACT_GELU_TANH) go(k_act_bwd<T, SGNN_ACT_GELU_TANH>);
  else if (act == SGNN_ACT_SILU) go(k_act_bwd<T, SGNN_ACT_SILU>);
  else go(k_act_bwd<T, SGNN_ACT_NONE>);
}

bool act_ok(int32_t act) { return act >= SGNN_ACT_NONE && act <= SGNN_ACT_SILU; }
size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

Gemm forward(int32_t dtype, int64_t M, int64_t N, int64_t K) {
  Gemm g;
  g.dtype = dtype;
  g.M = M, g.N = N, g.K = K;
  return g;
}
Gemm dgrad(int32_t dtype, int64_t M, int64_t N, int64_t K) {  // dx[M][K] = dz[M][N] w[N][K]
  Gemm g;
  g.dtype = dtype;
  g.M = M, g.N = K, g.K = N;
  g.b_cols = true;
  return g;
}
Gemm wgrad(int32_t dtype, int64_t M, int64_t N, int64_t K) {  // dw[N][K] = dz^T x
  Gemm g;
  g.dtype = dtype;
  g.M = N, g.N = K, g.K = M;
  g.a_cols = g.b_cols = true;
  return g;
}

// Workspace of the backward pass: dz, the partial sums of db, and the products' own.
struct BwdLayout {
  size_t dz, partial, gemm, total;
  BwdLayout(int32_t dtype, int64_t M, int64_t N, int64_t K, int32_t act) {
    dz = act == SGNN_ACT_NONE ? 0 : pad256(dtype_size(dtype) * (size_t)M * (size_t)N);
    partial = pad256(sizeof(float) * (size_t)((M + kRows - 1) / kRows) * (size_t)N);
    gemm = std::max(gemm_workspace_bytes(dgrad(dtype, M, N, K)), gemm_workspace_bytes(wgrad(dtype, M, N, K)));
    total = dz + partial + gemm;
  }
};

}  // namespace

extern "C" size_t sgnn_linear_workspace_bytes(int32_t dtype, int64_t M, int64_t N, int64_t K) {
  if (!sgnn::dtype_ok(dtype) || M <= 0 || N <= 0 || K <= 0) return 0;
  return sgnn::gemm_workspace_bytes(forward(dtype, M, N, K));
}

extern "C" int sgnn_linear(int32_t dtype, int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const void* w,
                           int64_t ldw, const void* bias, int32_t act, const void* residual, int64_t ldr, void* z,
                           void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype) || !act_ok(act)) return set_error(SGNN_ERR_INVALID, "linear: unknown dtype or activation");
  if (M < 0 || N < 0 || K < 0) return set_error(SGNN_ERR_INVALID, "linear: negative size");
  if (M == 0 || N == 0) return SGNN_OK;
  if (!y || ldy < N || (residual && ldr < N)) return set_error(SGNN_ERR_INVALID, "linear: bad output or residual");
  if (K > 0 && (!x || !w || ldx < K || ldw < K)) return set_error(SGNN_ERR_INVALID, "linear: bad operand");
  if (workspace_bytes < sgnn_linear_workspace_bytes(dtype, M, N, K))
    return set_error(SGNN_ERR_INVALID, "linear: workspace smaller than sgnn_linear_workspace_bytes");
  Gemm g = forward(dtype, M, N, K);
  g.A = x, g.lda = ldx;
  g.B = w, g.ldb = ldw;
  g.bias = bias, g.act = act;
  g.res = residual, g.ldr = ldr;
  g.z = z, g.C = y, g.ldc = ldy;
  return gemm_run(g, workspace, workspace_bytes, stream);
}

extern "C" size_t sgnn_linear_bwd_workspace_bytes(int32_t dtype, int64_t M, int64_t N, int64_t K, int32_t act) {
  if (!sgnn::dtype_ok(dtype) || !act_ok(act) || M <= 0 || N <= 0 || K < 0) return 0;
  return BwdLayout(dtype, M, N, K, act).total;
}

extern "C" int sgnn_linear_bwd(int32_t dtype, int64_t M, int64_t N, int64_t K, const void* dy, int64_t ldd,
                               const void* z, int32_t act, const void* x, int64_t ldx, const void* w, int64_t ldw,
                               void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype) || !act_ok(act)) return set_error(SGNN_ERR_INVALID, "linear_bwd: unknown dtype or activation");
  if (M < 0 || N < 0 || K < 0) return set_error(SGNN_ERR_INVALID, "linear_bwd: negative size");
  if (M > 0 && N > 0 && (!dy || ldd < N || (act != SGNN_ACT_NONE && !z)))
    return set_error(SGNN_ERR_INVALID, "linear_bwd: bad dy or z");
  if (K > 0 && ((dx && N > 0 && (!w || ldw < K)) || (dw && M > 0 && (!x || ldx < K))))
    return set_error(SGNN_ERR_INVALID, "linear_bwd: bad operand");
  if (workspace_bytes < sgnn_linear_bwd_workspace_bytes(dtype, M, N, K, act))
    return set_error(SGNN_ERR_INVALID, "linear_bwd: workspace smaller than sgnn_linear_bwd_workspace_bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const BwdLayout at(dtype, std::max<int64_t>(M, 0), N, K, act);
  char* ws = static_cast<char*>(workspace);
  const int64_t nblk = (M + kRows - 1) / kRows;
  const void* up = dy;      // dz and its leading dimension
  int64_t ldu = ldd;
  if (N > 0 && M > 0 && (act != SGNN_ACT_NONE || db)) {
    if (nblk > 65535) return set_error(SGNN_ERR_UNSUPPORTED, "linear_bwd: more than 8M rows");
    with_type(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      T* dz = act == SGNN_ACT_NONE ? nullptr : reinterpret_cast<T*>(ws);
      launch_act_bwd<T>(act, dim3((unsigned)((N + kThreads - 1) / kThreads), (unsigned)nblk), s,
                        static_cast<const T*>(dy), ldd, static_cast<const T*>(z), M, N, dz,
                        db ? reinterpret_cast<float*>(ws + at.dz) : nullptr);
      return 0;
    });
    if (act != SGNN_ACT_NONE) up = ws, ldu = N;
  }
  if (db && N > 0)
    with_type(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      hipLaunchKernelGGL(k_sum_partials<T>, dim3((unsigned)((N + kThreads - 1) / kThreads)), dim3(kThreads), 0, s,
                         reinterpret_cast<const float*>(ws + at.dz), nblk, N, static_cast<T*>(db));
      return 0;
    });
  const int st = check_launch("linear_bwd");
  if (st != SGNN_OK) return st;
  char* gws = ws + at.dz + at.partial;
  if (dx) {
    Gemm g = dgrad(dtype, M, N, K);
    g.A = up, g.lda = ldu;
    g.B = w, g.ldb = ldw;
    g.C = dx, g.ldc = K;
    const int e = gemm_run(g, gws, at.gemm, stream);
    if (e != SGNN_OK) return e;
  }
  if (dw) {
    Gemm g = wgrad(dtype, M, N, K);
    g.A = up, g.lda = ldu;
    g.B = x, g.ldb = ldx;
    g.C = dw, g.ldc = K;
    return gemm_run(g, gws, at.gemm, stream);
  }
  return SGNN_OK;
}
