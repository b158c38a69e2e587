// sgnn_linear and its backward pass (include/sgnn.h): y = act(x w^T + bias) + residual.
//   dz = dy act'(z)   dx = dz w   dw = dz^T x   db = sum_m dz
// The three products run in gemm.hip; here is the pass over dy that forms dz and the bias gradient's sums.
#include "gemm.h"
#include "ops_types.h"

namespace {
using namespace sgnn;

constexpr int kThreads = 256;

// How the pass over dy is cut: `lanes` threads side by side take a 16-byte piece each of a row, 256 / lanes rows at
// once; `strips` such column strips, `blocks` row blocks.  About 2048 workgroups (8 per CU) keep enough loads in
// flight for the memory's rate; the row blocks are also the partial sums of db, so there are at most 512, of four
// passes at least.
struct ActCut {
  int lanes;
  int64_t strips, blocks;
  ActCut(size_t size, int64_t M, int64_t N) {
    const int64_t pieces = std::max<int64_t>(1, (N * (int64_t)size + 15) / 16);  // one of no columns where N = 0
    lanes = 16;
    while (lanes < kThreads && lanes < pieces) lanes *= 2;
    strips = (pieces + lanes - 1) / lanes;
    const int64_t passes = (M + kThreads / lanes - 1) / (kThreads / lanes);
    blocks = std::max<int64_t>(1, std::min({(passes + 3) / 4, (int64_t)512, (2048 + strips - 1) / strips}));
  }
};

// dz = dy act'(z), for lo != 0 as two planes of its half, lo values apart (split2; dy times a slope of up to 1.13 may leave
// the type's range), and the column sums of this workgroup's rows: every thread over its rows in order, then the
// threads of one column in order.  Reads dy and the slopes, writes dz: bounded by memory (200003 x 128 fp32 52 us,
// 5.9 TB/s; 8192 x 8192 bf16, two planes, 162 us, 4.1 TB/s -- formed inside the two products instead, dz would be computed and its
// inputs read twice, at every tile's pace).  Slopes rather than z are kept by the forward: it has the activation's
// functions at hand, and this pass none.  They are fp32 for every type: in the tails of gelu and silu a slope is far below
// 1, where fixed point of 16 bits leaves nothing of it.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_act_bwd(const T* dy, int64_t ldd, const float* slope, int64_t M, int64_t N,
                                                      int lanes, T* dz, int64_t lo, float* partial) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float sums[kThreads * V];
  const int rows = kThreads / lanes, lane = threadIdx.x % lanes, row = threadIdx.x / lanes;
  const int64_t c = ((int64_t)blockIdx.x * lanes + lane) * V;
  const int cnt = (int)min((int64_t)V, N - c);
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.0f;
  if (cnt > 0) {
    // four rows are loaded before the first is used
    constexpr int U = 4;
    const int64_t step = (int64_t)gridDim.y * rows;
    for (int64_t r0 = (int64_t)blockIdx.y * rows + row; r0 < M; r0 += U * step) {
      u32x4 up[U];
      float t[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = r0 + u * step;
        up[u] = u32x4{0, 0, 0, 0};
        if (r >= M) continue;
        up[u] = load_raw(dy + r * ldd + c, cnt);
        if (slope) load_some<V>(slope + r * N + c, cnt, t[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = r0 + u * step;
        if (r >= M) continue;
        float v[V];
        unpack<T>(up[u], v);
        if (slope) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] *= lo ? 0.5f * t[u][i] : t[u][i];
          if (lo == 0) {
            store_some<V>(dz + r * N + c, cnt, v);
          } else if constexpr (sizeof(T) == 2) {
            float h[V], l[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
              T hi, low;
              split2(v[i], hi, low);
              h[i] = to_float(hi), l[i] = to_float(low);
              v[i] *= 2.0f;
            }
            store_some<V>(dz + r * N + c, cnt, h);
            store_some<V>(dz + lo + r * N + c, cnt, l);
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += v[i];
      }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int i = 0; i < V; ++i) sums[threadIdx.x * V + i] = s[i];
  __syncthreads();
  if (row != 0 || cnt <= 0) return;
  for (int q = 1; q < rows; ++q)
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] += sums[(q * lanes + lane) * V + i];
  float* o = partial + (int64_t)blockIdx.y * N + c;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < cnt) o[i] = s[i];
}

// The row blocks' sums of every column, in order: 7 us for 512 x 8192.
template <typename T>
__global__ __launch_bounds__(kSumThreads) void k_bias_grad(const float* partial, int64_t nblk, int64_t N, T* out) {
  sum_partials(partial, nblk, N, [&](int64_t c, float s) { out[c] = from_float<T>(s); });
}

// A launch has fewer than 2^32 threads: k_bias_grad takes 64 per column, the products' tiles 4 per row of one column.
constexpr int64_t kMostRows = (int64_t)1 << 30, kMostCols = (int64_t)1 << 25;
bool too_many(int64_t M, int64_t N, int64_t K) { return M > kMostRows || std::max(N, K) > kMostCols; }

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

// Workspace of the backward pass: dz (two planes of 16-bit types but for slopes of 0 and 1), the partial sums of db, and
// the products' own.
struct BwdLayout {
  size_t plane, dz, partial, gemm, total;
  bool two;
  BwdLayout(int32_t dtype, bool slopes_01, int64_t M, int64_t N, int64_t K, bool has_slope) {
    two = has_slope && dtype != SGNN_F32 && !slopes_01;
    plane = !has_slope ? 0 : pad256(dtype_size(dtype) * (size_t)M * (size_t)N);
    dz = two ? 2 * plane : plane;
    partial = pad256(sizeof(float) * (size_t)ActCut(dtype_size(dtype), M, N).blocks * (size_t)N);
    gemm = std::max(gemm_workspace_bytes(dgrad(dtype, M, N, K)), gemm_workspace_bytes(wgrad(dtype, M, N, K)));
    total = dz + partial + gemm;
  }
};

bool take_slopes_01(int32_t& dtype) {
  const bool set = (dtype & SGNN_SLOPES_01) != 0;
  dtype &= ~SGNN_SLOPES_01;
  return set;
}

}  // namespace

extern "C" size_t sgnn_linear_workspace_bytes(int32_t dtype, int64_t M, int64_t N, int64_t K) {
  if (!sgnn::dtype_ok(dtype) || M <= 0 || N <= 0 || K <= 0) return 0;
  return sgnn::gemm_workspace_bytes(forward(dtype, M, N, K));
}

extern "C" int sgnn_linear(int32_t dtype, int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const void* w,
                           int64_t ldw, const void* bias, int32_t act, const void* residual, int64_t ldr, float* slope,
                           void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype) || !act_ok(act)) return set_error(SGNN_ERR_INVALID, "linear: unknown dtype or activation");
  if (M < 0 || N < 0 || K < 0) return set_error(SGNN_ERR_INVALID, "linear: negative size");
  if (too_many(M, N, K)) return set_error(SGNN_ERR_UNSUPPORTED, "linear: more than 2^30 rows or 2^25 columns");
  if (M == 0 || N == 0) return SGNN_OK;
  if (!y || ldy < N || (residual && ldr < N)) return set_error(SGNN_ERR_INVALID, "linear: bad output or residual");
  if (K > 0 && (!x || !w || ldx < K || ldw < K)) return set_error(SGNN_ERR_INVALID, "linear: bad operand");
  const size_t need = sgnn_linear_workspace_bytes(dtype, M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(SGNN_ERR_INVALID, "linear: workspace smaller than sgnn_linear_workspace_bytes");
  Gemm g = forward(dtype, M, N, K);
  g.A = x, g.lda = ldx;
  g.B = w, g.ldb = ldw;
  g.bias = bias, g.act = act;
  g.res = residual, g.ldr = ldr;
  g.slope = slope, g.C = y, g.ldc = ldy;
  return gemm_run(g, workspace, workspace_bytes, stream);
}

extern "C" size_t sgnn_linear_bwd_workspace_bytes(int32_t dtype, int64_t M, int64_t N, int64_t K, int32_t has_slope) {
  const bool slopes_01 = take_slopes_01(dtype);
  if (!sgnn::dtype_ok(dtype) || M <= 0 || N <= 0 || K < 0) return 0;
  return BwdLayout(dtype, slopes_01, M, N, K, has_slope != 0).total;
}

extern "C" int sgnn_linear_bwd(int32_t dtype, int64_t M, int64_t N, int64_t K, const void* dy, int64_t ldd,
                               const float* slope, const void* x, int64_t ldx, const void* w, int64_t ldw, void* dx,
                               void* dw, void* db, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sgnn;
  const int32_t asked = dtype;
  const bool slopes_01 = take_slopes_01(dtype);
  if (!dtype_ok(dtype)) return set_error(SGNN_ERR_INVALID, "linear_bwd: unknown dtype");
  if (M < 0 || N < 0 || K < 0) return set_error(SGNN_ERR_INVALID, "linear_bwd: negative size");
  if (too_many(M, N, K)) return set_error(SGNN_ERR_UNSUPPORTED, "linear_bwd: more than 2^30 rows or 2^25 columns");
  if (M > 0 && N > 0 && (!dy || ldd < N)) return set_error(SGNN_ERR_INVALID, "linear_bwd: bad dy");
  if (K > 0 && ((dx && N > 0 && (!w || ldw < K)) || (dw && M > 0 && (!x || ldx < K))))
    return set_error(SGNN_ERR_INVALID, "linear_bwd: bad operand");
  const size_t need = sgnn_linear_bwd_workspace_bytes(asked, M, N, K, slope != nullptr);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(SGNN_ERR_INVALID, "linear_bwd: workspace smaller than sgnn_linear_bwd_workspace_bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const BwdLayout at(dtype, slopes_01, M, N, K, slope != nullptr);
  char* ws = static_cast<char*>(workspace);
  const void* up = dy;      // dz and its leading dimension
  int64_t ldu = ldd, lo = 0;
  if (N > 0 && (slope || db)) {
    with_type(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      const ActCut cut(sizeof(T), M, N);
      float* partial = db ? reinterpret_cast<float*>(ws + at.dz) : nullptr;
      if (M > 0) {
        hipLaunchKernelGGL(k_act_bwd<T>, dim3((unsigned)cut.strips, (unsigned)cut.blocks), dim3(kThreads), 0, s,
                           static_cast<const T*>(dy), ldd, slope, M, N, cut.lanes, reinterpret_cast<T*>(ws),
                           at.two ? (int64_t)(at.plane / sizeof(T)) : 0, partial);
        if (slope) up = ws, ldu = N, lo = at.two ? (int64_t)at.plane : 0;
      }
      if (db)
        hipLaunchKernelGGL(k_bias_grad<T>, dim3(sum_grid(N)), dim3(kSumThreads), 0, s, partial,
                           M > 0 ? cut.blocks : 0, N, static_cast<T*>(db));
      return 0;
    });
    const int st = check_launch("linear_bwd");
    if (st != SGNN_OK) return st;
  }
  char* gws = ws + at.dz + at.partial;
  if (dx) {
    Gemm g = dgrad(dtype, M, N, K);
    g.A = up, g.lda = ldu, g.lo = lo;
    g.B = w, g.ldb = ldw;
    g.C = dx, g.ldc = K;
    const int e = gemm_run(g, gws, at.gemm, stream);
    if (e != SGNN_OK) return e;
  }
  if (dw) {
    Gemm g = wgrad(dtype, M, N, K);
    g.A = up, g.lda = ldu, g.lo = lo;
    g.B = x, g.ldb = ldx;
    g.C = dw, g.ldc = K;
    return gemm_run(g, gws, at.gemm, stream);
  }
  return SGNN_OK;
}
