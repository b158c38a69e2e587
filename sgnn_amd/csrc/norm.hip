// sgnn_norm and its backward pass (include/sgnn.h): LayerNorm over rows, with the reductions of the weight's and
// the bias's gradient in the pass over the rows that forms dx.
#include "ops_types.h"

namespace {
using namespace sgnn;

// Rows are held in registers: G lanes per row (16, 64, or a workgroup of 256 or 512), NC 16-byte pieces per lane,
// piece j of lane i at column (j G + i) V.  Forward and backward read every input once and write every output once:
// both are bounded by memory, where a copy reaches 6.2 TB/s: 200003 x 128 fp32 34 us forward (6.0 TB/s) and 52 + 5
// backward (5.9); 16384 x 4096 bf16 52 us (5.2) and 84 + 9 (4.8: gamma and the sums hold the registers that another row
// in flight would need, and every row has its barrier).
constexpr int threads_of(int G) { return G > 256 ? G : 256; }

// Sum over a row's G lanes; `red` is 2 x 16 floats of LDS, `turn` the half to use (the other may still be read).
template <int G>
SGNN_DEV float group_sum(float v, float* red, int turn) {
  if constexpr (G <= 64) return lanes_sum<G>(v);
  v = lanes_sum<64>(v);
  float* r = red + 16 * turn;
  if (lane_id() == 0) r[wave_id()] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < G / 64; ++w) s += r[w];
  return s;
}

// Mean, then the variance of the differences (both from registers), then the outputs; kRows rows per group of lanes
// in turn, so that gamma and beta are read once for them.
template <typename T, typename W, int G, int NC>
__global__ __launch_bounds__(threads_of(G)) void k_norm(const T* x, int64_t ldx, int64_t n, int width, const W* gamma,
                                                        const W* beta, const T* residual, int64_t ldr, float eps, T* y,
                                                        float* mean_out, float* rstd_out, int rows_per) {
  constexpr int V = 16 / sizeof(T), kGroups = threads_of(G) / G;
  __shared__ float red[32];
  const int i = threadIdx.x % G;
  float ga[NC][V], be[NC][V];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (j * G + i) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ga[j][e] = 1.0f, be[j][e] = 0.0f;
    if (gamma) load_some<V>(gamma + c, width - c, ga[j]);
    if (beta) load_some<V>(beta + c, width - c, be[j]);
  }
  const int64_t r0 = (int64_t)blockIdx.x * rows_per * kGroups + threadIdx.x / G;
  for (int q = 0; q < rows_per; ++q) {
    const int64_t r = r0 + (int64_t)q * kGroups;
    if (r >= n) break;  // the lanes of one row leave together
    float v[NC][V];
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + i) * V;
      load_some<V>(x + r * ldx + c, width - c, v[j]);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[j][e];
    const float mean = group_sum<G>(s, red, 0) / width;
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[j][e] -= mean;
        if ((j * G + i) * V + e < width) s += v[j][e] * v[j][e];
      }
    const float rstd = 1.0f / sqrtf(group_sum<G>(s, red, 1) / width + eps);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + i) * V;
      if (c >= width) continue;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = v[j][e] * rstd * ga[j][e] + be[j][e];
      if (residual) {
        float t[V];
        load_some<V>(residual + r * ldr + c, width - c, t);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] += t[e];
      }
      store_some<V>(y + r * width + c, width - c, o);
    }
    if (i == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
  }
}

// Two sums over a row's G lanes at once; turn: as in group_sum.
template <int G>
SGNN_DEV void group_sum2(float& a, float& b, float* red, int turn) {
  a = lanes_sum<G <= 64 ? G : 64>(a);
  b = lanes_sum<G <= 64 ? G : 64>(b);
  if constexpr (G > 64) {
    float* r = red + 2 * (G / 64) * turn;
    if (lane_id() == 0) r[2 * wave_id()] = a, r[2 * wave_id() + 1] = b;
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) a += r[2 * w], b += r[2 * w + 1];
  }
}

// dx, and this workgroup's share of dgamma and dbeta: every lane sums its own columns over its rows (rows blockIdx,
// + gridDim ... in order), the groups of one workgroup are added in order in LDS, and the workgroups' sums go to
// partial [workgroup][2][width].  A row waits in registers as it was loaded (16-bit values packed) and is unpacked for
// its sums and again for dx; the next row is loaded before this one's sums are waited for.
template <typename T, typename W, int G, int NC>
__global__ __launch_bounds__(threads_of(G)) void k_norm_bwd(const T* dy, int64_t ldd, const T* x, int64_t ldx,
                                                            const float* mean, const float* rstd, const W* gamma,
                                                            int64_t n, int width, T* dx, float* partial) {
  constexpr int V = 16 / sizeof(T), kGroups = threads_of(G) / G;
  __shared__ float red[G > 64 ? 4 * G / 64 : 1];
  __shared__ float join[kGroups > 1 ? (kGroups - 1) * G * NC * V : 1];
  const int i = threadIdx.x % G, grp = threadIdx.x / G;
  float ga[NC][V], dg[NC][V], db[NC][V];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (j * G + i) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ga[j][e] = 1.0f, dg[j][e] = 0.0f, db[j][e] = 0.0f;
    if (gamma) load_some<V>(gamma + c, width - c, ga[j]);
  }
  const int64_t step = (int64_t)gridDim.x * kGroups;
  u32x4 nx[NC], nu[NC];
  float nmu = 0.0f, nrs = 0.0f;
  const auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + i) * V;
      nx[j] = load_raw(x + r * ldx + c, width - c);
      nu[j] = load_raw(dy + r * ldd + c, width - c);
    }
    nmu = mean[r], nrs = rstd[r];
  };
  int64_t r = (int64_t)blockIdx.x * kGroups + grp;
  if (r < n) load(r);
  for (int turn = 0; r < n; r += step, turn ^= 1) {
    u32x4 vx[NC], vu[NC];
    const float mu = nmu, rs = nrs;
#pragma unroll
    for (int j = 0; j < NC; ++j) vx[j] = nx[j], vu[j] = nu[j];
    if (r + step < n) load(r + step);
    float sg = 0.0f, sgh = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      float xv[V], up[V];
      unpack<T>(vx[j], xv);
      unpack<T>(vu[j], up);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // columns past the row read as 0 in dy: nothing of theirs is summed
        const float hat = (xv[e] - mu) * rs, g = up[e] * ga[j][e];
        dg[j][e] += up[e] * hat;
        db[j][e] += up[e];
        sg += g;
        sgh += g * hat;
      }
    }
    if (dx) {
      group_sum2<G>(sg, sgh, red, turn);
      sg /= width, sgh /= width;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = (j * G + i) * V;
        if (c >= width) continue;
        float xv[V], o[V];
        // unpacked anew: the floats of the first time would be twice the registers across the barrier
        asm volatile("" : "+v"(vx[j]), "+v"(vu[j]));
        unpack<T>(vx[j], xv);
        unpack<T>(vu[j], o);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = rs * (o[e] * ga[j][e] - sg - (xv[e] - mu) * rs * sgh);
        store_some<V>(dx + r * width + c, width - c, o);
      }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&a)[NC][V] = which == 0 ? dg : db;
    if constexpr (kGroups > 1) {
      if (grp > 0)
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) join[((grp - 1) * NC * V + j * V + e) * G + i] = a[j][e];
      __syncthreads();
      if (grp == 0)
        for (int q = 0; q < kGroups - 1; ++q)
#pragma unroll
          for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) a[j][e] += join[(q * NC * V + j * V + e) * G + i];
      __syncthreads();
    }
    if (grp == 0)
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = (j * G + i) * V;
        if (c < width) store_some<V>(partial + ((int64_t)blockIdx.x * 2 + which) * width + c, width - c, a[j]);
      }
  }
}

// Rows longer than 512 lanes hold: a workgroup per row, read again for each of the steps (from L2 where it is still
// there).
constexpr int kMaxWidth = 8192, kWide = 1024;

template <typename T>
SGNN_DEV float at_or(const T* p, int c, float none) {
  return p ? to_float(p[c]) : none;
}

template <typename T, typename W>
__global__ __launch_bounds__(kWide) void k_norm_wide(const T* x, int64_t ldx, int64_t n, int width, const W* gamma,
                                                     const W* beta, const T* residual, int64_t ldr, float eps, T* y,
                                                     float* mean_out, float* rstd_out) {
  __shared__ float red[32];
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
    const T* p = x + r * ldx;
    float s = 0.0f;
    for (int c = threadIdx.x; c < width; c += kWide) s += to_float(p[c]);
    const float mean = group_sum<kWide>(s, red, 0) / width;
    s = 0.0f;
    for (int c = threadIdx.x; c < width; c += kWide) {
      const float d = to_float(p[c]) - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(group_sum<kWide>(s, red, 1) / width + eps);
    for (int c = threadIdx.x; c < width; c += kWide) {
      const float o = (to_float(p[c]) - mean) * rstd * at_or(gamma, c, 1.0f) + at_or(beta, c, 0.0f);
      y[r * width + c] = from_float<T>(o + (residual ? to_float(residual[r * ldr + c]) : 0.0f));
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(kWide) void k_norm_bwd_wide(const T* dy, int64_t ldd, const T* x, int64_t ldx,
                                                         const float* mean, const float* rstd, const W* gamma,
                                                         int64_t n, int width, T* dx) {
  __shared__ float red[2][32];
  int turn = 0;
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x, turn ^= 1) {
    const float mu = mean[r], rs = rstd[r];
    float sg = 0.0f, sgh = 0.0f;
    for (int c = threadIdx.x; c < width; c += kWide) {
      const float g = to_float(dy[r * ldd + c]) * at_or(gamma, c, 1.0f);
      sg += g;
      sgh += g * (to_float(x[r * ldx + c]) - mu) * rs;
    }
    sg = group_sum<kWide>(sg, red[0], turn) / width;
    sgh = group_sum<kWide>(sgh, red[1], turn) / width;
    for (int c = threadIdx.x; c < width; c += kWide) {
      const float g = to_float(dy[r * ldd + c]) * at_or(gamma, c, 1.0f);
      dx[r * width + c] = from_float<T>(rs * (g - sg - (to_float(x[r * ldx + c]) - mu) * rs * sgh));
    }
  }
}

// One thread per column over every gridDim.x-th row.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_sums_wide(const T* dy, int64_t ldd, const T* x, int64_t ldx,
                                                        const float* mean, const float* rstd, int64_t n, int width,
                                                        float* partial) {
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= width) return;
  float dg = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
    const float g = to_float(dy[r * ldd + c]);
    dg += g * (to_float(x[r * ldx + c]) - mean[r]) * rstd[r];
    db += g;
  }
  partial[(int64_t)blockIdx.x * 2 * width + c] = dg;
  partial[(int64_t)blockIdx.x * 2 * width + width + c] = db;
}

template <typename W>
__global__ __launch_bounds__(kSumThreads) void k_norm_reduce(const float* partial, int64_t nblk, int width, W* dgamma,
                                                             W* dbeta) {
  sum_partials(partial, nblk, 2 * (int64_t)width, [&](int64_t c, float s) {
    if (c < width) {
      if (dgamma) dgamma[c] = from_float<W>(s);
    } else if (dbeta) {
      dbeta[c - width] = from_float<W>(s);
    }
  });
}

constexpr int kMostWidth = 1 << 23;  // the column blocks of k_norm_sums_wide are the grid's second dimension (65535)

// Lanes per row and pieces per lane: the fewest lanes that leave a lane at most 16 values (the backward pass holds
// gamma and its two sums of them).
struct NormCut {
  int G, NC;  // G = 0: the wide kernels
  NormCut(size_t size, int width) {
    G = width <= 256 ? 16 : width <= 1024 ? 64 : width <= 4096 ? 256 : width <= kMaxWidth ? 512 : 0;
    const int per = G ? (width + G - 1) / G * (int)size : 0;  // bytes per lane
    NC = per <= 16 ? 1 : per <= 32 ? 2 : 4;
  }
};

// Workgroups of the backward pass, which are also the partial sums: as many as the registers of 4, 8 or 16 values per
// lane let reside at once, never more than there are rows for (1024 and 2048 before, where a second round of fewer
// workgroups followed: 16384 x 4096 bf16 88 + 12 us, 50000 x 1024 bf16 69 us in all against 60).
int64_t bwd_blocks(const NormCut& cut, size_t size, int64_t n) {
  const int64_t groups = cut.G == 0 || cut.G > 256 ? 1 : 256 / cut.G;
  const int values = cut.NC * 16 / (int)size;
  const int64_t most = 256 * (cut.G == 0 ? 2 : cut.G > 256 ? (values <= 4 ? 3 : values <= 8 ? 2 : 1) : values <= 4 ? 8 : values <= 8 ? 5 : 3);
  return std::max<int64_t>(1, std::min(most, (n + groups - 1) / groups));
}

template <typename T, typename F>
void with_cut(const NormCut& cut, F f) {
  const auto nc = [&](auto g) {
    if (cut.NC == 1) f(g, std::integral_constant<int, 1>{});
    else if (cut.NC == 2) f(g, std::integral_constant<int, 2>{});
    else if constexpr (sizeof(T) == 4) f(g, std::integral_constant<int, 4>{});  // 16 values are two pieces of 16 bits
  };
  if (cut.G == 16) nc(std::integral_constant<int, 16>{});
  else if (cut.G == 64) nc(std::integral_constant<int, 64>{});
  else if (cut.G == 256) nc(std::integral_constant<int, 256>{});
  else nc(std::integral_constant<int, 512>{});
}

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
  if (width > kMostWidth) return set_error(SGNN_ERR_UNSUPPORTED, "norm: more than 8M columns");
  if (n == 0) return SGNN_OK;
  if (!x || !y || ldx < width || (residual && ldr < width)) return set_error(SGNN_ERR_INVALID, "norm: bad operand");
  with_types(dtype, wdtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    const NormCut cut(sizeof(T), width);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const T *in = static_cast<const T*>(x), *res = static_cast<const T*>(residual);
    const W *ga = static_cast<const W*>(gamma), *be = static_cast<const W*>(beta);
    T* out = static_cast<T*>(y);
    if (cut.G == 0) {
      hipLaunchKernelGGL((k_norm_wide<T, W>), dim3((unsigned)std::min<int64_t>(n, 4096)), dim3(kWide), 0, s, in, ldx, n,
                         width, ga, be, res, ldr, eps, out, mean, rstd);
      return 0;
    }
    with_cut<T>(cut, [&](auto g, auto nc) {
      constexpr int G = decltype(g)::value, NC = decltype(nc)::value, kGroups = threads_of(G) / G;
      // several rows per group once there are enough for 16 workgroups on every CU; as many as keep a launch below 2^32
      // threads
      const int64_t per = std::max<int64_t>(1, std::min<int64_t>(4, n / (kGroups * 4096))) + n / kGroups / (1 << 22);
      hipLaunchKernelGGL((k_norm<T, W, G, NC>), dim3((unsigned)((n + kGroups * per - 1) / (kGroups * per))),
                         dim3(threads_of(G)), 0, s, in, ldx, n, width, ga, be, res, ldr, eps, out, mean, rstd, (int)per);
    });
    return 0;
  });
  return check_launch("norm");
}

extern "C" size_t sgnn_norm_bwd_workspace_bytes(int64_t n, int32_t width) {
  if (n <= 0 || width <= 0) return 0;
  const auto blocks = [&](size_t size) { return bwd_blocks(NormCut(size, width), size, n); };
  return sizeof(float) * 2 * (size_t)width * (size_t)std::max(blocks(2), blocks(4));
}

extern "C" int sgnn_norm_bwd(int32_t dtype, int32_t wdtype, const void* dy, int64_t ldd, const void* x, int64_t ldx,
                             const float* mean, const float* rstd, const void* gamma, int64_t n, int32_t width,
                             void* dx, void* dgamma, void* dbeta, void* workspace, size_t workspace_bytes,
                             void* stream) {
  using namespace sgnn;
  if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != SGNN_F32))
    return set_error(SGNN_ERR_INVALID, "norm_bwd: unknown dtype, or a weight type that is neither dtype nor fp32");
  if (n < 0 || width < 1) return set_error(SGNN_ERR_INVALID, "norm_bwd: bad size");
  if (width > kMostWidth) return set_error(SGNN_ERR_UNSUPPORTED, "norm_bwd: more than 8M columns");
  if (n > 0 && (!dy || !x || !mean || !rstd || ldd < width || ldx < width))
    return set_error(SGNN_ERR_INVALID, "norm_bwd: bad operand");
  const bool sums = dgamma || dbeta;
  if (sums && n > 0 && (!workspace || workspace_bytes < sgnn_norm_bwd_workspace_bytes(n, width)))
    return set_error(SGNN_ERR_INVALID, "norm_bwd: workspace smaller than sgnn_norm_bwd_workspace_bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  with_types(dtype, wdtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    const NormCut cut(sizeof(T), width);
    const int64_t nblk = n > 0 ? bwd_blocks(cut, sizeof(T), n) : 0;
    const T *up = static_cast<const T*>(dy), *in = static_cast<const T*>(x);
    const W* ga = static_cast<const W*>(gamma);
    T* out = static_cast<T*>(dx);
    if (n > 0 && cut.G == 0) {
      if (dx)
        hipLaunchKernelGGL((k_norm_bwd_wide<T, W>), dim3((unsigned)std::min<int64_t>(n, 4096)), dim3(kWide), 0, s, up,
                           ldd, in, ldx, mean, rstd, ga, n, width, out);
      if (sums)
        hipLaunchKernelGGL(k_norm_sums_wide<T>, dim3((unsigned)nblk, (unsigned)((width + 255) / 256)), dim3(256), 0, s,
                           up, ldd, in, ldx, mean, rstd, n, width, part);
    } else if (n > 0 && (dx || sums)) {
      with_cut<T>(cut, [&](auto g, auto nc) {
        constexpr int G = decltype(g)::value, NC = decltype(nc)::value;
        hipLaunchKernelGGL((k_norm_bwd<T, W, G, NC>), dim3((unsigned)nblk), dim3(threads_of(G)), 0, s, up, ldd, in, ldx,
                           mean, rstd, ga, n, width, out, part);
      });
    }
    if (sums)
      hipLaunchKernelGGL(k_norm_reduce<W>, dim3(sum_grid(2 * (int64_t)width)), dim3(kSumThreads), 0, s, part, nblk,
                         width, static_cast<W*>(dgamma), static_cast<W*>(dbeta));
    return 0;
  });
  return check_launch("norm_bwd");
}
