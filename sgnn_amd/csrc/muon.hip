// sgnn_newton_schulz (include/sgnn.h): X = in / (|in|_F + eps), then X <- Q X, Q = a I + b G + c G^2, G = X X^T.
//
// A matrix taller than wide takes the same steps from its other side, X <- X Q with G = X^T X: no transposition.
// X, G and Q are kept as fp16 planes of the value times 2^10; the singular values of X stay below 1.3, so that all of
// them fit.  fp32 and fp16 matrices have two planes, hi + lo, 22 bits of every value that is not tiny against 1 and an
// absolute 2^-35 below that, and products hi hi + hi lo + lo hi: good to 2^-22, below what an fp32 sum of some hundred
// products loses.  bf16 matrices have the hi plane alone, a third of the instructions: its 11 bits are 3 more than
// their elements have, and a I inside Q keeps the sum a X + (b G + c G^2) X, whose terms cancel to a fifth near 1,
// out of the rounding.  The planes are padded with zeros to whole tiles (zeros stay zeros under the steps), so nothing
// is checked inside the products; the last one writes the caller's type from its fp32 sums.
#include "gemm_tile.h"

namespace {
using namespace sgnn;

constexpr float kScale = 1024.0f, kInvScale = 1.0f / 1024.0f;
constexpr int kMaxGroup = 32;  // matrices of one shape per launch (their pointers are kernel arguments)
constexpr int kNormParts = 64; // partial sums of squares per matrix

struct Group {
  int32_t rows, cols, count;
  const void* in[kMaxGroup];
  void* out[kMaxGroup];
  int64_t ld_in[kMaxGroup], ld_out[kMaxGroup];
};

// Sums of squares in 64 bits: the square of a gradient leaves fp32's range long before the gradient does.
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(Group g, double* part) {
  __shared__ double red[4];
  constexpr int V = 16 / sizeof(T);
  const int b = blockIdx.y;
  const T* in = static_cast<const T*>(g.in[b]);
  const int per = (g.cols + V - 1) / V;
  const int64_t total = (int64_t)g.rows * per;
  double s = 0.0;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / per;
    const int c = (int)(t - r * per) * V;
    float v[V];
    load_some<V>(in + r * g.ld_in[b] + c, g.cols - c, v);
#pragma unroll
    for (int i = 0; i < V; ++i) s += (double)v[i] * (double)v[i];
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane_id() == 0) red[wave_id()] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[b * gridDim.x + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// Eight values times scale into the planes, at a 16-byte address.
template <int P>
SGNN_DEV void put_planes(f16_t* p, int64_t plane, const float* v, float scale) {
  typedef f16_t h8 __attribute__((ext_vector_type(8)));
  h8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = v[i] * scale;
    const f16_t h = (f16_t)x;
    hi[i] = h, lo[i] = (f16_t)(x - (float)h);
  }
  *reinterpret_cast<h8*>(p) = hi;
  if constexpr (P == 2) *reinterpret_cast<h8*>(p + plane) = lo;
}

// The planes of in / (|in|_F + eps), zero in the padding; one thread per 8 columns.  Without steps (x null) the
// values go to out.
template <typename T, int P>
__global__ __launch_bounds__(256) void k_ns_begin(Group g, const double* part, int nparts, float eps, f16_t* x,
                                                  int64_t plane, int64_t batch, int64_t ld, int64_t rows_padded) {
  const int b = blockIdx.y;
  double s = 0.0;
  for (int i = 0; i < nparts; ++i) s += part[b * nparts + i];
  const float norm = (float)sqrt(s) + eps;
  const T* in = static_cast<const T*>(g.in[b]);
  const int64_t per = ld / 8, total = rows_padded * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / per, c = (t - r * per) * 8;
    const bool there = r < g.rows && c < g.cols;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (there) load_some<8>(in + r * g.ld_in[b] + c, (int)(g.cols - c), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = norm == 0.0f ? 0.0f : v[i] / norm;  // only zeros have the norm 0
    if (x)
      put_planes<P>(x + b * batch + r * ld + c, plane, v, kScale);
    else if (there)
      store_some<8>(static_cast<T*>(g.out[b]) + r * g.ld_out[b] + c, (int)(g.cols - c), v);
  }
}

// C = alpha A B^T + beta R + diag I on planes, all of them padded to whole tiles; last: into last's outputs instead.
struct NsGemm {
  const f16_t *A, *B, *R;
  f16_t* C;
  int64_t lda, ldb, ldc, plane_a, plane_b, plane_c, batch_a, batch_b, batch_c;  // R is laid out as C
  int32_t K, tiles_m, tiles_n, last_dtype;  // last_dtype: -1 but for the last product
  float alpha, beta, diag;
  Group last;
};

// BT x BT outputs by four waves.  P planes per operand (1: hi alone).  SYM: the product is symmetric; only the tiles
// on and above the diagonal are formed and each is written to both sides.
template <int P, bool AC, bool BC, int BT, bool SYM>
__global__ __launch_bounds__(256) void k_ns_gemm(NsGemm g) {
  constexpr int BK = 64 / P, kThreads = 256, TT = BT / 2 / 16;
  using TA = Tile16<BT, BK, AC>;
  using TB = Tile16<BT, BK, BC>;
  constexpr int kStage = 2 * P * TA::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
  const int w = wave_id(), wm = w >> 1, wn = w & 1, l = lane_id();
  int tm, tn;
  if constexpr (SYM) {  // row tm of the triangle holds tiles_n - tm tiles
    int t = blockIdx.x;
    tm = 0;
    while (t >= g.tiles_n - tm) t -= g.tiles_n - tm, ++tm;
    tn = tm + t;
  } else {  // XCD x (workgroups x, x + 8, ...) takes the x-th contiguous share of the tiles, column tiles first
    const int total = g.tiles_m * g.tiles_n, xcd = blockIdx.x & 7, q = total >> 3, r = total & 7;
    const int t = xcd * q + min(xcd, r) + (blockIdx.x >> 3);
    tm = t / g.tiles_n, tn = t - tm * g.tiles_n;
  }
  const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane(tm) * BT;
  const int64_t n0 = (int64_t)__builtin_amdgcn_readfirstlane(tn) * BT;
  const int64_t b = blockIdx.z;

  f32x4 acc[TT][TT];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  constexpr int PER = BT * BK / 8 / kThreads;
  uint32_t oa[PER], ob[PER];
  TA::template offsets<kThreads>(oa, g.lda, BT, 0);
  TB::template offsets<kThreads>(ob, g.ldb, BT, 0);
  const char* pa = reinterpret_cast<const char*>(g.A + b * g.batch_a + (AC ? m0 : m0 * g.lda));
  const char* pb = reinterpret_cast<const char*>(g.B + b * g.batch_b + (BC ? n0 : n0 * g.ldb));
  const int64_t sa = 2 * BK * (AC ? g.lda : 1), sb = 2 * BK * (BC ? g.ldb : 1);
  const auto stage = [&](char* to, int blk) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      TA::template direct<kThreads>(to + p * TA::kBytes, pa + 2 * p * g.plane_a + blk * sa, oa);
      TB::template direct<kThreads>(to + (P + p) * TA::kBytes, pb + 2 * p * g.plane_b + blk * sb, ob);
    }
  };
  const int blocks = g.K / BK;
  char* here = lds;
  char* there = lds + kStage;
  stage(here, 0);
  for (int blk = 0; blk < blocks; ++blk) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (blk + 1 < blocks) stage(there, blk + 1);
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      s16x8 fa[P][TT], fb[P][TT];
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          fa[p][i] = TA::frag(here + p * TA::kBytes, (wm * TT + i) * 16, kk);
          fb[p][i] = TB::frag(here + (P + p) * TA::kBytes, (wn * TT + i) * 16, kk);
        }
      if constexpr (P == 2) {
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int j = 0; j < TT; ++j) acc[i][j] = mfma16<f16_t>(fb[1][j], fa[0][i], acc[i][j]);
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int j = 0; j < TT; ++j) acc[i][j] = mfma16<f16_t>(fb[0][j], fa[1][i], acc[i][j]);
      }
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = mfma16<f16_t>(fb[0][j], fa[0][i], acc[i][j]);
    }
    char* t = here;
    here = there, there = t;
  }
  __syncthreads();
  // through LDS by 16 rows of m (as in gemm.hip), so that every load and store is 16 bytes of a row
  constexpr int kPieces = 4 * TT, kMask = kPieces - 1;
  float* buf = reinterpret_cast<float*>(lds) + w * 16 * 16 * TT;
  const float alpha = g.alpha * kInvScale * kInvScale;
  const f16_t* R = g.R ? g.R + b * g.batch_c : nullptr;
  f16_t* C = g.C + b * g.batch_c;
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    const int lm = l & 15;
#pragma unroll
    for (int j = 0; j < TT; ++j)
      *reinterpret_cast<f32x4*>(buf + lm * 16 * TT + ((4 * j + (l >> 4)) ^ (lm & kMask)) * 4) = acc[i][j];
    __builtin_amdgcn_wave_barrier();
    const int64_t mi = m0 + (wm * TT + i) * 16, ni = n0 + wn * TT * 16;
#pragma unroll 1
    for (int t = l; t < 16 * kPieces / 2; t += 64) {
      const int r = t / (kPieces / 2), p = t % (kPieces / 2) * 2;
      float* at0 = buf + r * 16 * TT + (p ^ (r & kMask)) * 4;
      float* at1 = buf + r * 16 * TT + ((p + 1) ^ (r & kMask)) * 4;
      const f32x4 v0 = *reinterpret_cast<const f32x4*>(at0), v1 = *reinterpret_cast<const f32x4*>(at1);
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = alpha * v0[e], v[4 + e] = alpha * v1[e];
      const int64_t m = mi + r, n = ni + 4 * p, at = m * g.ldc + n;
      if constexpr (SYM) {
        if (R) {
          float hi[8], lo[8];
          load_vec(R + at, hi);
          if constexpr (P == 2) load_vec(R + g.plane_c + at, lo);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] += g.beta * kInvScale * (P == 2 ? hi[e] + lo[e] : hi[e]);
            if (n + e == m) v[e] += g.diag;
          }
        }
        // the values back into the buffer for the mirrored tile
        *reinterpret_cast<f32x4*>(at0) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(at1) = f32x4{v[4], v[5], v[6], v[7]};
        put_planes<P>(C + at, g.plane_c, v, kScale);
      } else if (g.last_dtype < 0) {
        put_planes<P>(C + at, g.plane_c, v, kScale);
      } else if (m < g.last.rows && n < g.last.cols) {
        const int64_t to = m * g.last.ld_out[b] + n;
        const int cnt = (int)(g.last.cols - n);
        if constexpr (P == 1) store_some<8>(static_cast<bf16_t*>(g.last.out[b]) + to, cnt, v);
        else if (g.last_dtype == SGNN_F32) store_some<8>(static_cast<float*>(g.last.out[b]) + to, cnt, v);
        else store_some<8>(static_cast<f16_t*>(g.last.out[b]) + to, cnt, v);
      }
    }
    __builtin_amdgcn_wave_barrier();
    if constexpr (SYM) {
      if (tm != tn) {
#pragma unroll 1
        for (int t = l; t < 2 * 16 * TT; t += 64) {  // column n of the tile, 8 of its 16 m
          const int n = t >> 1, r0 = (t & 1) * 8;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int r = r0 + e;
            v[e] = buf[r * 16 * TT + ((n >> 2) ^ (r & kMask)) * 4 + (n & 3)];
          }
          put_planes<P>(C + (ni + n) * g.ldc + mi + r0, g.plane_c, v, kScale);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
}

template <int P, bool AC, bool BC, bool SYM>
void launch_gemm(const NsGemm& g, int bt, int count, hipStream_t s) {
  const int tiles = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
  const dim3 grid((unsigned)tiles, 1, (unsigned)count);
  if (bt == 128) hipLaunchKernelGGL((k_ns_gemm<P, AC, BC, 128, SYM>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((k_ns_gemm<P, AC, BC, 64, SYM>), grid, dim3(256), 0, s, g);
}

size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

// A group's workspace: the norms' partial sums, X twice, G and Q, each two planes.
struct NsLayout {
  int bt;
  int64_t rows, cols, side;  // padded; side: of G
  size_t norms, x, g, total;
  NsLayout(int32_t r, int32_t c, int count) {
    const int64_t small = std::min(r, c), large = std::max(r, c);
    // 128-tiles read half as much per product; the smaller ones pad less and fill the CUs sooner
    bt = (small * large + 128 * 128 - 1) / (128 * 128) * count >= 192 && small > 64 ? 128 : 64;
    rows = (r + bt - 1) / bt * bt, cols = (c + bt - 1) / bt * bt, side = std::min(rows, cols);
    norms = pad256(sizeof(double) * kNormParts * count);
    x = pad256(2 * sizeof(f16_t) * rows * cols * count);
    g = pad256(2 * sizeof(f16_t) * side * side * count);
    total = norms + 2 * x + 2 * g;
  }
};

// The matrices from i on that share a launch: one shape, next to each other.
int32_t run_of(const sgnn_matrix* mats, int32_t count, int32_t i) {
  int32_t n = 1;
  while (i + n < count && n < kMaxGroup && mats[i + n].rows == mats[i].rows && mats[i + n].cols == mats[i].cols) ++n;
  return n;
}

template <typename T>
void orthogonalise(const Group& grp, int32_t steps, float a, float b, float c, float eps, char* ws, hipStream_t s) {
  const NsLayout at(grp.rows, grp.cols, grp.count);
  const bool tall = grp.rows > grp.cols;
  double* norms = reinterpret_cast<double*>(ws);
  f16_t* x = reinterpret_cast<f16_t*>(ws + at.norms);
  f16_t* next = reinterpret_cast<f16_t*>(ws + at.norms + at.x);
  f16_t* gram = reinterpret_cast<f16_t*>(ws + at.norms + 2 * at.x);
  f16_t* poly = reinterpret_cast<f16_t*>(ws + at.norms + 2 * at.x + at.g);
  const int64_t batch_x = at.rows * at.cols, plane_x = batch_x * grp.count;
  const int64_t batch_g = at.side * at.side, plane_g = batch_g * grp.count;
  const auto blocks = [](int64_t items, int64_t most) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, most));
  };
  const int parts = (int)blocks((int64_t)grp.rows * grp.cols / 8, kNormParts);
  hipLaunchKernelGGL(k_ns_norm<T>, dim3(parts, grp.count), dim3(256), 0, s, grp, norms);
  constexpr int P = std::is_same_v<T, bf16_t> ? 1 : 2;
  hipLaunchKernelGGL((k_ns_begin<T, P>), dim3(blocks(batch_x / 8, 4096), grp.count), dim3(256), 0, s, grp, norms, parts,
                     eps, steps > 0 ? x : nullptr, plane_x, batch_x, at.cols, at.rows);
  for (int32_t k = 0; k < steps; ++k) {
    NsGemm g{};
    g.last_dtype = -1;
    g.tiles_m = g.tiles_n = (int32_t)(at.side / at.bt);
    g.A = g.B = x, g.lda = g.ldb = at.cols, g.plane_a = g.plane_b = plane_x, g.batch_a = g.batch_b = batch_x;
    g.C = gram, g.ldc = at.side, g.plane_c = plane_g, g.batch_c = batch_g;
    g.alpha = 1.0f;
    g.K = (int32_t)(tall ? at.rows : at.cols);
    if (tall) launch_gemm<P, true, true, true>(g, at.bt, grp.count, s);
    else launch_gemm<P, false, false, true>(g, at.bt, grp.count, s);
    g.A = g.B = g.R = gram, g.lda = g.ldb = at.side, g.plane_a = g.plane_b = plane_g, g.batch_a = g.batch_b = batch_g;
    g.C = poly;
    g.alpha = c, g.beta = b, g.diag = a;
    g.K = (int32_t)at.side;
    launch_gemm<P, false, false, true>(g, at.bt, grp.count, s);
    g.R = nullptr, g.C = next, g.ldc = at.cols, g.plane_c = plane_x, g.batch_c = batch_x;
    g.alpha = 1.0f;
    g.tiles_m = (int32_t)(at.rows / at.bt), g.tiles_n = (int32_t)(at.cols / at.bt);
    if (k + 1 == steps) {
      g.last_dtype = std::is_same_v<T, float> ? SGNN_F32 : std::is_same_v<T, bf16_t> ? SGNN_BF16 : SGNN_F16;
      g.last = grp;
    }
    if (tall) {  // X Q: Q is symmetric, its rows are its columns
      g.A = x, g.lda = at.cols, g.plane_a = plane_x, g.batch_a = batch_x;
      g.B = poly;
      launch_gemm<P, false, false, false>(g, at.bt, grp.count, s);
    } else {     // Q X
      g.A = poly;
      g.B = x, g.ldb = at.cols, g.plane_b = plane_x, g.batch_b = batch_x;
      launch_gemm<P, false, true, false>(g, at.bt, grp.count, s);
    }
    std::swap(x, next);
  }
}

}  // namespace

extern "C" size_t sgnn_newton_schulz_workspace_bytes(const sgnn_matrix* mats, int32_t count) {
  size_t most = 0;
  for (int32_t i = 0, n; mats && i < count; i += n) {
    n = run_of(mats, count, i);
    if (mats[i].rows > 0 && mats[i].cols > 0) most = std::max(most, NsLayout(mats[i].rows, mats[i].cols, n).total);
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
    // the tiles' 32-bit offsets: 64 lines of 2 bytes a value
    if (std::max(t.rows, t.cols) > (1 << 22)) return set_error(SGNN_ERR_UNSUPPORTED, "newton_schulz: more than 4M rows or columns");
  }
  if (workspace_bytes < sgnn_newton_schulz_workspace_bytes(mats, count))
    return set_error(SGNN_ERR_INVALID, "newton_schulz: workspace smaller than sgnn_newton_schulz_workspace_bytes");
  for (int32_t i = 0, n; i < count; i += n) {
    n = run_of(mats, count, i);
    if (mats[i].rows == 0 || mats[i].cols == 0) continue;
    Group grp;
    grp.rows = mats[i].rows, grp.cols = mats[i].cols, grp.count = n;
    for (int32_t k = 0; k < n; ++k) {
      grp.in[k] = mats[i + k].in, grp.out[k] = mats[i + k].out;
      grp.ld_in[k] = mats[i + k].ld_in, grp.ld_out[k] = mats[i + k].ld_out;
    }
    with_type(dtype, [&](auto* t) {
      orthogonalise<std::remove_pointer_t<decltype(t)>>(grp, steps, a, b, c, eps, static_cast<char*>(workspace),
                                                        static_cast<hipStream_t>(stream));
      return 0;
    });
    const int st = check_launch("newton_schulz");
    if (st != SGNN_OK) return st;
  }
  return SGNN_OK;
}
