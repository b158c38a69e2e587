// sgnn_newton_schulz (include/sgnn.h): X = in / (|in|_F + eps), then X <- Q X, Q = a I + b G + c G^2, G = X X^T.
//
// A matrix taller than wide takes the same steps from its other side, X <- X Q with G = X^T X: no transposition.
// X, G and Q are kept as two fp16 planes, hi + lo, of the value times 2^10; the singular values of X stay below 1.3, so
// that all of them fit: 22 bits of every value that is not tiny against 1 and an absolute 2^-35 below that.  Products
// are hi hi + hi lo + lo hi, good to 2^-22, below what an fp32 sum of some hundred products loses, and a I inside Q
// keeps the sum a X + (b G + c G^2) X, whose terms cancel to a fifth near 1, out of the rounding.  This holds for every
// type of matrix: with the hi plane alone bf16 ones took 537 us instead of 1250 to 1380 (4096 x 2048), but fifteen roundings to
// 11 bits come out beside the one of the result (error 0.0028 instead of 0.0017 for a small matrix).  The planes are
// padded with zeros to whole tiles (zeros stay zeros under the steps), so nothing is checked inside the products; the
// last one writes the caller's type from its fp32 sums.
#include "gemm_tile.h"

namespace {
using namespace sgnn;

constexpr float kScale = 1024.0f, kInvScale = 1.0f / 1024.0f;
constexpr int kPlanes = 2;     // hi, lo
constexpr int kMaxGroup = 32;  // matrices of one shape per launch (their pointers are kernel arguments)
constexpr int kNormParts = 256; // partial sums of squares per matrix, at most

struct Group {
  int32_t rows, cols, count;
  const void* in[kMaxGroup];
  void* out[kMaxGroup];
  int64_t ld_in[kMaxGroup], ld_out[kMaxGroup];
};

// Sums of squares in 64 bits: the square of a gradient leaves fp32's range long before the gradient does.  Up to 256
// partial sums a matrix, so that k_ns_begin adds them with one thread each (2048 x 4096 bf16: 8.3 us, 10.4 with one load
// under way).
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(Group g, double* part) {
  __shared__ double red[4];
  constexpr int V = 16 / sizeof(T);
  const int b = blockIdx.y;
  const T* in = static_cast<const T*>(g.in[b]);
  const int per = (g.cols + V - 1) / V;
  const int64_t total = (int64_t)g.rows * per;
  double s = 0.0;
  constexpr int U = 4;  // loads under way before the first is used
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t t0 = (int64_t)blockIdx.x * 256 + threadIdx.x; t0 < total; t0 += U * step) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = min(t0 + u * step, total - 1);
      const int64_t r = total < (1LL << 32) ? (int64_t)((uint32_t)t / (uint32_t)per) : t / per;
      const int c = (int)(t - r * per) * V;
      raw[u] = load_raw(in + r * g.ld_in[b] + c, g.cols - c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u * step >= total) break;
      float v[V];
      unpack<T>(raw[u], v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += (double)v[i] * (double)v[i];
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane_id() == 0) red[wave_id()] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[b * gridDim.x + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// |in|_F + eps from the sum of squares.  A norm can pass fp32's range where no element does: it and the elements are
// then brought down by 2^64 first.
struct Norm {
  float down, norm;
  SGNN_DEV Norm(double squares, float eps) {
    const double n = sqrt(squares);
    down = n > 1e38 ? 0x1p-64f : 1.0f;
    norm = (float)(n * down) + eps * down;
  }
  SGNN_DEV float of(float v) const { return norm == 0.0f ? 0.0f : v * down / norm; }  // only zeros have the norm 0
};

// Eight values times scale into the planes, at a 16-byte address.
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
  *reinterpret_cast<h8*>(p + plane) = lo;
}

// The planes of in / (|in|_F + eps), zero in the padding; one thread per 8 columns.  Without steps (x null) the
// values go to out.
template <typename T>
__global__ __launch_bounds__(256) void k_ns_begin(Group g, const double* part, int nparts, float eps, f16_t* x,
                                                  int64_t plane, int64_t batch, int64_t ld, int64_t rows_padded) {
  __shared__ double red[4];
  const int b = blockIdx.y;
  double s = (int)threadIdx.x < nparts ? part[b * nparts + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane_id() == 0) red[wave_id()] = s;
  __syncthreads();
  s = red[0] + red[1] + red[2] + red[3];
  const Norm norm(s, eps);
  const T* in = static_cast<const T*>(g.in[b]);
  const int64_t per = ld / 8, total = rows_padded * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / per, c = (t - r * per) * 8;
    const bool there = r < g.rows && c < g.cols;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (there) load_some<8>(in + r * g.ld_in[b] + c, (int)(g.cols - c), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = norm.of(v[i]);
    if (x)
      put_planes(x + b * batch + r * ld + c, plane, v, kScale);
    else if (there)
      store_some<8>(static_cast<T*>(g.out[b]) + r * g.ld_out[b] + c, (int)(g.cols - c), v);
  }
}

// acc[j] += the products of 32 k: A's rows a_hi + a_lo by B's b[0][j] + b[1][j].  A matrix instruction lines its products
// up with what it adds them to and drops what falls below: with the running sum as its addend a sum of some thousand
// products lost 1e-6 of itself, always towards 0.  So each starts from zero and its 32 k are added by the vector units.
template <int N>
SGNN_DEV void add_products(f32x4 (&acc)[N], const s16x8 (&b)[kPlanes][N], s16x8 a_hi, s16x8 a_lo) {
  f32x4 t[N];
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = mfma16<f16_t>(b[1][j], a_hi, f32x4{0, 0, 0, 0});
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = mfma16<f16_t>(b[0][j], a_lo, t[j]);
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = mfma16<f16_t>(b[0][j], a_hi, t[j]);
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] += t[j];
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

// BT x BT outputs by four waves.  SYM: the product is symmetric; only the tiles on and above the diagonal are formed and
// each is written to both sides.
// KG groups of four waves take every KG-th block of k each, with LDS of their own, and are added in order at the end:
// these products have few tiles (36 of 128 x 128 in the triangle of 1024), and one wave per SIMD leaves memory's and
// LDS's latencies in the open.  One group instead of two, all five steps in us: 1024 x 1024 301 / 225, 2048 x 4096
// 1507 / 1228, 4096 x 4096 5253 / 4646; two of 2048 x 4096 2379 / 2420.  2048 x 4096: X X^T 87 to 98 us
// (136 tiles of 256 CUs; three times 18 GFLOP formed), G^2 55 to 60, Q X 107 to 116 (three times 34 GFLOP, 890 to 960
// TFLOP/s): bounded by the CUs without a tile and by LDS reads beside the matrix instructions.
constexpr int KG = 2;
template <bool AC, bool BC, int BT, bool SYM>
__global__ __launch_bounds__(256 * KG) void k_ns_gemm(NsGemm g) {
  constexpr int P = kPlanes, BK = 32, kThreads = 256, TT = BT / 2 / 16;
  using TA = Tile16<BT, BK, AC>;
  using TB = Tile16<BT, BK, BC>;
  constexpr int kStage = 2 * P * TA::kBytes;
  __shared__ __attribute__((aligned(16))) char all[2 * KG * kStage];
  const int kg = wave_id() >> 2, w = wave_id() & 3, wm = w >> 1, wn = w & 1, l = lane_id(), tid = threadIdx.x & 255;
  char* lds = all + kg * 2 * kStage;
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
  TA::template offsets<kThreads>(oa, g.lda, BT, 0, tid);
  TB::template offsets<kThreads>(ob, g.ldb, BT, 0, tid);
  const char* pa = reinterpret_cast<const char*>(g.A + b * g.batch_a + (AC ? m0 : m0 * g.lda));
  const char* pb = reinterpret_cast<const char*>(g.B + b * g.batch_b + (BC ? n0 : n0 * g.ldb));
  const int64_t sa = 2 * BK * (AC ? g.lda : 1), sb = 2 * BK * (BC ? g.ldb : 1);
  const auto stage = [&](char* to, int blk) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      TA::template direct<kThreads>(to + p * TA::kBytes, pa + 2 * p * g.plane_a + blk * sa, oa, tid);
      TB::template direct<kThreads>(to + (P + p) * TA::kBytes, pb + 2 * p * g.plane_b + blk * sb, ob, tid);
    }
  };
  const int blocks = g.K / BK;
  if (kg < blocks) stage(lds, kg);
  for (int round = 0; round * KG < blocks; ++round) {
    const int blk = round * KG + kg;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (blk + KG < blocks) stage(lds + ((round & 1) ^ 1) * kStage, blk + KG);
    if (blk >= blocks) continue;
    const char* here = lds + (round & 1) * kStage;
    s16x8 fa[P][TT], fb[P][TT];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        fa[p][i] = TA::frag(here + p * TA::kBytes, (wm * TT + i) * 16, 0);
        fb[p][i] = TB::frag(here + (P + p) * TA::kBytes, (wn * TT + i) * 16, 0);
      }
#pragma unroll
    for (int i = 0; i < TT; ++i) add_products<TT>(acc[i], fb, fa[0][i], fa[1][i]);
  }
  __syncthreads();
  f32x4* sums = reinterpret_cast<f32x4*>(all) + ((kg - 1) * 4 + w) * TT * TT * 64 + l;
  static_assert((KG - 1) * 4 * TT * TT * 64 * 16 <= 2 * KG * kStage, "the groups' sums fit");
  if (kg > 0)
#pragma unroll
    for (int i = 0; i < TT * TT; ++i) sums[64 * i] = acc[i / TT][i % TT];
  __syncthreads();
  if (kg > 0) return;
  for (int q = 1; q < KG; ++q)
#pragma unroll
    for (int i = 0; i < TT * TT; ++i) acc[i / TT][i % TT] += sums[(q * 4 * TT * TT + i) * 64];
  // the epilogue's buffers are this wave's own part of what it has read
  // through LDS by 16 rows of m (as in gemm.hip), so that every load and store is 16 bytes of a row
  constexpr int kPieces = 4 * TT, kMask = kPieces - 1;
  float* buf = reinterpret_cast<float*>(all) + w * TT * TT * 256;
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
          load_vec(R + g.plane_c + at, lo);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] += g.beta * kInvScale * (hi[e] + lo[e]);
            if (n + e == m) v[e] += g.diag;
          }
        }
        // the values back into the buffer for the mirrored tile
        *reinterpret_cast<f32x4*>(at0) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(at1) = f32x4{v[4], v[5], v[6], v[7]};
        put_planes(C + at, g.plane_c, v, kScale);
      } else if (g.last_dtype < 0) {
        put_planes(C + at, g.plane_c, v, kScale);
      } else if (m < g.last.rows && n < g.last.cols) {
        const int64_t to = m * g.last.ld_out[b] + n;
        const int cnt = (int)(g.last.cols - n);
        if (g.last_dtype == SGNN_BF16) store_some<8>(static_cast<bf16_t*>(g.last.out[b]) + to, cnt, v);
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
          put_planes(C + (ni + n) * g.ldc + mi + r0, g.plane_c, v, kScale);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
}

template <bool AC, bool BC, bool SYM>
void launch_gemm(const NsGemm& g, int bt, int count, hipStream_t s) {
  const auto tiles = [&](int m, int n) { return SYM ? m * (m + 1) / 2 : m * n; };
  const dim3 grid((unsigned)tiles(g.tiles_m, g.tiles_n), 1, (unsigned)count);
  if (bt == 128) hipLaunchKernelGGL((k_ns_gemm<AC, BC, 128, SYM>), grid, dim3(256 * KG), 0, s, g);
  else hipLaunchKernelGGL((k_ns_gemm<AC, BC, 64, SYM>), grid, dim3(256 * KG), 0, s, g);
}

// ----------------------------------------------------------------------------- small matrices
// All steps of one matrix in one workgroup of eight waves, for sides that fit its LDS: X [m][n] and G / Q [m][m] as planes
// with rows of n + 8 and m + 8 values (an odd number of 16-byte pieces, so that 16 rows' pieces fall on different banks),
// m <= n in whole 32s, zeros in the padding.  A tall matrix is laid down transposed.  Each wave has up to NB times
// 32 x 32 of a product in registers, in blocks of 16 BI x 32; G and X are read along k from their rows, X as the second factor transposed
// (ds_read_b64_tr_b16).  One launch instead of 2 + 3 per step, whose latency is all a small matrix costs: 64 x 64 fp32
// 22 us against 60 by tiles; bounded by the chain of LDS reads, matrix instructions and barriers, about 4 us a step.
constexpr int kMaxSmall = 48, kSmallThreads = 512, kSmallWaves = kSmallThreads / 64, kMaxLds = 160 * 1024 - 256;
struct SmallArgs {
  sgnn_matrix mats[kMaxSmall];
};

inline int pad32(int v) { return (v + 31) & ~31; }
inline size_t small_lds(int rows, int cols) {
  const size_t m = pad32(std::min(rows, cols)), n = pad32(std::max(rows, cols));
  return 2 * (size_t)kPlanes * m * ((n + 8) + (m + 8));
}
inline int small_blocks(int rows, int cols) { return pad32(std::min(rows, cols)) / 32 * (pad32(std::max(rows, cols)) / 32); }
// A short side of 128 fills the waves with blocks of 64 x 32, which read a quarter less of LDS than those of 32 x 32.
inline bool full_side(int rows, int cols) { return pad32(std::min(rows, cols)) == 128; }
inline bool small_ok(int rows, int cols) {
  return std::min(rows, cols) <= 128 && std::max(rows, cols) <= 4096 && small_blocks(rows, cols) <= 6 * kSmallWaves &&
         small_lds(rows, cols) <= kMaxLds;
}

// acc = the 16 BI x 32 block (a0, b0) of A B^T, A's rows from LDS, B's from LDS (BT: its columns), over K.
template <bool BT, int BI>
SGNN_DEV void small_block(f32x4 (&acc)[BI][2], const char* A, int lda, int plane_a, const char* B, int ldb, int plane_b,
                          int a0, int b0, int K) {
  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < BI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  constexpr int P = kPlanes;
  s16x8 fa[2][P][BI], fb[2][P][2];
  const auto load = [&](int h, int k0) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < BI; ++i)
        fa[h][p][i] = *reinterpret_cast<const s16x8*>(A + p * plane_a + 2 * ((a0 + 16 * i + (l & 15)) * lda + k0 + 8 * (l >> 4)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (!BT) {
          fb[h][p][i] = *reinterpret_cast<const s16x8*>(B + p * plane_b + 2 * ((b0 + 16 * i + (l & 15)) * ldb + k0 + 8 * (l >> 4)));
        } else {
          const char* at = B + p * plane_b + 2 * ((k0 + 8 * (l >> 4) + ((l & 15) >> 2)) * ldb + b0 + 16 * i + 4 * (l & 3));
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SGNN_LDS s16x4*)(at));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SGNN_LDS s16x4*)(at + 8 * ldb));
          fb[h][p][i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
    }
  };
  const auto multiply = [&](int h) {
#pragma unroll
    for (int i = 0; i < BI; ++i) add_products<2>(acc[i], fb[h], fa[h][0][i], fa[h][1][i]);
  };
  // the next 32 k are read under this one's products (past the end: the last ones again)
  load(0, 0);
  for (int k0 = 0; k0 < K; k0 += 64) {
    load(1, min(k0 + 32, K - 32));
    multiply(0);
    if (k0 + 32 >= K) break;
    load(0, min(k0 + 64, K - 32));
    multiply(1);
  }
}

// The block's values times scale into planes of LDS.
template <int BI>
SGNN_DEV void small_put(char* C, int ldc, int plane, const f32x4 (&acc)[BI][2], int a0, int b0, float scale) {
  typedef f16_t h4 __attribute__((ext_vector_type(4)));
  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < BI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      h4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = acc[i][j][r] * scale;
        const f16_t h = (f16_t)v;
        hi[r] = h, lo[r] = (f16_t)(v - (float)h);
      }
      char* at = C + 2 * ((a0 + 16 * i + (l & 15)) * ldc + b0 + 16 * j + 4 * (l >> 4));
      *reinterpret_cast<h4*>(at) = hi;
      *reinterpret_cast<h4*>(at + plane) = lo;
    }
}

// A wave's q-th block, computed where it is used (hoisted out of the steps, all blocks' addresses at once would not fit
// the registers).
SGNN_DEV int block_of(int w, int q) {
  int b = w + q * kSmallWaves;
  asm volatile("" : "+s"(b));
  return b;
}

constexpr float kDown = kInvScale * kInvScale;  // of a product of two scaled planes

// The planes of Q = ca I + cb G + cc G^2 into LDS at G, from this wave's blocks g of kScale^2 G.
template <int NG, int BI>
SGNN_DEV void small_poly(f32x4 (&g)[NG][BI][2], char* G, int ldg, int plane_g, int m, float ca, float cb, float cc) {
  const int l = lane_id(), w = wave_id(), mb = m / (16 * BI), gblocks = mb * (m / 32);
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    const int b = block_of(w, q);
    if (b < gblocks) small_put(G, ldg, plane_g, g[q], b % mb * 16 * BI, b / mb * 32, kInvScale);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    const int b = block_of(w, q);
    if (b < gblocks) {
      f32x4 h[BI][2];
      const int a0 = b % mb * 16 * BI, b0 = b / mb * 32;
      small_block<false>(h, G, ldg, plane_g, G, ldg, plane_g, a0, b0, m);
#pragma unroll
      for (int i = 0; i < BI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool diag = a0 + 16 * i + (l & 15) == b0 + 16 * j + 4 * (l >> 4) + r;
            g[q][i][j][r] = cb * (g[q][i][j][r] * kDown) + cc * (h[i][j][r] * kDown) + (diag ? ca : 0.0f);
          }
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    const int b = block_of(w, q);
    if (b < gblocks) small_put(G, ldg, plane_g, g[q], b % mb * 16 * BI, b / mb * 32, kScale);
  }
  __syncthreads();
}

// A block of kScale^2 X, at (r0, c0) of the matrix as it lies in LDS, into the caller's matrix.
template <typename T, int BI>
SGNN_DEV void small_out(const f32x4 (&x)[BI][2], T* out, int64_t ld, int rows, int cols, bool tall, int r0, int c0) {
  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < BI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = r0 + 16 * i + (l & 15), c = c0 + 16 * j + 4 * (l >> 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = x[i][j][e] * kDown;
        if (tall) {
          if (r < cols && c + e < rows) out[(int64_t)(c + e) * ld + r] = from_float<T>(v);
        } else if (r < rows && c + e < cols) {
          out[(int64_t)r * ld + c + e] = from_float<T>(v);
        }
      }
    }
}

template <typename T, int NB, int BI>
__global__ __launch_bounds__(kSmallThreads) void k_ns_small(SmallArgs args, int steps, float ca, float cb, float cc,
                                                            float eps) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ double red[kSmallWaves];
  constexpr int V = 16 / sizeof(T), P = kPlanes;
  const sgnn_matrix& mat = args.mats[blockIdx.x];
  const bool tall = mat.rows > mat.cols;
  const int m = (min(mat.rows, mat.cols) + 31) & ~31, n = (max(mat.rows, mat.cols) + 31) & ~31;
  const int ldx = n + 8, ldg = m + 8, plane_x = 2 * m * ldx, plane_g = 2 * m * ldg;
  char *X = lds, *G = lds + P * plane_x;
  const int w = wave_id(), l = lane_id();
  const T* in = static_cast<const T*>(mat.in);

  for (int t = threadIdx.x; t < P * plane_x / 16; t += kSmallThreads)
    *reinterpret_cast<u32x4*>(X + 16 * t) = u32x4{0, 0, 0, 0};
  __syncthreads();
  // the elements' bits into their places (upper halves in the hi plane, lower ones in the lo plane) and the sum of
  // squares, in 64 bits as in k_ns_norm
  const int per = (mat.cols + V - 1) / V, pieces = mat.rows * per;
  double s = 0.0;
#pragma unroll 4
  for (int t = threadIdx.x; t < pieces; t += kSmallThreads) {
    const int r = t / per, c = (t - r * per) * V;
    float v[V];
    load_some<V>(in + (int64_t)r * mat.ld_in + c, mat.cols - c, v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s += (double)v[e] * (double)v[e];
      if (c + e >= mat.cols) continue;
      char* at = X + 2 * (tall ? (c + e) * ldx + r : r * ldx + c + e);
      const uint32_t bits = __builtin_bit_cast(uint32_t, v[e]);
      *reinterpret_cast<uint16_t*>(at) = bits >> 16;
      *reinterpret_cast<uint16_t*>(at + plane_x) = bits;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (l == 0) red[w] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < kSmallWaves; ++i) s += red[i];
  const Norm norm(s, eps);
  // the bits into the planes of the value / norm
  for (int t = threadIdx.x; t < plane_x / 16; t += kSmallThreads) {
    const u32x4 hi = *reinterpret_cast<u32x4*>(X + 16 * t), lo = *reinterpret_cast<u32x4*>(X + plane_x + 16 * t);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t up = hi[e >> 1] >> (16 * (e & 1)) << 16, low = lo[e >> 1] >> (16 * (e & 1)) & 0xffffu;
      v[e] = norm.of(__builtin_bit_cast(float, up | low));
    }
    put_planes(reinterpret_cast<f16_t*>(X + 16 * t), plane_x / 2, v, kScale);
  }
  __syncthreads();

  if (steps == 0) {
    T* out = static_cast<T*>(mat.out);
    for (int t = threadIdx.x; t < mat.rows * mat.cols; t += kSmallThreads) {
      const int r = t / mat.cols, c = t - r * mat.cols;
      const f16_t* at = reinterpret_cast<const f16_t*>(X) + (tall ? c * ldx + r : r * ldx + c);
      out[(int64_t)r * mat.ld_out + c] = from_float<T>((to_float(at[0]) + to_float(at[plane_x / 2])) * kInvScale);
    }
  }
  constexpr int NG = 4 / BI, NX = 2 * NB / BI;
  const int mb = m / (16 * BI), gblocks = mb * (m / 32), xblocks = mb * (n / 32);
  for (int step = 0; step < steps; ++step) {
    f32x4 g[NG][BI][2], x[NX][BI][2];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const int b = block_of(w, q);
      if (b < gblocks) small_block<false>(g[q], X, ldx, plane_x, X, ldx, plane_x, b % mb * 16 * BI, b / mb * 32, n);
    }
    small_poly(g, G, ldg, plane_g, m, ca, cb, cc);
#pragma unroll
    for (int q = 0; q < NX; ++q) {
      const int b = block_of(w, q);
      if (b < xblocks) small_block<true>(x[q], G, ldg, plane_g, X, ldx, plane_x, b % mb * 16 * BI, b / mb * 32, m);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NX; ++q) {
      const int b = block_of(w, q);
      if (b >= xblocks) continue;
      const int r0 = b % mb * 16 * BI, c0 = b / mb * 32;
      if (step + 1 < steps) small_put(X, ldx, plane_x, x[q], r0, c0, kInvScale);
      else small_out<T>(x[q], static_cast<T*>(mat.out), mat.ld_out, mat.rows, mat.cols, tall, r0, c0);
    }
    __syncthreads();
  }
}

template <typename T>
int launch_small(const sgnn_matrix* mats, int count, int32_t steps, float a, float b, float c, float eps, hipStream_t s) {
  SmallArgs args;
  size_t bytes = 0;
  int blocks = 0;
  for (int i = 0; i < count; ++i) {
    args.mats[i] = mats[i];
    bytes = std::max(bytes, small_lds(mats[i].rows, mats[i].cols));
    blocks = std::max(blocks, small_blocks(mats[i].rows, mats[i].cols));
  }
  const auto go = [&](auto kernel) {
    // the attribute belongs to the device that is current
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds) !=
        hipSuccess)
      return check_launch("newton_schulz");
    hipLaunchKernelGGL(kernel, dim3((unsigned)count), dim3(kSmallThreads), bytes, s, args, steps, a, b, c, eps);
    return check_launch("newton_schulz");
  };
  if (full_side(mats[0].rows, mats[0].cols))
    return blocks <= 2 * kSmallWaves ? go(k_ns_small<T, 2, 4>) : go(k_ns_small<T, 6, 4>);
  return blocks <= 2 * kSmallWaves ? go(k_ns_small<T, 2, 2>) : go(k_ns_small<T, 6, 2>);
}

// ----------------------------------------------------------------------------- short and long matrices
// A matrix whose short side fits as above but whose long one does not: a workgroup per kChunk of its long side.  G is the
// sum of the chunks' X_c X_c^T, so one launch per step does: add the chunks' shares of G (in order, every workgroup for
// itself), form Q, X_c <- Q X_c, and its share of the next G -- 2 + steps launches for 2 + 3 steps, 12 to 16 us each,
// bounded as the small kernel is.  fp32 by chunks / by tiles, us: one 32 x 2048 53 / 143, 64 x 1024 57 / 100, 128 x 384
// 92 / 87, 128 x 2048 132 / 163; ten 128 x 384 98 / 98, 128 x 2048 160 / 210; 32 of 128 x 384 110 / 115, 128 x 2048
// 384 / 390.  Beyond 16 chunks the sums of G's shares, which every workgroup reads, can cost more than the launches saved:
// 128 x 4096 177 / 256, but 32 of them 833 / 656, and the number of matrices must not decide, or it would their bits.
//   shares [matrix][chunk][32 x 32 block of G][4][lane] as the accumulators hold them; x: planes [matrix][m][ld]
constexpr int kChunk = 128, kMaxChunks = 16;
inline bool chunk_ok(int rows, int cols) {
  return std::min(rows, cols) <= 128 && std::max(rows, cols) <= kChunk * kMaxChunks;
}
inline int chunks_of(int rows, int cols) { return (std::max(rows, cols) + kChunk - 1) / kChunk; }
inline size_t chunk_lds(int m) { return 2 * (size_t)kPlanes * m * ((kChunk + 8) + (m + 8)); }

struct ChunkArgs {
  const double* norms;
  f16_t* x;
  const float* from;  // the shares of this step's G (null: the first launch, which has the norms instead)
  float* to;          // of the next one (null: the last step)
  int64_t plane;
  int32_t nparts, m, ld;
  float ca, cb, cc, eps;
};

template <typename T, int BI>
__global__ __launch_bounds__(kSmallThreads) void k_ns_chunk(Group grp, ChunkArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ double red[kSmallWaves];
  constexpr int V = 16 / sizeof(T), P = kPlanes;
  const int l = lane_id(), w = wave_id(), mat = blockIdx.y, c0 = blockIdx.x * kChunk;
  constexpr int NG = 4 / BI;
  const int m = a.m, mb = m / (16 * BI), gblocks = mb * (m / 32), xblocks = mb * (kChunk / 32);
  const int ldx = kChunk + 8, ldg = m + 8, plane_x = 2 * m * ldx, plane_g = 2 * m * ldg;
  char *X = lds, *G = lds + P * plane_x;
  const bool tall = grp.rows > grp.cols;
  f16_t* home = a.x + (int64_t)mat * m * a.ld + c0;
  f32x4 g[NG][BI][2];

  if (a.from) {
    // X's loads go out before those of the shares
    constexpr int kPer = 128 * (kChunk / 8) / kSmallThreads;
    u32x4 px[P][kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = i * kSmallThreads + threadIdx.x, r = min(t / (kChunk / 8), m - 1), c = t % (kChunk / 8) * 8;
#pragma unroll
      for (int p = 0; p < P; ++p) px[p][i] = *reinterpret_cast<const u32x4*>(home + p * a.plane + (int64_t)r * a.ld + c);
    }
    const f32x4* from = reinterpret_cast<const f32x4*>(a.from) + (int64_t)mat * gridDim.x * gblocks * 128 * BI + l;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const int b = block_of(w, q);
      if (b >= gblocks) continue;
#pragma unroll
      for (int i = 0; i < 2 * BI; ++i) g[q][i >> 1][i & 1] = f32x4{0, 0, 0, 0};
#pragma unroll 2
      for (int c = 0; c < (int)gridDim.x; ++c)
#pragma unroll
        for (int i = 0; i < 2 * BI; ++i) g[q][i >> 1][i & 1] += from[((int64_t)c * gblocks + b) * 128 * BI + 64 * i];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = i * kSmallThreads + threadIdx.x, r = t / (kChunk / 8), c = t % (kChunk / 8) * 8;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (r < m) *reinterpret_cast<u32x4*>(X + p * plane_x + 2 * (r * ldx + c)) = px[p][i];
    }
    __syncthreads();
    small_poly(g, G, ldg, plane_g, m, a.ca, a.cb, a.cc);
    f32x4 x[NG][BI][2];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const int b = block_of(w, q);
      if (b < xblocks) small_block<true>(x[q], G, ldg, plane_g, X, ldx, plane_x, b % mb * 16 * BI, b / mb * 32, m);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const int b = block_of(w, q);
      if (b >= xblocks) continue;
      if (a.to)
        small_put(X, ldx, plane_x, x[q], b % mb * 16 * BI, b / mb * 32, kInvScale);
      else
        small_out<T>(x[q], static_cast<T*>(grp.out[mat]), grp.ld_out[mat], grp.rows, grp.cols, tall, b % mb * 16 * BI,
                     c0 + b / mb * 32);
    }
    if (!a.to) return;
  } else {
    double s = (int)threadIdx.x < a.nparts ? a.norms[mat * a.nparts + threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (l == 0) red[w] = s;
    for (int t = threadIdx.x; t < P * plane_x / 16; t += kSmallThreads)
      *reinterpret_cast<u32x4*>(X + 16 * t) = u32x4{0, 0, 0, 0};
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int i = 0; i < kSmallWaves; ++i) s += red[i];
    const Norm norm(s, a.eps);
    // this chunk of the caller's matrix: rows r0 .. of it where it is tall, columns where it is wide
    const int r0 = tall ? c0 : 0, rows = tall ? min(kChunk, grp.rows - c0) : grp.rows;
    const int k0 = tall ? 0 : c0, cols = tall ? grp.cols : min(kChunk, grp.cols - c0);
    const T* in = static_cast<const T*>(grp.in[mat]) + (int64_t)r0 * grp.ld_in[mat] + k0;
    const int per = (cols + V - 1) / V, pieces = rows * per;
    constexpr int U = 4;  // loads under way before the first is used
    for (int t0 = threadIdx.x; t0 < pieces; t0 += U * kSmallThreads) {
      u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = min(t0 + u * kSmallThreads, pieces - 1), r = t / per, c = (t - r * per) * V;
        raw[u] = load_raw(in + (int64_t)r * grp.ld_in[mat] + c, cols - c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kSmallThreads, r = t / per, c = (t - r * per) * V;
        if (t >= pieces) break;
        float v[V];
        unpack<T>(raw[u], v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (c + e >= cols) continue;
          char* at = X + 2 * (tall ? (c + e) * ldx + r : r * ldx + c + e);
          const float y = norm.of(v[e]) * kScale;
          const f16_t h = (f16_t)y;
          *reinterpret_cast<f16_t*>(at) = h;
          *reinterpret_cast<f16_t*>(at + plane_x) = (f16_t)(y - (float)h);
        }
      }
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < m * (kChunk / 8); t += kSmallThreads) {
    const int r = t / (kChunk / 8), c = t % (kChunk / 8) * 8;
#pragma unroll
    for (int p = 0; p < P; ++p)
      *reinterpret_cast<u32x4*>(home + p * a.plane + (int64_t)r * a.ld + c) =
          *reinterpret_cast<const u32x4*>(X + p * plane_x + 2 * (r * ldx + c));
  }
  f32x4* to = reinterpret_cast<f32x4*>(a.to) + ((int64_t)mat * gridDim.x + blockIdx.x) * gblocks * 128 * BI + l;
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    const int b = block_of(w, q);
    if (b >= gblocks) continue;
    small_block<false>(g[q], X, ldx, plane_x, X, ldx, plane_x, b % mb * 16 * BI, b / mb * 32, kChunk);
#pragma unroll
    for (int i = 0; i < 2 * BI; ++i) to[(int64_t)b * 128 * BI + 64 * i] = g[q][i >> 1][i & 1];
  }
}

// ----------------------------------------------------------------------------- large matrices
size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

// A group's workspace: the norms' partial sums, X twice, G and Q, each two planes.
struct NsLayout {
  int bt;
  int64_t rows, cols, side;  // padded; side: of G
  size_t norms, x, g, total;
  NsLayout(int32_t r, int32_t c, int count) {
    const int64_t small = std::min(r, c), large = std::max(r, c);
    // 128-tiles read half as much per product; the smaller ones pad less and fill the CUs sooner (fp32, 128 / 64, us:
    // 2048 x 2048 763 / 885, twelve 512 x 768 411 / 399, 1536 x 2048 643 / 538, 512 x 512 267 / 140)
    bt = (small * large + 128 * 128 - 1) / (128 * 128) * count >= 256 && small > 64 ? 128 : 64;
    rows = (r + bt - 1) / bt * bt, cols = (c + bt - 1) / bt * bt, side = std::min(rows, cols);
    norms = pad256(sizeof(double) * kNormParts * count);
    x = pad256(2 * sizeof(f16_t) * rows * cols * count);
    g = pad256(2 * sizeof(f16_t) * side * side * count);
    total = norms + 2 * x + 2 * g;
  }
};

// The same for a group by chunks: the norms' partial sums, X, G's shares twice.
struct ChunkLayout {
  int chunks, m, ld;
  size_t norms, x, share, total;
  ChunkLayout(int32_t r, int32_t c, int count) {
    chunks = chunks_of(r, c), m = pad32(std::min(r, c)), ld = chunks * kChunk;
    norms = pad256(sizeof(double) * kNormParts * count);
    x = pad256(2 * sizeof(f16_t) * (size_t)m * ld * count);
    share = pad256(sizeof(float) * (size_t)m * m * chunks * count);
    total = norms + x + 2 * share;
  }
};
size_t group_bytes(int32_t r, int32_t c, int count) {  // steps 0 of a matrix by chunks takes the large path's layout
  const size_t large = NsLayout(r, c, count).total;
  return chunk_ok(r, c) ? std::max(large, ChunkLayout(r, c, count).total) : large;
}

unsigned blocks_for(int64_t items, int64_t most) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, most));
}

template <typename T>
int by_chunks(const Group& grp, int32_t steps, float a, float b, float c, float eps, char* ws, hipStream_t s) {
  const ChunkLayout at(grp.rows, grp.cols, grp.count);
  double* norms = reinterpret_cast<double*>(ws);
  float *from = reinterpret_cast<float*>(ws + at.norms + at.x), *to = reinterpret_cast<float*>(ws + at.norms + at.x + at.share);
  const size_t lds = chunk_lds(at.m);
  ChunkArgs g{norms, reinterpret_cast<f16_t*>(ws + at.norms), nullptr, to, (int64_t)at.m * at.ld * grp.count,
              (int32_t)blocks_for((int64_t)grp.rows * grp.cols / 16, kNormParts), at.m, at.ld, a, b, c, eps};
  hipLaunchKernelGGL(k_ns_norm<T>, dim3((unsigned)g.nparts, grp.count), dim3(256), 0, s, grp, norms);
  const auto go = [&](auto kernel) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds) !=
        hipSuccess)
      return check_launch("newton_schulz");
    for (int32_t k = 0; k <= steps; ++k) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)at.chunks, (unsigned)grp.count), dim3(kSmallThreads), lds, s, grp, g);
      std::swap(from, to);
      g.from = from, g.to = k + 1 < steps ? to : nullptr;
    }
    return check_launch("newton_schulz");
  };
  return full_side(grp.rows, grp.cols) ? go(k_ns_chunk<T, 4>) : go(k_ns_chunk<T, 2>);
}

// The matrices from i on that share a launch: small ones of any shape, or large ones of one shape; an empty one is a run
// of its own.
int32_t run_of(const sgnn_matrix* mats, int32_t count, int32_t i) {
  int32_t n = 1;
  if (mats[i].rows == 0 || mats[i].cols == 0) return n;
  if (small_ok(mats[i].rows, mats[i].cols)) {
    while (i + n < count && n < kMaxSmall && mats[i + n].rows > 0 && mats[i + n].cols > 0 &&
           small_ok(mats[i + n].rows, mats[i + n].cols) &&
           full_side(mats[i + n].rows, mats[i + n].cols) == full_side(mats[i].rows, mats[i].cols))
      ++n;
    return n;
  }
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
  const int parts = (int)blocks_for((int64_t)grp.rows * grp.cols / 16, kNormParts);
  hipLaunchKernelGGL(k_ns_norm<T>, dim3(parts, grp.count), dim3(256), 0, s, grp, norms);
  hipLaunchKernelGGL(k_ns_begin<T>, dim3(blocks_for(batch_x / 8, 4096), grp.count), dim3(256), 0, s, grp, norms, parts,
                     eps, steps > 0 ? x : nullptr, plane_x, batch_x, at.cols, at.rows);
  for (int32_t k = 0; k < steps; ++k) {
    NsGemm g{};
    g.last_dtype = -1;
    g.tiles_m = g.tiles_n = (int32_t)(at.side / at.bt);
    g.A = g.B = x, g.lda = g.ldb = at.cols, g.plane_a = g.plane_b = plane_x, g.batch_a = g.batch_b = batch_x;
    g.C = gram, g.ldc = at.side, g.plane_c = plane_g, g.batch_c = batch_g;
    g.alpha = 1.0f;
    g.K = (int32_t)(tall ? at.rows : at.cols);
    if (tall) launch_gemm<true, true, true>(g, at.bt, grp.count, s);
    else launch_gemm<false, false, true>(g, at.bt, grp.count, s);
    g.A = g.B = g.R = gram, g.lda = g.ldb = at.side, g.plane_a = g.plane_b = plane_g, g.batch_a = g.batch_b = batch_g;
    g.C = poly;
    g.alpha = c, g.beta = b, g.diag = a;
    g.K = (int32_t)at.side;
    launch_gemm<false, false, true>(g, at.bt, grp.count, s);
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
      launch_gemm<false, false, false>(g, at.bt, grp.count, s);
    } else {     // Q X
      g.A = poly;
      g.B = x, g.ldb = at.cols, g.plane_b = plane_x, g.batch_b = batch_x;
      launch_gemm<false, true, false>(g, at.bt, grp.count, s);
    }
    std::swap(x, next);
  }
}

}  // namespace

extern "C" size_t sgnn_newton_schulz_workspace_bytes(const sgnn_matrix* mats, int32_t count) {
  size_t most = 0;
  for (int32_t i = 0, n; mats && i < count; i += n) {
    n = run_of(mats, count, i);
    if (mats[i].rows > 0 && mats[i].cols > 0 && !small_ok(mats[i].rows, mats[i].cols))
      most = std::max(most, group_bytes(mats[i].rows, mats[i].cols, n));
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
  const size_t need = sgnn_newton_schulz_workspace_bytes(mats, count);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(SGNN_ERR_INVALID, "newton_schulz: workspace smaller than sgnn_newton_schulz_workspace_bytes");
  for (int32_t i = 0, n; i < count; i += n) {
    n = run_of(mats, count, i);
    if (mats[i].rows == 0 || mats[i].cols == 0) continue;
    if (small_ok(mats[i].rows, mats[i].cols)) {
      const int st = with_type(dtype, [&](auto* t) {
        return launch_small<std::remove_pointer_t<decltype(t)>>(mats + i, n, steps, a, b, c, eps,
                                                                static_cast<hipStream_t>(stream));
      });
      if (st != SGNN_OK) return st;
      continue;
    }
    Group grp;
    grp.rows = mats[i].rows, grp.cols = mats[i].cols, grp.count = n;
    for (int32_t k = 0; k < n; ++k) {
      grp.in[k] = mats[i + k].in, grp.out[k] = mats[i + k].out;
      grp.ld_in[k] = mats[i + k].ld_in, grp.ld_out[k] = mats[i + k].ld_out;
    }
    const int st = with_type(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      char* ws = static_cast<char*>(workspace);
      hipStream_t s = static_cast<hipStream_t>(stream);
      if (steps > 0 && chunk_ok(grp.rows, grp.cols)) return by_chunks<T>(grp, steps, a, b, c, eps, ws, s);
      orthogonalise<T>(grp, steps, a, b, c, eps, ws, s);
      return check_launch("newton_schulz");
    });
    if (st != SGNN_OK) return st;
  }
  return SGNN_OK;
}
