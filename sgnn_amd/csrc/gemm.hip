// One matrix product for every operand type and storage order (gemm.h).
//
//   k_gemm16     bf16 / fp16 operands on v_mfma_f32_16x16x32: double-buffered LDS tiles of 64 k, filled by the
//                direct-to-LDS loads where the operands' rows are 16-byte aligned, through registers elsewhere
//   k_gemm32     fp32 operands as three bf16 parts each (8 + 8 + 8 bits, split exactly while they are staged), six
//                bf16 products per fp32 one
//   k_gemm_rows  up to 32 rows of x: the waves stream their shares of w's rows into registers, LDS only for the join
//
// Both tiled kernels hold D[n][m] (w's rows on the accumulators' rows, x's on the lanes): a lane then has four
// consecutive n of one m, which go through LDS once more so that the epilogue's loads and stores are whole
// 16-byte pieces of rows at any alignment.
#include "gemm.h"

#include "gemm_tile.h"

namespace {
using namespace sgnn;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct GemmArgs {
  const void *A, *B, *bias, *res;
  float* slope;
  void* C;
  float* part;  // split-K partials [split][M][N] (null: one split, the epilogue in place)
  int64_t lda, ldb, ldr, ldc, M, N, K;
  int32_t act, nsplit, tiles_m, tiles_n;
  int64_t lo;  // of A's two planes (gemm.h)
};

// ----------------------------------------------------------------------------- epilogue
template <int ACT, typename T, int V>
SGNN_DEV void act_row(const GemmArgs& g, int64_t at, int cnt, float (&v)[V]) {
  if (g.slope) {
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) act_both<ACT, true, sizeof(T) == 2>(v[i], v[i], s[i]);
    store_some<V>(g.slope + at, cnt, s);
  } else {
    float unused;
#pragma unroll
    for (int i = 0; i < V; ++i) act_both<ACT, false, sizeof(T) == 2>(v[i], v[i], unused);
  }
}

// The bias of columns n .., zeros where there is none; cnt of them exist.
template <typename T, int V>
SGNN_DEV void load_bias(const GemmArgs& g, int64_t n, int cnt, float (&t)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = 0.0f;
  if (g.bias && cnt > 0) load_some<V>(static_cast<const T*>(g.bias) + n, cnt, t);
}

// V = 16 bytes' consecutive outputs (m, n ..) of one lane; cnt of them exist.
template <typename T, int V>
SGNN_DEV void finish(const GemmArgs& g, int64_t m, int64_t n, float (&v)[V], const float (&bias)[V], int cnt) {
  float t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] += bias[i];
  switch (g.act) {  // the same for every lane
    case SGNN_ACT_RELU: act_row<SGNN_ACT_RELU, T>(g, m * g.N + n, cnt, v); break;
    case SGNN_ACT_GELU: act_row<SGNN_ACT_GELU, T>(g, m * g.N + n, cnt, v); break;
    case SGNN_ACT_GELU_TANH: act_row<SGNN_ACT_GELU_TANH, T>(g, m * g.N + n, cnt, v); break;
    case SGNN_ACT_SILU: act_row<SGNN_ACT_SILU, T>(g, m * g.N + n, cnt, v); break;
    default: act_row<SGNN_ACT_NONE, T>(g, m * g.N + n, cnt, v); break;
  }
  if (g.res) {
    load_some<V>(static_cast<const T*>(g.res) + m * g.ldr + n, cnt, t);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += t[i];
  }
  store_some<V>(static_cast<T*>(g.C) + m * g.ldc + n, cnt, v);
}

// A wave's accumulators (TM x TN sub-tiles of 16 x 16, lane l: m = l & 15, n = 4 (l >> 4) + r) to memory, RP sub-tile
// rows at a time through `buf` (16 RP x 16 TN floats of its own).  16-byte pieces are XORed with m, so that the 16
// rows of one write, which are a multiple of all banks apart, fall on different ones.
template <typename T, int RP, int TM, int TN>
SGNN_DEV void write_tile(const GemmArgs& g, float* buf, const f32x4 (&acc)[TM][TN], int split, int64_t m0,
                         int64_t n0) {
  static_assert(TM % RP == 0, "whole rounds");
  const int l = lane_id();
  constexpr int kPieces = 4 * TN;  // 16-byte pieces per row of 16 TN floats
  constexpr int kMask = kPieces - 1 < 15 ? kPieces - 1 : 15;
  // a lane's columns are the same in every row it takes, so their bias is loaded once
  constexpr int V = 16 / sizeof(T), kPer = V / 4, kAcross = kPieces / kPer;
  static_assert(64 % kAcross == 0, "whole rows of pieces per wave");
  const int64_t n_mine = n0 + 4 * kPer * (l % kAcross);
  const int cnt = (int)min((int64_t)V, g.N - n_mine);
  float bias[V];
  if (!g.part) load_bias<T>(g, n_mine, cnt, bias);
#pragma unroll
  for (int round = 0; round < TM / RP; ++round) {
#pragma unroll
    for (int i = 0; i < RP; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int r = 16 * i + (l & 15), piece = (4 * j + (l >> 4)) ^ (r & kMask);
        *reinterpret_cast<f32x4*>(buf + r * 16 * TN + piece * 4) = acc[round * RP + i][j];
      }
    __builtin_amdgcn_wave_barrier();
    const int64_t mr = m0 + 16 * RP * round;
    if (g.part) {
#pragma unroll 1
      for (int t = l; t < 16 * RP * kPieces; t += 64) {
        const int r = t / kPieces, p = t % kPieces;
        const f32x4 f = *reinterpret_cast<const f32x4*>(buf + r * 16 * TN + (p ^ (r & kMask)) * 4);
        const int64_t m = mr + r, n = n0 + 4 * p;
        const float v[4] = {f[0], f[1], f[2], f[3]};
        if (m < g.M && n < g.N)
          store_some<4>(g.part + ((int64_t)split * g.M + m) * g.N + n, (int)min((int64_t)4, g.N - n), v);
      }
    } else {
#pragma unroll 2
      for (int r = l / kAcross; r < 16 * RP; r += 64 / kAcross) {
        const int p = l % kAcross * kPer;
        float v[V];
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const f32x4 f = *reinterpret_cast<const f32x4*>(buf + r * 16 * TN + ((p + q) ^ (r & kMask)) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * q + e] = f[e];
        }
        if (mr + r < g.M && cnt > 0) finish<T>(g, mr + r, n_mine, v, bias, cnt);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Workgroup -> tile.  Consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its own: XCD x takes the
// x-th contiguous share of the tiles, in groups of 8 row tiles by all column tiles, so that the tiles resident on
// one L2 share their operands' rows.
SGNN_DEV void tile_of(const GemmArgs& g, int& tm, int& tn) {
  const int total = g.tiles_m * g.tiles_n, id = blockIdx.x;
  const int xcd = id & 7, q = total >> 3, r = total & 7;
  const int t = xcd * q + min(xcd, r) + (id >> 3);
  constexpr int kGroup = 8;
  const int per = kGroup * g.tiles_n, grp = t / per, rest = t - grp * per;
  const int rows = min(kGroup, g.tiles_m - grp * kGroup);
  const int col = rest / rows;
  tn = __builtin_amdgcn_readfirstlane(col);
  tm = __builtin_amdgcn_readfirstlane(grp * kGroup + rest - col * rows);
}

// This workgroup's blocks of k.
SGNN_DEV void blocks_of(const GemmArgs& g, int bk, int split, int& first, int& last) {
  const int64_t blocks = (g.K + bk - 1) / bk;
  first = __builtin_amdgcn_readfirstlane((int)(blocks * split / g.nsplit));
  last = __builtin_amdgcn_readfirstlane((int)(blocks * (split + 1) / g.nsplit));
}

// ----------------------------------------------------------------------------- 16-bit operands
// BM x BN outputs per workgroup, WM x WN waves.  DIRECT: both operands' lines are 16-byte aligned (and in the cols
// layout a multiple of 8 rows): LDS is filled without passing registers but for the last, partial block of k.
// NST stages of LDS: NST - 1 blocks are under way while one is worked on.  Two suffice where a block's products take
// longer than memory; the small tile has four.
// 8192 x 8192 x 2048 in bf16 (275 GFLOP; the library's products take 187 to 230 us): x w^T with gelu and its slopes 290
// to 330 us, dy w 230 to 260, dy^T x 234 to 260; with two planes of dz 409 to 480 and 403 to 496.  No bank conflicts are left; the matrix units are busy 50 to 60 % of the
// time, and the rest is LDS's latency after each block's barrier, which all waves meet together, and, forward, the
// epilogue's 402 MB.  Memory is not waited for: four stages of 32 k took 334 / 248 / 244 us at their fastest, where these
// two of 64 k took 290 / 230 / 230; the next block's loads issued behind the first fragments' reads took 292 / 226 / 237.
template <typename T, bool ACOLS, bool BCOLS, int BM, int BN, int WM, int WN, bool DIRECT, int NST>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_gemm16(GemmArgs g) {
  constexpr int BK = 64, kThreads = 64 * WM * WN;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  using TA = Tile16<BM, BK, ACOLS>;
  using TB = Tile16<BN, BK, BCOLS>;
  constexpr int kStage = TA::kBytes + TB::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[NST * kStage];  // stages of A's and B's tiles
  constexpr int RP = TM < 4 ? TM : 4, kBuf = RP * 16 * 16 * TN;
  static_assert(kBuf * 4 * WM * WN <= NST * kStage, "the epilogue's buffers fit");
  const int w = wave_id(), wm = w / WN, wn = w % WN;
  int tm, tn;
  tile_of(g, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int split = blockIdx.z;
  const char* A = static_cast<const char*>(g.A);
  const char* B = static_cast<const char*>(g.B);
  int first, last;
  blocks_of(g, BK, split, first, last);
  const int planes = BCOLS && g.lo != 0 ? 2 : 1;

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  // Two planes of A: the products of lo over all of k, brought to hi's scale, then those of hi.  A lo of 0 times an
  // infinite operand is NaN where hi's product is infinite, so of lo's sums only finite ones count.
  const auto settle = [&] {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        f32x4& v = acc[i][j];
        const float odd = (v[0] - v[0]) + (v[1] - v[1]) + (v[2] - v[2]) + (v[3] - v[3]);  // 0 where all four are finite
        v *= 1.0f / (1 << kLoBits<T>);
        if (odd == 0.0f) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = v[r] - v[r] == 0.0f ? v[r] : 0.0f;
      }
  };

  const auto compute = [&](const char* a) {
    const char* b = a + TA::kBytes;
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      s16x8 fa[TM], fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = TB::frag(b, (wn * TN + j) * 16, kk);
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = TA::frag(a, (wm * TM + i) * 16, kk);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma16<T>(fb[j], fa[i], acc[i][j]);
    }
    if constexpr (TM >= 4) order_products<TM, TN, ACOLS ? 2 : 1, BCOLS ? 2 : 1>();
  };
  constexpr int PA = BM * BK / 8 / kThreads, PB = BN * BK / 8 / kThreads;
  const auto fetch = [&](u32x4(&va)[PA], u32x4(&vb)[PB], int blk, int64_t plane) {
    TA::template fetch<kThreads>(va, A + plane, g.lda, g.M, g.K, m0, (int64_t)blk * BK);
    TB::template fetch<kThreads>(vb, B, g.ldb, g.N, g.K, n0, (int64_t)blk * BK);
  };
  const auto put = [&](char* a, const u32x4(&va)[PA], const u32x4(&vb)[PB]) {
    TA::template put<kThreads>(a, va);
    TB::template put<kThreads>(a + TA::kBytes, vb);
  };
  // One barrier per block: past it, this block's tiles are whole and the stage before it is read by no wave any more.
  if constexpr (DIRECT) {
    uint32_t oa[PA], ob[PB];
    TA::template offsets<kThreads>(oa, g.lda, g.M, m0);
    TB::template offsets<kThreads>(ob, g.ldb, g.N, n0);
    const char* pa = A + 2 * (ACOLS ? m0 : m0 * g.lda);
    const char* pb = B + 2 * (BCOLS ? n0 : n0 * g.ldb);
    const int64_t sa = 2 * BK * (ACOLS ? g.lda : 1), sb = 2 * BK * (BCOLS ? g.ldb : 1);
    // step t of the planes' blocks of k one after the other
    const int blocks = last - first, total = planes * blocks;
    const auto stage = [&](char* a, int t) {
      const int64_t plane = planes == 2 && t < blocks ? g.lo : 0;
      const int blk = first + (t < blocks ? t : t - blocks);
      if ((int64_t)(blk + 1) * BK <= g.K) {
        TA::template direct<kThreads>(a, pa + plane + blk * sa, oa);
        TB::template direct<kThreads>(a + TA::kBytes, pb + blk * sb, ob);
      } else {  // its loads are waited for here, and with them all before them
        u32x4 va[PA], vb[PB];
        fetch(va, vb, blk, plane);
        put(a, va, vb);
      }
    };
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
      if (i < total) stage(lds + i * kStage, i);
    int at = 0;
    for (int t = 0; t < total; ++t) {
      wait_stages<PA + PB, NST - 2>(total - 1 - t);
      __syncthreads();
      if (t + NST - 1 < total) stage(lds + (at == 0 ? NST - 1 : at - 1) * kStage, t + NST - 1);
      if (planes == 2 && t == blocks) settle();
      compute(lds + at * kStage);
      at = at == NST - 1 ? 0 : at + 1;
    }
  } else {
    // Whole blocks, DEPTH of them waiting in registers (their loads stand outside any branch: past the end the last block
    // is loaded again; or the compiler waits for all of them at each use); then the partial block of k (or all, of an
    // operand too narrow for 16 bytes) one after the other.  The order of k is that of the direct loads, so an output
    // has the same bits at any alignment.
    static_assert(NST == 2, "two stages");
    constexpr int DEPTH = BM > 64 ? 2 : 4;
    const bool plain = TA::plain(g.lda, g.M) && TB::plain(g.ldb, g.N);
    const int whole = plain ? min(last, (int)(g.K / BK)) : first;
    u32x4 va[DEPTH][PA], vb[DEPTH][PB];
#pragma unroll 1
    for (int p = planes - 1; p >= 0; --p) {
      const int64_t plane = p == 1 ? g.lo : 0;
      if (planes == 2 && p == 0) settle();
      if (first < whole) {
        uint32_t oa[PA], ob[PB], move_a, move_b;
        TA::template places<kThreads>(oa, move_a, g.lda, g.M, m0);
        TB::template places<kThreads>(ob, move_b, g.ldb, g.N, n0);
        const char* pa = A + plane + 2 * (ACOLS ? m0 - TA::lead(m0) : m0 * g.lda);
        const char* pb = B + 2 * (BCOLS ? n0 - TB::lead(n0) : n0 * g.ldb);
        const int64_t sa = 2 * BK * (ACOLS ? g.lda : 1), sb = 2 * BK * (BCOLS ? g.ldb : 1);
        const bool edge_a = m0 + BM > g.M, edge_b = n0 + BN > g.N;
        const auto get = [&](u32x4(&a)[PA], u32x4(&b)[PB], int blk) {
          blk = min(blk, whole - 1);
          TA::fetch_whole(a, pa + blk * sa, oa);
          TB::fetch_whole(b, pb + blk * sb, ob);
        };
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) get(va[u], vb[u], first + u);
        for (int blk = first; blk < whole; blk += DEPTH) {
#pragma unroll
          for (int u = 0; u < DEPTH; ++u) {
            // past the end: the same block once more, whose products are not formed
            char* a = lds + (u & 1) * kStage;
            TA::template put_moved<kThreads>(a, va[u], move_a, edge_a);
            TB::template put_moved<kThreads>(a + TA::kBytes, vb[u], move_b, edge_b);
            get(va[u], vb[u], blk + u + DEPTH);
            __syncthreads();
            if (blk + u < whole) compute(a);
          }
        }
        __syncthreads();
      }
      for (int blk = max(whole, first); blk < last; ++blk) {
        fetch(va[0], vb[0], blk, plane);
        put(lds, va[0], vb[0]);
        __syncthreads();
        compute(lds);
        __syncthreads();
      }
    }
  }
  if (planes == 2) {  // of half of A
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] *= 2.0f;
  }
  __syncthreads();
  write_tile<T, RP>(g, reinterpret_cast<float*>(lds) + w * kBuf, acc, split, m0 + wm * TM * 16,
                    n0 + wn * TN * 16);
}

// ----------------------------------------------------------------------------- fp32 operands
// v = hi + mid + lo, each the leading 8 bits of what is left (truncated, so every difference is exact).
SGNN_DEV void split3(f32x4 v, u32x2& hi, u32x2& mid, u32x2& lo) {
  uint32_t h[4], m[4], q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = v[i];
    h[i] = __builtin_bit_cast(uint32_t, x);
    const float r = x - __builtin_bit_cast(float, h[i] & 0xffff0000u);
    m[i] = __builtin_bit_cast(uint32_t, r);
    q[i] = __builtin_bit_cast(uint32_t, r - __builtin_bit_cast(float, m[i] & 0xffff0000u));
  }
  // the upper halves of two words as one: bytes 2, 3 of the first, then of the second
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    hi[i] = __builtin_amdgcn_perm(h[2 * i + 1], h[2 * i], 0x07060302u);
    mid[i] = __builtin_amdgcn_perm(m[2 * i + 1], m[2 * i], 0x07060302u);
    lo[i] = __builtin_amdgcn_perm(q[2 * i + 1], q[2 * i], 0x07060302u);
  }
}

// R rows by 32 k as three planes of bf16, 64 bytes a row.  Rows layout: row r's chunk c (8 k) at slot c ^ ((r >> 2) & 3).
// Cols layout, whose writers hold four rows each and write one of them at a time: the rows 4 i + e of one e stand next
// to each other, chunk c at slot c ^ e.  In both the 16 rows' chunks of one read, and 32 lanes' pieces of one write,
// cover all banks.
template <int R, bool COLS>
struct Tile32 {
  static constexpr int BK = 32, kPlane = R * BK * 2, kBytes = 3 * kPlane;
  static SGNN_DEV int at(int row, int k) {  // byte of element (row, k)
    if constexpr (COLS) return ((row & 3) * (R / 4) + (row >> 2)) * 64 + (((k >> 3) ^ (row & 3)) * 16) + (k & 7) * 2;
    return row * 64 + (((k >> 3) ^ ((row >> 2) & 3)) * 16) + (k & 7) * 2;
  }
  // Cols: this thread's block of KPER k by four rows.  Four threads side by side read 64 bytes of a line; the next bits
  // are the k, so that 32 lanes write 32 different 8 (4) byte pieces of 256 bytes.
  template <int KPER>
  static SGNN_DEV int block_k() { return (threadIdx.x >> 2) % (BK / KPER) * KPER; }
  template <int KPER>
  static SGNN_DEV int block_row() { return ((threadIdx.x >> 2) / (BK / KPER) * 4 + (threadIdx.x & 3)) * 4; }
  // Rows: KPER x four k of one row.  Cols: one block of KPER k (two or four) by four rows.  Whole blocks as Tile16's.
  static SGNN_DEV bool plain(int64_t ld, int64_t rows) { return ld < kNear && (!COLS || rows >= 4); }
  static SGNN_DEV int lead(int64_t r0) { return COLS && r0 > 0 ? 4 : 0; }
  template <int THREADS, int KPER>
  static SGNN_DEV void places(uint32_t (&o)[KPER], int& move, int64_t ld, int64_t rows, int64_t r0) {
    const int left = (int)min(rows - r0, (int64_t)R);
    move = 0;
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      if constexpr (COLS) {
        const int line = block_k<KPER>() + i, col = block_row<KPER>(), from = min(col, left - 4);
        move = min(col - from, 4);
        o[i] = 4 * ((uint32_t)line * (uint32_t)ld + (uint32_t)(lead(r0) + from));
      } else {
        const int q = i * THREADS + threadIdx.x;
        o[i] = 4 * ((uint32_t)min(q / 8, left - 1) * (uint32_t)ld + q % 8 * 4);
      }
    }
  }
  template <int KPER>
  static SGNN_DEV void fetch_whole(f32x4 (&v)[KPER], const char* first, const uint32_t (&o)[KPER]) {
#pragma unroll
    for (int i = 0; i < KPER; ++i)
      v[i] = __builtin_bit_cast(f32x4, (u32x4)*reinterpret_cast<const u32x4_any*>(first + o[i]));
  }
  template <int THREADS, int KPER>
  static SGNN_DEV void put_moved(char* lds, const f32x4 (&v)[KPER], int move, bool edge) {
    if (!COLS || !edge) return put<THREADS>(lds, v);
    f32x4 t[KPER];
#pragma unroll
    for (int i = 0; i < KPER; ++i) t[i] = __builtin_bit_cast(f32x4, move_down(__builtin_bit_cast(u32x4, v[i]), 4 * move));
    put<THREADS>(lds, t);
  }
  template <int THREADS, int KPER>
  static SGNN_DEV void fetch(f32x4 (&v)[KPER], const float* src, int64_t ld, int64_t rows, int64_t K, int64_t r0,
                             int64_t k0) {
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      int64_t line, col, lines, most;
      if constexpr (COLS) {
        line = k0 + block_k<KPER>() + i, col = r0 + block_row<KPER>(), lines = K, most = rows;
      } else {
        const int q = i * THREADS + threadIdx.x;
        line = r0 + q / 8, col = k0 + q % 8 * 4, lines = rows, most = K;
      }
      f32x4 t = {0, 0, 0, 0};
      if (line < lines && col < most) {
        const float* p = src + line * ld + col;
        if (col + 4 <= most) {
          t = __builtin_bit_cast(f32x4, (u32x4)*reinterpret_cast<const u32x4_any*>(p));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < most) t[e] = p[e];
        }
      }
      v[i] = t;
    }
  }
  template <int THREADS, int KPER>
  static SGNN_DEV void put(char* lds, const f32x4 (&v)[KPER]) {
    u32x2 hi, mid, lo;
    if constexpr (!COLS) {
#pragma unroll
      for (int i = 0; i < KPER; ++i) {
        const int q = i * THREADS + threadIdx.x, o = at(q / 8, q % 8 * 4);
        split3(v[i], hi, mid, lo);
        *reinterpret_cast<u32x2*>(lds + o) = hi;
        *reinterpret_cast<u32x2*>(lds + kPlane + o) = mid;
        *reinterpret_cast<u32x2*>(lds + 2 * kPlane + o) = lo;
      }
    } else {
      static_assert(KPER == 2 || KPER == 4, "a block's k fit one LDS word or two");
      const int k = block_k<KPER>(), r = block_row<KPER>();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int o = at(r + e, k);
        if constexpr (KPER == 4) {
          split3(f32x4{v[0][e], v[1][e], v[2][e], v[3][e]}, hi, mid, lo);
          *reinterpret_cast<u32x2*>(lds + o) = hi;
          *reinterpret_cast<u32x2*>(lds + kPlane + o) = mid;
          *reinterpret_cast<u32x2*>(lds + 2 * kPlane + o) = lo;
        } else {
          split3(f32x4{v[0][e], v[1][e], 0.0f, 0.0f}, hi, mid, lo);
          *reinterpret_cast<uint32_t*>(lds + o) = hi[0];
          *reinterpret_cast<uint32_t*>(lds + kPlane + o) = mid[0];
          *reinterpret_cast<uint32_t*>(lds + 2 * kPlane + o) = lo[0];
        }
      }
    }
  }
  static SGNN_DEV s16x8 frag(const char* lds, int plane, int r) {
    const int l = lane_id();
    return *reinterpret_cast<const s16x8*>(lds + plane * kPlane + at(r + (l & 15), 8 * (l >> 4)));
  }
};

// Sub-tiles of a wave's accumulators (at m0, n0) with a value that is not finite are formed once more over k0 .. k1 with
// fp32 matrix instructions, straight from memory, and those values replaced.  Nothing is shared between sub-tiles, as few
// products need it.  2048^3 forward and backward take 0.36 ms, of NaN alone 3.6.
constexpr int kRedo = 4;  // k per lane and step
template <bool ACOLS, bool BCOLS, int TM, int TN>
SGNN_DEV void redo_non_finite(const GemmArgs& g, f32x4 (&acc)[TM][TN], int64_t m0, int64_t n0, int64_t k0, int64_t k1) {
  static_assert(TM * TN <= 32, "a bit per sub-tile");
  uint32_t odd_tiles = 0;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const f32x4 v = acc[i][j];
      // x - x is 0 for finite x alone
      const float odd = (v[0] - v[0]) + (v[1] - v[1]) + (v[2] - v[2]) + (v[3] - v[3]);
      if (__any(odd != 0.0f)) odd_tiles |= 1u << (i * TN + j);
    }
  const int l = lane_id();
  const float *A = static_cast<const float*>(g.A), *B = static_cast<const float*>(g.B);
  while (odd_tiles) {  // the same in every lane
    const int t = __builtin_ctz(odd_tiles);
    odd_tiles &= odd_tiles - 1;
    const int64_t m = m0 + t / TN * 16 + (l & 15), n = n0 + t % TN * 16 + (l & 15), kl = k0 + kRedo * (l >> 4);
    const int64_t step_a = ACOLS ? g.lda : 1, step_b = BCOLS ? g.ldb : 1;
    const float* pa = A + (ACOLS ? m : m * g.lda) + kl * step_a;
    const float* pb = B + (BCOLS ? n : n * g.ldb) + kl * step_b;
    int64_t left = k1 - kl;  // of this lane's k
    const bool there_a = m < g.M, there_b = n < g.N;
    f32x4 s = {0, 0, 0, 0};
#pragma unroll 1
    for (int64_t k = k0; k < k1; k += 4 * kRedo) {
      float a[kRedo], b[kRedo];
#pragma unroll
      for (int e = 0; e < kRedo; ++e) {
        a[e] = there_a && e < left ? pa[e * step_a] : 0.0f;
        b[e] = there_b && e < left ? pb[e * step_b] : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < kRedo; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(b[e], a[e], s, 0, 0, 0);
      pa += 4 * kRedo * step_a, pb += 4 * kRedo * step_b, left -= 4 * kRedo;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (t == i * TN + j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!(acc[i][j][r] - acc[i][j][r] == 0.0f)) acc[i][j][r] = s[r];
  }
}

// a b = sum of the parts' products; left out are mid lo, lo mid and lo lo, below 2^-22 of |a b| together.
// An infinite operand gives inf - inf = NaN in its parts, and a part of 0 times infinity is one too: outputs that
// are not finite are formed once more (redo_non_finite).
// NST = 2 stages of LDS: the next block is split and written while this one's products run; a matrix instruction takes
// 16 cycles, in which a wave issues three others (4096^3: 630 to 670 us, 205 to 218 TFLOP/s; 765 with one stage, where split and
// products take turns and the two waves of a SIMD fall into step; other mixtures asked of the scheduler: 704 to 733).
// NST = 1: half the LDS, so two workgroups per CU, one's epilogue beside the other's products: better where k is short
// (200003 x 384 x 128, silu: 180 us against 211).
template <bool ACOLS, bool BCOLS, int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_gemm32(GemmArgs g) {
  constexpr int BK = 32, kThreads = 64 * WM * WN;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  using TA = Tile32<BM, ACOLS>;
  using TB = Tile32<BN, BCOLS>;
  constexpr int kStage = TA::kBytes + TB::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[NST * kStage];
  constexpr int RP = 2, kBuf = RP * 16 * 16 * TN;
  static_assert(kBuf * 4 * WM * WN <= NST * kStage, "the epilogue's buffers fit");
  const int w = wave_id(), wm = w / WN, wn = w % WN;
  int tm, tn;
  tile_of(g, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int split = blockIdx.z;
  const float* A = static_cast<const float*>(g.A);
  const float* B = static_cast<const float*>(g.B);
  int first, last;
  blocks_of(g, BK, split, first, last);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  constexpr int PA = BM * BK / 4 / kThreads, PB = BN * BK / 4 / kThreads;
  f32x4 va[PA], vb[PB];
  const auto compute = [&](const char* sa) {
    const char* sb = sa + TA::kBytes;
    s16x8 fb[TN][3];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int p = 0; p < 3; ++p) fb[j][p] = TB::frag(sb, p, (wn * TN + j) * 16);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      s16x8 fa[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) fa[p] = TA::frag(sa, p, (wm * TM + i) * 16);
      // Smallest products first, from zero, and added by the vector units: a matrix instruction drops what lies far below
      // the sum it adds to, which took the small parts out of long sums (4096^3 of positive values: off by 1e-5, now by
      // 1.5e-7, at 2 to 7 % more time).
      f32x4 t[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = mfma16<bf16_t>(fb[j][2], fa[0], f32x4{0, 0, 0, 0});
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = mfma16<bf16_t>(fb[j][0], fa[2], t[j]);
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = mfma16<bf16_t>(fb[j][1], fa[1], t[j]);
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = mfma16<bf16_t>(fb[j][1], fa[0], t[j]);
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = mfma16<bf16_t>(fb[j][0], fa[1], t[j]);
#pragma unroll
      for (int j = 0; j < TN; ++j) t[j] = mfma16<bf16_t>(fb[j][0], fa[0], t[j]);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] += t[j];
    }
  };
  // As in k_gemm16: whole blocks without branches, then the partial one (or all, of an operand too narrow).
  const bool plain = TA::plain(g.lda, g.M) && TB::plain(g.ldb, g.N);
  const int whole = plain ? min(last, (int)(g.K / BK)) : first;
  if (first < whole) {
    uint32_t oa[PA], ob[PB];
    int move_a, move_b;
    TA::template places<kThreads>(oa, move_a, g.lda, g.M, m0);
    TB::template places<kThreads>(ob, move_b, g.ldb, g.N, n0);
    const char* pa = reinterpret_cast<const char*>(A + (ACOLS ? m0 - TA::lead(m0) : m0 * g.lda));
    const char* pb = reinterpret_cast<const char*>(B + (BCOLS ? n0 - TB::lead(n0) : n0 * g.ldb));
    const int64_t step_a = 4 * BK * (ACOLS ? g.lda : 1), step_b = 4 * BK * (BCOLS ? g.ldb : 1);
    const bool edge_a = m0 + BM > g.M, edge_b = n0 + BN > g.N;
    const auto get = [&](f32x4(&a)[PA], f32x4(&b)[PB], int blk) {
      blk = min(blk, whole - 1);
      TA::fetch_whole(a, pa + blk * step_a, oa);
      TB::fetch_whole(b, pb + blk * step_b, ob);
    };
    const auto place = [&](char* a, const f32x4(&x)[PA], const f32x4(&y)[PB]) {
      TA::template put_moved<kThreads>(a, x, move_a, edge_a);
      TB::template put_moved<kThreads>(a + TA::kBytes, y, move_b, edge_b);
    };
    get(va, vb, first);
    if constexpr (NST == 1) {
      for (int blk = first; blk < whole; ++blk) {
        place(lds, va, vb);
        get(va, vb, blk + 1);
        __syncthreads();
        compute(lds);
        __syncthreads();
      }
    } else {
      place(lds, va, vb);
      get(va, vb, first + 1);
      __syncthreads();
      char *here = lds, *there = lds + kStage;
      for (int blk = first; blk < whole; ++blk) {
        // after the last block: it once more, into the stage that is not read again
        compute(here);
        place(there, va, vb);
        get(va, vb, blk + 2);
        __syncthreads();
        char* t = here;
        here = there, there = t;
      }
    }
  }
  for (int blk = max(whole, first); blk < last; ++blk) {
    TA::template fetch<kThreads>(va, A, g.lda, g.M, g.K, m0, (int64_t)blk * BK);
    TB::template fetch<kThreads>(vb, B, g.ldb, g.N, g.K, n0, (int64_t)blk * BK);
    TA::template put<kThreads>(lds, va);
    TB::template put<kThreads>(lds + TA::kBytes, vb);
    __syncthreads();
    compute(lds);
    __syncthreads();
  }
  __syncthreads();
  redo_non_finite<ACOLS, BCOLS>(g, acc, m0 + wm * TM * 16, n0 + wn * TN * 16, (int64_t)first * BK,
                                min((int64_t)last * BK, g.K));
  write_tile<float, RP>(g, reinterpret_cast<float*>(lds) + w * kBuf, acc, split, m0 + wm * TM * 16,
                        n0 + wn * TN * 16);
}

// ----------------------------------------------------------------------------- few rows
// M <= 16 MT rows of x, both operands with k contiguous: a workgroup takes 16 MT columns n, its W waves every W-th block
// of k, straight from memory into the matrix instructions' registers (a lane reads 32 or 64 bytes of one row of w at a
// time, a row's four lanes 128 or 256), and the waves' sums are added in order through LDS.  Bounded by w's bytes: one row
// by 4096 x 4096 bf16 takes 8 to 9 us, 3.9 TB/s, of which some 3 are launch and first latency (tiles of 64: 21 us).
template <typename T, int MT, int W>
__global__ __launch_bounds__(64 * W) void k_gemm_rows(GemmArgs g) {
  constexpr bool k32 = sizeof(T) == 4;
  constexpr int BK = 64, V = 16 / sizeof(T), kLoads = 16 / V, U = MT == 1 ? 2 : 1;  // a lane's 16 k of a block
  __shared__ float part[W][16 * MT][16 * MT + 4];
  const int l = lane_id(), w = wave_id(), i = l & 15, kl = 16 * (l >> 4);
  const int64_t n0 = (int64_t)blockIdx.x * 16 * MT;
  const T* A = static_cast<const T*>(g.A);
  const T* B = static_cast<const T*>(g.B);
  f32x4 acc[MT][MT];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b) acc[a][b] = f32x4{0, 0, 0, 0};
  // 16 k of a row from k, as loaded; zeros past K and for rows that are not there
  const auto load = [&](u32x4(&v)[kLoads], const T* p, int64_t k, bool there) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int64_t c = k + q * V;
      v[q] = u32x4{0, 0, 0, 0};
      if (!there || c >= g.K) continue;
      if (c + V <= g.K) {
        v[q] = *reinterpret_cast<const u32x4_any*>(p + c);
      } else {
        typedef T TV __attribute__((ext_vector_type(V)));
        TV t = __builtin_bit_cast(TV, v[q]);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c + e < g.K) t[e] = p[c + e];
        v[q] = __builtin_bit_cast(u32x4, t);
      }
    }
  };
  for (int64_t k0 = (int64_t)w * BK; k0 < g.K; k0 += (int64_t)W * BK * U) {
    u32x4 xa[U][MT][kLoads], wb[U][MT][kLoads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + (int64_t)u * W * BK + kl;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t n = n0 + 16 * t + i, m = 16 * t + i;
        load(wb[u][t], B + n * g.ldb, k, n < g.N);
        load(xa[u][t], A + m * g.lda, k, m < g.M);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < kLoads; ++q)
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
          for (int b = 0; b < MT; ++b) {
            if constexpr (k32) {
              const f32x4 p = __builtin_bit_cast(f32x4, wb[u][b][q]), x = __builtin_bit_cast(f32x4, xa[u][a][q]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[e], x[e], acc[a][b], 0, 0, 0);
            } else {
              acc[a][b] = mfma16<T>(__builtin_bit_cast(s16x8, wb[u][b][q]), __builtin_bit_cast(s16x8, xa[u][a][q]), acc[a][b]);
            }
          }
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b)
      *reinterpret_cast<f32x4*>(&part[w][16 * a + i][16 * b + 4 * (l >> 4)]) = acc[a][b];
  __syncthreads();
  constexpr int kPer = 16 * MT / V;  // 16-byte pieces of an output row
  for (int t = threadIdx.x; t < 16 * MT * kPer; t += 64 * W) {
    const int m = t / kPer, c = t % kPer * V;
    if (m >= g.M || n0 + c >= g.N) continue;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.0f;
    for (int q = 0; q < W; ++q)
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += part[q][m][c + e];
    const int cnt = (int)min((int64_t)V, g.N - n0 - c);
    float bias[V];
    load_bias<T>(g, n0 + c, cnt, bias);
    finish<T>(g, m, n0 + c, v, bias, cnt);
  }
}

// ----------------------------------------------------------------------------- split k
// Partials summed, then the epilogue: 32 pieces of 16 output bytes per workgroup, eight threads per piece that sum an
// eighth of the splits each, in order, and are added in order.
constexpr int kJoinParts = 8;
template <typename T>
__global__ __launch_bounds__(32 * kJoinParts) void k_gemm_join(GemmArgs g) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float sums[kJoinParts][32][V + 1];
  const int64_t per = (g.N + V - 1) / V, total = g.M * per;
  const int i = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * 32 + i;
  const int64_t m = t / per, n = (t - m * per) * V;
  const int cnt = t < total ? (int)min((int64_t)V, g.N - n) : 0;
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = 0.0f;
  if (cnt > 0) {
    const int s0 = g.nsplit * part / kJoinParts, s1 = g.nsplit * (part + 1) / kJoinParts;
    const float* p = g.part + ((int64_t)s0 * g.M + m) * g.N + n;
#pragma unroll 4
    for (int s = s0; s < s1; ++s, p += g.M * g.N) {
      float u[V];
      load_some<V>(p, cnt, u);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += u[e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sums[part][i][e] = v[e];
  __syncthreads();
  if (part != 0 || cnt <= 0) return;
  for (int q = 1; q < kJoinParts; ++q)
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] += sums[q][i][e];
  float bias[V];
  load_bias<T>(g, n, cnt, bias);
  finish<T>(g, m, n, v, bias, cnt);
}

// ----------------------------------------------------------------------------- choice and launch
struct Plan {
  int bm, bn, nsplit;
};

// The larger tile moves fewer bytes per product through LDS and L2, the smaller ones fill the 256 CUs sooner.  Square
// outputs, x w^T, in us:
//   256 x 256 (16 bits) or 128 x 128, k 2048: 169 of the larger tiles 51 / 56, 100 of them 59 / 32; k 512: 196 tiles
//   22.5 / 23.4, 169 21.9 / 21.3.
//   256 x 128 (fp32) or 128 x 128, 512 of the larger tiles: k 1024 160 / 168, k 256 58 / 55; 128 of them, k 1024 66 / 68.
//   128 x 128 or 64 x 64: 16 bits, k 1024: 144 of the larger tiles 15 / 16, 100 of them 23 / 10; k 16384: 36 tiles
//   42 / 44, 1 tile 12 / 9.  fp32, k 512: 400 tiles 44 / 55, 144 34 / 26; k 4096: 36 tiles 41 / 49, 4 tiles 23 / 14.  With
//   64 rows or columns half of the larger tile is empty (dw of 100000 rows, 64 x 192, fp32: 48 / 36).
// k is split over workgroups where the tiles leave CUs idle: one workgroup per CU, and two where k is long enough to pay
// for the partial sums (128 x 128, two / one, us: bf16 2048^2, k 1024 38 / 16; 1536^2, k 16384 91 / 164; fp32 2048^2,
// k 512 49 / 36; 1536^2, k 1024 47 / 61).
Plan plan_of(const Gemm& g) {
  const auto tiles = [&](int bm, int bn) { return ((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn); };
  const int bk = g.dtype == SGNN_F32 ? 32 : 64;
  Plan p{64, 64, 1};
  const bool f32 = g.dtype == SGNN_F32;
  const bool long_k = std::min(g.M, g.N) > 64 && g.K >= (f32 ? 2048 : 8192) && tiles(128, 128) * g.K >= (f32 ? 1 << 16 : 1 << 18);
  if (!f32 && tiles(256, 256) >= 192) p = {256, 256, 1};
  else if (f32 && tiles(256, 128) >= 256 && g.K >= 1024) p = {256, 128, 1};
  else if (tiles(128, 128) >= (f32 ? 256 : 128) || long_k) p = {128, 128, 1};
  const int64_t blocks = (g.K + bk - 1) / bk, wgs = p.bm != 256 && blocks >= (f32 ? 32 : 64) ? 512 : 256;
  const int64_t want = wgs / std::max<int64_t>(1, tiles(p.bm, p.bn));
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({want, blocks / 8, 256}));
  return p;
}

template <typename T, bool AC, bool BC>
void launch_tiles(const GemmArgs& g, const Plan& p, dim3 grid, bool direct, hipStream_t s) {
  if constexpr (std::is_same_v<T, float>) {
    if (p.bm == 256)
      hipLaunchKernelGGL((k_gemm32<AC, BC, 256, 128, 4, 2, 2>), grid, dim3(512), 0, s, g);
    else if (p.bm == 128)
      hipLaunchKernelGGL((k_gemm32<AC, BC, 128, 128, 2, 2, 1>), grid, dim3(256), 0, s, g);
    else
      hipLaunchKernelGGL((k_gemm32<AC, BC, 64, 64, 2, 2, 2>), grid, dim3(256), 0, s, g);
  } else {
    if (p.bm == 256)
      hipLaunchKernelGGL((k_gemm16<T, AC, BC, 256, 256, 2, 4, true, 2>), grid, dim3(512), 0, s, g);
    else if (p.bm == 128 && direct)
      hipLaunchKernelGGL((k_gemm16<T, AC, BC, 128, 128, 2, 2, true, 2>), grid, dim3(256), 0, s, g);
    else if (p.bm == 128)
      hipLaunchKernelGGL((k_gemm16<T, AC, BC, 128, 128, 2, 2, false, 2>), grid, dim3(256), 0, s, g);
    else if (direct)
      hipLaunchKernelGGL((k_gemm16<T, AC, BC, 64, 64, 2, 2, true, 4>), grid, dim3(256), 0, s, g);
    else
      hipLaunchKernelGGL((k_gemm16<T, AC, BC, 64, 64, 2, 2, false, 2>), grid, dim3(256), 0, s, g);
  }
}

// The row kernel: 32 rows at most, both operands with k contiguous.
bool rows_ok(const Gemm& g) { return !g.a_cols && !g.b_cols && g.M <= 32; }

template <typename T>
void launch_rows(const GemmArgs& g, hipStream_t s) {
  // a wave per 128 of k, up to eight
  const bool many = g.K > 512;
  const auto go = [&](auto kernel, int mt, int w) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((g.N + 16 * mt - 1) / (16 * mt))), dim3(64 * w), 0, s, g);
  };
  if (g.M <= 16) {
    if (many) go(k_gemm_rows<T, 1, 8>, 1, 8);
    else go(k_gemm_rows<T, 1, 4>, 1, 4);
  } else {
    if (many) go(k_gemm_rows<T, 2, 8>, 2, 8);
    else go(k_gemm_rows<T, 2, 4>, 2, 4);
  }
}

// Whether the direct-to-LDS loads serve an operand: 16-byte lines whose offsets within a tile fit 32 bits.
bool direct_ok(const void* p, int64_t ld, bool cols, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld < kNear &&
         (!cols || rows % 8 == 0);
}

}  // namespace

namespace sgnn {

size_t gemm_workspace_bytes(const Gemm& g) {
  if (g.M <= 0 || g.N <= 0 || g.K <= 0 || rows_ok(g)) return 0;
  const int s = plan_of(g).nsplit;
  return s > 1 ? sizeof(float) * (size_t)s * (size_t)g.M * (size_t)g.N : 0;
}

int gemm_run(const Gemm& g, void* workspace, size_t workspace_bytes, void* stream) {
  if (g.M == 0 || g.N == 0) return SGNN_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  GemmArgs a{g.A, g.B, g.bias, g.res, g.slope, g.C, nullptr, g.lda, g.ldb, g.ldr, g.ldc, g.M, g.N, g.K,
             g.act, 1, 0, 0, g.lo};
  if (rows_ok(g)) {
    with_type(g.dtype, [&](auto* t) {
      launch_rows<std::remove_pointer_t<decltype(t)>>(a, s);
      return 0;
    });
    return check_launch("gemm");
  }
  Plan p = plan_of(g);
  const bool direct = direct_ok(g.A, g.lda, g.a_cols, g.M) && direct_ok(g.B, g.ldb, g.b_cols, g.N);
  if (!direct && p.bm == 256 && g.dtype != SGNN_F32) p.bm = p.bn = 128;
  const int64_t tm = (g.M + p.bm - 1) / p.bm, tn = (g.N + p.bn - 1) / p.bn;
  if (tm > INT32_MAX / tn || g.K > (int64_t)INT32_MAX * 32)
    return set_error(SGNN_ERR_UNSUPPORTED, "gemm: more than 2^31 tiles or blocks of k");
  a.nsplit = p.nsplit, a.tiles_m = (int32_t)tm, a.tiles_n = (int32_t)tn;
  if (p.nsplit > 1) {
    if (!workspace || workspace_bytes < gemm_workspace_bytes(g))
      return set_error(SGNN_ERR_INVALID, "gemm: workspace too small");
    a.part = static_cast<float*>(workspace);
  }
  const dim3 grid((unsigned)(tm * tn), 1, (unsigned)p.nsplit);
  with_type(g.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!g.a_cols && !g.b_cols) launch_tiles<T, false, false>(a, p, grid, direct, s);
    else if (!g.a_cols) launch_tiles<T, false, true>(a, p, grid, direct, s);
    else launch_tiles<T, true, true>(a, p, grid, direct, s);
    if (p.nsplit > 1) {
      const int64_t items = g.M * ((g.N + 16 / (int64_t)sizeof(T) - 1) / (16 / (int64_t)sizeof(T)));
      hipLaunchKernelGGL(k_gemm_join<T>, dim3((unsigned)((items + 31) / 32)), dim3(32 * kJoinParts), 0, s, a);
    }
    return 0;
  });
  return check_launch("gemm");
}

}  // namespace sgnn
