// The 16-bit tiles that the matrix products stage through LDS (gemm.hip, muon.hip), and their matrix instruction.
#pragma once
#include "ops_types.h"

namespace sgnn {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define SGNN_LDS __attribute__((address_space(3)))

template <typename T>
SGNN_DEV f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  if constexpr (std::is_same_v<T, bf16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
}

// Leading dimensions below this keep a tile's byte offsets in 32 bits (256 lines of 4 bytes a value at most).
constexpr int64_t kNear = 1 << 22;

// One operand's tile in LDS: R rows (m or n) by BK of k, in 16-byte chunks.
//   rows layout (k contiguous in memory): row r's chunk c (8 k) at slot c ^ swizzle(r)
//   cols layout (m / n contiguous): k's chunk c (8 rows) at slot c ^ 2 h(k); read back transposed
// The swizzles put the pieces that one LDS instruction touches at a time on different banks.
template <int R, int BK, bool COLS>
struct Tile16 {
  static constexpr int kChunks = COLS ? R / 8 : BK / 8;  // chunks per line of memory (a row, or a k)
  static constexpr int kLines = COLS ? BK : R;
  static constexpr int kBytes = R * BK * 2;
  static SGNN_DEV int swizzle(int line) {
    if constexpr (COLS) return (2 * ((line & 3) | ((line >> 1) & 4))) & (kChunks - 1);
    return kChunks == 8 ? (line >> 1) & 7 : (line >> 2) & 3;
  }

  // Chunk q of the tile (in LDS order) holds memory's line q / kChunks, chunk (q % kChunks) ^ swizzle.  offsets():
  // this lane's chunks' bytes from the tile's first element, the same for every block of k.  Lines and chunks past
  // the last row read another one's data: their outputs are not stored.
  template <int THREADS, int KPER>
  static SGNN_DEV void offsets(uint32_t (&o)[KPER], int64_t ld, int64_t rows, int64_t r0, int tid = threadIdx.x) {
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      const int q = i * THREADS + tid;
      const int line = q / kChunks, c = (q % kChunks) ^ swizzle(line);
      const int left = (int)min(rows - r0, (int64_t)R);
      o[i] = 2 * (COLS ? (uint32_t)line * (uint32_t)ld + min(8 * c, left - 8)
                       : (uint32_t)min(line, left - 1) * (uint32_t)ld + 8 * c);
    }
  }
  // first: the block's first element.  The loads' 64 x 16 bytes land at m0 in lane order; they are written as
  // instructions, as the compiler makes every later LDS read wait for the builtin's.  The caller waits (vmcnt); no other code of
  // these kernels has a value in m0.
  template <int THREADS, int KPER>
  static SGNN_DEV void direct(const char* lds, const char* first, const uint32_t (&o)[KPER], int tid = threadIdx.x) {
    const uint64_t at = (uint64_t)first;
    const uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(
          (uint32_t)(uintptr_t)(const SGNN_LDS char*)lds + (i * THREADS + tid / 64 * 64) * 16);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(to), "v"(o[i]), "s"(base)
                   : "memory");
    }
  }

  // The same through registers, at any alignment: whole blocks of k by places(), like offsets().  In cols the chunks that
  // the last row cuts, or that lie past it, are read 8 rows from the end and moved into place by put_moved(); `move`
  // holds their distances, 4 bits each.  first: `lead` rows (0 or 8, as places() says) before the tile's first.
  static SGNN_DEV bool plain(int64_t ld, int64_t rows) { return ld < kNear && (!COLS || rows >= 8); }
  static SGNN_DEV int lead(int64_t r0) { return COLS && r0 > 0 ? 8 : 0; }
  template <int THREADS, int KPER>
  static SGNN_DEV void places(uint32_t (&o)[KPER], uint32_t& move, int64_t ld, int64_t rows, int64_t r0) {
    const int left = (int)min(rows - r0, (int64_t)R);
    move = 0;
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      const int q = i * THREADS + threadIdx.x;
      const int line = q / kChunks, c = (q % kChunks) ^ swizzle(line);
      if constexpr (COLS) {
        const int from = min(8 * c, left - 8);  // down to -7 where r0 > 0
        move |= (uint32_t)min(8 * c - from, 8) << (4 * i);
        o[i] = 2 * ((uint32_t)line * (uint32_t)ld + (uint32_t)(lead(r0) + from));
      } else {
        o[i] = 2 * ((uint32_t)min(line, left - 1) * (uint32_t)ld + 8 * c);
      }
    }
  }
  template <int KPER>
  static SGNN_DEV void fetch_whole(u32x4 (&v)[KPER], const char* first, const uint32_t (&o)[KPER]) {
#pragma unroll
    for (int i = 0; i < KPER; ++i) v[i] = *reinterpret_cast<const u32x4_any*>(first + o[i]);
  }
  template <int THREADS, int KPER>
  static SGNN_DEV void put_moved(char* lds, const u32x4 (&v)[KPER], uint32_t move, bool edge) {
    if (!COLS || !edge) return put<THREADS>(lds, v);
    u32x4 t[KPER];
#pragma unroll
    for (int i = 0; i < KPER; ++i) t[i] = move_down(v[i], 2 * (move >> (4 * i) & 15));
    put<THREADS>(lds, t);
  }
  // Any block, with zeros past K (and past the last row, in cols).
  template <int THREADS, int KPER>
  static SGNN_DEV void fetch(u32x4 (&v)[KPER], const char* src, int64_t ld, int64_t rows, int64_t K, int64_t r0,
                             int64_t k0) {
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      const int q = i * THREADS + threadIdx.x;
      const int line = q / kChunks, c = (q % kChunks) ^ swizzle(line);
      const int64_t gl = (COLS ? k0 : r0) + line, gc = (COLS ? r0 : k0) + 8 * c;
      const int64_t lines = COLS ? K : rows, most = COLS ? rows : K;
      u32x4 t = {0, 0, 0, 0};
      if (gl < lines && gc < most) {
        const char* p = src + 2 * (gl * ld + gc);
        if (gc + 8 <= most) {
          t = *reinterpret_cast<const u32x4_any*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (gc + e < most) t[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
        }
      }
      v[i] = t;
    }
  }
  template <int THREADS, int KPER>
  static SGNN_DEV void put(char* lds, const u32x4 (&v)[KPER]) {
#pragma unroll
    for (int i = 0; i < KPER; ++i) *reinterpret_cast<u32x4*>(lds + (i * THREADS + threadIdx.x) * 16) = v[i];
  }

  // Fragment of 16 rows from r (a multiple of 16) by 32 k from 32 kk: lane l has row l & 15, k 8 (l >> 4) .. + 7.
  static SGNN_DEV s16x8 frag(const char* lds, int r, int kk) {
    const int l = lane_id();
    if constexpr (!COLS) {
      const int row = r + (l & 15);
      return *reinterpret_cast<const s16x8*>(lds + (row * kChunks + ((4 * kk + (l >> 4)) ^ swizzle(row))) * 16);
    } else {
      // ds_read_b64_tr_b16: lanes 4 j .. 4 j + 3 of a group of 16 read 16 rows of k + j, lane i gets row i of 4 k
      const int k = 32 * kk + 8 * (l >> 4) + ((l & 15) >> 2);
      const int at = (k * kChunks + ((r / 8 + ((l & 3) >> 1)) ^ swizzle(k))) * 16 + (l & 1) * 8;
      // k + 4 has the same swizzle
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SGNN_LDS s16x4*)(lds + at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SGNN_LDS s16x4*)(lds + at + 4 * kChunks * 16));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// The order asked of the scheduler for the products of two steps of 32 k (TM x TN sub-tiles, RA / RB LDS reads per
// fragment): fragments are read two rows of products ahead of their use.  Left to itself the compiler reads each right
// before its products, with LDS's latency in the open.
template <int TM, int TN, int RA, int RB>
SGNN_DEV void order_products() {
  constexpr int kMfma = 0x008, kRead = 0x100, kNext = (TM * RA + TN * RB + TM - 1) / TM;
  __builtin_amdgcn_sched_group_barrier(kRead, TN * RB + 2 * RA, 0);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, TN, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, kNext, 0);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMfma, TN, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, RA, 0);
  }
}

// Waits until at most `keep` stages' direct loads (PER of this wave each) are under way.
template <int PER, int MOST>
SGNN_DEV void wait_stages(int keep) {
  static_assert(MOST <= 2 && PER * MOST < 64, "vmcnt's range");
  if (MOST >= 2 && keep >= 2) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(PER * 2) : "memory");
  else if (MOST >= 1 && keep >= 1) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(PER) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
}

}  // namespace sgnn
