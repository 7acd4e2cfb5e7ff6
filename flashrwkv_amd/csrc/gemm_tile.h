// Tiled 16-bit matrix product for gfx950: one workgroup's BP x BQ tile of
//   D[p][q] = sum_k A[p][k] B[q][k],   fp32 accumulators,
// with v_mfma_f32_16x16x32 (bf16 or fp16 operands).
//
// Either operand may lie in memory with k contiguous ("k-major": rows are p or
// q) or with p / q contiguous ("x-major": rows are k). Tiles of 64 k go from
// HBM straight into LDS (16 bytes a lane, no registers), NS stages deep: at
// step t the workgroup waits for stage t, starts the load of stage t + NS - 1
// into the buffer that step t - 1 has read, and multiplies stage t.
//
// LDS holds a stage unpadded (the load writes 64 consecutive 16-byte pieces a
// wave), so bank conflicts are avoided by which piece goes where:
//   k-major  row x of 64 k = 8 pieces; piece c lies at c ^ ((x >> 1) & 7).
//            An operand read takes one piece of 16 consecutive rows: rows x
//            and x + 1 lie in different halves of the 64 banks, and the 8 row
//            pairs in different pieces.
//   x-major  row k of BX x = BX/16 granules of 32 bytes; granule c lies at
//            c ^ f(k), f(k) = (k & 3) | ((k >> 3) & 1) << 2. A transposing read
//            (ds_read_b64_tr_b16) takes one granule of rows 8g + 0..3 for the
//            lane groups g: f differs over the 8 rows of a half wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wkv7_device.h"

namespace frwkv {
namespace gemm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;      // k of one LDS stage
constexpr int kThreads = 512;  // 8 waves, two a SIMD

enum class Major { kK, kX };

template <typename T>
__device__ __forceinline__ f32x4 mfma(i16x8 a, i16x8 b, f32x4 c) {
  if constexpr (__is_same(T, Bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// One operand in memory. `rows` and `cols` bound what may be read: a k-major
// operand has `rows` values of p / q, an x-major one `rows` values of k and
// `cols` of p / q (a multiple of 8). Reads beyond a bound are turned to the
// last row or to column 0; what they bring has to be multiplied by zeros or
// land in rows and columns of D that the caller drops.
struct Operand {
  const uint16_t* data;
  int64_t ld;  // elements between rows
  int32_t rows;
  int32_t cols;
};

// 64 lanes x 16 bytes from per-lane addresses to LDS bytes [lds, lds + 1024).
// The hardware adds lane * 16 to the address in m0, which is wave-uniform. In
// asm because the compiler, unable to tell the stages apart, puts a wait for
// the whole queue before every LDS read that follows the builtin.
__device__ __forceinline__ void load_to_lds(const void* src, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(src), "s"(lds));
}

// Waits until at most kLeft of this wave's loads are outstanding and its LDS
// reads have returned, then for the workgroup.
template <int kLeft>
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kLeft) : "memory");
}

// The loads of one operand's stages by the whole workgroup.
template <Major M, int BX>
struct Loader {
  static constexpr int kRounds = BX * 8 / kThreads;
  static constexpr int kBytes = BX * kStep * 2;
  static_assert(kRounds >= 1, "a stage is at least one piece a thread");
  static_assert(M == Major::kK || BX >= 128, "x-major rows hold at least 8 granules");

  const uint16_t* src[kRounds];  // k-major: this thread's rows; x-major: its column
  int64_t ld;
  int32_t row;
  int32_t last;

  __device__ __forceinline__ void init(const Operand& op, int x0, int k0) {
    const int tid = threadIdx.x;
    if constexpr (M == Major::kK) {
      const int piece = (tid & 7) ^ ((tid >> 4) & 7);
#pragma unroll
      for (int j = 0; j < kRounds; ++j) {
        int r = x0 + j * (kThreads / 8) + (tid >> 3);
        r = r < op.rows ? r : op.rows - 1;
        src[j] = op.data + r * op.ld + k0 + piece * 8;
      }
    } else {
      constexpr int kPieces = BX / 8;
      row = k0 + tid / kPieces;
      last = op.rows - 1;
      ld = op.ld;
      const int at = tid % kPieces;
      const int k = tid / kPieces;
      const int f = (k & 3) | (((k >> 3) & 1) << 2);
      int x = x0 + (((at >> 1) ^ f) << 4) + ((at & 1) << 3);
      x = x < op.cols ? x : 0;
      src[0] = op.data + x;
    }
  }

  // Starts the loads of the next stage (stages are taken in order).
  __device__ __forceinline__ void next(uint32_t lds) {
    const uint32_t base =
        lds + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)) * 1024u;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const uint16_t* p;
      if constexpr (M == Major::kK) {
        p = src[j];
        src[j] += kStep;
      } else {
        int r = row + j * (kThreads / (BX / 8));
        r = r < last ? r : last;
        p = src[0] + r * ld;
      }
      load_to_lds(p, base + static_cast<uint32_t>(j) * (kThreads * 16u));
    }
    if constexpr (M == Major::kX) row += kStep;
  }
};

// Operand registers of 16 x 32 blocks read from a stage. Lane (g = lane / 16,
// n = lane % 16) holds x = n, k = 8g .. 8g + 7 of the block.
template <Major M, int BX>
struct Reader {
  uint32_t at[M == Major::kK ? 2 : 8];

  // x0: the wave's first x in the tile, a multiple of 16.
  __device__ __forceinline__ void init(int x0) {
    const int lane = threadIdx.x & 63;
    const int g = lane >> 4, n = lane & 15;
    if constexpr (M == Major::kK) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        at[kk] = (x0 + n) * (kStep * 2) + (((kk * 4 + g) ^ (n >> 1)) << 4);
      }
    } else {
      const int f = (n >> 2) | ((g & 1) << 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        at[i] = (8 * g + (n >> 2)) * (BX * 2) + (((x0 / 16 + i) ^ f) << 5) + ((n & 3) << 3);
      }
    }
  }

  // Block i (x0 + 16 i ..), k half kk of the stage at LDS address `stage`.
  __device__ __forceinline__ i16x8 read(const char* stage, int i, int kk) const {
    if constexpr (M == Major::kK) {
      return *reinterpret_cast<const i16x8*>(stage + at[kk] + i * (16 * kStep * 2));
    } else {
      typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
      const char* p = stage + at[i] + kk * (32 * BX * 2);
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 4 * BX * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// A workgroup's product. WP x WQ waves, each with TP x TQ blocks of 16 x 16;
// acc[i][j] of lane (g, n) is D[p0 + 16 i + 4 g + r][q0 + 16 j + n], r = 0..3,
// p0 = BP / WP * (wave / WQ), q0 = BQ / WQ * (wave % WQ).
template <typename T, Major MA, Major MB, int BP, int BQ, int WP, int WQ, int NS>
struct Tile {
  static constexpr int kBP = BP, kBQ = BQ, kWP = WP, kWQ = WQ;
  static constexpr int TP = BP / WP / 16;
  static constexpr int TQ = BQ / WQ / 16;
  static constexpr int kStageBytes = (BP + BQ) * kStep * 2;
  static constexpr int kLdsBytes = NS * kStageBytes;
  static_assert(WP * WQ * 64 == kThreads, "8 waves");
  static_assert(MA == Major::kK || TP <= 8, "x-major block addresses");
  static_assert(MB == Major::kK || TQ <= 8, "x-major block addresses");
  static_assert(kLdsBytes <= 160 * 1024, "LDS of a CU");

  using LoadA = Loader<MA, BP>;
  using LoadB = Loader<MB, BQ>;
  static constexpr int kLoads = LoadA::kRounds + LoadB::kRounds;

  f32x4 acc[TP][TQ];

  static __device__ __forceinline__ int wave() {
    return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  }
  static __device__ __forceinline__ int wave_p0() { return (wave() / WQ) * (BP / WP); }
  static __device__ __forceinline__ int wave_q0() { return (wave() % WQ) * (BQ / WQ); }

  // steps: number of 64-k stages from k0 on (at least 1). smem: kLdsBytes.
  __device__ __forceinline__ void run(const Operand& a, const Operand& b, int p0, int q0, int k0,
                                      int steps, char* smem) {
    const uint32_t lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
    LoadA la;
    LoadB lb;
    la.init(a, p0, k0);
    lb.init(b, q0, k0);
    Reader<MA, BP> ra;
    Reader<MB, BQ> rb;
    ra.init(wave_p0());
    rb.init(wave_q0());
#pragma unroll
    for (int i = 0; i < TP; ++i) {
#pragma unroll
      for (int j = 0; j < TQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
      if (s < steps) {
        la.next(lds + s * kStageBytes);
        lb.next(lds + s * kStageBytes + LoadA::kBytes);
      }
    }
    int read_at = 0, load_at = NS - 1;
    for (int t = 0; t < steps; ++t) {
      if (NS > 2 && t + NS - 1 <= steps) {
        wait_and_barrier<(NS - 2) * kLoads>();
      } else {
        wait_and_barrier<0>();
      }
      if (t + NS - 1 < steps) {
        la.next(lds + load_at * kStageBytes);
        lb.next(lds + load_at * kStageBytes + LoadA::kBytes);
      }
      const char* sa = smem + read_at * kStageBytes;
      const char* sb = sa + LoadA::kBytes;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        i16x8 af[TP], bf[TQ];
#pragma unroll
        for (int j = 0; j < TQ; ++j) bf[j] = rb.read(sb, j, kk);
#pragma unroll
        for (int i = 0; i < TP; ++i) af[i] = ra.read(sa, i, kk);
#pragma unroll
        for (int i = 0; i < TP; ++i) {
#pragma unroll
          for (int j = 0; j < TQ; ++j) acc[i][j] = mfma<T>(af[i], bf[j], acc[i][j]);
        }
      }
      read_at = read_at + 1 == NS ? 0 : read_at + 1;
      load_at = load_at + 1 == NS ? 0 : load_at + 1;
    }
  }
};

// Workgroups go round the 8 XCDs in turn; this gives each XCD one contiguous
// run of tile numbers, so that tiles sharing operands share its L2.
__device__ __forceinline__ int xcd_run(int block, int total) {
  const int each = total / 8, rest = total % 8;
  const int xcd = block % 8;
  return xcd * each + (xcd < rest ? xcd : rest) + block / 8;
}

// Tile number -> (p, q): groups of 4 p tiles, p fastest, so that the 32 tiles
// of an XCD's CUs are 4 x 8.
__device__ __forceinline__ void tile_of(int id, int np, int nq, int& p, int& q) {
  const int group = id / (4 * nq);
  const int first = group * 4;
  const int height = np - first < 4 ? np - first : 4;
  const int within = id - group * 4 * nq;
  p = first + within % height;
  q = within / height;
}

}  // namespace gemm
}  // namespace frwkv
