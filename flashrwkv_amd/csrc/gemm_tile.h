// Tiled 16-bit matrix product for gfx950: one workgroup's BP x BQ tile of
//   D[p][q] = sum_k A[p][k] B[q][k],   fp32 accumulators,
// with v_mfma_f32_16x16x32 (bf16 or fp16 operands).
//
// Either operand may lie in memory with k contiguous ("k-major": rows are p or
// q) or with p / q contiguous ("x-major": rows are k). Tiles of 64 k go from
// HBM straight into LDS (16 bytes a lane, no registers) up to NS stages ahead.
//
// Large products are bound by the matrix units and by the clock that their power
// allows: 8192 x 65536 x 4096 bf16 in 256 x 256 tiles runs at 1302 TFLOP/s with k-major
// operands, units busy 74% of the cycles at 1.67 GHz. 256 x 256 by 8 waves of 128 x 64
// is the largest tile whose accumulators (128 registers) leave room for two sets
// of operands; with one set, loads, LDS reads and matrix instructions one after the other,
// it was 58% at 1.91 GHz. v_mfma_f32_32x32x16 in the same tile was 6 to 8% slower.
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
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
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

// One operand in memory: `rows` rows of `ld` elements (rows are p or q of a
// k-major operand, k of an x-major one). Rows beyond the last read as zeros.
// Reads of an x-major operand may go past a row's end into the next row: they
// land in rows and columns of D that the caller drops.
struct Operand {
  const uint16_t* data;
  int64_t ld;
  int32_t rows;
};

// 64 lanes x 16 bytes from a buffer to LDS bytes [lds, lds + 1024): the hardware
// adds lane * 16 to the address in m0, which is wave-uniform, and writes zeros
// for lanes whose offset lies beyond the buffer. In asm because the compiler,
// unable to tell the stages apart, puts a wait for the whole queue before every
// LDS read that follows the builtin. The compiler writes m0 itself, as the block's
// operand, so it knows what stands there (saved and restored in the block, as a
// register that cannot be declared as written, the small tiles were 2% slower); a
// load reads m0 one wait state after its write at the earliest.
// kStream: not kept in the caches.
template <bool kStream>
__device__ __forceinline__ void load_to_lds(u32x4 buffer, uint32_t offset, uint32_t lds) {
  if constexpr (kStream) {
    asm volatile(
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen nt lds"
        :
        : "v"(offset), "s"(buffer), "{m0}"(lds));
  } else {
    asm volatile(
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen lds"
        :
        : "v"(offset), "s"(buffer), "{m0}"(lds));
  }
}

// Waits until at most kLeft of this wave's loads are outstanding and its LDS
// reads have returned, then for the workgroup.
template <int kLeft>
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kLeft) : "memory");
}

// The loads of one operand's stages by the whole workgroup: 16-byte pieces, one
// a thread and round. A thread's offset from the round's first row never
// changes; the rounds' and stages' first rows are scalars.
template <Major M, int BX, bool kTurn, bool kStream = false>
struct Loader {
  static constexpr int kRounds = BX * 8 / kThreads;
  static constexpr int kBytes = BX * kStep * 2;
  static constexpr int kRoundRows = M == Major::kK ? kThreads / 8 : kThreads / (BX / 8);
  static_assert(kRounds >= 1, "a stage is at least one piece a thread");
  static_assert(M == Major::kK || BX >= 128, "x-major rows hold at least 8 granules");
  static_assert(M == Major::kK || !kTurn, "k-major operands turn");

  const char* base;  // the next stage's first row (k-major: at its first k)
  int32_t row_bytes;
  int32_t left;      // rows from there on
  int32_t into;      // x-major: bytes of base into its row
  uint32_t offset;   // of this thread's piece from a round's first row
  uint32_t wave_lds;

  int32_t ahead;     // kTurn: stages until the product's k begins again
  int32_t span;

  // turn < steps: the stage that is taken first (kTurn).
  __device__ __forceinline__ void init(const Operand& op, int x0, int k0, int steps, int turn) {
    const int tid = threadIdx.x;
    if (kTurn) {
      ahead = steps - turn;
      span = steps * (kStep * 2);
    }
    row_bytes = static_cast<int32_t>(op.ld * 2);
    const int first = M == Major::kK ? x0 : k0;
    into = 2 * (M == Major::kK ? k0 : x0);
    left = op.rows - first;
    base = reinterpret_cast<const char*>(op.data) + static_cast<int64_t>(first) * row_bytes + into;
    if (kTurn) base += turn * (kStep * 2);
    wave_lds = __builtin_amdgcn_readfirstlane(tid >> 6) * 1024u;
    if constexpr (M == Major::kK) {
      offset = static_cast<uint32_t>(tid >> 3) * row_bytes + (((tid & 7) ^ ((tid >> 4) & 7)) << 4);
    } else {
      const int at = tid % (BX / 8), k = tid / (BX / 8);
      const int f = (k & 3) | (((k >> 3) & 1) << 2);
      offset = static_cast<uint32_t>(k) * row_bytes + (((at >> 1) ^ f) << 5) + ((at & 1) << 4);
    }
  }

  // Starts round j of the next stage's loads; there = 0: of zeros, for a stage
  // beyond the last.
  __device__ __forceinline__ void load(int j, int there, uint32_t lds) const {
    const char* from = base + static_cast<int64_t>(j * kRoundRows) * row_bytes;
    // The buffer ends where the round's last row does, if not before it.
    int rows = left - j * kRoundRows;
    rows = rows < kRoundRows + 1 ? rows : kRoundRows + 1;
    int bytes = M == Major::kK ? (rows - 1) * row_bytes + kStep * 2 : rows * row_bytes - into;
    bytes = rows > 0 && there ? bytes : 0;
    const uint64_t address = reinterpret_cast<uint64_t>(from);
    const u32x4 buffer = {static_cast<uint32_t>(address), static_cast<uint32_t>(address >> 32),
                          static_cast<uint32_t>(bytes), 0x00020000u};
    load_to_lds<kStream>(buffer, offset, lds + j * (kThreads * 16u) + wave_lds);
  }
  // Moves on to the stage after it.
  __device__ __forceinline__ void next() {
    if constexpr (M == Major::kK) {
      base += kStep * 2;
      if (kTurn) {
        ahead -= 1;
        base -= ahead == 0 ? span : 0;
      }
    } else {
      base += static_cast<int64_t>(kStep) * row_bytes;
      left -= kStep;
    }
  }
};

// Operand registers of 16 x 32 blocks read from a stage. Lane (g = lane / 16,
// n = lane % 16) holds x = n, k = 8g .. 8g + 7 of the block.
template <Major M, int BX, int kBlocks>
struct Reader {
  uint32_t at[M == Major::kK ? 2 : kBlocks];

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
      for (int i = 0; i < kBlocks; ++i) {
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
template <typename T, Major MA, Major MB, int BP, int BQ, int WP, int WQ, int NS,
          bool kTurn = false, bool kStream = false>
struct Tile {
  static constexpr bool kTurns = kTurn;
  // The same with A's loads past the caches.
  using Streaming = Tile<T, MA, MB, BP, BQ, WP, WQ, NS, kTurn, true>;
  static constexpr int kBP = BP, kBQ = BQ, kWP = WP, kWQ = WQ;
  static constexpr int TP = BP / WP / 16;
  static constexpr int TQ = BQ / WQ / 16;
  static constexpr int kStageBytes = (BP + BQ) * kStep * 2;
  static constexpr int kLdsBytes = NS * kStageBytes;
  static_assert(WP * WQ * 64 == kThreads, "8 waves");
  static_assert(kLdsBytes <= 160 * 1024, "LDS of a CU");

  using LoadA = Loader<MA, BP, kTurn, kStream>;
  using LoadB = Loader<MB, BQ, kTurn>;
  static constexpr int kLoads = LoadA::kRounds + LoadB::kRounds;

  f32x4 acc[TP][TQ];

  static __device__ __forceinline__ int wave() {
    return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  }
  static __device__ __forceinline__ int wave_p0() { return (wave() / WQ) * (BP / WP); }
  static __device__ __forceinline__ int wave_q0() { return (wave() % WQ) * (BQ / WQ); }
  // Lane l holds of D the columns column(j), j < TQ, and in them the rows row(i) .. + 3.
  static __device__ __forceinline__ int row(int i) {
    return wave_p0() + 16 * i + 4 * static_cast<int>((threadIdx.x & 63) >> 4);
  }
  static __device__ __forceinline__ int column(int j) {
    return wave_q0() + 16 * j + static_cast<int>(threadIdx.x & 15);
  }

  // A product is begin (starts the loads of its first stages), arrive (this
  // wave's have arrived) and multiply. Between begin and arrive a workgroup can
  // finish the tile before: its accumulators are its own until multiply, and
  // the LDS beyond kLdsBytes is not touched.
  //
  // steps: number of 64-k stages from k0 on; 0 leaves zeros. turn: which of them
  // comes first, the others follow round (kTurn).
  __device__ __forceinline__ void begin(const Operand& a, const Operand& b, int p0, int q0, int k0,
                                        int steps_, char* smem, int turn = 0) {
    lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
    steps = steps_;
    la.init(a, p0, k0, steps, turn);
    lb.init(b, q0, k0, steps, turn);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) load(la, lb, l, s < steps, lds + s * kStageBytes);
      la.next();
      lb.next();
    }
  }

  static __device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(0)"); }

  // A stage is two halves of 32 k. While a half's matrix instructions run, the
  // other half's operands come from LDS into the registers that the half
  // before used, and in the second half the loads of stage t + NS start into
  // the buffer that stage t has left. One barrier a stage, between the halves:
  // there stage t + 1 has arrived and every wave has read all of stage t.
  __device__ __forceinline__ void multiply(const char* smem) {
    Reader<MA, BP, TP> ra;
    Reader<MB, BQ, TQ> rb;
    ra.init(wave_p0());
    rb.init(wave_q0());
#pragma unroll
    for (int i = 0; i < TP; ++i) {
#pragma unroll
      for (int j = 0; j < TQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
    i16x8 fa[2][TP], fb[2][TQ];
#pragma unroll
    for (int r = 0; r < TP + TQ; ++r) fetch(ra, rb, smem, r, 0, fa[0], fb[0]);
    int at = 0;
    for (int t = 0; t < steps; ++t) {
      const char* stage = smem + at * kStageBytes;
      const int after = at + 1 == NS ? 0 : at + 1;
#pragma unroll
      for (int i = 0; i < TP; ++i) {
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = mfma<T>(fa[0][i], fb[0][j], acc[i][j]);
#pragma unroll
        for (int r = i * kReads; r < (i + 1) * kReads && r < TP + TQ; ++r) {
          fetch(ra, rb, stage, r, 1, fa[1], fb[1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_and_barrier<(NS - 2) * kLoads>();
      const int there = t + NS < steps;
      const char* next = smem + after * kStageBytes;
#pragma unroll
      for (int i = 0; i < TP; ++i) {
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = mfma<T>(fa[1][i], fb[1][j], acc[i][j]);
#pragma unroll
        for (int l = i * kStarts; l < (i + 1) * kStarts && l < kLoads; ++l) {
          load(la, lb, l, there, lds + at * kStageBytes);
        }
#pragma unroll
        for (int r = i * kReads; r < (i + 1) * kReads && r < TP + TQ; ++r) {
          fetch(ra, rb, next, r, 0, fa[0], fb[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      la.next();
      lb.next();
      at = after;
    }
    wait_and_barrier<0>();
  }

 private:
  LoadA la;
  LoadB lb;
  uint32_t lds;
  int steps;

  // LDS reads and started loads beside each block row of matrix instructions.
  static constexpr int kReads = (TP + TQ + TP - 1) / TP;
  static constexpr int kStarts = (kLoads + TP - 1) / TP;

  static __device__ __forceinline__ void load(const LoadA& la, const LoadB& lb, int l, int there,
                                              uint32_t lds) {
    if (l < LoadA::kRounds) {
      la.load(l, there, lds);
    } else {
      lb.load(l - LoadA::kRounds, there, lds + LoadA::kBytes);
    }
  }
  // Operand r of a half: the q blocks first, which all matrix instructions use.
  template <typename RA, typename RB>
  static __device__ __forceinline__ void fetch(const RA& ra, const RB& rb, const char* stage,
                                               int r, int kk, i16x8 (&fa)[TP], i16x8 (&fb)[TQ]) {
    if (r < TQ) {
      fb[r] = rb.read(stage + LoadA::kBytes, r, kk);
    } else {
      fa[r - TQ] = ra.read(stage, r - TQ, kk);
    }
  }
};

// Stores column j of a tile's lanes as 16 bits: element (p, q) of the tile to
// to[q * ld + p], for q < columns and p < rows (a multiple of 32). quad[i] holds
// rows row(i) .. + 3: 8 bytes a lane, 32 bytes apart. Exchanged between odd and
// even groups of 16 lanes, quads i and i + 1 become 16 consecutive bytes a lane
// and 64 a column; half the stores and half the requests to L2 (a backward of
// 1000 x 50277 x 2560: 797 -> 764 us).
template <typename G>
__device__ __forceinline__ void store_column(uint16_t* to, int64_t ld, int rows, int columns,
                                             int j, const uint2 (&quad)[G::TP]) {
  static_assert(G::TP % 2 == 0, "quads go in pairs");
  const int g = static_cast<int>((threadIdx.x & 63) >> 4);
  const int first = G::wave_p0() + 16 * (g & 1) + 8 * (g >> 1);
  const int q = G::column(j);
  uint16_t* column = to + q * ld;
#pragma unroll
  for (int i = 0; i < G::TP; i += 2) {
    const auto x = __builtin_amdgcn_permlane16_swap(quad[i].x, quad[i + 1].x, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(quad[i].y, quad[i + 1].y, false, false);
    const int p = first + 16 * i;
    if (q < columns && p < rows) {
      *reinterpret_cast<uint4*>(column + p) = make_uint4(x[0], y[0], x[1], y[1]);
    }
  }
}

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
