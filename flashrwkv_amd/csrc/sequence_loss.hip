// Losses over packed sequences of token log probabilities: the clipped policy
// loss with a KL term, and the preference loss of paired sequences.
//
// Policy, token i with log probability x, that of the policy that sampled it
// o, a reference's f, advantage A and entropy H; d = x - o, r = e^d:
//   l = -min(r A, clamp(r, 1 - low, 1 + high) A) + kl k3(f - x) - ew H
// (A < 0 with a dual clip: at most -dual A), k3(t) = e^t - 1 - t;
//   dl/dx = -[not clipped] r A + kl (1 - e^(f - x)),  dl/dH = -ew.
// Clipped: A > 0 and d > log(1 + high), A < 0 and (d < log(1 - low) or
// d > log dual). Reduced over the tokens that take part (mean, sum), over the
// sequences that have such tokens (mean of each one's mean), or not.
//
// Preference, sequences 2p chosen and 2p + 1 rejected:
//   s_b = sum (x - f) over b's tokens (its mean where asked for),
//   m = beta (s_2p - s_2p+1) - margin,
//   l = -(1 - eps) log sigma(m) - eps log sigma(-m), max(0, 1 - m) or
//       ((m - 1/2) / beta)^2,
//   dl/dx_i = dl/dm beta (+ or -) (/ count).
//
// d decides on which side of a border a token is. Differences of logs are exact up
// to one rounding; where a rounded one falls on a rounded border, both are taken in
// 64 bits. Exponentials and a token's loss are in 32 bits, sums over tokens in 64.
//
// A wave takes a tile of 64 x kRounds consecutive tokens with all loads under
// way at once, and finds the sequence of its first token by itself, 64 offsets a
// step. Sums of a sequence go tile by tile: tile t and sequence b meet in piece
// t + b, a number that no other meeting has and that is consecutive for a
// sequence's tiles, so a second pass adds them in order without atomics. The
// offsets stand on the device and are not trusted: every index that is made from
// them is bounded, and offsets that do not start at 0, fall or go past the last
// token make a reduced loss and the gradients of all tokens NaN.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "capi_internal.h"
#include "wkv7_device.h"

namespace frwkv {
namespace {

constexpr int kWaves = 4;           // of a workgroup of the token kernels
constexpr int kJoinThreads = 1024;
constexpr int kJoinWaves = kJoinThreads / 64;
constexpr int kMostJoins = 64;      // workgroups that join
constexpr int kMany = 4;            // rounds of a tile of a large call
constexpr int kFew = 2;
constexpr int kNone = -1;           // a column that is not there

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// A lane's 32 bits moved by a DPP pattern, 0 where it has no source.
template <int kPattern, int kRows>
__device__ __forceinline__ int32_t moved(int32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, kPattern, kRows, 0xf, true);
}

template <int kPattern, int kRows, typename T>
__device__ __forceinline__ T moved_of(T x) {
  int32_t part[sizeof(T) / 4];
  __builtin_memcpy(part, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) part[i] = moved<kPattern, kRows>(part[i]);
  __builtin_memcpy(&x, part, sizeof(T));
  return x;
}

// The sum over the wave, the same for all lanes. By row shifts and row broadcasts,
// which stay in the vector unit: through LDS the six steps of a 64-bit sum are
// twelve dependent trips.
template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
  x += moved_of<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: lane 15 of a row of 16 has its sum
  x += moved_of<0x112, 0xf>(x);
  x += moved_of<0x114, 0xf>(x);
  x += moved_of<0x118, 0xf>(x);
  x += moved_of<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
  x += moved_of<0x143, 0xc>(x);
  int32_t part[sizeof(T) / 4];
  __builtin_memcpy(part, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) part[i] = __builtin_amdgcn_readlane(part[i], 63);
  __builtin_memcpy(&x, part, sizeof(T));
  return x;
}

// A vector of a type that is known at run time, the same for all threads.
struct Column {
  const void* data;
  int dtype;  // FRWKV_DTYPE_*, or kNone
  __host__ __device__ bool given() const { return dtype != kNone; }
};

// log2 of a tile's tokens.
__host__ __device__ constexpr int shift_of(int rounds) { return rounds == 1 ? 6 : 1 + shift_of(rounds / 2); }

// A tile of 64 x kRounds tokens: where it begins and how many there are.
template <int kRounds>
struct Tile {
  int64_t first;
  int32_t left;
  __device__ __forceinline__ Tile(int64_t tile, int64_t tokens) {
    first = tile * (64 * kRounds);
    left = static_cast<int32_t>(min(tokens - first, int64_t{64 * kRounds}));
  }
  __device__ __forceinline__ bool empty() const { return left <= 0; }
  __device__ __forceinline__ bool has(int r) const { return 64 * r + lane_id() < left; }
  // to[r] = from[token of round r], the last one for those beyond it. Whole tiles are
  // read at constant distances from one address.
  template <typename S, typename D>
  __device__ __forceinline__ void fetch(const S* from, D (&to)[kRounds]) const {
    from += first;
    if (left == 64 * kRounds) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) to[r] = from[64 * r + lane_id()];
    } else {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) to[r] = from[min(64 * r + lane_id(), left - 1)];
    }
  }
  __device__ __forceinline__ void fetch(const Column& from, uint32_t (&to)[kRounds]) const {
    if (from.dtype == FRWKV_DTYPE_F32) {
      fetch(static_cast<const uint32_t*>(from.data), to);
    } else {
      fetch(static_cast<const uint16_t*>(from.data), to);
    }
  }
  __device__ __forceinline__ void fetch_part(const uint8_t* mask, bool (&part)[kRounds]) const {
    uint32_t here[kRounds];
    if (mask != nullptr) fetch(mask, here);
#pragma unroll
    for (int r = 0; r < kRounds; ++r) part[r] = has(r) && (mask == nullptr || here[r] != 0);
  }
};

__device__ __forceinline__ uint32_t bits_at(const Column& c, int64_t i) {
  return c.dtype == FRWKV_DTYPE_F32 ? static_cast<const uint32_t*>(c.data)[i]
                                    : static_cast<const uint16_t*>(c.data)[i];
}

__device__ __forceinline__ float value_of(const Column& c, uint32_t bits) {
  if (c.dtype == FRWKV_DTYPE_F32) return __uint_as_float(bits);
  if (c.dtype == FRWKV_DTYPE_BF16) return bf16_to_f32(bits);
  return f16_to_f32(static_cast<uint16_t>(bits));
}

__device__ __forceinline__ void store_at(void* data, int dtype, int64_t i, float x) {
  if (dtype == FRWKV_DTYPE_F32) {
    static_cast<float*>(data)[i] = x;
  } else if (dtype == FRWKV_DTYPE_BF16) {
    static_cast<uint16_t*>(data)[i] = from_f32<Bf16>(x);
  } else {
    static_cast<uint16_t*>(data)[i] = from_f32<F16>(x);
  }
}

// Tokens, and the sequences they are packed into (cu null: none).
struct Packed {
  int64_t n;
  const int32_t* cu;   // [sequences + 1]
  int32_t sequences;
  const uint8_t* mask; // null: all
};

// The last sequence that starts at or before token i, or `sequences` behind the
// last one's end; by the whole wave.
__device__ __forceinline__ int32_t sequence_of(const Packed& p, int64_t i) {
  int32_t at = 0, left = p.sequences + 1;
  while (left > 1) {
    const int32_t step = (left + 63) / 64;
    const int32_t mine = lane_id() * step;
    const int hits = __popcll(__ballot(mine < left && p.cu[at + min(mine, left - 1)] <= i));
    const int32_t skip = hits > 0 ? (hits - 1) * step : 0;
    at += skip;
    left = min(step, left - skip);
  }
  return at;
}

// Sequences of a tile's tokens, a round of 64 at a time.
template <int kRounds>
__device__ __forceinline__ void sequences_of(const Packed& p, int64_t first,
                                             int32_t (&id)[kRounds]) {
  int32_t s = sequence_of(p, first), from = s;
  // The next 64 ends, a lane each.
  const auto window = [&] { return p.cu[min(from + 1 + lane_id(), p.sequences)]; };
  int32_t ends = window();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + 64 * r + lane_id();
    const int64_t last = min(first + 64 * r + 63, p.n - 1);
    id[r] = s;
    while (s < p.sequences) {
      if (s - from == 64) {
        from = s;
        ends = window();
      }
      const int32_t end = __builtin_amdgcn_readlane(ends, s - from);
      if (end > last) break;
      id[r] += i >= end ? 1 : 0;
      ++s;
    }
  }
}

struct Piece {
  double sum;
  int64_t count;
};

// Adds a tile's values up by sequence. add() takes the rounds in order.
struct Pieces {
  Piece* at;          // of this tile: [sequence]
  int32_t sequences;
  int32_t open;       // the sequence that sum and count belong to
  double sum = 0.0;   // a lane's share
  int32_t count = 0;

  __device__ __forceinline__ void put(int32_t id, double x, int32_t n) {
    if (id < sequences) at[id] = {x, n};
  }
  __device__ __forceinline__ void add(int32_t id, double x, bool part) {
    int32_t n = part ? 1 : 0;
    const int32_t last = __builtin_amdgcn_readlane(id, 63);
    if (last == open) {  // the round is the open sequence's
      sum += x;
      count += n;
      return;
    }
    const double before = wave_sum(sum);
    const int32_t count_before = wave_sum(count);
    if (__builtin_amdgcn_readfirstlane(id) != open && lane_id() == 0) {
      put(open, before, count_before);  // it ended where the round begins
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double y = __shfl_up(x, off, 64);
      const int32_t m = __shfl_up(n, off, 64);
      const int32_t other = __shfl_up(id, off, 64);
      if (lane_id() >= off && other == id) {
        x += y;
        n += m;
      }
    }
    if (id == open) {
      x += before;
      n += count_before;
    }
    const int32_t next = __shfl_down(id, 1, 64);
    if (lane_id() < 63 && next != id) put(id, x, n);
    open = last;
    sum = lane_id() == 63 ? x : 0.0;
    count = lane_id() == 63 ? n : 0;
  }
  __device__ __forceinline__ void end() {
    const double x = wave_sum(sum);
    const int32_t n = wave_sum(count);
    if (lane_id() == 0) put(open, x, n);
  }
};

// Whether sequence b's offsets are ones that a caller may give.
__device__ __forceinline__ bool in_order(const Packed& p, int32_t b) {
  const int32_t from = p.cu[b], to = p.cu[b + 1];
  return from >= 0 && from <= to && to <= p.n && (b > 0 || from == 0);
}

// Sum of a sequence's pieces: up to kOwnPieces by the lane that asks, others by
// the wave. All lanes call; b < 0 asks for none.
constexpr int kOwnPieces = 64;
constexpr int kAtOnce = 8;  // of them under way

__device__ __forceinline__ Piece sum_of(const Packed& p, const Piece* pieces, int tile_shift,
                                        int64_t tiles, int32_t b) {
  Piece out{0.0, 0};
  int64_t from = 0, to = 0;  // tiles
  if (b >= 0 && in_order(p, b) && p.cu[b] < p.cu[b + 1]) {
    from = p.cu[b] >> tile_shift;
    to = min(static_cast<int64_t>((p.cu[b + 1] - 1) >> tile_shift) + 1, tiles);
  }
  const bool own = to - from <= kOwnPieces;
  if (own) {
    for (int64_t t = from; t < to; t += kAtOnce) {
      Piece x[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) x[u] = pieces[min(t + u, to - 1) + b];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (t + u < to) {
          out.sum += x[u].sum;
          out.count += x[u].count;
        }
      }
    }
  }
  uint64_t others = __ballot(!own);
  while (others != 0) {
    const int who = __ffsll(static_cast<unsigned long long>(others)) - 1;
    others &= others - 1;
    const int32_t of = __shfl(b, who, 64);
    const int64_t end = __shfl(to, who, 64);
    double x = 0.0;
    int64_t n = 0;
#pragma unroll 4
    for (int64_t t = __shfl(from, who, 64) + lane_id(); t < end; t += 64) {
      const Piece y = pieces[t + of];
      x += y.sum;
      n += y.count;
    }
    x = wave_sum(x);
    n = wave_sum(n);
    if (lane_id() == who) out = {x, n};
  }
  return out;
}

// ------------------------------------------------------------------ policy
struct Policy {
  Column x, old, advantage, reference, entropy;
  bool per_sequence;  // advantages are
  float above, below, far;   // borders: log(1 + high), log(1 - low), log dual
  double above_exact, below_exact, far_exact;
  float most, least, dual;   // 1 + high, 1 - low; dual 0: none
  float kl, ew;
};

// Sums over a workgroup's tokens, and what the call returns of them.
enum { kLoss, kCount, kBad, kRatio, kClipped, kOld, kReference, kSums };
constexpr int kMetrics = 4;  // the last of them, over the count

// e^t, e^t - 1 and k3 = e^t - 1 - t, without a branch. e^t = 2^n (1 + r log 2), n the
// rounded t log2 e and r what that left out; the differences lose all digits near 0
// and are taken up to |t| = 1 from k3's series, whose terms fall quickly (nine of them: 5e-8 of
// the sum at 1).
struct Exponential {
  float e, less_one, k3;
};

__device__ __forceinline__ Exponential exponential(float t) {
  constexpr float kLog2ELow = 1.9259629911266175e-8f;  // log2 e - kLog2E
  const float n = t * kLog2E;
  const float r = fmaf(t, kLog2ELow, fmaf(t, kLog2E, -n));
  const float power = __builtin_amdgcn_exp2f(n);
  // Beyond, the power is 0 or infinite and r may be NaN.
  const float e = fabsf(n) < 128.0f ? fmaf(power * 0.69314718f, r, power) : power;
  float s = 1.0f / 3628800.0f;
  s = fmaf(s, t, 1.0f / 362880.0f);
  s = fmaf(s, t, 1.0f / 40320.0f);
  s = fmaf(s, t, 1.0f / 5040.0f);
  s = fmaf(s, t, 1.0f / 720.0f);
  s = fmaf(s, t, 1.0f / 120.0f);
  s = fmaf(s, t, 1.0f / 24.0f);
  s = fmaf(s, t, 1.0f / 6.0f);
  s = fmaf(s, t, 0.5f);
  const float near = t * t * s;
  const bool small = fabsf(t) < 1.0f;
  const float less_one = small ? t + near : e - 1.0f;
  return {small ? 1.0f + less_one : e, less_one, small ? near : less_one - t};
}

// A token's surrogate, as a loss and its slope in x.
struct Term {
  float loss, slope;
  float ratio, k3;
  bool clipped;
};

__device__ __forceinline__ Term policy_term(const Policy& a, float x, float old,
                                            float advantage) {
  Term out;
  const float d = x - old;
  const bool gains = advantage > 0.0f, loses = advantage < 0.0f;
  const bool dual = a.dual > 0.0f && loses;
  out.clipped = (gains && d > a.above) || (loses && d < a.below) || (dual && d > a.far);
  // Rounding keeps the order, so a rounded d beside a rounded border decides; d on
  // it is compared in 64 bits.
  const bool on = d == a.above || d == a.below || d == a.far;
  if (__builtin_expect(__ballot(on) != 0, 0)) {
    const double exact = static_cast<double>(x) - static_cast<double>(old);
    const bool clipped = (gains && exact > a.above_exact) || (loses && exact < a.below_exact) ||
                         (dual && exact > a.far_exact);
    if (on) out.clipped = clipped;
  }
  const Exponential r = exponential(d);
  const float plain = r.e * advantage;
  const float bounded = fminf(fmaxf(r.e, a.least), a.most) * advantage;
  // NaN stays NaN.
  float gain = bounded < plain ? bounded : plain;
  if (dual && gain < a.dual * advantage) gain = a.dual * advantage;
  out.loss = -gain;
  out.slope = out.clipped ? 0.0f : -plain;
  out.ratio = r.e;
  out.k3 = r.k3;
  return out;
}

// What the forward leaves for the backward, and its scratch.
struct Saved {
  float* share;   // [1]  what a token's slope is multiplied by, NaN for bad offsets
  float* weight;  // [sequences] the same of each sequence, beside share
  float* slope;   // [n]  dl/dx, 0 for tokens that take no part
};

struct Scratch {
  int32_t* done;   // workgroups of the join that have ended
  double* sums;    // [workgroups][kSums]
  double* joins;   // [kMostJoins][3]
  Piece* pieces;   // [tiles + sequences]
};

struct PolicyOut {
  float* loss;      // [1], or [n]
  float* metrics;   // [kMetrics], or null
  int reduction;
  bool slopes;
};

// Adds `values` up over the workgroup; the result is the first wave's.
template <int kBlockWaves, int kValues>
__device__ __forceinline__ void workgroup_sum(double (&values)[kValues], double* shared) {
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int v = 0; v < kValues; ++v) {
    const double x = wave_sum(values[v]);
    if (lane_id() == 0) shared[v * kBlockWaves + wave] = x;
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int v = 0; v < kValues; ++v) {
      values[v] = wave_sum(lane_id() < kBlockWaves ? shared[v * kBlockWaves + lane_id()] : 0.0);
    }
  }
  __syncthreads();
}

template <int kRounds>
__device__ __forceinline__ void policy_tile(const Policy& a, const Packed& p, const PolicyOut& o,
                                            const Saved& s, const Scratch& w, int64_t index,
                                            double (&sums)[kSums]) {
  const Tile<kRounds> tile(index, p.n);
  if (tile.empty()) return;
  uint32_t x[kRounds], old[kRounds], advantage[kRounds], reference[kRounds], entropy[kRounds];
  bool part[kRounds];
  tile.fetch(a.x, x);
  tile.fetch(a.old, old);
  if (!a.per_sequence) tile.fetch(a.advantage, advantage);
  if (a.reference.given()) tile.fetch(a.reference, reference);
  if (a.entropy.given()) tile.fetch(a.entropy, entropy);
  tile.fetch_part(p.mask, part);
  const bool by_sequence = o.reduction == FRWKV_REDUCE_SEQUENCE_MEAN;
  int32_t id[kRounds];
  if (by_sequence || a.per_sequence) {
    sequences_of<kRounds>(p, tile.first, id);
#pragma unroll
    for (int r = 0; r < kRounds; ++r) part[r] = part[r] && id[r] < p.sequences;
    if (a.per_sequence) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        advantage[r] = bits_at(a.advantage, min(id[r], p.sequences - 1));
      }
    }
  } else if (p.cu != nullptr) {  // which sequence does not matter, only whether one
    const int64_t end = p.cu[p.sequences] - tile.first;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) part[r] = part[r] && 64 * r + lane_id() < end;
  }
  // Vector by vector: what is the same for all tokens is asked once a tile.
  float losses[kRounds], slopes[kRounds];
  double ratio = 0.0, old_kl = 0.0, reference_kl = 0.0;
  int32_t count = 0, clipped = 0;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const Term t = policy_term(a, value_of(a.x, x[r]), value_of(a.old, old[r]),
                               value_of(a.advantage, advantage[r]));
    losses[r] = t.loss;
    slopes[r] = t.slope;
    // What stands in a token that takes no part, NaN included, ends here.
    ratio += part[r] ? t.ratio : 0.0f;
    old_kl += part[r] ? t.k3 : 0.0f;
    clipped += part[r] && t.clipped ? 1 : 0;
    count += part[r] ? 1 : 0;
  }
  if (a.reference.given()) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const Exponential q =
          exponential(value_of(a.reference, reference[r]) - value_of(a.x, x[r]));
      if (a.kl != 0.0f) {  // or only looked at, and 0 of an infinite k3 would be NaN
        losses[r] = fmaf(a.kl, q.k3, losses[r]);
        slopes[r] = fmaf(-a.kl, q.less_one, slopes[r]);
      }
      reference_kl += part[r] ? q.k3 : 0.0f;
    }
  }
  if (a.entropy.given()) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      losses[r] = fmaf(-a.ew, value_of(a.entropy, entropy[r]), losses[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) losses[r] = part[r] ? losses[r] : 0.0f;
  if (o.slopes) {
    float* to = s.slope + tile.first;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (tile.has(r)) to[64 * r + lane_id()] = part[r] ? slopes[r] : 0.0f;
    }
  }
  if (o.reduction == FRWKV_REDUCE_NONE) {
    float* to = o.loss + tile.first;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (tile.has(r)) to[64 * r + lane_id()] = losses[r];
    }
  }
  double loss = 0.0;
  if (by_sequence) {
    Pieces pieces;
    pieces.at = w.pieces + index;
    pieces.sequences = p.sequences;
    pieces.open = __builtin_amdgcn_readfirstlane(id[0]);
#pragma unroll
    for (int r = 0; r < kRounds; ++r) pieces.add(id[r], losses[r], part[r]);
    pieces.end();
  } else {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) loss += losses[r];
  }
  sums[kLoss] = loss;
  sums[kCount] = count;
  sums[kRatio] = ratio;
  sums[kClipped] = clipped;
  sums[kOld] = old_kl;
  sums[kReference] = reference_kl;
}

// Offsets that may not be, of a thread's share of the sequences.
__device__ __forceinline__ double bad_offsets(const Packed& p, int64_t thread, int64_t threads) {
  if (p.cu == nullptr) return 0.0;
  double bad = 0.0;
  for (int64_t b = thread; b < p.sequences; b += threads) {
    if (!in_order(p, static_cast<int32_t>(b))) bad = 1.0;
  }
  return bad;
}

// A workgroup's part of the sequences, for the mean over them: {sum of their means,
// how many have tokens}.
__device__ __forceinline__ void join_sequences(const Packed& p, const PolicyOut& o,
                                               const Saved& s, const Scratch& w, int tile_shift,
                                               int64_t tiles, int64_t wave, int64_t waves,
                                               double (&found)[2]) {
  if (o.reduction != FRWKV_REDUCE_SEQUENCE_MEAN) return;
  // Few sequences are one a wave, many 64.
  const int64_t each = min(max((p.sequences + waves - 1) / waves, int64_t{1}), int64_t{64});
  for (int64_t at = wave * each; at < p.sequences; at += waves * each) {
    const bool mine = lane_id() < each && at + lane_id() < p.sequences;
    const int32_t b = mine ? static_cast<int32_t>(at) + lane_id() : -1;
    const Piece x = sum_of(p, w.pieces, tile_shift, tiles, b);
    if (mine) {
      s.weight[b] = x.count > 0 ? static_cast<float>(1.0 / static_cast<double>(x.count)) : 0.0f;
      if (x.count > 0) {
        found[0] += x.sum / static_cast<double>(x.count);
        found[1] += 1.0;
      }
    }
  }
}

__device__ __forceinline__ void write_policy(const PolicyOut& o, const Saved& s,
                                             const double (&sums)[kSums],
                                             const double (&found)[2]) {
  const bool by_sequence = o.reduction == FRWKV_REDUCE_SEQUENCE_MEAN;
  const float bad = sums[kBad] > 0.0 ? __builtin_nanf("") : 0.0f;
  const double over = by_sequence ? found[1] : sums[kCount];
  const bool mean = by_sequence || o.reduction == FRWKV_REDUCE_MEAN;
  const double share = mean ? (over > 0.0 ? 1.0 / over : 0.0) : 1.0;
  *s.share = static_cast<float>(share) + bad;
  if (o.reduction != FRWKV_REDUCE_NONE) {
    const double total = by_sequence ? found[0] : sums[kLoss];
    *o.loss = static_cast<float>(over > 0.0 ? total * share : 0.0) + bad;
  }
  if (o.metrics != nullptr) {
    const double by = sums[kCount] > 0.0 ? 1.0 / sums[kCount] : 0.0;
#pragma unroll
    for (int q = 0; q < kMetrics; ++q) {
      o.metrics[q] = static_cast<float>(sums[kRatio + q] * by) + bad;
    }
  }
}

// Losses and slopes of all tokens. kAlone: one workgroup takes them all and
// joins them, which saves the second launch. kPlain: all vectors are fp32, known to the
// compiler; a type that is looked at for each value costs scalar instructions and branches (4M
// tokens with 16-bit old and reference columns: 26.5 us, for 17 MB less).
// 4M tokens with a reference and a mask in 24 us: 89 MB at 3.7 TB/s, 185 vector
// instructions for 64 tokens. With a wave's sums in 32 bits it is 21 and 154, but two
// ratios of 3e38 have a mean and no such sum, and terms that cancel lose their digits.
template <int kRounds, int kBlockWaves, bool kAlone, bool kPlain>
__global__ __launch_bounds__(kBlockWaves * 64) void policy_tokens_kernel(Policy a, Packed p,
                                                                         PolicyOut o, Saved s,
                                                                         Scratch w,
                                                                         int64_t tiles) {
  __shared__ double shared[kBlockWaves * kSums];
  constexpr int kThreads = kBlockWaves * 64;
  const int64_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (kPlain) {
    a.x.dtype = a.old.dtype = a.advantage.dtype = FRWKV_DTYPE_F32;
    if (a.reference.given()) a.reference.dtype = FRWKV_DTYPE_F32;
    if (a.entropy.given()) a.entropy.dtype = FRWKV_DTYPE_F32;
  }
  double sums[kSums] = {};
  policy_tile<kRounds>(a, p, o, s, w,
                       static_cast<int64_t>(blockIdx.x) * kBlockWaves + wave, sums);
  sums[kBad] = bad_offsets(p, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x,
                           static_cast<int64_t>(gridDim.x) * kThreads);
  workgroup_sum<kBlockWaves>(sums, shared);
  if constexpr (kAlone) {
    double found[2] = {};
    join_sequences(p, o, s, w, shift_of(kRounds), tiles, wave, kBlockWaves, found);
    workgroup_sum<kBlockWaves>(found, shared);
    if (threadIdx.x == 0) write_policy(o, s, sums, found);
  } else if (threadIdx.x == 0) {
#pragma unroll
    for (int v = 0; v < kSums; ++v) w.sums[blockIdx.x * kSums + v] = sums[v];
    if (blockIdx.x == 0) *w.done = 0;
  }
}

// Whether this is the last of the launch's workgroups to end, which then has all of
// their sums.
template <int kValues>
__device__ __forceinline__ bool last_with_all(double (&found)[kValues], const Scratch& w,
                                              double* shared) {
  __shared__ bool last;
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int v = 0; v < kValues; ++v) {
      __hip_atomic_store(w.joins + blockIdx.x * kValues + v, found[v], __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    }
    last = __hip_atomic_fetch_add(w.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
           static_cast<int32_t>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return false;
#pragma unroll
  for (int v = 0; v < kValues; ++v) {
    found[v] = threadIdx.x < gridDim.x
                   ? __hip_atomic_load(w.joins + threadIdx.x * kValues + v, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT)
                   : 0.0;
  }
  workgroup_sum<kJoinWaves>(found, shared);
  return true;
}

// Bound by latency: the workgroups' sums, and of a mean over sequences the pieces, in
// two or three dependent trips to memory. 4096 workgroups' sums (4M tokens): 5 us; 64
// sequences of 800 tokens, by sequence: 7.
__global__ __launch_bounds__(kJoinThreads) void policy_join_kernel(Packed p, PolicyOut o, Saved s,
                                                                   Scratch w, int tile_shift,
                                                                   int64_t tiles,
                                                                   int32_t blocks) {
  __shared__ double shared[kJoinWaves * kSums];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  double found[2] = {};
  join_sequences(p, o, s, w, tile_shift, tiles,
                 static_cast<int64_t>(blockIdx.x) * kJoinWaves + wave,
                 static_cast<int64_t>(gridDim.x) * kJoinWaves, found);
  if (o.reduction == FRWKV_REDUCE_SEQUENCE_MEAN) {
    workgroup_sum<kJoinWaves>(found, shared);
    if (!last_with_all(found, w, shared)) return;
  }
  double sums[kSums] = {};
  for (int32_t b = threadIdx.x; b < blocks; b += kJoinThreads) {
#pragma unroll
    for (int v = 0; v < kSums; ++v) sums[v] += w.sums[b * kSums + v];
  }
  workgroup_sum<kJoinWaves>(sums, shared);
  if (threadIdx.x == 0) write_policy(o, s, sums, found);
}

// Gradients of x (slope times what the loss gives it) and of the entropies. 4M tokens in
// 8 us: 34 MB at 4.2 TB/s.
struct PolicyGrad {
  const float* upstream;  // [1], or [n]
  void* x;                // null: not wanted
  int x_dtype;
  void* entropy;
  int entropy_dtype;
  float ew;
  int reduction;
};

template <int kRounds>
__global__ __launch_bounds__(kWaves * 64) void policy_grad_kernel(Packed p, PolicyGrad g,
                                                                  Saved s) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile<kRounds> tile(static_cast<int64_t>(blockIdx.x) * kWaves + wave, p.n);
  if (tile.empty()) return;
  float slope[kRounds], up[kRounds];
  bool part[kRounds];
  if (g.x != nullptr) tile.fetch(s.slope, slope);
  if (g.reduction == FRWKV_REDUCE_NONE) {
    tile.fetch(g.upstream, up);
  } else {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) up[r] = *g.upstream;
  }
  tile.fetch_part(g.entropy != nullptr ? p.mask : nullptr, part);
  const float share = *s.share;
  const bool bad = share != share;  // offsets that may not be: NaN for all tokens
#pragma unroll
  for (int r = 0; r < kRounds; ++r) up[r] *= share;
  const bool by_sequence = g.reduction == FRWKV_REDUCE_SEQUENCE_MEAN;
  if (by_sequence) {
    int32_t id[kRounds];
    sequences_of<kRounds>(p, tile.first, id);
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      part[r] = part[r] && id[r] < p.sequences;
      up[r] *= s.weight[min(id[r], p.sequences - 1)];
    }
  } else if (g.entropy != nullptr && p.cu != nullptr) {
    const int64_t end = p.cu[p.sequences] - tile.first;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) part[r] = part[r] && 64 * r + lane_id() < end;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (!tile.has(r)) continue;
    const int64_t i = tile.first + 64 * r + lane_id();
    // A slope of 0, as a token without part has, stays 0 under any upstream.
    if (g.x != nullptr) {
      const float grad = slope[r] == 0.0f ? 0.0f : slope[r] * up[r];
      store_at(g.x, g.x_dtype, i, bad ? share : grad);
    }
    if (g.entropy != nullptr) {
      const float grad = part[r] ? -g.ew * up[r] : 0.0f;
      store_at(g.entropy, g.entropy_dtype, i, bad ? share : grad);
    }
  }
}

// -------------------------------------------------------------- preference
struct Preference {
  Column x, reference;
  double beta, margin, smoothing;
  int kind;
  bool normalize;
};

struct PreferenceOut {
  float* loss;     // [1], or [pairs]
  float* rewards;  // [pairs][2]
  int reduction;
};

// What the backward multiplies the upstream gradient by: coefficient x share.
struct PreferenceSaved {
  float* share;        // [1]
  float* coefficient;  // [2 pairs]
};

template <int kRounds>
__device__ __forceinline__ void preference_tile(const Preference& a, const Packed& p, Piece* all,
                                                int64_t index) {
  const Tile<kRounds> tile(index, p.n);
  if (tile.empty()) return;
  uint32_t x[kRounds], reference[kRounds];
  bool part[kRounds];
  tile.fetch(a.x, x);
  if (a.reference.given()) tile.fetch(a.reference, reference);
  tile.fetch_part(p.mask, part);
  int32_t id[kRounds];
  sequences_of<kRounds>(p, tile.first, id);
  Pieces pieces;
  pieces.at = all + index;
  pieces.sequences = p.sequences;
  pieces.open = __builtin_amdgcn_readfirstlane(id[0]);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    double d = value_of(a.x, x[r]);
    if (a.reference.given()) d -= static_cast<double>(value_of(a.reference, reference[r]));
    pieces.add(id[r], part[r] ? d : 0.0, part[r]);
  }
  pieces.end();
}

// Loss of one pair and its slope in m.
__device__ __forceinline__ void preference_term(const Preference& a, double m, double& loss,
                                                double& slope) {
  if (a.kind == FRWKV_PREFERENCE_SIGMOID) {
    const double e = exp(-fabs(m));  // both log sigmas from it, no overflow
    const double soft = log1p(e), eps = a.smoothing;
    loss = (1.0 - eps) * (soft + fmax(-m, 0.0));
    // Without smoothing the term is not there: m is infinite where the rejected answer
    // cannot be, and 0 of it would be NaN.
    if (eps != 0.0) loss += eps * (soft + fmax(m, 0.0));
    // sigma(m) - 1 = -sigma(-m), of which the smaller one keeps its digits.
    const double small = e / (1.0 + e), large = 1.0 / (1.0 + e);
    slope = eps * (m > 0.0 ? large : small) - (1.0 - eps) * (m > 0.0 ? small : large);
  } else if (a.kind == FRWKV_PREFERENCE_HINGE) {
    loss = fmax(1.0 - m, 0.0);
    slope = m < 1.0 ? -1.0 : 0.0;
  } else {
    const double t = (m - 0.5) / a.beta;
    loss = t * t;
    slope = 2.0 * t / a.beta;
  }
  if (m != m) loss = slope = m;
}

// A workgroup's part of the pairs: {sum of losses, pairs that take part, bad
// offsets}. A lane has one sequence, even ones the chosen.
__device__ __forceinline__ void join_pairs(const Preference& a, const Packed& p,
                                           const PreferenceOut& o, const PreferenceSaved& s,
                                           const Piece* pieces, int tile_shift, int64_t tiles,
                                           int64_t wave, int64_t waves, double (&found)[3]) {
  int64_t each = (p.sequences / 2 + waves - 1) / waves;
  each = 2 * min(max(each, int64_t{1}), int64_t{32});
  for (int64_t at = wave * each; at < p.sequences; at += waves * each) {
    const bool mine = lane_id() < each && at + lane_id() < p.sequences;
    const int32_t b = mine ? static_cast<int32_t>(at) + lane_id() : -1;
    if (mine && !in_order(p, b)) found[2] += 1.0;
    const Piece x = sum_of(p, pieces, tile_shift, tiles, b);
    const double by = a.normalize && x.count > 0 ? 1.0 / static_cast<double>(x.count) : 1.0;
    const double reward = a.beta * (x.sum * by);
    const double other = __shfl_xor(reward, 1, 64);
    const int64_t other_count = __shfl_xor(x.count, 1, 64);
    const bool rejected = (lane_id() & 1) != 0;
    const bool part = x.count > 0 && other_count > 0;
    const double m = (rejected ? other - reward : reward - other) - a.margin;
    double loss = 0.0, slope = 0.0;
    if (part) preference_term(a, m, loss, slope);
    if (mine) {
      s.coefficient[b] = static_cast<float>((rejected ? -slope : slope) * a.beta * by);
      o.rewards[b] = static_cast<float>(reward);
      if (!rejected) {
        if (o.reduction == FRWKV_REDUCE_NONE) o.loss[b / 2] = static_cast<float>(loss);
        found[0] += loss;
        found[1] += part ? 1.0 : 0.0;
      }
    }
  }
}

__device__ __forceinline__ void write_preference(const PreferenceOut& o, const PreferenceSaved& s,
                                                 const double (&found)[3]) {
  const float bad = found[2] > 0.0 ? __builtin_nanf("") : 0.0f;
  const bool mean = o.reduction == FRWKV_REDUCE_MEAN;
  const double share = mean ? (found[1] > 0.0 ? 1.0 / found[1] : 0.0) : 1.0;
  *s.share = static_cast<float>(share) + bad;
  if (o.reduction != FRWKV_REDUCE_NONE) {
    *o.loss = static_cast<float>(found[1] > 0.0 ? found[0] * share : 0.0) + bad;
  }
}

// The sums of log ratios. 2M tokens with a reference and a mask in 8 us, 19 MB: bound by
// the way to them (two or three steps of the search, a window of offsets, the tokens).
// kAlone: one workgroup takes them all and joins them.
template <int kRounds, int kBlockWaves, bool kAlone>
__global__ __launch_bounds__(kBlockWaves * 64) void preference_tokens_kernel(
    Preference a, Packed p, PreferenceOut o, PreferenceSaved s, Scratch w, int64_t tiles) {
  const int64_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  preference_tile<kRounds>(a, p, w.pieces,
                           static_cast<int64_t>(blockIdx.x) * kBlockWaves + wave);
  if constexpr (kAlone) {
    __shared__ double shared[kBlockWaves * 3];
    __syncthreads();
    double found[3] = {};
    join_pairs(a, p, o, s, w.pieces, shift_of(kRounds), tiles, wave, kBlockWaves, found);
    workgroup_sum<kBlockWaves>(found, shared);
    if (threadIdx.x == 0) write_preference(o, s, found);
  } else if (blockIdx.x == 0 && threadIdx.x == 0) {
    *w.done = 0;
  }
}

// Losses and slopes of the pairs. Bound by latency: 512 pairs of 9 pieces a sequence in
// 11 us, 64 pairs in 6.5; more workgroups would have to join their sums in turn.
__global__ __launch_bounds__(kJoinThreads) void preference_join_kernel(
    Preference a, Packed p, PreferenceOut o, PreferenceSaved s, Scratch w, int tile_shift,
    int64_t tiles) {
  __shared__ double shared[kJoinWaves * 3];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  double found[3] = {};
  join_pairs(a, p, o, s, w.pieces, tile_shift, tiles,
             static_cast<int64_t>(blockIdx.x) * kJoinWaves + wave,
             static_cast<int64_t>(gridDim.x) * kJoinWaves, found);
  workgroup_sum<kJoinWaves>(found, shared);
  if (!last_with_all(found, w, shared)) return;
  if (threadIdx.x == 0) write_preference(o, s, found);
}

// A sequence's coefficient to its tokens. 2M tokens in 7 us, as the forward bound by the
// way to the coefficient.
template <int kRounds>
__global__ __launch_bounds__(kWaves * 64) void preference_grad_kernel(
    Packed p, PreferenceSaved s, const float* __restrict__ upstream, bool per_pair,
    void* grad_x, int x_dtype) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile<kRounds> tile(static_cast<int64_t>(blockIdx.x) * kWaves + wave, p.n);
  if (tile.empty()) return;
  bool part[kRounds];
  tile.fetch_part(p.mask, part);
  const float share = *s.share;
  const bool bad = share != share;  // offsets that may not be: NaN for all tokens
  int32_t id[kRounds];
  sequences_of<kRounds>(p, tile.first, id);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int32_t b = min(id[r], p.sequences - 1);
    const float c = s.coefficient[b];
    const bool here = part[r] && id[r] < p.sequences && c != 0.0f;
    const float up = upstream[per_pair ? b / 2 : 0] * share;
    if (tile.has(r)) {
      const float grad = here ? c * up : 0.0f;
      store_at(grad_x, x_dtype, tile.first + 64 * r + lane_id(), bad ? share : grad);
    }
  }
}

// ------------------------------------------------------------------- sizes
constexpr int64_t kMostTokens = (int64_t{1} << 31) - 1;
constexpr int64_t kMostSequences = int64_t{1} << 30;
// Tiles are short until those of kFew rounds fill the GPU's 1024 SIMDs twice (4M tokens,
// policy forward: 28 us with 8 rounds, 25 with 4, whose fewer registers let more waves in).
constexpr int64_t kFewTokens = int64_t{1024} * 64 * kFew * 2;
// One workgroup's tokens: 16 waves of kFew or kMany rounds.
constexpr int64_t kAloneFew = 16 * 64 * kFew;
constexpr int64_t kAloneMany = 16 * 64 * kMany;

int rounds_of(int64_t tokens) {
  if (tokens <= kAloneFew) return kFew;
  if (tokens <= kAloneMany) return kMany;
  return tokens <= kFewTokens ? kFew : kMany;
}

int64_t tiles_of(int64_t tokens) {
  const int64_t each = 64 * rounds_of(tokens);
  return (tokens + each - 1) / each;
}

unsigned blocks_of(int64_t tiles) { return static_cast<unsigned>((tiles + kWaves - 1) / kWaves); }

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

bool sizes_fit(int64_t tokens, int64_t sequences) {
  return tokens > 0 && tokens <= kMostTokens && sequences >= 0 && sequences <= kMostSequences;
}

Saved saved_of(char* p, int64_t tokens, int64_t sequences, size_t* bytes) {
  const size_t weight = 256, slope = weight + aligned(static_cast<size_t>(sequences) * 4);
  *bytes = slope + aligned(static_cast<size_t>(tokens) * 4);
  return {reinterpret_cast<float*>(p), reinterpret_cast<float*>(p + weight),
          reinterpret_cast<float*>(p + slope)};
}

PreferenceSaved preference_saved_of(char* p, int64_t sequences, size_t* bytes) {
  *bytes = 256 + aligned(static_cast<size_t>(sequences) * 4);
  return {reinterpret_cast<float*>(p), reinterpret_cast<float*>(p + 256)};
}

Scratch scratch_of(char* p, int64_t tokens, int64_t sequences, size_t* bytes) {
  const int64_t tiles = tiles_of(tokens);
  const size_t sums = 256;
  const size_t joins = sums + aligned(static_cast<size_t>(blocks_of(tiles)) * kSums * 8);
  const size_t pieces = joins + aligned(kMostJoins * 3 * 8);
  *bytes = pieces + aligned(static_cast<size_t>(tiles + sequences) * sizeof(Piece));
  return {reinterpret_cast<int32_t*>(p), reinterpret_cast<double*>(p + sums),
          reinterpret_cast<double*>(p + joins), reinterpret_cast<Piece*>(p + pieces)};
}

// Workgroups of a join, 64 sequences a wave: up to 1024 need no other workgroup,
// whose sums would take two trips through memory.
unsigned joins_of(int64_t sequences) {
  return static_cast<unsigned>(
      std::clamp<int64_t>((sequences + kJoinThreads - 1) / kJoinThreads, 1, kMostJoins));
}

bool known_dtype(int dtype) {
  return dtype == FRWKV_DTYPE_F32 || dtype == FRWKV_DTYPE_F16 || dtype == FRWKV_DTYPE_BF16;
}

// A vector's type and place; one that may be missing is so where its place is null.
int check_column(const char* what, const char* name, int dtype, const void* data, bool optional,
                 Column* out) {
  if (data == nullptr && optional) {
    *out = {nullptr, kNone};
    return FRWKV_OK;
  }
  if (data == nullptr) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
  }
  if (!known_dtype(dtype)) {
    return set_error(FRWKV_ERR_UNSUPPORTED, "%s: %s must be float32, float16 or bfloat16", what,
                     name);
  }
  *out = {data, dtype};
  return FRWKV_OK;
}

int check_sizes(const char* what, int64_t tokens, int64_t sequences) {
  if (tokens <= 0 || tokens > kMostTokens) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: tokens must be in [1, 2^31), got %lld", what,
                     static_cast<long long>(tokens));
  }
  if (sequences < 0 || sequences > kMostSequences) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: sequences must be in [0, 2^30], got %lld", what,
                     static_cast<long long>(sequences));
  }
  return FRWKV_OK;
}

int check_memory(const char* what, const char* name, const void* p, size_t have, size_t need) {
  if (p == nullptr || have < need) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: %s of %zu bytes given, %zu needed", what,
                     name, p == nullptr ? size_t{0} : have, need);
  }
  if (reinterpret_cast<uintptr_t>(p) % 256 != 0) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: %s must be 256-byte aligned", what, name);
  }
  return FRWKV_OK;
}

// f(rounds) for the tiles of these tokens.
template <typename F>
void with_rounds(int64_t tokens, F&& f) {
  if (rounds_of(tokens) == kFew) {
    f(std::integral_constant<int, kFew>{});
  } else {
    f(std::integral_constant<int, kMany>{});
  }
}

}  // namespace
}  // namespace frwkv

extern "C" {

size_t frwkv_policy_loss_saved_bytes(int64_t tokens, int64_t sequences) {
  if (!frwkv::sizes_fit(tokens, sequences)) return 0;
  size_t bytes = 0;
  (void)frwkv::saved_of(nullptr, tokens, sequences, &bytes);
  return bytes;
}

size_t frwkv_preference_loss_saved_bytes(int64_t pairs) {
  if (pairs <= 0 || pairs > frwkv::kMostSequences / 2) return 0;
  size_t bytes = 0;
  (void)frwkv::preference_saved_of(nullptr, 2 * pairs, &bytes);
  return bytes;
}

size_t frwkv_sequence_loss_workspace_bytes(int64_t tokens, int64_t sequences) {
  if (!frwkv::sizes_fit(tokens, sequences)) return 0;
  size_t bytes = 0;
  (void)frwkv::scratch_of(nullptr, tokens, sequences, &bytes);
  return bytes;
}

int frwkv_policy_loss_forward(int64_t tokens, int64_t sequences, const int32_t* cu_seqlens,
                              const uint8_t* mask, int log_probs_dtype, const void* log_probs,
                              int old_dtype, const void* old_log_probs, int advantages_dtype,
                              const void* advantages, int advantages_per_sequence,
                              int reference_dtype, const void* reference_log_probs,
                              int entropy_dtype, const void* entropy, double clip_low,
                              double clip_high, double dual_clip, float kl_weight,
                              float entropy_weight, int reduction, float* loss, float* metrics,
                              int want_slopes, void* saved, size_t saved_bytes, void* workspace,
                              size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_policy_loss_forward";
  int rc = check_sizes(what, tokens, sequences);
  if (rc != FRWKV_OK) return rc;
  if ((cu_seqlens != nullptr) != (sequences > 0)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: cu_seqlens and a number of sequences go together", what);
  }
  if (reduction < FRWKV_REDUCE_NONE || reduction > FRWKV_REDUCE_SEQUENCE_MEAN) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: unknown reduction %d", what, reduction);
  }
  if ((reduction == FRWKV_REDUCE_SEQUENCE_MEAN || advantages_per_sequence) && sequences == 0) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: cu_seqlens is null", what);
  }
  Policy a{};
  rc = check_column(what, "log_probs", log_probs_dtype, log_probs, false, &a.x);
  if (rc == FRWKV_OK) {
    rc = check_column(what, "old_log_probs", old_dtype, old_log_probs, false, &a.old);
  }
  if (rc == FRWKV_OK) {
    rc = check_column(what, "advantages", advantages_dtype, advantages, false, &a.advantage);
  }
  if (rc == FRWKV_OK) {
    rc = check_column(what, "reference_log_probs", reference_dtype, reference_log_probs, true,
                      &a.reference);
  }
  if (rc == FRWKV_OK) rc = check_column(what, "entropy", entropy_dtype, entropy, true, &a.entropy);
  if (rc != FRWKV_OK) return rc;
  if (entropy_weight == 0.0f) a.entropy = {nullptr, kNone};  // whatever it holds
  if (!(clip_low >= 0.0 && clip_low <= 1.0) || !(clip_high >= 0.0 && clip_high <= 1e30)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: clip_low must be in [0, 1] and clip_high in [0, 1e30]", what);
  }
  if (dual_clip != 0.0 && !(dual_clip > 1.0 && dual_clip <= 1e30)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: dual_clip must be 0 or in (1, 1e30]", what);
  }
  if (!std::isfinite(kl_weight) || !std::isfinite(entropy_weight)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: weights must be finite", what);
  }
  if (!loss) return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: loss is null", what);
  size_t need = 0;
  const Saved s = saved_of(static_cast<char*>(saved), tokens, sequences, &need);
  rc = check_memory(what, "saved", saved, saved_bytes, need);
  if (rc != FRWKV_OK) return rc;
  const Scratch w = scratch_of(static_cast<char*>(workspace), tokens, sequences, &need);
  rc = check_memory(what, "workspace", workspace, workspace_bytes, need);
  if (rc != FRWKV_OK) return rc;
  a.per_sequence = advantages_per_sequence != 0;
  a.above_exact = std::log1p(clip_high);
  a.below_exact = std::log1p(-clip_low);
  a.far_exact = dual_clip > 0.0 ? std::log(dual_clip) : a.above_exact;
  a.above = static_cast<float>(a.above_exact);
  a.below = static_cast<float>(a.below_exact);
  a.far = static_cast<float>(a.far_exact);
  a.most = static_cast<float>(1.0 + clip_high);
  a.least = static_cast<float>(1.0 - clip_low);
  a.dual = static_cast<float>(dual_clip);
  a.kl = kl_weight;
  a.ew = entropy_weight;
  const Packed p{tokens, cu_seqlens, static_cast<int32_t>(sequences), mask};
  const PolicyOut o{loss, metrics, reduction, want_slopes != 0};
  const int64_t tiles = tiles_of(tokens);
  const hipStream_t q = static_cast<hipStream_t>(stream);
  bool plain = true;
  for (const Column* c : {&a.x, &a.old, &a.advantage, &a.reference, &a.entropy}) {
    plain = plain && (!c->given() || c->dtype == FRWKV_DTYPE_F32);
  }
  const auto run = [&](auto rounds, auto all_plain) {
    constexpr int kRounds = decltype(rounds)::value;
    constexpr bool kPlain = decltype(all_plain)::value;
    if (tiles <= kJoinWaves) {
      hipLaunchKernelGGL((policy_tokens_kernel<kRounds, kJoinWaves, true, kPlain>), dim3(1),
                         dim3(kJoinThreads), 0, q, a, p, o, s, w, tiles);
      return;
    }
    const unsigned blocks = blocks_of(tiles);
    hipLaunchKernelGGL((policy_tokens_kernel<kRounds, kWaves, false, kPlain>), dim3(blocks),
                       dim3(kWaves * 64), 0, q, a, p, o, s, w, tiles);
    const unsigned joins = reduction == FRWKV_REDUCE_SEQUENCE_MEAN ? joins_of(sequences) : 1;
    hipLaunchKernelGGL(policy_join_kernel, dim3(joins), dim3(kJoinThreads), 0, q, p, o, s, w,
                       shift_of(kRounds), tiles, static_cast<int32_t>(blocks));
  };
  with_rounds(tokens, [&](auto rounds) {
    if (plain) {
      run(rounds, std::true_type{});
    } else {
      run(rounds, std::false_type{});
    }
  });
  return check_launch("policy loss forward");
}

int frwkv_policy_loss_backward(int64_t tokens, int64_t sequences, const int32_t* cu_seqlens,
                               const uint8_t* mask, float entropy_weight, int reduction,
                               const float* grad_loss, const void* saved, size_t saved_bytes,
                               int log_probs_dtype, void* grad_log_probs, int entropy_dtype,
                               void* grad_entropy, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_policy_loss_backward";
  int rc = check_sizes(what, tokens, sequences);
  if (rc != FRWKV_OK) return rc;
  if ((cu_seqlens != nullptr) != (sequences > 0)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: cu_seqlens and a number of sequences go together", what);
  }
  if (reduction < FRWKV_REDUCE_NONE || reduction > FRWKV_REDUCE_SEQUENCE_MEAN ||
      (reduction == FRWKV_REDUCE_SEQUENCE_MEAN && sequences == 0)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: unknown reduction %d", what, reduction);
  }
  if (!grad_loss) return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: grad_loss is null", what);
  if ((grad_log_probs && !known_dtype(log_probs_dtype)) ||
      (grad_entropy && !known_dtype(entropy_dtype))) {
    return set_error(FRWKV_ERR_UNSUPPORTED,
                     "%s: gradients must be float32, float16 or bfloat16", what);
  }
  size_t need = 0;
  // The forward's buffer is only read here.
  const Saved s = saved_of(const_cast<char*>(static_cast<const char*>(saved)), tokens, sequences,
                           &need);
  rc = check_memory(what, "saved", saved, saved_bytes, need);
  if (rc != FRWKV_OK) return rc;
  if (!grad_log_probs && !grad_entropy) return FRWKV_OK;
  const Packed p{tokens, cu_seqlens, static_cast<int32_t>(sequences), mask};
  const PolicyGrad g{grad_loss,     grad_log_probs, log_probs_dtype, grad_entropy,
                     entropy_dtype, entropy_weight, reduction};
  with_rounds(tokens, [&](auto rounds) {
    hipLaunchKernelGGL((policy_grad_kernel<decltype(rounds)::value>),
                       dim3(blocks_of(tiles_of(tokens))), dim3(kWaves * 64), 0,
                       static_cast<hipStream_t>(stream), p, g, s);
  });
  return check_launch("policy loss backward");
}

int frwkv_preference_loss_forward(int64_t tokens, int64_t pairs, const int32_t* cu_seqlens,
                                  const uint8_t* mask, int log_probs_dtype,
                                  const void* log_probs, int reference_dtype,
                                  const void* reference_log_probs, double beta, double margin,
                                  double label_smoothing, int kind, int normalize, int reduction,
                                  float* loss, float* rewards, void* saved, size_t saved_bytes,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_preference_loss_forward";
  int rc = check_sizes(what, tokens, 2 * std::clamp(pairs, int64_t{-1}, kMostSequences));
  if (rc != FRWKV_OK) return rc;
  if (pairs == 0 || !cu_seqlens || !loss || !rewards) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument or no pairs", what);
  }
  if (reduction < FRWKV_REDUCE_NONE || reduction > FRWKV_REDUCE_SUM) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: unknown reduction %d", what, reduction);
  }
  if (kind < FRWKV_PREFERENCE_SIGMOID || kind > FRWKV_PREFERENCE_SQUARED) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: unknown kind %d", what, kind);
  }
  if (!(beta > 0.0 && beta <= 1e30 && beta >= 1e-30) || !std::isfinite(margin) ||
      !(label_smoothing >= 0.0 && label_smoothing <= 0.5)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: beta must be positive, margin finite and label_smoothing in [0, 0.5]",
                     what);
  }
  Preference a{};
  rc = check_column(what, "log_probs", log_probs_dtype, log_probs, false, &a.x);
  if (rc == FRWKV_OK) {
    rc = check_column(what, "reference_log_probs", reference_dtype, reference_log_probs, true,
                      &a.reference);
  }
  if (rc != FRWKV_OK) return rc;
  const int64_t sequences = 2 * pairs;
  size_t need = 0;
  const PreferenceSaved s = preference_saved_of(static_cast<char*>(saved), sequences, &need);
  rc = check_memory(what, "saved", saved, saved_bytes, need);
  if (rc != FRWKV_OK) return rc;
  const Scratch w = scratch_of(static_cast<char*>(workspace), tokens, sequences, &need);
  rc = check_memory(what, "workspace", workspace, workspace_bytes, need);
  if (rc != FRWKV_OK) return rc;
  a.beta = beta;
  a.margin = margin;
  a.smoothing = label_smoothing;
  a.kind = kind;
  a.normalize = normalize != 0;
  const Packed p{tokens, cu_seqlens, static_cast<int32_t>(sequences), mask};
  const PreferenceOut o{loss, rewards, reduction};
  const int64_t tiles = tiles_of(tokens);
  const hipStream_t q = static_cast<hipStream_t>(stream);
  with_rounds(tokens, [&](auto rounds) {
    constexpr int kRounds = decltype(rounds)::value;
    if (tiles <= kJoinWaves) {
      hipLaunchKernelGGL((preference_tokens_kernel<kRounds, kJoinWaves, true>), dim3(1),
                         dim3(kJoinThreads), 0, q, a, p, o, s, w, tiles);
      return;
    }
    hipLaunchKernelGGL((preference_tokens_kernel<kRounds, kWaves, false>), dim3(blocks_of(tiles)),
                       dim3(kWaves * 64), 0, q, a, p, o, s, w, tiles);
    hipLaunchKernelGGL(preference_join_kernel, dim3(joins_of(sequences)), dim3(kJoinThreads), 0, q,
                       a, p, o, s, w, shift_of(kRounds), tiles);
  });
  return check_launch("preference loss forward");
}

int frwkv_preference_loss_backward(int64_t tokens, int64_t pairs, const int32_t* cu_seqlens,
                                   const uint8_t* mask, int reduction, const float* grad_loss,
                                   const void* saved, size_t saved_bytes, int log_probs_dtype,
                                   void* grad_log_probs, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_preference_loss_backward";
  int rc = check_sizes(what, tokens, 2 * std::clamp(pairs, int64_t{-1}, kMostSequences));
  if (rc != FRWKV_OK) return rc;
  if (pairs == 0 || !cu_seqlens || !grad_loss || !grad_log_probs) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument or no pairs", what);
  }
  if (reduction < FRWKV_REDUCE_NONE || reduction > FRWKV_REDUCE_SUM) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: unknown reduction %d", what, reduction);
  }
  if (!known_dtype(log_probs_dtype)) {
    return set_error(FRWKV_ERR_UNSUPPORTED,
                     "%s: gradients must be float32, float16 or bfloat16", what);
  }
  size_t need = 0;
  const PreferenceSaved s = preference_saved_of(
      const_cast<char*>(static_cast<const char*>(saved)), 2 * pairs, &need);
  rc = check_memory(what, "saved", saved, saved_bytes, need);
  if (rc != FRWKV_OK) return rc;
  const Packed p{tokens, cu_seqlens, static_cast<int32_t>(2 * pairs), mask};
  with_rounds(tokens, [&](auto rounds) {
    hipLaunchKernelGGL((preference_grad_kernel<decltype(rounds)::value>),
                       dim3(blocks_of(tiles_of(tokens))), dim3(kWaves * 64), 0,
                       static_cast<hipStream_t>(stream), p, s, grad_loss,
                       reduction == FRWKV_REDUCE_NONE, grad_log_probs, log_probs_dtype);
  });
  return check_launch("preference loss backward");
}

}  // extern "C"
