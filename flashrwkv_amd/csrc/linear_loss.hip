// Losses of a language model's head from its hidden rows: softmax cross
// entropy and distillation from a teacher's top logits, both over the whole
// vocabulary and both without keeping the logits.
//
// With z = h W^T (rows i, vocabulary v), s = 1 / T (1 for cross entropy) and a
// sparse target b_i (one entry 1 for cross entropy; the K shares p_ik =
// softmax over the row's present teacher logits / T for distillation):
//   lse_i = log sum_v exp(s z_iv)
//   loss_i = T^2 (lse_i + sum_k p_ik (log p_ik - s z_i,k))
//   dL/dz_iv = w_i T (exp(s z_iv - lse_i) - b_iv),  w_i the upstream weight
//   dh = dz W,  dW = dz^T h.
//
// Rows that take no part (target = ignore_index; no teacher entry) are left
// out at the start: the hidden rows of the others are copied together (2 N C
// elements moved against 2 N V C operations a product), so masked rows cost
// nothing afterwards and what stands in them reaches nothing. How many rows
// are left stays on the device; grids are sized for all rows and tiles past
// the count end at once.
//
// Forward: one product h W^T whose epilogue keeps the maximum and the sum of
// exponentials of each tile's columns, row by row; a second kernel joins the
// tiles. A row's one target logit is taken from the accumulators that hold it;
// K > 1 of them are dot products of their own (fp32).
// Backward, for one piece of the vocabulary after another: the product again,
// its epilogue turning logits into dz of the piece (16 bits, [rows][piece]);
// the target entries are overwritten from the fp32 target logits, so that
// p - b does not lose digits where the two are close; then dz W into fp32 slabs,
// one a split of it, to which each piece adds (their sum, in order, is dh), and
// dz^T h, which is dW's rows.
// Everything is summed in fp32 in a fixed order; dz is the only rounding to
// 16 bits before the outputs, as a matrix operand has to be (relative error at
// most 2^-8 an entry for bf16, independent between entries).
#include <algorithm>
#include <type_traits>

#include "capi_internal.h"
#include "gemm_tile.h"
#include "wkv7_device.h"

namespace frwkv {
namespace {

using gemm::f32x4;
using gemm::Major;
using gemm::Operand;

constexpr float kLn2 = 0.69314718055994531f;
constexpr int kRowPad = 256;       // rows of workspaces, and a product's largest tile
constexpr int kVocabTile = 256;    // pieces of the vocabulary are whole multiples of it
constexpr int kFewest = 32;        // rows that take part up to here: see Twice below
constexpr int kScanThreads = 1024;
constexpr int kCus = 256;
constexpr int kMostSplits = 16;
constexpr float kNaN = __builtin_nanf("");

__host__ __device__ constexpr int64_t round_up(int64_t x, int64_t to) {
  return (x + to - 1) / to * to;
}

template <typename T>
__device__ __forceinline__ void unpack8(uint4 q, float (&out)[8]) {
  const uint16_t* s = reinterpret_cast<const uint16_t*>(&q);
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = to_f32<T>(s[e]);
}

template <typename T>
__device__ __forceinline__ float low(uint32_t pair) {
  return to_f32<T>(static_cast<uint16_t>(pair & 0xffffu));
}

template <typename T>
__device__ __forceinline__ float high(uint32_t pair) {
  return to_f32<T>(static_cast<uint16_t>(pair >> 16));
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
  return x;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

// (maximum, sum of 2^(scale (x - maximum))) of two sets; a sum of 0 is an empty set.
// Here as wherever an exponential is taken the difference comes before the scale: it
// is exact near the maximum, while a rounded scale x maximum is off by a part of
// itself, which is all of the exponent where logits over T are beyond 2^24.
__device__ __forceinline__ float2 joined(float2 a, float2 b, float scale) {
  if (b.y == 0.0f) return a;
  if (a.y == 0.0f) return b;
  const float top = fmaxf(a.x, b.x);
  return make_float2(top, a.y * __builtin_amdgcn_exp2f((a.x - top) * scale) +
                              b.y * __builtin_amdgcn_exp2f((b.x - top) * scale));
}

// Twice: where the two terms of row m of a few stand in dz, 16 rows' first terms
// and then their second ones, so that a lane of any tile that holds the one holds
// the other. The hidden rows stand in the same order from kTermRows on.
constexpr int kTermRows = 2 * kFewest;
__device__ __forceinline__ int term_row(int m, int term) {
  return (m & 15) + 2 * (m & ~15) + 16 * term;
}

// What the forward leaves for the backward. Row indices m count the rows that
// take part, in order; i is the row's place in the caller's tensors.
struct Saved {
  int32_t* count;   // [1]     rows that take part
  int32_t* cut;     // [1]     columns of the forward that large tiles take
  int32_t* done;    // [1]     workgroups of join_tiles_kernel that have ended
  int32_t* row;     // [pad]   m -> i
  int32_t* place;   // [N]     i -> m, or -1
  int32_t* part;    // [N]     distillation: whether row i takes part
  int32_t* index;   // [N][K]  target tokens (by i); -1 absent, V or more out of range
  float* share;     // [N][K]  p (by i)
  float* target;    // [N][K]  b at that token: the sum of p over equal tokens (by i)
  float* base;      // [N]     sum p log p (by i)
  float* lse;       // [pad]   T log sum exp(z / T), never below the maximum of z (by m)
  float* logit;     // [pad][K] z at the target tokens (by m)
  uint16_t* hidden; // [pad][C] the rows that take part, zeros after the last up to a tile;
                    // of a few also their term_row order, zeros between, from kTermRows on
};

struct Layout {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};

Saved saved_of(char* p, int64_t n, int64_t c, int64_t k, size_t* bytes) {
  const int64_t pad = round_up(n, kRowPad);
  Layout l;
  Saved s;
  const size_t count = l.take(4), cut = l.take(4), done = l.take(4);
  const size_t row = l.take(pad * 4), place = l.take(n * 4), part = l.take(n * 4);
  const size_t index = l.take(n * k * 4), share = l.take(n * k * 4);
  const size_t target = l.take(n * k * 4), base = l.take(n * 4), lse = l.take(pad * 4);
  const size_t logit = l.take(pad * k * 4), hidden = l.take(pad * c * 2);
  s.count = reinterpret_cast<int32_t*>(p + count);
  s.cut = reinterpret_cast<int32_t*>(p + cut);
  s.done = reinterpret_cast<int32_t*>(p + done);
  s.row = reinterpret_cast<int32_t*>(p + row);
  s.place = reinterpret_cast<int32_t*>(p + place);
  s.part = reinterpret_cast<int32_t*>(p + part);
  s.index = reinterpret_cast<int32_t*>(p + index);
  s.share = reinterpret_cast<float*>(p + share);
  s.target = reinterpret_cast<float*>(p + target);
  s.base = reinterpret_cast<float*>(p + base);
  s.lse = reinterpret_cast<float*>(p + lse);
  s.logit = reinterpret_cast<float*>(p + logit);
  s.hidden = reinterpret_cast<uint16_t*>(p + hidden);
  *bytes = l.bytes;
  return s;
}

// -------------------------------------------------- tile sizes and their times
enum class Size { kNarrow64, kNarrow128, kFewRows, kSmall, kLarge };

struct TileTime {
  int32_t p, q;
  float step_us, fixed_us;  // of 64 k, and of a tile's start and end beside them
};

// Measured on products that fill the GPU for many rounds.
__host__ __device__ constexpr TileTime time_of(Size s) {
  return s == Size::kNarrow64    ? TileTime{64, 64, 0.4f, 3.0f}
         : s == Size::kNarrow128 ? TileTime{128, 64, 0.7f, 3.0f}
         : s == Size::kFewRows   ? TileTime{256, 64, 1.0f, 3.0f}
         : s == Size::kSmall     ? TileTime{128, 128, 0.6f, 3.0f}
                                 : TileTime{256, 256, 1.65f, 5.0f};
}

// kSmall's are fewer than 2^30, checked at the entry points; the narrow ones that
// size_of counts before it takes them can be four times as many.
__host__ __device__ inline int64_t tiles_of(Size s, int32_t p, int32_t q) {
  const TileTime t = time_of(s);
  return static_cast<int64_t>((p + t.p - 1) / t.p) * ((q + t.q - 1) / t.q);
}

__host__ __device__ inline float product_us(Size s, int32_t p, int32_t q, int32_t steps) {
  const int64_t rounds = (tiles_of(s, p, q) + kCus - 1) / kCus;
  return static_cast<float>(rounds) *
         (static_cast<float>(steps) * time_of(s).step_us + time_of(s).fixed_us);
}

// How a product over a range of the vocabulary is tiled: `first` columns with
// large tiles, the rest with small ones. Large tiles leave a last round with few
// of them; small ones, less efficient by half but four times as many, take its
// place where that is faster (forward of 1000 x 50277 x 2560, 3.1 rounds: 248 ->
// 233 us).
struct Cut {
  int32_t first;
  float us;
};

// Tile sizes that may be used.
struct Sizes {
  bool small, large;
};

// vocab: columns of the range; across: the other extent (rows or channels).
__host__ __device__ inline Cut cut_of(int32_t vocab, int32_t across, int32_t steps, Sizes sizes) {
  if (!sizes.large || (sizes.small && across <= time_of(Size::kSmall).q)) {
    return {0, product_us(Size::kSmall, vocab, across, steps)};
  }
  const float large = product_us(Size::kLarge, vocab, across, steps);
  if (!sizes.small) return {vocab, large};
  const float small = product_us(Size::kSmall, vocab, across, steps);
  Cut best = small < large ? Cut{0, small} : Cut{vocab, large};
  const int64_t full = tiles_of(Size::kLarge, vocab, across) / kCus * kCus;
  const int32_t first = static_cast<int32_t>(full / ((across + 255) / 256) * 256);
  if (first > 0 && first < vocab) {
    const float both = product_us(Size::kLarge, first, across, steps) +
                       product_us(Size::kSmall, vocab - first, across, steps) + 3.0f;
    if (both < best.us) best = {first, both};
  }
  return best;
}

constexpr Sizes kBothSizes = {true, true};

// Of the products over rows, those whose tiles, narrow as they are, fill the GPU at
// most once have the narrowest such ones: what bounds them is how many loads are
// under way (scoring 8 rows of 4096 channels, 64 x 64, 128 x 64 and 256 x 64 tiles:
// 8192 tokens 27, 30 and 43 us, 32768 tokens 77, 59 and 72, 65536 tokens 127, 112
// and 106). Otherwise few rows have tiles of 64 of them, and kSmall stands for a cut.
inline Size size_of(int32_t vocab, int32_t rows) {
  for (Size size : {Size::kNarrow64, Size::kNarrow128}) {
    if (tiles_of(size, vocab, rows) <= kCus) return size;
  }
  return rows <= time_of(Size::kFewRows).q ? Size::kFewRows : Size::kSmall;
}

// For products over the rows that take part the device decides the cut, where their
// count is (777 rows, of which 520 take part, 20011 x 768: forward and backward
// 138 -> 127 us). A launch that finds no columns of its own ends at once, which takes
// 4 us; sizes that no count from half of the rows on asks for are not launched.
inline Sizes sizes_of(int32_t vocab, int32_t rows, int32_t steps) {
  Sizes sizes = {false, false};
  if (size_of(vocab, rows) != Size::kSmall) return {true, false};
  for (int eighths = 4; eighths <= 8; ++eighths) {
    const Cut cut = cut_of(vocab, (rows * eighths + 7) / 8, steps, kBothSizes);
    sizes.large |= cut.first > 0;
    sizes.small |= cut.first < vocab;
  }
  return sizes;
}

// The columns that a kernel of tiles G takes of `columns`, cut at *cut.
template <typename G>
__device__ __forceinline__ void own_columns(const int32_t* cut, int32_t& from, int32_t& columns) {
  from = 0;
  if (G::kBQ == 64) return;  // all of them
  if (G::kBQ == 256) {
    columns = *cut;
  } else {
    from = *cut;
    columns -= from;
  }
}

// ---------------------------------------------------------------- targets
__device__ __forceinline__ int32_t as_token(int64_t t, int32_t vocab) {
  // Negative tokens are absent for distillation and out of range for cross
  // entropy, whose caller has taken ignore_index out before.
  return t < 0 ? -1 : t >= vocab ? vocab : static_cast<int32_t>(t);
}

// Distillation, a wave a row: shares from the teacher's logits. An entry is
// present where its token is not negative and its logit not -inf; a row
// without one takes no part. The gradients of tokens that occur twice in a row take
// the sum of their shares, found by comparing all pairs, four of them a step (2 rows
// of 116 entries: 5.7 us, one by one 13); the loss is a sum over the entries. Dynamic
// LDS: K tokens and K shares a wave, rounded up to four.
template <typename T, typename Index>
__global__ __launch_bounds__(256) void teacher_targets_kernel(
    const typename IoTraits<T>::storage* __restrict__ logits, const Index* __restrict__ indices,
    int32_t n, int32_t k, int32_t vocab, float inv_temperature, Saved s) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + wave;
  const int room = static_cast<int>(round_up(k, 4));
  int32_t* tokens = reinterpret_cast<int32_t*>(smem) + wave * 2 * room;
  float* shares = reinterpret_cast<float*>(tokens + room);
  const int64_t at = static_cast<int64_t>(i) * k;
  float top = -__builtin_inff();
  bool any = false;
  if (i < n) {
    for (int j = lane; j < k; j += 64) {
      const float x = to_f32<T>(logits[at + j]);
      const int32_t token = x == -__builtin_inff() ? -1 : as_token(indices[at + j], vocab);
      tokens[j] = token;
      shares[j] = x;
      if (token >= 0) {
        any = true;
        top = fmaxf(top, x);
      }
    }
  }
  const bool part = __ballot(any) != 0;
  // From the maximum before 1 / T, which can take the lowest finite logit to -inf.
  top = wave_max(top);
  float total = 0.0f;
  if (i < n) {
    for (int j = lane; j < k; j += 64) {
      shares[j] = (shares[j] - top) * inv_temperature;
      total += tokens[j] >= 0 ? __builtin_amdgcn_exp2f(shares[j] * kLog2E) : 0.0f;
    }
  }
  total = wave_sum(total);
  const float log_total = __logf(total);
  float base = 0.0f;
  if (i < n) {
    for (int j = lane; j < k; j += 64) {
      float p = 0.0f;
      if (part && tokens[j] >= 0) {
        const float log_p = shares[j] - log_total;
        p = __builtin_amdgcn_exp2f(log_p * kLog2E);
        base += p == 0.0f ? 0.0f : p * log_p;
      }
      shares[j] = p;
    }
  }
  base = wave_sum(base);
  if (lane < room - k) tokens[k + lane] = -2;  // no token's
  __syncthreads();
  if (i >= n) return;
  for (int j = lane; j < k; j += 64) {
    const int32_t token = tokens[j];
    float sum = 0.0f;
#pragma unroll 4
    for (int q = 0; q < room; q += 4) {
      const int4 t = *reinterpret_cast<const int4*>(tokens + q);
      const float4 p = *reinterpret_cast<const float4*>(shares + q);
      sum += t.x == token ? p.x : 0.0f;
      sum += t.y == token ? p.y : 0.0f;
      sum += t.z == token ? p.z : 0.0f;
      sum += t.w == token ? p.w : 0.0f;
    }
    s.index[at + j] = token;
    s.share[at + j] = shares[j];
    s.target[at + j] = sum;
  }
  if (lane == 0) {
    s.part[i] = part;
    s.base[i] = base;
  }
}

// Which rows take part, and what is noted of one that stands in no tensor yet.
// Cross entropy: one entry a row, share 1.
template <typename Index>
struct Labels {
  const Index* targets;
  int64_t ignore;
  __device__ __forceinline__ bool part(int32_t i) const { return targets[i] != ignore; }
  __device__ __forceinline__ void note(int32_t i, int32_t vocab, const Saved& s) const {
    const int64_t t = targets[i];
    const int32_t token = as_token(t, vocab);
    s.index[i] = t != ignore && token < 0 ? vocab : token;
    s.share[i] = 1.0f;
    s.target[i] = 1.0f;
    s.base[i] = 0.0f;
  }
};

// Distillation, behind teacher_targets_kernel.
struct Teacher {
  const int32_t* parts;
  __device__ __forceinline__ bool part(int32_t i) const { return parts[i] != 0; }
  __device__ __forceinline__ void note(int32_t, int32_t, const Saved&) const {}
};

// What the numbering of the rows needs to know of the product.
struct Rows {
  int32_t n, vocab, steps;
  Sizes sizes;      // launched for it
  float* row_loss;  // not null: 0 for the rows that take no part
};

__device__ __forceinline__ void note_count(const Rows& d, int32_t count, const Saved& s) {
  *s.count = count;
  *s.cut = cut_of(d.vocab, count, d.steps, d.sizes).first;
  *s.done = 0;
}

// Numbers the rows that take part, in order. One workgroup: 5 us for 2048 rows, 13
// for 8192, beside products of milliseconds.
template <typename Source>
__global__ __launch_bounds__(kScanThreads) void number_rows_kernel(Source source, Rows d, Saved s) {
  __shared__ int32_t waves[kScanThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t before = 0;
  for (int32_t first = 0; first < d.n; first += kScanThreads) {
    const int32_t i = first + static_cast<int32_t>(threadIdx.x);
    const bool part = i < d.n && source.part(i);
    const uint64_t mask = __ballot(part);
    if (lane == 0) waves[wave] = __popcll(mask);
    __syncthreads();
    int32_t m = before + __popcll(mask & ((1ull << lane) - 1));
    int32_t all = 0;
#pragma unroll
    for (int w = 0; w < kScanThreads / 64; ++w) {
      if (w < wave) m += waves[w];
      all += waves[w];
    }
    if (i < d.n) {
      source.note(i, d.vocab, s);
      s.place[i] = part ? m : -1;
      if (!part && d.row_loss != nullptr) d.row_loss[i] = 0.0f;
    }
    if (part) s.row[m] = i;
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) note_count(d, before, s);
}

// The same by every workgroup for itself, for up to kOwnNumbers rows: a launch less
// (with the sum over rows in join_tiles_kernel, forward of 300 x 2000 x 768: 20.7 ->
// 19.3 us). m: how many take part before row `mine`; count: of all. Returns whether
// `mine` does.
constexpr int kOwnNumbers = 1024;
constexpr int kGatherThreads = 256;

template <typename Source>
__device__ __forceinline__ bool own_number(const Source& source, int32_t n, int32_t mine,
                                           int32_t& m, int32_t& count) {
  constexpr int kWaves = kGatherThreads / 64, kTurns = kOwnNumbers / kGatherThreads;
  __shared__ uint64_t masks[kTurns * kWaves];
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int32_t i = u * kGatherThreads + static_cast<int32_t>(threadIdx.x);
    const uint64_t mask = __ballot(i < n && source.part(i));
    if ((threadIdx.x & 63) == 0) masks[u * kWaves + wave] = mask;
  }
  __syncthreads();
  m = count = 0;
  bool part = false;
#pragma unroll
  for (int g = 0; g < kTurns * kWaves; ++g) {
    const uint64_t mask = masks[g];
    count += __popcll(mask);
    const int32_t at = mine - 64 * g;
    if (at >= 64) m += __popcll(mask);
    if (at >= 0 && at < 64) {
      m += __popcll(mask & ((1ull << at) - 1));
      part = (mask >> at & 1) != 0;
    }
  }
  return part;
}

// Copies the hidden rows that take part together (zeros for the rows that fill up
// the last tile; few rows once more for each term) and computes their K > 1
// target logits, kGather a workgroup, a wave each (NaN for a token out of range).
// blockIdx.x: a row i of the caller's, which the workgroup numbers itself (kOwn),
// or a row m; blockIdx.y: the tokens.
// Bound by the K weight rows a row where rows are many (4096 of 64 tokens of 2048
// channels: 151 us, 7.1 TB/s), by one read of a weight row where they are few (6
// rows of 94 tokens of 3712 channels, forward and backward with all of a row's
// tokens in one workgroup: 191 us, so: 120 us).
constexpr int kGather = 4;

template <typename T, bool kOwn, typename Source>
__global__ __launch_bounds__(kGatherThreads) void gather_rows_kernel(
    const uint16_t* __restrict__ hidden, const uint16_t* __restrict__ weight, int32_t c,
    int32_t k, Source source, Rows d, Saved s) {
  const int block = blockIdx.x;
  const bool first = blockIdx.y == 0;
  if (!first && block >= d.n) return;
  int32_t m = block, i = 0, count;
  bool part;
  if constexpr (kOwn) {
    i = block;
    part = own_number(source, d.n, i, m, count);
    if (first && threadIdx.x == 0) {
      if (block == 0) note_count(d, count, s);
      if (i < d.n) {
        source.note(i, d.vocab, s);
        s.place[i] = part ? m : -1;
        if (!part && d.row_loss != nullptr) d.row_loss[i] = 0.0f;
      }
      if (part) s.row[m] = i;
    }
  } else {
    count = *s.count;
    part = m < count;
    if (part) i = s.row[m];
  }
  const auto fill = [&](int row, const uint16_t* from) {
    uint16_t* to = s.hidden + static_cast<int64_t>(row) * c;
    for (int x = threadIdx.x * 8; x < c; x += kGatherThreads * 8) {
      *reinterpret_cast<uint4*>(to + x) =
          from == nullptr ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(from + x);
    }
  };
  const uint16_t* from = hidden + static_cast<int64_t>(i) * c;
  if (first) {
    const bool twice = count <= kFewest;
    // term_row's inverse: the row whose copy stands in this one.
    const int at = block - kTermRows;
    const bool copied = twice && at >= 0 && at < kTermRows && (at & 15) + (at >> 5) * 16 < count;
    if (block >= count && block < round_up(count, kRowPad) && !copied) fill(block, nullptr);
    if (part) fill(m, from);
    if (part && twice) {
      fill(kTermRows + term_row(m, 0), from);
      fill(kTermRows + term_row(m, 1), from);
    }
  }
  if (!part) return;
  if (k == 1) {  // one out of range; lse_tiles_kernel writes the others
    if (threadIdx.x == 0) s.logit[m] = kNaN;
    return;
  }
  const int j = static_cast<int>(blockIdx.y) * kGather + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (j >= k) return;
  const int32_t token = s.index[static_cast<int64_t>(i) * k + j];
  float z = token >= d.vocab ? kNaN : 0.0f;
  if (token >= 0 && token < d.vocab) {
    const uint16_t* w = weight + static_cast<int64_t>(token) * c;
    float sum = 0.0f;
    for (int x0 = lane * 8; x0 < c; x0 += 2048) {
      uint4 h4[4], w4[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = x0 + 512 * u;
        h4[u] = w4[u] = make_uint4(0, 0, 0, 0);
        if (x < c) {
          h4[u] = *reinterpret_cast<const uint4*>(from + x);
          w4[u] = *reinterpret_cast<const uint4*>(w + x);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float a[8], b[8];
        unpack8<T>(h4[u], a);
        unpack8<T>(w4[u], b);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(a[e], b[e], sum);
      }
    }
    z = wave_sum(sum);
  }
  if (lane == 0) s.logit[static_cast<int64_t>(m) * k + j] = z;
}

// ------------------------------------------------------------- products
// Tile shapes, chosen on the host by the time they would take (see plan_of).
template <typename T, Major MA, Major MB>
using LargeTile = gemm::Tile<T, MA, MB, 256, 256, 2, 4, 2>;
template <typename T, Major MA, Major MB>
using SmallTile = gemm::Tile<T, MA, MB, 128, 128, 2, 4, 4>;
// Few rows only stream the weight, and every workgroup starting at the first k
// hits the same memory channels where rows are a power of two apart: they
// start at different ones (scoring 1 row, 65536 x 2048, from memory: 79 -> 63 us;
// for the large tile, bound by the products, it costs 1%). So do the narrow tiles,
// with more stages under way.
template <typename T, Major MA, Major MB>
using Narrow64Tile = gemm::Tile<T, MA, MB, 64, 64, 2, 4, 8, true>;
template <typename T, Major MA, Major MB>
using Narrow128Tile = gemm::Tile<T, MA, MB, 128, 64, 4, 2, 6, true>;
template <typename T, Major MA, Major MB>
using FewRowsTile = gemm::Tile<T, MA, MB, 256, 64, 8, 1, 3, MA == Major::kK && MB == Major::kK>;

// The tiles of a product over rows m, whose count stands on the device: the
// workgroups of a launch of at most one a CU take them in turn. While a
// workgroup finishes a tile, the first stages of its next one are on their way.
__host__ __device__ __forceinline__ int tiles_along(int size, int tile) {
  return (size + tile - 1) / tile;
}

// Where this lane's accumulators hold a token: 16 i + r, or -1. p0: the tile's
// first token, left: tokens from there on.
template <typename G>
__device__ __forceinline__ int own_row(int token, int p0, int left) {
  const int at = token - p0, row = at - G::row(0);
  return token >= 0 && at < left && row >= 0 && row < 16 * G::TP && (row & 15) < 4 ? row : -1;
}

// D[v][m] of a vocabulary range: per tile of v and row m the maximum of z and
// the sum of 2^(scale (z - maximum)), scale = s log2 e, to part[tile][m]. one: rows
// have one target each, whose logit goes to s.logit as it stands here, so that
// it cancels against a maximum that it is.
// Bound by the matrix units for many rows (8192 x 65536 x 4096 bf16: 3.38 ms, 1302
// TFLOP/s) and by the weight's read for few (1 row of 2048 channels, 65536 tokens:
// 44 to 49 us, 5.5 to 6.1 TB/s). A tile's exponentials take 2 of its 5 us beside the
// product.
template <typename G, typename T>
__global__ __launch_bounds__(gemm::kThreads, 2) void lse_tiles_kernel(
    Operand w, Operand h, int32_t c, float scale, bool one, float2* __restrict__ part,
    int64_t pad, Saved s) {
  __shared__ __attribute__((aligned(1024))) char smem[G::kLdsBytes];
  __shared__ float maxima[G::kWP][G::kBQ], sums[G::kWP][G::kBQ];
  int vocab0;
  own_columns<G>(s.cut, vocab0, w.rows);
  w.data += static_cast<int64_t>(vocab0) * w.ld;
  part += vocab0 / 256 * pad;  // behind the large tiles'
  const int rows = *s.count;
  const int np = tiles_along(w.rows, G::kBP);
  const int nq = tiles_along(rows, G::kBQ), total = np * nq, steps = c / gemm::kStep;
  int id = blockIdx.x;
  if (id >= total) return;
  G tile;
  int tp, tq;
  gemm::tile_of(gemm::xcd_run(id, total), np, nq, tp, tq);
  tile.begin(w, h, tp * G::kBP, tq * G::kBQ, 0, steps, smem, G::kTurns ? tp % steps : 0);
  G::arrive();
  while (true) {
    const int p0 = tp * G::kBP, q0 = tq * G::kBQ;
    int token[G::TQ];
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      const int m = q0 + G::column(j);
      token[j] = one && m < rows ? s.index[s.row[m]] : -1;
    }
    tile.multiply(smem);
    // The compiler's wait for these comes here, not behind the loads that
    // begin starts, which it does not count.
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) asm volatile("" : "+v"(token[j]));
    const int64_t to = static_cast<int64_t>(tp) * pad + q0;
    id += gridDim.x;
    if (id < total) {
      gemm::tile_of(gemm::xcd_run(id, total), np, nq, tp, tq);
      tile.begin(w, h, tp * G::kBP, tq * G::kBQ, 0, steps, smem, G::kTurns ? tp % steps : 0);
    }
    const int left = w.rows - p0;
    if (left < G::kBP) {  // the last columns do not exist
#pragma unroll
      for (int i = 0; i < G::TP; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool here = G::row(i) + r < left;
#pragma unroll
          for (int j = 0; j < G::TQ; ++j) {
            tile.acc[i][j][r] = here ? tile.acc[i][j][r] : -__builtin_inff();
          }
        }
      }
    }
    const int wp = G::wave() / G::kWQ;
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < G::TP; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, tile.acc[i][j][r]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // -inf everywhere (columns beyond the vocabulary): a sum of 0, not NaN.
      const float from = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < G::TP; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sum += __builtin_amdgcn_exp2f((tile.acc[i][j][r] - from) * scale);
        }
      }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if ((threadIdx.x & 63) < 16) {
        maxima[wp][G::column(j)] = top;
        sums[wp][G::column(j)] = sum;
      }
    }
    G::arrive();
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      const int own = own_row<G>(token[j], vocab0 + p0, left);
      if (__ballot(own >= 0) == 0) continue;
      float z = 0.0f;
#pragma unroll
      for (int i = 0; i < G::TP; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) z = own == 16 * i + r ? tile.acc[i][j][r] : z;
      }
      if (own >= 0) s.logit[q0 + G::column(j)] = z;
    }
    __syncthreads();
    for (int q = threadIdx.x; q < G::kBQ; q += gemm::kThreads) {
      float top = maxima[0][q];
#pragma unroll
      for (int x = 1; x < G::kWP; ++x) top = fmaxf(top, maxima[x][q]);
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < G::kWP; ++x) {
        const float s = sums[x][q];
        if (s != 0.0f) sum += s * __builtin_amdgcn_exp2f((maxima[x][q] - top) * scale);
      }
      part[to + q] = make_float2(top, sum);
    }
    if (id >= total) return;
  }
}

// D[v][m] of a piece of the vocabulary: dz[m][v] = coef_m 2^(scale (z - lse_m)),
// zero for rows and columns that are not there. Bound as the forward is:
// 8192 x 32768 x 4096 in 1.75 ms, 1260 TFLOP/s. The 256 x 256 form has 10 values more
// than registers: 44 MB of scratch written beside 537 of dz.
//
// Twice: rounding dz to 16 bits is one error for all elements that a target
// entry dominates, up to 2^-9 of the entry 1 for bf16. Over many rows such
// errors average out below the outputs' own rounding; in a few rows one can be
// twice that. Up to kFewest rows that take part leave half of a tile's columns
// unused, so there dz has two terms, the rounded value and what is left of it, and
// the products add both at no cost (bf16 gradients of 3 weighted rows,
// 3001 x 512: up to 3.8e-3 off with one term, 1.7e-3 with two, the outputs' own
// rounding). More rows would need a product of twice as many: they keep one term.
template <typename G, typename T>
__global__ __launch_bounds__(gemm::kThreads, 2) void softmax_grad_kernel(
    Operand w, Operand h, const int32_t* __restrict__ cut, int32_t c, float scale,
    const float* __restrict__ coef, uint16_t* __restrict__ dz, int64_t ld, Saved s) {
  __shared__ __attribute__((aligned(1024))) char smem[G::kLdsBytes];
  int at;
  own_columns<G>(cut, at, w.rows);
  w.data += static_cast<int64_t>(at) * w.ld;
  dz += at;
  const int rows = *s.count;
  const int np = tiles_along(w.rows, G::kBP);
  const int nq = tiles_along(rows, G::kBQ), total = np * nq, steps = c / gemm::kStep;
  int id = blockIdx.x;
  if (id >= total) return;
  G tile;
  int tp, tq;
  gemm::tile_of(gemm::xcd_run(id, total), np, nq, tp, tq);
  tile.begin(w, h, tp * G::kBP, tq * G::kBQ, 0, steps, smem, G::kTurns ? tp % steps : 0);
  G::arrive();
  while (true) {
    const int p0 = tp * G::kBP, q0 = tq * G::kBQ;
    float from[G::TQ], co[G::TQ];
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      const int m = q0 + G::column(j);
      from[j] = m < rows ? s.lse[m] : 0.0f;
      co[j] = m < rows ? coef[m] : 0.0f;
    }
    tile.multiply(smem);
    // The compiler's wait for these comes here, not behind the loads that
    // begin starts, which it does not count.
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) asm volatile("" : "+v"(from[j]), "+v"(co[j]));
    id += gridDim.x;
    if (id < total) {
      gemm::tile_of(gemm::xcd_run(id, total), np, nq, tp, tq);
      tile.begin(w, h, tp * G::kBP, tq * G::kBQ, 0, steps, smem, G::kTurns ? tp % steps : 0);
    }
    const int left = w.rows - p0;
    const bool all = left >= G::kBP && rows - q0 >= G::kBQ;
    const bool twice = rows <= kFewest;
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      const bool here = q0 + G::column(j) < rows;
      const auto term = [&](bool second, uint2 (&out)[G::TP]) {
#pragma unroll
        for (int i = 0; i < G::TP; ++i) {
          float x[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[r] = co[j] * __builtin_amdgcn_exp2f((tile.acc[i][j][r] - from[j]) * scale);
            if (!all) x[r] = here && G::row(i) + r < left ? x[r] : 0.0f;
          }
          out[i] = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
          if (second) {
            out[i] = make_uint2(
                pack2<T>(x[0] - low<T>(out[i].x), x[1] - high<T>(out[i].x)),
                pack2<T>(x[2] - low<T>(out[i].y), x[3] - high<T>(out[i].y)));
          }
        }
      };
      uint2 out[G::TP];
      term(false, out);
      // The next tile's loads are waited for before the first store, which
      // would have to be waited for with them.
      if (j == 0) G::arrive();
      uint16_t* to = dz + q0 * ld + p0;
      if (!twice) {
        gemm::store_column<G>(to, ld, G::kBP, G::kBQ, j, out);
        continue;
      }
      // Sixteen rows' block of columns, and where their first terms stand from it.
      const int block = G::wave_q0() + 16 * j;
      if (block >= kFewest) continue;
      to += block * ld;
      gemm::store_column<G>(to, ld, G::kBP, G::kBQ, j, out);
      term(true, out);
      gemm::store_column<G>(to + 16 * ld, ld, G::kBP, G::kBQ, j, out);
    }
    if (id >= total) return;
  }
}

// The entries of dz that have a target: coef (p - b) in fp32 from the fp32
// logit, over what the product's epilogue wrote (which as a part of that epilogue
// costs more, 2 to 4% of a backward, than this launch's 5 us). A thread an entry; equal
// tokens of a row write the same value.
template <typename T>
__global__ __launch_bounds__(256) void target_grad_kernel(int32_t k, int32_t vocab0,
                                                          int32_t columns, float scale,
                                                          const float* __restrict__ coef,
                                                          uint16_t* __restrict__ dz, int64_t ld,
                                                          Saved s) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t m = e / k;
  const int32_t count = *s.count;
  if (m >= count) return;
  const int64_t at = static_cast<int64_t>(s.row[m]) * k + (e - m * k);
  const int32_t v = s.index[at] - vocab0;
  if (s.index[at] < 0 || v < 0 || v >= columns) return;
  const float p = __builtin_amdgcn_exp2f((s.logit[e] - s.lse[m]) * scale);
  const float x = coef[m] * (p - s.target[at]);
  const uint16_t rounded = from_f32<T>(x);
  if (count > kFewest) {
    dz[m * ld + v] = rounded;
    return;
  }
  const int row = static_cast<int>(m);
  dz[term_row(row, 0) * ld + v] = rounded;
  dz[term_row(row, 1) * ld + v] = from_f32<T>(x - to_f32<T>(rounded));
}

// dz W has (C / tile) x (rows / tile) tiles, often fewer than CUs, over a long k:
// k is split so that the rounds of tiles are full, by the estimate
//   rounds x (steps of a split x step_us + fixed_us) + splits x slab_us,
// a slab being written and read once. The host allocates room for the splits
// of all rows; how many the rows that take part want, fewer rows more of them,
// is found where their count is known.
struct Splitting {
  int32_t steps;  // of a whole piece
  int32_t across; // tiles over C
  int32_t tile;   // rows of a tile
  float step_us, fixed_us, row_slab_us;
  int64_t room;   // rows of all slabs
};

__host__ __device__ inline float split_us(const Splitting& x, int64_t rows, int32_t s) {
  const int64_t tiles = (rows + x.tile - 1) / x.tile * x.across;
  return static_cast<float>((tiles * s + kCus - 1) / kCus) *
             (static_cast<float>((x.steps + s - 1) / s) * x.step_us + x.fixed_us) +
         static_cast<float>(s) * static_cast<float>(rows) * x.row_slab_us;
}

__host__ __device__ inline bool may_split(const Splitting& x, int64_t rows, int32_t s) {
  return s == 1 || (x.steps / s >= 8 && s * rows <= x.room);
}

int32_t splits_of(const Splitting& x, int64_t rows) {
  int32_t best = 1;
  for (int32_t s = 2; s <= kMostSplits; ++s) {
    if (may_split(x, rows, s) && split_us(x, rows, s) < split_us(x, rows, best)) best = s;
  }
  return best;
}

// The same by one wave, a lane a choice.
__device__ __forceinline__ int32_t wave_splits_of(const Splitting& x, int64_t rows) {
  const int lane = threadIdx.x & 63;
  int32_t best = lane + 1;
  float least = lane < kMostSplits && may_split(x, rows, best) ? split_us(x, rows, best) : 3e38f;
#pragma unroll
  for (int off = 1; off < kMostSplits; off <<= 1) {
    const float us = __shfl_xor(least, off, 64);
    const int32_t s = __shfl_xor(best, off, 64);
    if (us < least || (us == least && s < best)) {
      least = us;
      best = s;
    }
  }
  return __shfl(best, 0, 64);
}

// The columns of a piece of the backward, and the tile sizes launched over them:
// [0] of the pieces before the last, [1] of the last one.
struct Pieces {
  int32_t columns[2];
  Sizes sizes[2];
  int32_t steps;
};

// D[c][m] = sum over a split's vocabulary of W[v][c] dz[m][v], to slab [m][c]
// of the split (fp32), added to what the pieces before left there: they run one
// after the other, and every element has one owner in each. Bound by the matrix units: 8192 x 32768 x 4096 in 1.69 ms, 1299
// TFLOP/s, in one split.
template <typename G, typename T>
__global__ __launch_bounds__(gemm::kThreads, 2) void hidden_grad_kernel(
    Operand w, Operand dz, const int32_t* __restrict__ count,
    const int32_t* __restrict__ split_count, int32_t steps, int32_t whole_steps, int32_t np,
    bool add, int32_t c, float* __restrict__ slabs) {
  __shared__ __attribute__((aligned(1024))) char smem[G::kLdsBytes];
  const int rows = *count;
  const int splits = *split_count;
  const int split_steps = (whole_steps + splits - 1) / splits;
  const int nq = tiles_along(rows, G::kBQ), each = np * nq, total = each * splits;
  const int64_t slab = static_cast<int64_t>(rows) * c;
  int id = blockIdx.x;
  if (id >= total) return;
  G tile;
  int tp, tq, split;
  const auto begin = [&] {
    const int at = gemm::xcd_run(id, total);
    split = at / each;
    gemm::tile_of(at - split * each, np, nq, tp, tq);
    const int first = split * split_steps;
    const int left = steps - first;
    tile.begin(w, dz, tp * G::kBP, tq * G::kBQ, first * gemm::kStep,
               left < split_steps ? left : split_steps, smem);
  };
  begin();
  G::arrive();
  while (true) {
    tile.multiply(smem);
    const int p0 = tp * G::kBP, q0 = tq * G::kBQ;
    float* out = slabs + split * slab;
    id += gridDim.x;
    if (id < total) {
      begin();
      G::arrive();
    }
    static_assert(G::TQ % 2 == 0, "a lane holds both terms");
    const bool twice = rows <= kFewest;
    if (twice) {  // both terms of dz
#pragma unroll
      for (int j = 0; j < G::TQ; j += 2) {
#pragma unroll
        for (int i = 0; i < G::TP; ++i) tile.acc[i][j] += tile.acc[i][j + 1];
      }
    }
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      int m = q0 + G::column(j);
      if (twice) m = j % 2 == 0 ? (m & 15) + m / 32 * 16 : rows;
      if (m >= rows) continue;
      f32x4* to = reinterpret_cast<f32x4*>(out + static_cast<int64_t>(m) * c + p0 + G::row(0));
      if (add) {
#pragma unroll
        for (int i = 0; i < G::TP; ++i) {
          if (p0 + G::row(i) < c) tile.acc[i][j] += to[4 * i];
        }
      }
#pragma unroll
      for (int i = 0; i < G::TP; ++i) {
        if (p0 + G::row(i) < c) to[4 * i] = tile.acc[i][j];
      }
    }
    if (id >= total) return;
  }
}

// dh[i][c] = scale x sum of the slabs of row place[i], in order; zeros for
// rows that took no part. Bound by the slabs' read: one of 8192 x 4096 in 38 us, 5.3
// TB/s with the output.
template <typename T>
__global__ __launch_bounds__(256) void hidden_grad_rows_kernel(
    const float* __restrict__ slabs, const int32_t* __restrict__ rows,
    const int32_t* __restrict__ split_count, int32_t c, int64_t n,
    const float* __restrict__ scale, const int32_t* __restrict__ place, uint16_t* __restrict__ dh) {
  const int64_t quads = n * (c / 4), slab = static_cast<int64_t>(*rows) * c;
  const int count = *split_count;
  const float by = *scale;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < quads;
       e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t i = e / (c / 4);
    const int64_t x = (e - i * (c / 4)) * 4;
    const int32_t m = place[i];
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (m >= 0) {
      for (int s = 0; s < count; ++s) {
        sum += *reinterpret_cast<const f32x4*>(slabs + s * slab + static_cast<int64_t>(m) * c + x);
      }
      sum *= by;
    }
    *reinterpret_cast<uint2*>(dh + i * c + x) =
        make_uint2(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]));
  }
}

// D[c][v] = sum_m h[m][c] dz[m][v]: dW of a piece of the vocabulary. Both operands
// are x-major, twice the LDS reads of the others: 8192 x 32768 x 4096 in 1.80 ms, 1223
// TFLOP/s (a library product of that layout: 1084 to 1136).
template <typename G, typename T>
__global__ __launch_bounds__(gemm::kThreads, 2) void weight_grad_kernel(
    Operand h, Operand dz, const int32_t* __restrict__ count, int32_t columns, int32_t c,
    const float* __restrict__ scale, uint16_t* __restrict__ dw) {
  __shared__ __attribute__((aligned(1024))) char smem[G::kLdsBytes];
  const int rows = *count;
  const int steps = static_cast<int>(round_up(rows, gemm::kStep) / gemm::kStep);
  if (rows <= kFewest) {  // both terms of dz, and the hidden rows in their order
    h.data += kTermRows * h.ld;
    h.rows -= kTermRows;
  }
  const int np = tiles_along(c, G::kBP), nq = tiles_along(columns, G::kBQ), total = np * nq;
  int id = blockIdx.x;
  G tile;
  int tp, tq;
  gemm::tile_of(gemm::xcd_run(id, total), np, nq, tp, tq);
  tile.begin(h, dz, tp * G::kBP, tq * G::kBQ, 0, steps, smem);
  G::arrive();
  const float by = *scale;
  while (true) {
    tile.multiply(smem);
    const int p0 = tp * G::kBP, q0 = tq * G::kBQ;
    id += gridDim.x;
    if (id < total) {
      gemm::tile_of(gemm::xcd_run(id, total), np, nq, tp, tq);
      tile.begin(h, dz, tp * G::kBP, tq * G::kBQ, 0, steps, smem);
      G::arrive();
    }
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
      uint2 out[G::TP];
#pragma unroll
      for (int i = 0; i < G::TP; ++i) {
        const f32x4 y = tile.acc[i][j] * by;
        out[i] = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
      }
      gemm::store_column<G>(dw + static_cast<int64_t>(q0) * c + p0, c, c - p0, columns - q0, j,
                            out);
    }
    if (id >= total) return;
  }
}

// -------------------------------------------------------- row reductions
// A workgroup takes 32 rows, 32 threads a row: joins the tiles' maxima and
// sums to lse[m], and the row's loss, to row_loss (by i) or into the sum of all
// rows. A thread has 8 tiles under way at a time, all of those of 65536 columns.
// In the loss the target logits are taken from the row's maximum, a difference
// that is exact where they are close, and not from lse, whose rounding alone
// (half a unit of 16 in base 2) is 1e-6 of a loss near 1.
// The last workgroup to end adds the workgroups' sums, in their order: a launch
// less than a kernel of its own. Bound by latency: 5 to 7 us up to 1000 rows, 16 us
// for 8192 rows of 256 tiles (17 MB).
__global__ __launch_bounds__(1024) void join_tiles_kernel(const float2* __restrict__ part,
                                                          int32_t vocab, int32_t rest_tile,
                                                          int64_t pad, int32_t k, float scale,
                                                          float temperature, bool mean,
                                                          float* row_loss, float* loss,
                                                          float* partial, Saved s) {
  __shared__ float2 shared[32][33];
  __shared__ float losses[32];
  __shared__ bool last;
  const int q = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int m = blockIdx.x * 32 + q;
  const int count = *s.count;
  if (static_cast<int>(blockIdx.x) * 32 >= count) {
    if (count == 0 && blockIdx.x == 0 && threadIdx.x == 0 && loss != nullptr) *loss = 0.0f;
    return;
  }
  const int cut = *s.cut;
  const int tiles = tiles_along(cut, 256) + tiles_along(vocab - cut, rest_tile);
  float2 all = make_float2(-__builtin_inff(), 0.0f);
  if (m < count) {
    for (int t = slice; t < tiles; t += 256) {
      float2 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        x[u] = t + 32 * u < tiles ? part[(t + 32 * u) * pad + m]
                                  : make_float2(-__builtin_inff(), 0.0f);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) all = joined(all, x[u], scale);
    }
  }
  shared[q][slice] = all;
  __syncthreads();
  // 32 rows by 32 slices, turned: 32 lanes join a row's slices.
  const int row = threadIdx.x >> 5, lane = threadIdx.x & 31;
  all = shared[row][lane];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    all = joined(all, make_float2(__shfl_xor(all.x, off, 64), __shfl_xor(all.y, off, 64)),
                 scale);
  }
  // The lanes' orders differ: the first one's result.
  const float top = __shfl(all.x, threadIdx.x & 32, 64);
  const int mine = blockIdx.x * 32 + row;
  float term = 0.0f;
  int64_t i = 0;
  if (mine < count) {
    i = s.row[mine];
    for (int j = lane; j < k; j += 32) {
      const float p = s.share[i * k + j], z = s.logit[static_cast<int64_t>(mine) * k + j];
      // Absent entries have p = 0; one out of range has z = NaN.
      if (p != 0.0f || z != z) term = fmaf(p, (top - z) * scale, term);
    }
  }
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) term += __shfl_xor(term, off, 64);
  if (lane == 0) {
    float value = 0.0f;
    if (mine < count) {
      const float log_sum = __builtin_amdgcn_logf(all.y);
      // A target out of range makes its row NaN in the backward too.
      s.lse[mine] = term == term ? top + log_sum / scale : term;
      // T twice: T^2 by itself can be beyond fp32.
      value = temperature * (temperature * ((term + log_sum) * kLn2 + s.base[i]));
      if (row_loss != nullptr) row_loss[i] = value;
    }
    losses[row] = value;
  }
  if (loss == nullptr) return;
  __syncthreads();
  const int blocks = (count + 31) / 32;
  if (threadIdx.x < 64) {
    const float sum = wave_sum(threadIdx.x < 32 ? losses[threadIdx.x] : 0.0f);
    if (threadIdx.x == 0) {
      __hip_atomic_store(partial + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(s.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             blocks - 1;
    }
  }
  __syncthreads();
  if (!last || threadIdx.x >= 64) return;
  float sum = 0.0f;
  for (int b = threadIdx.x; b < blocks; b += 64) {
    sum += __hip_atomic_load(partial + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  sum = wave_sum(sum);
  if (threadIdx.x == 0) *loss = mean ? sum / static_cast<float>(count) : sum;
}

// coef[m] multiplies (p - b) of row m in dz, *scale the finished gradients;
// together they are the row's upstream weight x T (/ count for a mean).
// One weight for all rows: all of it is in the scale, so that dz is p - b
// itself, whose target entries (near -1 where p is small) round to 16 bits with
// little error and not all with the same one. Weights of their own: in coef,
// divided by a power of two near the largest one.
// 2^up on top of that keeps fp16's small entries normal numbers: |coef (p - b)|
// is at most 2^14, and 2^-28 of that is the smallest one.
__global__ __launch_bounds__(kScanThreads) void row_coefficients_kernel(
    const float* __restrict__ upstream, bool per_row, bool mean, float temperature, int up,
    Splitting splitting, Pieces pieces, float* __restrict__ coef, float* __restrict__ scale,
    int32_t* __restrict__ splits, int32_t* __restrict__ cuts, Saved s) {
  __shared__ float waves[kScanThreads / 64];
  const int n = *s.count;
  if (threadIdx.x < 64) {
    const int32_t most = wave_splits_of(splitting, n);
    if (threadIdx.x == 0) *splits = most;
  } else if (threadIdx.x < 66) {
    const int which = threadIdx.x - 64;
    cuts[which] = cut_of(pieces.columns[which], n, pieces.steps, pieces.sizes[which]).first;
  }
  const float by = mean ? temperature / static_cast<float>(n > 0 ? n : 1) : temperature;
  const float lift = ldexpf(1.0f, up);
  if (!per_row) {
    for (int m = threadIdx.x; m < n; m += kScanThreads) coef[m] = lift;
    if (threadIdx.x == 0) *scale = *upstream * by / lift;
    return;
  }
  // A weight of 1e30 or more, infinite ones among them, has gradients beyond fp16 by
  // itself; the others' power of two is chosen without it, or they would be as well.
  float top = 0.0f;
  for (int m = threadIdx.x; m < n; m += kScanThreads) {
    const float x = fabsf(upstream[s.row[m]] * by);
    top = x < 1e30f ? fmaxf(top, x) : top;
  }
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScanThreads / 64; ++w) top = fmaxf(top, waves[w]);
  const int exponent = top > 1e-30f ? static_cast<int>(ceilf(__builtin_amdgcn_logf(top))) : 0;
  const float divide = ldexpf(1.0f, up - exponent);
  for (int m = threadIdx.x; m < n; m += kScanThreads) {
    coef[m] = upstream[s.row[m]] * by * divide;
  }
  if (threadIdx.x == 0) *scale = ldexpf(1.0f, exponent - up);
}

// ---------------------------------------------------------------- launches
// How the backward goes through the vocabulary.
struct Plan {
  int32_t columns;  // of a piece, a multiple of kVocabTile
  int32_t pieces;
  int32_t splits;   // of a piece's columns in dz W, for all rows
  Size hidden;
};

// dz of a piece up to kCachedBytes is written and read in the last-level cache;
// beyond, its traffic is partly hidden by the products (4096 x 65536 x 2048 in
// pieces of 128, 256 and 512 MB: 2612, 2700, 2675 us; 8192 x 65536 x 4096, whose
// slabs weigh more: 9784, 9749, 9715 us). A slab is written in each piece and read
// once after it.
constexpr int64_t kCachedBytes = int64_t{192} << 20;
constexpr int64_t kMostBytes = int64_t{512} << 20;
constexpr double kGradBytesPerUs = 20.0e6;
constexpr double kSlabBytesPerUs = 4.0e6;

Splitting splitting_of(Size size, int64_t columns, int64_t c, int64_t room) {
  const TileTime t = time_of(size);
  return {static_cast<int32_t>(columns / gemm::kStep), static_cast<int32_t>((c + t.p - 1) / t.p),
          t.q, t.step_us, t.fixed_us, static_cast<float>(4.0 * c / kSlabBytesPerUs), room};
}

bool few(int64_t n) { return n <= time_of(Size::kFewRows).q; }

double rows_us(int32_t columns, int32_t rows, int32_t steps) {
  const Size size = size_of(columns, rows);
  return size == Size::kSmall ? cut_of(columns, rows, steps, kBothSizes).us
                              : product_us(size, columns, rows, steps);
}

Plan plan_of(int64_t n, int64_t c, int64_t vocab) {
  const int64_t all = round_up(vocab, kVocabTile), pad = round_up(n, kRowPad);
  const int64_t steps_c = c / gemm::kStep, steps_n = (n + gemm::kStep - 1) / gemm::kStep;
  Plan best{};
  double least = 1e300;
  int32_t last = 0;
  for (int64_t pieces = 1; pieces <= all / kVocabTile; ++pieces) {
    Plan p;
    p.columns = static_cast<int32_t>(round_up((all + pieces - 1) / pieces, kVocabTile));
    p.pieces = static_cast<int32_t>((all + p.columns - 1) / p.columns);
    if (p.columns == last) continue;
    last = p.columns;
    const int64_t bytes = pad * p.columns * 2;
    if (bytes > kMostBytes && p.columns > kVocabTile) continue;
    double us = 12.0 + rows_us(p.columns, n, steps_c) +
                cut_of(p.columns, c, steps_n, kBothSizes).us +
                (bytes > kCachedBytes ? 3 * bytes / kGradBytesPerUs : 0.0);
    double hidden = 1e300;
    for (Size size : {Size::kFewRows, Size::kSmall, Size::kLarge}) {
      if ((size == Size::kFewRows) != few(n)) continue;
      const Splitting x = splitting_of(size, p.columns, c, kMostSplits * n);
      const int32_t splits = splits_of(x, n);
      const double t = split_us(x, n, splits);
      if (t >= hidden) continue;
      hidden = t;
      p.splits = splits;
      p.hidden = size;
    }
    us = (us + hidden) * p.pieces;
    if (us < least) {
      least = us;
      best = p;
    }
    if (bytes < kCachedBytes / 8) break;  // smaller pieces only add launches
  }
  return best;
}

// Rows of the slabs: a slab more than all rows want, so that a part of the
// rows, which want more splits, can have them.
int64_t slab_rows(const Plan& plan, int64_t n) {
  return plan.splits == 1 ? n : (plan.splits + 1) * n;
}

struct ForwardWork {
  float2* part;
  float* partial;
};

ForwardWork forward_work(char* p, int64_t n, int64_t vocab, size_t* bytes) {
  const int64_t pad = round_up(n, kRowPad);
  Layout l;
  const int64_t tile = time_of(size_of(vocab, n)).p;
  const size_t part = l.take((vocab + tile - 1) / tile * pad * 8);
  const size_t partial = l.take(pad / 32 * 4);
  *bytes = l.bytes;
  return {reinterpret_cast<float2*>(p + part), reinterpret_cast<float*>(p + partial)};
}

struct BackwardWork {
  float* coef;
  float* scale;
  int32_t* splits;
  int32_t* cuts;
  uint16_t* dz;
  float* slabs;
};

BackwardWork backward_work(char* p, int64_t n, int64_t c, const Plan& plan, bool hidden,
                           size_t* bytes) {
  const int64_t pad = round_up(n, kRowPad);
  Layout l;
  const size_t coef = l.take(pad * 4), scale = l.take(4), splits = l.take(4);
  const size_t cuts = l.take(8);
  const size_t dz = l.take(pad * plan.columns * 2);
  const size_t slabs =
      l.take(hidden ? static_cast<size_t>(slab_rows(plan, n)) * c * 4 : 0);
  *bytes = l.bytes;
  return {reinterpret_cast<float*>(p + coef), reinterpret_cast<float*>(p + scale),
          reinterpret_cast<int32_t*>(p + splits), reinterpret_cast<int32_t*>(p + cuts),
          reinterpret_cast<uint16_t*>(p + dz), reinterpret_cast<float*>(p + slabs)};
}

struct Shape {
  int32_t n, c, vocab, k;
};

int grid_of(int64_t tiles) { return static_cast<int>(std::min<int64_t>(tiles, kCus)); }

// f(tile type) for a size.
template <typename T, Major MA, Major MB, typename F>
void with_tile(Size size, F&& f) {
  switch (size) {
    case Size::kFewRows:
      if constexpr (MB == Major::kK) f(static_cast<FewRowsTile<T, MA, MB>*>(nullptr));
      return;
    case Size::kNarrow64:
      if constexpr (MA == Major::kK && MB == Major::kK) {
        f(static_cast<Narrow64Tile<T, MA, MB>*>(nullptr));
      }
      return;
    case Size::kNarrow128:
      if constexpr (MA == Major::kK && MB == Major::kK) {
        f(static_cast<Narrow128Tile<T, MA, MB>*>(nullptr));
      }
      return;
    case Size::kSmall:
      return f(static_cast<SmallTile<T, MA, MB>*>(nullptr));
    case Size::kLarge:
      return f(static_cast<LargeTile<T, MA, MB>*>(nullptr));
  }
}

// f(tile type, grid) for the sizes that a product over `vocab` columns and
// `rows` rows may be cut into on the device.
template <typename T, typename F>
void for_sizes(int32_t vocab, int32_t rows, int32_t steps, F&& f) {
  const auto launch = [&](Size size) {
    const int grid = grid_of(tiles_of(size, vocab, rows));
    with_tile<T, Major::kK, Major::kK>(size, [&](auto* tile) { f(tile, grid); });
  };
  const Size size = size_of(vocab, rows);
  if (size != Size::kSmall) return launch(size);
  const Sizes sizes = sizes_of(vocab, rows, steps);
  if (sizes.large) launch(Size::kLarge);
  if (sizes.small) launch(Size::kSmall);
}

template <typename T, typename Source>
int run_forward(const Shape& d, const Source& source, const void* hidden, const void* weight,
                float temperature, int reduction, float* loss, const Saved& s,
                const ForwardWork& w, hipStream_t stream) {
  const int64_t pad = round_up(d.n, kRowPad);
  const int steps = d.c / gemm::kStep;
  const float scale = kLog2E / temperature;
  float* row_loss = reduction == FRWKV_REDUCE_NONE ? loss : nullptr;
  const Rows rows{d.n, d.vocab, steps, sizes_of(d.vocab, d.n, steps), row_loss};
  const auto gather = [&](auto* kernel) {
    const int groups = d.k == 1 ? 1 : (d.k + kGather - 1) / kGather;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(pad), groups), dim3(kGatherThreads), 0,
                       stream, static_cast<const uint16_t*>(hidden),
                       static_cast<const uint16_t*>(weight), d.c, d.k, source, rows, s);
  };
  if (d.n <= kOwnNumbers) {
    gather(gather_rows_kernel<T, true, Source>);
  } else {
    hipLaunchKernelGGL((number_rows_kernel<Source>), dim3(1), dim3(kScanThreads), 0, stream,
                       source, rows, s);
    gather(gather_rows_kernel<T, false, Source>);
  }
  const Operand a{static_cast<const uint16_t*>(weight), d.c, d.vocab};
  const Operand b{s.hidden, d.c, static_cast<int32_t>(pad)};
  for_sizes<T>(d.vocab, d.n, steps, [&](auto* tile, int grid) {
    using G = std::remove_pointer_t<decltype(tile)>;
    hipLaunchKernelGGL((lse_tiles_kernel<G, T>), dim3(grid), dim3(gemm::kThreads), 0, stream, a, b,
                       d.c, scale, d.k == 1, w.part, pad, s);
  });
  hipLaunchKernelGGL(join_tiles_kernel, dim3((d.n + 31) / 32), dim3(1024), 0, stream, w.part,
                     d.vocab, time_of(size_of(d.vocab, d.n)).p, pad, d.k, scale,
                     temperature, reduction == FRWKV_REDUCE_MEAN, row_loss,
                     row_loss == nullptr ? loss : nullptr, w.partial, s);
  return check_launch("linear loss forward");
}

template <typename T>
void launch_piece(const Shape& d, const Plan& plan, int piece, const uint16_t* weight,
                  float scale, uint16_t* dh, uint16_t* dw, const Saved& s, const BackwardWork& w,
                  hipStream_t stream) {
  const int64_t pad = round_up(d.n, kRowPad);
  const int first = piece * plan.columns;
  const int columns = std::min(plan.columns, d.vocab - first);
  const int64_t ld = plan.columns;
  const uint16_t* from = weight + static_cast<int64_t>(first) * d.c;
  const Operand wp{from, d.c, columns};
  const Operand h{s.hidden, d.c, static_cast<int32_t>(pad)};
  const Operand dz{w.dz, ld, static_cast<int32_t>(pad)};
  const int32_t* cut = w.cuts + (piece + 1 == plan.pieces);
  for_sizes<T>(columns, d.n, d.c / gemm::kStep, [&](auto* tile, int grid) {
    using G = std::remove_pointer_t<decltype(tile)>;
    hipLaunchKernelGGL((softmax_grad_kernel<G, T>), dim3(grid), dim3(gemm::kThreads), 0, stream,
                       wp, h, cut, d.c, scale, w.coef, w.dz, ld, s);
  });
  const int64_t entries = static_cast<int64_t>(d.n) * d.k;
  hipLaunchKernelGGL((target_grad_kernel<T>), dim3(static_cast<unsigned>((entries + 255) / 256)),
                     dim3(256), 0, stream, d.k, first, columns, scale, w.coef, w.dz, ld, s);
  if (dh != nullptr) {
    const int steps = static_cast<int>(round_up(columns, gemm::kStep) / gemm::kStep);
    with_tile<T, Major::kX, Major::kK>(plan.hidden, [&](auto* tile) {
      using G = std::remove_pointer_t<decltype(tile)>;
      hipLaunchKernelGGL((hidden_grad_kernel<G, T>), dim3(kCus), dim3(gemm::kThreads), 0, stream,
                         wp, dz, s.count, w.splits, steps, plan.columns / gemm::kStep,
                         (d.c + G::kBP - 1) / G::kBP, piece > 0, d.c, w.slabs);
    });
  }
  if (dw != nullptr) {
    // Masks shorten its tiles and leave their number.
    const Cut cut = cut_of(columns, d.c, tiles_along(d.n, gemm::kStep), kBothSizes);
    const auto launch = [&](Size size, int32_t at, int32_t part) {
      if (part == 0) return;
      const Operand b{w.dz + at, ld, static_cast<int32_t>(pad)};
      with_tile<T, Major::kX, Major::kX>(size, [&](auto* tile) {
        using G = std::remove_pointer_t<decltype(tile)>;
        hipLaunchKernelGGL((weight_grad_kernel<G, T>), dim3(grid_of(tiles_of(size, d.c, part))),
                           dim3(gemm::kThreads), 0, stream, h, b, s.count,
                           part, d.c, w.scale, dw + static_cast<int64_t>(first + at) * d.c);
      });
    };
    launch(Size::kLarge, 0, cut.first);
    launch(Size::kSmall, cut.first, columns - cut.first);
  }
}

template <typename T>
int run_backward(const Shape& d, const void* weight, const float* upstream, bool per_row,
                 bool mean, float temperature, void* dh, void* dw, const Saved& s,
                 const Plan& plan, const BackwardWork& w, hipStream_t stream) {
  const float scale = kLog2E / temperature;
  const int steps = d.c / gemm::kStep, last = d.vocab - (plan.pieces - 1) * plan.columns;
  const Pieces pieces{{plan.columns, last},
                      {sizes_of(plan.columns, d.n, steps), sizes_of(last, d.n, steps)},
                      steps};
  hipLaunchKernelGGL(row_coefficients_kernel, dim3(1), dim3(kScanThreads), 0, stream, upstream,
                     per_row, mean, temperature, __is_same(T, F16) ? 14 : 0,
                     splitting_of(plan.hidden, plan.columns, d.c, slab_rows(plan, d.n)),
                     pieces,
                     w.coef, w.scale, w.splits, w.cuts, s);
  for (int p = 0; p < plan.pieces; ++p) {
    launch_piece<T>(d, plan, p, static_cast<const uint16_t*>(weight), scale,
                    static_cast<uint16_t*>(dh), static_cast<uint16_t*>(dw), s, w, stream);
  }
  if (dh != nullptr) {
    const int64_t quads = static_cast<int64_t>(d.n) * (d.c / 4);
    const int64_t blocks = std::min<int64_t>((quads + 255) / 256, 8192);
    hipLaunchKernelGGL((hidden_grad_rows_kernel<T>), dim3(static_cast<unsigned>(blocks)),
                       dim3(256), 0, stream, w.slabs, s.count, w.splits, d.c, d.n,
                       w.scale, s.place, static_cast<uint16_t*>(dh));
  }
  return check_launch("linear loss backward");
}

constexpr int64_t kMostRows = int64_t{1} << 23;  // a launch: less than 2^32 threads, 256 a row
constexpr int64_t kMostChannels = 65536;
constexpr int64_t kMostVocab = int64_t{1} << 28;
constexpr int64_t kMostTargets = 1024;

bool within(int64_t x, int64_t most) { return x > 0 && x <= most; }

// What one call takes of rows, channels, vocabulary and targets a row together.
bool sizes_fit(int64_t n, int64_t c, int64_t vocab, int64_t k) {
  if (!within(n, kMostRows) || !within(c, kMostChannels) || c % gemm::kStep != 0 ||
      !within(vocab, kMostVocab) || !within(k, kMostTargets)) {
    return false;
  }
  const int64_t tile = time_of(Size::kSmall).p;  // of the most tiles a product is cut into
  const int64_t tiles = round_up(vocab, tile) / tile * (round_up(n, tile) / tile);
  return tiles < (int64_t{1} << 30) && n * k < (int64_t{1} << 31);
}

int check_shape(const char* what, int io_dtype, int64_t n, int64_t c, int64_t vocab, int64_t k) {
  if (io_dtype != FRWKV_DTYPE_F16 && io_dtype != FRWKV_DTYPE_BF16) {
    return set_error(FRWKV_ERR_UNSUPPORTED, "%s: io dtype must be float16 or bfloat16", what);
  }
  if (!within(n, kMostRows)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: rows must be in [1, 2^23], got %lld", what,
                     static_cast<long long>(n));
  }
  if (!within(c, kMostChannels) || c % gemm::kStep != 0) {
    return set_error(FRWKV_ERR_UNSUPPORTED,
                     "%s: channels must be a multiple of 64, at most 65536, got %lld", what,
                     static_cast<long long>(c));
  }
  if (!within(vocab, kMostVocab)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: vocabulary must be in [1, 2^28], got %lld",
                     what, static_cast<long long>(vocab));
  }
  if (!within(k, kMostTargets)) {
    return set_error(FRWKV_ERR_UNSUPPORTED,
                     "%s: targets of a row must be in [1, 1024], got %lld", what,
                     static_cast<long long>(k));
  }
  if (!sizes_fit(n, c, vocab, k)) {
    return set_error(FRWKV_ERR_UNSUPPORTED,
                     "%s: rows x vocabulary or rows x targets too large for one call", what);
  }
  return FRWKV_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

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

int check_reduction(const char* what, int reduction) {
  if (reduction != FRWKV_REDUCE_NONE && reduction != FRWKV_REDUCE_MEAN &&
      reduction != FRWKV_REDUCE_SUM) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: unknown reduction %d", what, reduction);
  }
  return FRWKV_OK;
}

int check_temperature(const char* what, float t) {
  if (!(t > 0.0f) || t > 1e30f || t < 1e-30f) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: temperature must be positive and finite",
                     what);
  }
  return FRWKV_OK;
}

template <typename Source>
int forward(int io_dtype, const Shape& d, const Source& source, const void* hidden,
            const void* weight, float temperature, int reduction, float* loss, const Saved& s,
            void* workspace, hipStream_t stream) {
  size_t need = 0;
  const ForwardWork w = forward_work(static_cast<char*>(workspace), d.n, d.vocab, &need);
  return io_dtype == FRWKV_DTYPE_F16
             ? run_forward<F16>(d, source, hidden, weight, temperature, reduction, loss, s, w,
                                stream)
             : run_forward<Bf16>(d, source, hidden, weight, temperature, reduction, loss, s, w,
                                 stream);
}

// The checks that both forwards share, and the layout of what they leave.
int begin_forward(const char* what, int io_dtype, int64_t n, int64_t c, int64_t vocab, int64_t k,
                  const void* hidden, const void* weight, int reduction, const float* loss,
                  void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes,
                  Saved* s) {
  if (!hidden || !weight || !loss) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  }
  int rc = check_shape(what, io_dtype, n, c, vocab, k);
  if (rc == FRWKV_OK) rc = check_reduction(what, reduction);
  if (rc != FRWKV_OK) return rc;
  if (!aligned16(hidden) || !aligned16(weight)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: hidden and weight must be 16-byte aligned", what);
  }
  size_t need = 0;
  *s = saved_of(static_cast<char*>(saved), n, c, k, &need);
  rc = check_memory(what, "saved", saved, saved_bytes, need);
  if (rc != FRWKV_OK) return rc;
  (void)forward_work(nullptr, n, vocab, &need);
  return check_memory(what, "workspace", workspace, workspace_bytes, need);
}

}  // namespace
}  // namespace frwkv

extern "C" {

size_t frwkv_linear_loss_saved_bytes(int64_t rows, int64_t channels, int64_t top) {
  using namespace frwkv;
  if (!sizes_fit(rows, channels, 1, top)) return 0;
  size_t bytes = 0;
  (void)frwkv::saved_of(nullptr, rows, channels, top, &bytes);
  return bytes;
}

size_t frwkv_linear_loss_forward_workspace_bytes(int64_t rows, int64_t vocab) {
  using namespace frwkv;
  if (!sizes_fit(rows, gemm::kStep, vocab, 1)) return 0;
  size_t bytes = 0;
  (void)frwkv::forward_work(nullptr, rows, vocab, &bytes);
  return bytes;
}

size_t frwkv_linear_loss_backward_workspace_bytes(int64_t rows, int64_t channels, int64_t vocab,
                                                  int want_grad_hidden) {
  using namespace frwkv;
  if (!sizes_fit(rows, channels, vocab, 1)) return 0;
  size_t bytes = 0;
  (void)frwkv::backward_work(nullptr, rows, channels, frwkv::plan_of(rows, channels, vocab),
                             want_grad_hidden != 0, &bytes);
  return bytes;
}

int frwkv_linear_loss_backward_plan(int64_t rows, int64_t channels, int64_t vocab,
                                    int32_t* columns, int32_t* pieces, int32_t* splits,
                                    int32_t* tile_rows) {
  using namespace frwkv;
  const char* what = "frwkv_linear_loss_backward_plan";
  if (!columns || !pieces || !splits || !tile_rows) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  }
  const int rc = check_shape(what, FRWKV_DTYPE_BF16, rows, channels, vocab, 1);
  if (rc != FRWKV_OK) return rc;
  const Plan plan = plan_of(rows, channels, vocab);
  *columns = plan.columns;
  *pieces = plan.pieces;
  *splits = plan.splits;
  *tile_rows = time_of(plan.hidden).q;
  return FRWKV_OK;
}

int frwkv_linear_cross_entropy_forward(int io_dtype, int64_t rows, int64_t channels,
                                       int64_t vocab, const void* hidden, const void* weight,
                                       int target_bytes, const void* targets,
                                       int64_t ignore_index, int reduction, float* loss,
                                       void* saved, size_t saved_bytes, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_linear_cross_entropy_forward";
  Saved s;
  const int rc = begin_forward(what, io_dtype, rows, channels, vocab, 1, hidden, weight,
                               reduction, loss, saved, saved_bytes, workspace, workspace_bytes,
                               &s);
  if (rc != FRWKV_OK) return rc;
  if (!targets || (target_bytes != 4 && target_bytes != 8)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: targets must be int32 or int64", what);
  }
  const hipStream_t q = static_cast<hipStream_t>(stream);
  const int32_t n = static_cast<int32_t>(rows), v = static_cast<int32_t>(vocab);
  const Shape d{n, static_cast<int32_t>(channels), v, 1};
  if (target_bytes == 8) {
    const Labels<int64_t> labels{static_cast<const int64_t*>(targets), ignore_index};
    return forward(io_dtype, d, labels, hidden, weight, 1.0f, reduction, loss, s, workspace, q);
  }
  const Labels<int32_t> labels{static_cast<const int32_t*>(targets), ignore_index};
  return forward(io_dtype, d, labels, hidden, weight, 1.0f, reduction, loss, s, workspace, q);
}

int frwkv_linear_topk_distillation_forward(
    int io_dtype, int64_t rows, int64_t channels, int64_t vocab, int64_t top, const void* hidden,
    const void* weight, int teacher_dtype, const void* teacher_logits, int index_bytes,
    const void* teacher_indices, float temperature, int reduction, float* loss, void* saved,
    size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_linear_topk_distillation_forward";
  Saved s;
  int rc = begin_forward(what, io_dtype, rows, channels, vocab, top, hidden, weight, reduction,
                         loss, saved, saved_bytes, workspace, workspace_bytes, &s);
  if (rc == FRWKV_OK) rc = check_temperature(what, temperature);
  if (rc != FRWKV_OK) return rc;
  if (!teacher_logits || (teacher_dtype != FRWKV_DTYPE_F32 && teacher_dtype != FRWKV_DTYPE_F16 &&
                          teacher_dtype != FRWKV_DTYPE_BF16)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: teacher_logits must be float32, float16 or bfloat16", what);
  }
  if (!teacher_indices || (index_bytes != 4 && index_bytes != 8)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: teacher_indices must be int32 or int64",
                     what);
  }
  const hipStream_t q = static_cast<hipStream_t>(stream);
  const int32_t n = static_cast<int32_t>(rows), k = static_cast<int32_t>(top);
  const int32_t v = static_cast<int32_t>(vocab);
  const auto launch = [&](auto io, auto index) {
    using T = decltype(io);
    using I = decltype(index);
    using S = typename IoTraits<T>::storage;
    hipLaunchKernelGGL((teacher_targets_kernel<T, I>), dim3((n + 3) / 4), dim3(256),
                       static_cast<size_t>(round_up(k, 4)) * 32, q,
                       static_cast<const S*>(teacher_logits),
                       static_cast<const I*>(teacher_indices), n, k, v, 1.0f / temperature, s);
  };
  const auto with_index = [&](auto io) {
    if (index_bytes == 8) {
      launch(io, int64_t{});
    } else {
      launch(io, int32_t{});
    }
  };
  if (teacher_dtype == FRWKV_DTYPE_F32) {
    with_index(float{});
  } else if (teacher_dtype == FRWKV_DTYPE_F16) {
    with_index(F16{});
  } else {
    with_index(Bf16{});
  }
  return forward(io_dtype, Shape{n, static_cast<int32_t>(channels), v, k}, Teacher{s.part},
                 hidden, weight, temperature, reduction, loss, s, workspace, q);
}

int frwkv_linear_loss_backward(int io_dtype, int64_t rows, int64_t channels, int64_t vocab,
                               int64_t top, const void* weight, float temperature, int reduction,
                               const float* grad_loss, const void* saved, size_t saved_bytes,
                               void* grad_hidden, void* grad_weight, void* workspace,
                               size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_linear_loss_backward";
  if (!weight || !grad_loss) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  }
  int rc = check_shape(what, io_dtype, rows, channels, vocab, top);
  if (rc == FRWKV_OK) rc = check_reduction(what, reduction);
  if (rc == FRWKV_OK) rc = check_temperature(what, temperature);
  if (rc != FRWKV_OK) return rc;
  if (!aligned16(weight) || !aligned16(grad_hidden) || !aligned16(grad_weight)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: weight and gradients must be 16-byte aligned", what);
  }
  size_t need = 0;
  // The forward's buffer is only read here.
  const Saved s = saved_of(const_cast<char*>(static_cast<const char*>(saved)), rows, channels,
                           top, &need);
  rc = check_memory(what, "saved", saved, saved_bytes, need);
  if (rc != FRWKV_OK) return rc;
  const Plan plan = plan_of(rows, channels, vocab);
  const BackwardWork w = backward_work(static_cast<char*>(workspace), rows, channels, plan,
                                       grad_hidden != nullptr, &need);
  rc = check_memory(what, "workspace", workspace, workspace_bytes, need);
  if (rc != FRWKV_OK) return rc;
  if (!grad_hidden && !grad_weight) return FRWKV_OK;
  const bool mean = reduction == FRWKV_REDUCE_MEAN, per_row = reduction == FRWKV_REDUCE_NONE;
  const Shape d{static_cast<int32_t>(rows), static_cast<int32_t>(channels),
                static_cast<int32_t>(vocab), static_cast<int32_t>(top)};
  const hipStream_t q = static_cast<hipStream_t>(stream);
  return io_dtype == FRWKV_DTYPE_F16
             ? run_backward<F16>(d, weight, grad_loss, per_row, mean, temperature, grad_hidden,
                                 grad_weight, s, plan, w, q)
             : run_backward<Bf16>(d, weight, grad_loss, per_row, mean, temperature, grad_hidden,
                                  grad_weight, s, plan, w, q);
}

}  // extern "C"
