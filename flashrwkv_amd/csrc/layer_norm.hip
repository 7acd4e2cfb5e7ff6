// Layer norm over the channels of [rows, C] with the residual add in front of
// it, forward and backward, fp32 / fp16 / bf16.
//
//   s = x + residual, rounded to the io type (the stream as it is kept; s = x
//   without a residual), mean and var (biased) over C, rstd = 1/sqrt(var+eps)
//   y = (s - mean) rstd weight + bias
// and for upstream dy (and ds of the stream), xhat = (s - mean) rstd,
// g = dy weight:
//   dx = rstd (g - mean_C(g) - xhat mean_C(g xhat)) + ds   (= dresidual)
//   dweight = sum_rows dy xhat,  dbias = sum_rows dy.
//
// HBM-bound: x [, residual] -> y [, s] forward, dy, s [, ds] -> dx backward.
// A row is held in registers by 1, 4 or 16 waves, 8 or 16 elements a thread (C
// up to 16384), so each tensor passes once and the variance is taken about the
// mean. The backward's workgroups walk over rows and keep the
// weight's and bias' sums of their 16 columns a thread in registers; one row
// of 2 C partial sums a workgroup goes to memory and a second kernel adds
// those in order, so the result does not depend on timing.
// Measured at 16384 x 4096 bf16: forward with a residual 91 us (5.9 TB/s), backward with
// a gradient of the stream 115 us (4.7 TB/s), the columns' sums 5 us; a copy of 1 GiB
// reaches 5.1 TB/s. fp32 16384 x 4096: forward with a residual 204 us, backward with a
// gradient of the stream 206 us (5.2 TB/s both). One row: 5 us, latency of its two
// reductions and the launch. 2311 x 1000 fp32: 8, 11 and 4 us where the bytes take 7 in
// all, three launches of one row a wave, which are latency as well.
// The backward with 16 elements a thread, two workgroups a CU at 128 registers, keeps
// 5 values in scratch for fp32 (C 2049 to 4096), up to 13 for unaligned rows.
// Unaligned rows of 4097 channels, 16 waves of which half hold nothing, run at half the
// rate (16384 x 4097 bf16: 164 and 203 us).
#include <algorithm>
#include <type_traits>

#include "capi_internal.h"
#include "wkv7_device.h"

namespace frwkv {
namespace {

constexpr int kVec = 8;          // consecutive elements a thread
constexpr int kMaxBlocks = 512;  // of the backward: two a CU
constexpr int kMaxChannels = 16384;

template <typename T>
using Store = typename IoTraits<T>::storage;

// Eight consecutive elements as they lie in memory. Aligned rows (16 bytes, C a
// multiple of 8) are read and written in 16-byte pieces; others in what the
// hardware takes at any address, with a last piece of fewer than eight.
template <typename T, bool kAligned>
struct Piece {
  static constexpr int kWords = kVec * IoTraits<T>::kBytes / 16;
  uint4 word[kWords];
  // left: elements of the row from p on (1 or more).
  __device__ __forceinline__ void load(const Store<T>* p, int left) {
    if (kAligned) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) word[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if (left >= kVec) {
      __builtin_memcpy(word, p, sizeof(word));
    } else {
      Store<T> x[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] = e < left ? p[e] : Store<T>(0);
      __builtin_memcpy(word, x, sizeof(word));
    }
  }
  __device__ __forceinline__ void store(Store<T>* p, int left) const {
    if (kAligned) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = word[i];
    } else if (left >= kVec) {
      __builtin_memcpy(p, word, sizeof(word));
    } else {
      Store<T> x[kVec];
      __builtin_memcpy(x, word, sizeof(word));
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (e < left) p[e] = x[e];
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) word[i] = make_uint4(0, 0, 0, 0);
  }
  // Conversions before and after this one are not one value kept in registers.
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      asm volatile("" : "+v"(word[i].x), "+v"(word[i].y), "+v"(word[i].z), "+v"(word[i].w));
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (__is_same(T, float)) {
      const uint4 q = word[e / 4];
      return __uint_as_float(e % 4 == 0 ? q.x : e % 4 == 1 ? q.y : e % 4 == 2 ? q.z : q.w);
    } else {
      const uint32_t d = e / 2 == 0 ? word[0].x : e / 2 == 1 ? word[0].y
                         : e / 2 == 2 ? word[0].z : word[0].w;
      return to_f32<T>(static_cast<uint16_t>(e % 2 ? d >> 16 : d & 0xffffu));
    }
  }
  __device__ __forceinline__ void set(const float* x) {
    if constexpr (__is_same(T, float)) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        word[i] = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]),
                             __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3]));
      }
    } else {
      word[0] = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                           pack2<T>(x[6], x[7]));
    }
  }
};

// Whether element e of the piece at col < c belongs to the row.
template <bool kAligned>
__device__ __forceinline__ bool inside(int col, int e, int c) {
  return kAligned || col + e < c;
}

// Sum over the kWaves waves of a row; red holds kWaves floats of the row's
// own. Calls alternate between two such arrays, so that one barrier does.
template <int kWaves>
__device__ __forceinline__ float row_sum(float x, float* red, int wave) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
  if constexpr (kWaves > 1) {
    if ((threadIdx.x & 63) == 0) red[wave] = x;
    __syncthreads();
    x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x += red[w];
  }
  return x;
}

template <int kWaves>
constexpr int forward_threads() { return kWaves == 16 ? 1024 : 256; }
template <int kWaves>
constexpr int backward_threads() { return kWaves == 16 ? 1024 : 512; }

template <typename T, bool kAligned, int kWaves, int kE>
__global__ __launch_bounds__(forward_threads<kWaves>()) void layer_norm_forward_kernel(
    const Store<T>* __restrict__ x, const Store<T>* __restrict__ residual,
    const Store<T>* __restrict__ weight, const Store<T>* __restrict__ bias,
    Store<T>* __restrict__ y, Store<T>* __restrict__ stream, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, int64_t rows, int32_t c, float eps) {
  constexpr int kGroups = forward_threads<kWaves>() / (64 * kWaves);
  constexpr int kRow = 64 * kWaves;
  constexpr int kPieces = kE / kVec;
  __shared__ float red[2][kGroups][kWaves];
  const int group = threadIdx.x / kRow, t = threadIdx.x % kRow, wave = t >> 6;
  const float inv_c = 1.0f / static_cast<float>(c);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool here = row < rows;
    const int64_t at = (here ? row : 0) * c;
    float s[kE];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      Piece<T, kAligned> a, r;
      a.zero();
      r.zero();
      if (here && col < c) {
        a.load(x + at + col, c - col);
        if (residual != nullptr) r.load(residual + at + col, c - col);
      }
      float* own = s + j * kVec;
#pragma unroll
      for (int e = 0; e < kVec; ++e) own[e] = a.get(e);
      if (residual != nullptr) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) own[e] += r.get(e);
        a.set(own);
        if (here && col < c) a.store(stream + at + col, c - col);
#pragma unroll
        for (int e = 0; e < kVec; ++e) own[e] = a.get(e);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += own[e];
    }
    const float mean = row_sum<kWaves>(sum, red[0][group], wave) * inv_c;
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      if (col < c) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float d = s[j * kVec + e] - mean;
          s[j * kVec + e] = d;
          if (inside<kAligned>(col, e, c)) sq = fmaf(d, d, sq);
        }
      }
    }
    const float var = row_sum<kWaves>(sq, red[1][group], wave) * inv_c;
    const float rstd = 1.0f / __builtin_sqrtf(var + eps);
    if (!here) continue;
    if (mean_out != nullptr && t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      if (col < c) {
        Piece<T, kAligned> w, b, o;
        w.load(weight + col, c - col);
        b.load(bias + col, c - col);
        float out[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          out[e] = fmaf(s[j * kVec + e] * rstd, w.get(e), b.get(e));
        }
        o.set(out);
        o.store(y + at + col, c - col);
      }
    }
  }
}

// What the backward reads of a row, as it lies in memory (zeros where there is
// nothing).
template <typename T, bool kAligned, int kPieces, int kRow>
struct Row {
  Piece<T, kAligned> x[kPieces], up[kPieces], add[kPieces];
  float mu, rs;
  __device__ __forceinline__ void load(const Store<T>* s, const Store<T>* dy, const Store<T>* ds,
                                       const float* mean, const float* rstd, int64_t row,
                                       int64_t rows, int32_t c, int t) {
    const bool here = row < rows;
    const int64_t at = row * c;
    mu = here ? mean[row] : 0.0f;
    rs = here ? rstd[row] : 0.0f;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      x[j].zero();
      up[j].zero();
      add[j].zero();
      if (here && col < c) {
        x[j].load(s + at + col, c - col);
        up[j].load(dy + at + col, c - col);
        if (ds != nullptr) add[j].load(ds + at + col, c - col);
      }
    }
  }
};

// partial[block][0][c] = sum over the block's rows of dy xhat, [1][c] of dy.
// With 8 elements a thread the next row's loads are under way while a row is
// summed up and written; with 16 there are no registers for that, and the two
// workgroups of a CU cover for each other.
template <typename T, bool kAligned, int kWaves, int kE>
__global__ __launch_bounds__(backward_threads<kWaves>(), 4) void layer_norm_backward_kernel(
    const Store<T>* __restrict__ dy, const Store<T>* __restrict__ s,
    const Store<T>* __restrict__ ds, const Store<T>* __restrict__ weight,
    const float* __restrict__ mean, const float* __restrict__ rstd, Store<T>* __restrict__ dx,
    float* __restrict__ partial, int64_t rows, int32_t c) {
  constexpr int kThreads = backward_threads<kWaves>();
  constexpr int kGroups = kThreads / (64 * kWaves);
  constexpr int kRow = 64 * kWaves;
  constexpr int kPieces = kE / kVec;
  __shared__ float red[2][2][kGroups][kWaves];
  __shared__ float columns[kGroups > 1 ? kThreads * kE : 1];
  const int group = threadIdx.x / kRow, t = threadIdx.x % kRow, wave = t >> 6;
  const float inv_c = 1.0f / static_cast<float>(c);
  Piece<T, kAligned> w[kPieces];
  float pw[kE], pb[kE];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int col = (j * kRow + t) * kVec;
    w[j].zero();
    if (col < c) w[j].load(weight + col, c - col);
#pragma unroll
    for (int e = 0; e < kVec; ++e) pw[j * kVec + e] = pb[j * kVec + e] = 0.0f;
  }
  int side = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  constexpr bool kAhead = kE == 8;
  Row<T, kAligned, kPieces, kRow> now, next;
  if constexpr (kAhead) {
    next.load(s, dy, ds, mean, rstd, static_cast<int64_t>(blockIdx.x) * kGroups + group, rows, c,
              t);
  }
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < rows; first += step) {
    const int64_t row = first + group;
    if constexpr (kAhead) {
      now = next;
      next.load(s, dy, ds, mean, rstd, row + step, rows, c, t);
    } else {
      now.load(s, dy, ds, mean, rstd, row, rows, c, t);
    }
    float xh[kE];
    float sg = 0.0f, sgx = 0.0f;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      w[j].again();
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int k = j * kVec + e;
        const float u = now.up[j].get(e), g = u * w[j].get(e);
        xh[k] = col < c && inside<kAligned>(col, e, c) ? (now.x[j].get(e) - now.mu) * now.rs : 0.0f;
        pw[k] = fmaf(u, xh[k], pw[k]);
        pb[k] += u;
        sg += g;
        sgx = fmaf(g, xh[k], sgx);
      }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      sg += __shfl_xor(sg, off, 64);
      sgx += __shfl_xor(sgx, off, 64);
    }
    if constexpr (kWaves > 1) {
      // Two sets in turn: one barrier a row.
      if ((threadIdx.x & 63) == 0) {
        red[side][0][group][wave] = sg;
        red[side][1][group][wave] = sgx;
      }
      __syncthreads();
      sg = sgx = 0.0f;
#pragma unroll
      for (int q = 0; q < kWaves; ++q) {
        sg += red[side][0][group][q];
        sgx += red[side][1][group][q];
      }
      side ^= 1;
    }
    const float mg = sg * inv_c, mgx = sgx * inv_c;
    if (row >= rows) continue;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      now.up[j].again();
      w[j].again();
      if (col < c) {
        float o[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float g = now.up[j].get(e) * w[j].get(e);
          o[e] = fmaf(now.rs, g - mg - xh[j * kVec + e] * mgx, now.add[j].get(e));
        }
        Piece<T, kAligned> out;
        out.set(o);
        out.store(dx + row * c + col, c - col);
      }
    }
  }
  // The block's groups are added in order.
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* mine = which == 0 ? pw : pb;
    if constexpr (kGroups > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kE; ++e) columns[(group * kE + e) * kRow + t] = mine[e];
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int q = 1; q < kGroups; ++q) {
#pragma unroll
          for (int e = 0; e < kE; ++e) mine[e] += columns[(q * kE + e) * kRow + t];
        }
      }
    }
    if (group == 0) {
      float* to = partial + (static_cast<int64_t>(blockIdx.x) * 2 + which) * c;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int col = (j * kRow + t) * kVec;
        Piece<float, kAligned> out;
        out.set(mine + j * kVec);
        if (col < c) out.store(to + col, c - col);
      }
    }
  }
}

// Sum of the blocks' partial sums, in a fixed order: 32 columns a workgroup,
// 32 runs of up to 16 blocks, all of a run's loads under way together.
constexpr int kRuns = 32;
constexpr int kRunBlocks = kMaxBlocks / kRuns;

template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_columns_kernel(
    const float* __restrict__ partial, int32_t blocks, int32_t c, Store<T>* __restrict__ dweight,
    Store<T>* __restrict__ dbias) {
  __shared__ float runs[kRuns][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float x[kRunBlocks];
#pragma unroll
  for (int u = 0; u < kRunBlocks; ++u) {
    const int b = run + kRuns * u;
    x[u] = col < c && b < blocks
               ? partial[(static_cast<int64_t>(b) * 2 + blockIdx.y) * c + col] : 0.0f;
  }
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < kRunBlocks; ++u) sum += x[u];
  runs[run][lane] = sum;
  __syncthreads();
  // Turned: the 32 lanes of a half wave add a column's runs.
  sum = runs[lane][run];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) sum += __shfl_xor(sum, off, 64);
  const int mine = blockIdx.x * 32 + run;
  if (lane == 0 && mine < c) (blockIdx.y == 0 ? dweight : dbias)[mine] = from_f32<T>(sum);
}

// Waves and elements a thread that hold a row: the fewest that do, since lanes
// without elements cost time (16384 x 2560 in bf16, backward: 4 waves with 16
// elements 69 us, 8 with 8 elements 75; 65536 x 768: one wave with 16 elements
// 84, 4 with 8 elements 121; 16384 x 2048: 4 waves with 8 elements 48, with 16 51).
int waves_of(int64_t c) { return c <= 1024 ? 1 : c <= 4096 ? 4 : 16; }
int elements_of(int64_t c) { return c <= waves_of(c) * 64 * kVec ? kVec : 2 * kVec; }

int64_t backward_blocks(int64_t rows, int64_t c) {
  const int waves = waves_of(c);
  const int64_t groups = waves == 16 ? 1 : 8 / waves;
  return std::min<int64_t>((rows + groups - 1) / groups, waves == 16 ? kMaxBlocks / 2 : kMaxBlocks);
}

template <int kValue>
using Int = std::integral_constant<int, kValue>;

// f(aligned, waves a row, elements a thread)
template <typename F>
void with_shape(int64_t c, bool aligned, F&& f) {
  const int waves = waves_of(c), elements = elements_of(c);
  const auto with_waves = [&](auto is_aligned) {
    if (waves == 1 && elements == 8) f(is_aligned, Int<1>{}, Int<8>{});
    if (waves == 1 && elements == 16) f(is_aligned, Int<1>{}, Int<16>{});
    if (waves == 4 && elements == 8) f(is_aligned, Int<4>{}, Int<8>{});
    if (waves == 4 && elements == 16) f(is_aligned, Int<4>{}, Int<16>{});
    if (waves == 16 && elements == 8) f(is_aligned, Int<16>{}, Int<8>{});
    if (waves == 16 && elements == 16) f(is_aligned, Int<16>{}, Int<16>{});
  };
  if (aligned) {
    with_waves(Int<1>{});
  } else {
    with_waves(Int<0>{});
  }
}

template <typename F>
void with_type(int io_dtype, F&& f) {
  if (io_dtype == FRWKV_DTYPE_F32) f(float{});
  if (io_dtype == FRWKV_DTYPE_F16) f(F16{});
  if (io_dtype == FRWKV_DTYPE_BF16) f(Bf16{});
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <size_t N>
bool aligned_call(int64_t c, const void* const (&pointers)[N]) {
  for (const void* p : pointers) {
    if (!aligned16(p)) return false;
  }
  return c % kVec == 0;
}

int check_shape(const char* what, int io_dtype, int64_t rows, int64_t c) {
  if (io_dtype != FRWKV_DTYPE_F32 && io_dtype != FRWKV_DTYPE_F16 &&
      io_dtype != FRWKV_DTYPE_BF16) {
    return set_error(FRWKV_ERR_UNSUPPORTED, "%s: io dtype must be float32, float16 or bfloat16",
                     what);
  }
  if (rows <= 0) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: rows must be positive, got %lld", what,
                     static_cast<long long>(rows));
  }
  if (c <= 0 || c > kMaxChannels) {
    return set_error(FRWKV_ERR_UNSUPPORTED, "%s: channels must be in [1, 16384], got %lld", what,
                     static_cast<long long>(c));
  }
  return FRWKV_OK;
}

}  // namespace
}  // namespace frwkv

extern "C" {

int frwkv_layer_norm_forward(int io_dtype, int64_t rows, int64_t channels, const void* x,
                             const void* residual, const void* weight, const void* bias,
                             float eps, void* y, void* stream_out, float* mean, float* rstd,
                             void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_layer_norm_forward";
  if (!x || !weight || !bias || !y) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  }
  if ((residual == nullptr) != (stream_out == nullptr) || (mean == nullptr) != (rstd == nullptr)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: residual comes with stream_out, mean with rstd", what);
  }
  const int rc = check_shape(what, io_dtype, rows, channels);
  if (rc != FRWKV_OK) return rc;
  if (!(eps >= 0.0f) || eps > 1e30f) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", what);
  }
  const void* const all[] = {x, residual, weight, bias, y, stream_out};
  const int32_t c = static_cast<int32_t>(channels);
  with_type(io_dtype, [&](auto io) {
    using T = decltype(io);
    using S = Store<T>;
    with_shape(c, aligned_call(c, all), [&](auto aligned, auto waves, auto elements) {
      constexpr bool kAligned = decltype(aligned)::value != 0;
      constexpr int kWaves = decltype(waves)::value, kE = decltype(elements)::value;
      constexpr int kThreads = forward_threads<kWaves>();
      constexpr int kGroups = kThreads / (64 * kWaves);
      const int64_t blocks = std::min<int64_t>((rows + kGroups - 1) / kGroups, 1 << 20);
      hipLaunchKernelGGL((layer_norm_forward_kernel<T, kAligned, kWaves, kE>),
                         dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                         static_cast<hipStream_t>(stream), static_cast<const S*>(x),
                         static_cast<const S*>(residual), static_cast<const S*>(weight),
                         static_cast<const S*>(bias), static_cast<S*>(y),
                         static_cast<S*>(stream_out), mean, rstd, rows, c, eps);
    });
  });
  return check_launch("layer_norm_forward_kernel");
}

size_t frwkv_layer_norm_backward_workspace_bytes(int64_t rows, int64_t channels) {
  if (rows <= 0 || channels <= 0) return 0;
  return static_cast<size_t>(frwkv::backward_blocks(rows, channels)) * 2 * channels *
         sizeof(float);
}

int frwkv_layer_norm_backward(int io_dtype, int64_t rows, int64_t channels, const void* grad_y,
                              const void* normed, const void* grad_stream, const void* weight,
                              const float* mean, const float* rstd, void* grad_x,
                              void* grad_weight, void* grad_bias, void* workspace,
                              size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_layer_norm_backward";
  if (!grad_y || !normed || !weight || !mean || !rstd || !grad_x || !grad_weight || !grad_bias ||
      !workspace) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  }
  const int rc = check_shape(what, io_dtype, rows, channels);
  if (rc != FRWKV_OK) return rc;
  const size_t need = frwkv_layer_norm_backward_workspace_bytes(rows, channels);
  if (workspace_bytes < need || !aligned16(workspace)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: workspace of %zu bytes given, %zu needed (16-byte aligned)", what,
                     workspace_bytes, need);
  }
  const void* const all[] = {grad_y, normed, grad_stream, weight, grad_x};
  const int32_t c = static_cast<int32_t>(channels);
  const int64_t blocks = backward_blocks(rows, channels);
  const hipStream_t q = static_cast<hipStream_t>(stream);
  float* partial = static_cast<float*>(workspace);
  with_type(io_dtype, [&](auto io) {
    using T = decltype(io);
    using S = Store<T>;
    with_shape(c, aligned_call(c, all), [&](auto aligned, auto waves, auto elements) {
      constexpr bool kAligned = decltype(aligned)::value != 0;
      constexpr int kWaves = decltype(waves)::value, kE = decltype(elements)::value;
      hipLaunchKernelGGL((layer_norm_backward_kernel<T, kAligned, kWaves, kE>),
                         dim3(static_cast<unsigned>(blocks)), dim3(backward_threads<kWaves>()), 0,
                         q, static_cast<const S*>(grad_y), static_cast<const S*>(normed),
                         static_cast<const S*>(grad_stream), static_cast<const S*>(weight), mean,
                         rstd, static_cast<S*>(grad_x), partial, rows, c);
    });
    hipLaunchKernelGGL((layer_norm_columns_kernel<T>), dim3((c + 31) / 32, 2), dim3(1024), 0, q,
                       partial, static_cast<int32_t>(blocks), c, static_cast<S*>(grad_weight),
                       static_cast<S*>(grad_bias));
  });
  return check_launch("layer_norm_backward_kernel");
}

}  // extern "C"
