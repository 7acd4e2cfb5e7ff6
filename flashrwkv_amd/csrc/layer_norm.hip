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
// A row is held in registers by 1, 4 or 16 waves, 16 elements a thread (C up
// to 1024, 4096, 16384), so each tensor passes once and the variance is taken
// about the mean. The backward's workgroups walk over rows and keep the
// weight's and bias' sums of their 16 columns a thread in registers; one row
// of 2 C partial sums a workgroup goes to memory and a second kernel adds
// those in order, so the result does not depend on timing.
#include <algorithm>
#include <type_traits>

#include "capi_internal.h"
#include "wkv7_device.h"

namespace frwkv {
namespace {

constexpr int kEpt = 16;         // elements of a row a thread
constexpr int kMaxBlocks = 512;  // of the backward: two a CU

template <typename T>
using Store = typename IoTraits<T>::storage;

// kVec consecutive elements as they lie in memory; kVec 8 reads 16-byte pieces.
template <typename T, int kVec>
struct Piece {
  static constexpr int kWords = kVec == 1 ? 1 : kVec * IoTraits<T>::kBytes / 16;
  typedef typename std::conditional<kVec == 1, Store<T>, uint4>::type Word;
  Word word[kWords];
  __device__ __forceinline__ void load(const Store<T>* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) word[i] = reinterpret_cast<const Word*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) word[i] = Word{};
  }
  // Conversions before and after this one are not one value kept in registers.
  __device__ __forceinline__ void again() {
    if constexpr (kVec != 1) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        asm volatile("" : "+v"(word[i].x), "+v"(word[i].y), "+v"(word[i].z), "+v"(word[i].w));
      }
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (kVec == 1) {
      return to_f32<T>(word[0]);
    } else if constexpr (__is_same(T, float)) {
      const uint4 q = word[e / 4];
      return __uint_as_float(e % 4 == 0 ? q.x : e % 4 == 1 ? q.y : e % 4 == 2 ? q.z : q.w);
    } else {
      const uint32_t d = e / 2 == 0 ? word[0].x : e / 2 == 1 ? word[0].y
                         : e / 2 == 2 ? word[0].z : word[0].w;
      return to_f32<T>(static_cast<uint16_t>(e % 2 ? d >> 16 : d & 0xffffu));
    }
  }
};

template <typename T, int kVec>
__device__ __forceinline__ void load(const Store<T>* p, float* out) {
  Piece<T, kVec> x;
  x.load(p);
#pragma unroll
  for (int e = 0; e < kVec; ++e) out[e] = x.get(e);
}

template <typename T, int kVec>
__device__ __forceinline__ void store(Store<T>* p, const float* x) {
  if constexpr (kVec == 1) {
    *p = from_f32<T>(x[0]);
  } else if constexpr (__is_same(T, float)) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]),
                                              pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
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

template <typename T, int kVec, int kWaves>
__global__ __launch_bounds__(forward_threads<kWaves>()) void layer_norm_forward_kernel(
    const Store<T>* __restrict__ x, const Store<T>* __restrict__ residual,
    const Store<T>* __restrict__ weight, const Store<T>* __restrict__ bias,
    Store<T>* __restrict__ y, Store<T>* __restrict__ stream, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, int64_t rows, int32_t c, float eps) {
  constexpr int kGroups = forward_threads<kWaves>() / (64 * kWaves);
  constexpr int kRow = 64 * kWaves;
  __shared__ float red[2][kGroups][kWaves];
  const int group = threadIdx.x / kRow, t = threadIdx.x % kRow, wave = t >> 6;
  const float inv_c = 1.0f / static_cast<float>(c);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool here = row < rows;
    const int64_t at = (here ? row : 0) * c;
    float s[kEpt];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kEpt; j += kVec) {
      const int col = (j / kVec * kRow + t) * kVec;
#pragma unroll
      for (int e = 0; e < kVec; ++e) s[j + e] = 0.0f;
      if (here && col < c) {
        load<T, kVec>(x + at + col, s + j);
        if (residual != nullptr) {
          float r[kVec];
          load<T, kVec>(residual + at + col, r);
#pragma unroll
          for (int e = 0; e < kVec; ++e) s[j + e] = to_f32<T>(from_f32<T>(s[j + e] + r[e]));
          store<T, kVec>(stream + at + col, s + j);
        }
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum += s[j + e];
      }
    }
    const float mean = row_sum<kWaves>(sum, red[0][group], wave) * inv_c;
    float sq = 0.0f;
#pragma unroll
    for (int j = 0; j < kEpt; j += kVec) {
      const int col = (j / kVec * kRow + t) * kVec;
      if (col < c) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          s[j + e] -= mean;
          sq = fmaf(s[j + e], s[j + e], sq);
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
    for (int j = 0; j < kEpt; j += kVec) {
      const int col = (j / kVec * kRow + t) * kVec;
      if (col < c) {
        float w[kVec], b[kVec], o[kVec];
        load<T, kVec>(weight + col, w);
        load<T, kVec>(bias + col, b);
#pragma unroll
        for (int e = 0; e < kVec; ++e) o[e] = fmaf(s[j + e] * rstd, w[e], b[e]);
        store<T, kVec>(y + at + col, o);
      }
    }
  }
}

// partial[block][0][c] = sum over the block's rows of dy xhat, [1][c] of dy.
template <typename T, int kVec, int kWaves>
__global__ __launch_bounds__(backward_threads<kWaves>(), kVec == 1 ? 1 : 4) void layer_norm_backward_kernel(
    const Store<T>* __restrict__ dy, const Store<T>* __restrict__ s,
    const Store<T>* __restrict__ ds, const Store<T>* __restrict__ weight,
    const float* __restrict__ mean, const float* __restrict__ rstd, Store<T>* __restrict__ dx,
    float* __restrict__ partial, int64_t rows, int32_t c) {
  constexpr int kThreads = backward_threads<kWaves>();
  constexpr int kGroups = kThreads / (64 * kWaves);
  constexpr int kRow = 64 * kWaves;
  __shared__ float red[2][2][kGroups][kWaves];
  __shared__ float columns[kGroups > 1 ? kThreads * kEpt : 1];
  const int group = threadIdx.x / kRow, t = threadIdx.x % kRow, wave = t >> 6;
  const float inv_c = 1.0f / static_cast<float>(c);
  // What is only read again is kept as it lies in memory.
  constexpr int kPieces = kEpt / kVec;
  Piece<T, kVec> w[kPieces], up[kPieces], add[kPieces];
  float pw[kEpt], pb[kEpt];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int col = (j * kRow + t) * kVec;
    w[j].zero();
    if (col < c) w[j].load(weight + col);
#pragma unroll
    for (int e = 0; e < kVec; ++e) pw[j * kVec + e] = pb[j * kVec + e] = 0.0f;
  }
  int side = 0;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool here = row < rows;
    const int64_t at = (here ? row : 0) * c;
    const float mu = here ? mean[row] : 0.0f, rs = here ? rstd[row] : 0.0f;
    float xh[kEpt];
    float sg = 0.0f, sgx = 0.0f;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      Piece<T, kVec> x;
      x.zero();
      up[j].zero();
      add[j].zero();
      w[j].again();
      if (here && col < c) {
        x.load(s + at + col);
        up[j].load(dy + at + col);
        if (ds != nullptr) add[j].load(ds + at + col);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int k = j * kVec + e;
        const float u = up[j].get(e), g = u * w[j].get(e);
        xh[k] = col < c ? (x.get(e) - mu) * rs : 0.0f;
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
    if (!here) continue;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int col = (j * kRow + t) * kVec;
      up[j].again();
      w[j].again();
      if (col < c) {
        float o[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float g = up[j].get(e) * w[j].get(e);
          o[e] = fmaf(rs, g - mg - xh[j * kVec + e] * mgx, add[j].get(e));
        }
        store<T, kVec>(dx + at + col, o);
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
      for (int e = 0; e < kEpt; ++e) columns[(group * kEpt + e) * kRow + t] = mine[e];
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int q = 1; q < kGroups; ++q) {
#pragma unroll
          for (int e = 0; e < kEpt; ++e) mine[e] += columns[(q * kEpt + e) * kRow + t];
        }
      }
    }
    if (group == 0) {
      float* to = partial + (static_cast<int64_t>(blockIdx.x) * 2 + which) * c;
#pragma unroll
      for (int j = 0; j < kEpt; j += kVec) {
        const int col = (j / kVec * kRow + t) * kVec;
        if (col < c) store<float, kVec>(to + col, mine + j);
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

int waves_of(int64_t c) { return c <= 64 * kEpt ? 1 : c <= 256 * kEpt ? 4 : 16; }

int64_t backward_blocks(int64_t rows, int64_t c) {
  const int waves = waves_of(c);
  const int64_t groups = waves == 16 ? 1 : 8 / waves;
  return std::min<int64_t>((rows + groups - 1) / groups, waves == 16 ? kMaxBlocks / 2 : kMaxBlocks);
}

struct Call {
  int64_t rows;
  int32_t c;
  hipStream_t stream;
};

template <typename F>
void with_shape(int64_t c, bool vector, F&& f) {
  const int waves = waves_of(c);
  const auto with_waves = [&](auto vec) {
    if (waves == 1) f(vec, std::integral_constant<int, 1>{});
    if (waves == 4) f(vec, std::integral_constant<int, 4>{});
    if (waves == 16) f(vec, std::integral_constant<int, 16>{});
  };
  if (vector) {
    with_waves(std::integral_constant<int, 8>{});
  } else {
    with_waves(std::integral_constant<int, 1>{});
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
bool vector_call(int64_t c, const void* const (&pointers)[N]) {
  for (const void* p : pointers) {
    if (!aligned16(p)) return false;
  }
  return c % 8 == 0;
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
  if (c <= 0 || c > 1024 * kEpt) {
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
    with_shape(c, vector_call(c, all), [&](auto vec, auto waves) {
      constexpr int kVec = decltype(vec)::value, kWaves = decltype(waves)::value;
      constexpr int kThreads = forward_threads<kWaves>();
      constexpr int kGroups = kThreads / (64 * kWaves);
      const int64_t blocks = std::min<int64_t>((rows + kGroups - 1) / kGroups, 1 << 20);
      hipLaunchKernelGGL((layer_norm_forward_kernel<T, kVec, kWaves>),
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
    with_shape(c, vector_call(c, all), [&](auto vec, auto waves) {
      constexpr int kVec = decltype(vec)::value, kWaves = decltype(waves)::value;
      hipLaunchKernelGGL((layer_norm_backward_kernel<T, kVec, kWaves>),
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
