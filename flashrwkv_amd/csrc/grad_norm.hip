// The norm of many gradients together, and clipping by it.
//
//   norm = sqrt(sum over all tensors of x^2),  by = min(1, most / (norm + eps)),
//   y = x by  (in place, or to other tensors of types of their own).
// A norm that is not finite leaves by = 1: the gradients stay what they are, and
// the norm tells the caller.
//
// Memory bounds both passes: each tensor is read once for the norm and once more
// to be scaled. Tensors are cut into chunks of kChunk elements that workgroups
// take in turn, so that a list of small tensors and one large one are the same
// work; which tensor a chunk is of stands in the kernel's arguments, kEntries
// tensors a launch, and no table is copied to the device. Squares are summed in
// 64 bits: gradients beyond 1.8e19 or below 1e-23 have squares that 32 bits do not
// hold, and the sum of many of them loses nothing. Workgroups leave one sum each, added in their
// order: two calls give the same bits.
#include <algorithm>
#include <cmath>

#include "capi_internal.h"
#include "wkv7_device.h"

namespace frwkv {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;        // elements
constexpr int kEntries = 112;       // of a launch: 3.5 KB of arguments
constexpr int kMostGroups = 2048;   // workgroups of a launch
constexpr int kJoinThreads = 1024;

struct Entry {
  const void* from;
  void* to;
  int64_t numel;
  int32_t first;  // chunk
  uint8_t dtype, to_dtype;
  bool aligned, to_aligned;  // to 16 bytes
};

struct Table {
  Entry entry[kEntries];
  int32_t count, chunks;
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

template <int kBlock>
__device__ __forceinline__ double workgroup_sum(double x, double* shared) {
  x = wave_sum(x);
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kBlock / 64; ++w) sum += shared[w];
  __syncthreads();
  return sum;
}

// Eight consecutive elements.
template <typename T>
struct Eight {
  using S = typename IoTraits<T>::storage;
  static constexpr int kParts = 8 * sizeof(S) / 16;
  uint4 part[kParts];
  __device__ __forceinline__ void load(const void* from, int64_t i) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const S*>(from) + i);
#pragma unroll
    for (int q = 0; q < kParts; ++q) part[q] = p[q];
  }
  __device__ __forceinline__ void load_unaligned(const void* from, int64_t i, int64_t left) {
    S* e = reinterpret_cast<S*>(part);
#pragma unroll
    for (int q = 0; q < 8; ++q) e[q] = q < left ? static_cast<const S*>(from)[i + q] : S{0};
  }
  __device__ __forceinline__ float at(int e) const {
    return to_f32<T>(reinterpret_cast<const S*>(part)[e]);
  }
};

// f(type) for a dtype code.
template <typename F>
__device__ __forceinline__ void with_dtype(uint8_t dtype, F&& f) {
  if (dtype == FRWKV_DTYPE_F32) {
    f(float{});
  } else if (dtype == FRWKV_DTYPE_BF16) {
    f(Bf16{});
  } else {
    f(F16{});
  }
}

template <typename T>
__device__ __forceinline__ void chunk_squares(const Entry& e, int64_t first, double (&sum)[4]) {
  constexpr int kEach = kChunk / (8 * kThreads);
  const int64_t left = e.numel - first;
  Eight<T> x[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t i = first + (j * kThreads + threadIdx.x) * 8;
    const int64_t here = e.numel - i;
    if (e.aligned && (left >= kChunk || here >= 8)) {
      x[j].load(e.from, i);
    } else {
      x[j].load_unaligned(e.from, i, here);
    }
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const double v = x[j].at(q);
      sum[q & 3] = fma(v, v, sum[q & 3]);
    }
  }
}

// The entry of a chunk, from the last one on.
__device__ __forceinline__ int entry_of(const Table& t, int32_t chunk) {
  int at = 0, left = t.count;
  while (left > 1) {
    const int half = left / 2;
    if (t.entry[at + half].first <= chunk) {
      at += half;
      left -= half;
    } else {
      left = half;
    }
  }
  return at;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Table t, double* __restrict__ sums) {
  __shared__ double shared[kThreads / 64];
  double sum[4] = {};
  for (int32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const Entry& e = t.entry[entry_of(t, c)];
    with_dtype(e.dtype, [&](auto type) {
      chunk_squares<decltype(type)>(e, static_cast<int64_t>(c - e.first) * kChunk, sum);
    });
  }
  const double all = workgroup_sum<kThreads>((sum[0] + sum[1]) + (sum[2] + sum[3]), shared);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

__device__ __forceinline__ float factor_of(double total, double most, double eps) {
  const double norm = sqrt(total);
  if (!(norm < __builtin_inf())) return 1.0f;
  return static_cast<float>(fmin(1.0, most / (norm + eps)));
}

__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(const double* __restrict__ sums,
                                                                 int32_t groups, double most,
                                                                 double eps,
                                                                 float* __restrict__ norm,
                                                                 float* __restrict__ factor) {
  __shared__ double shared[kJoinThreads / 64];
  double sum = 0.0;
  for (int32_t g = threadIdx.x; g < groups; g += kJoinThreads) sum += sums[g];
  sum = workgroup_sum<kJoinThreads>(sum, shared);
  if (threadIdx.x == 0) {
    *norm = static_cast<float>(sqrt(sum));
    if (factor != nullptr) *factor = factor_of(sum, most, eps);
  }
}

template <typename T>
__device__ __forceinline__ void store_eight(void* to, int64_t i, int64_t left, bool aligned,
                                            const float (&y)[8]) {
  using S = typename IoTraits<T>::storage;
  S out[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) out[q] = from_f32<T>(y[q]);
  S* p = static_cast<S*>(to) + i;
  if (aligned && left >= 8) {
    constexpr int kParts = 8 * sizeof(S) / 16;
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      reinterpret_cast<uint4*>(p)[q] = reinterpret_cast<const uint4*>(out)[q];
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (q < left) p[q] = out[q];
  }
}

template <typename T, typename To>
__device__ __forceinline__ void scale_chunk(const Entry& e, int64_t first, float by) {
  constexpr int kEach = kChunk / (8 * kThreads);
  Eight<T> x[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t i = first + (j * kThreads + threadIdx.x) * 8;
    const int64_t here = e.numel - i;
    if (e.aligned && here >= 8) {
      x[j].load(e.from, i);
    } else {
      x[j].load_unaligned(e.from, i, here);
    }
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t i = first + (j * kThreads + threadIdx.x) * 8;
    float y[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) y[q] = x[j].at(q) * by;
    store_eight<To>(e.to, i, e.numel - i, e.to_aligned, y);
  }
}

// From the last chunk to the first: what the norm read last is still in the cache.
__global__ __launch_bounds__(kThreads) void scale_kernel(Table t,
                                                         const float* __restrict__ factor,
                                                         bool in_place) {
  const float by = *factor;
  if (in_place && by == 1.0f) return;
  for (int32_t c = t.chunks - 1 - static_cast<int32_t>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const Entry& e = t.entry[entry_of(t, c)];
    const int64_t first = static_cast<int64_t>(c - e.first) * kChunk;
    with_dtype(e.dtype, [&](auto type) {
      with_dtype(e.to_dtype, [&](auto to) {
        scale_chunk<decltype(type), decltype(to)>(e, first, by);
      });
    });
  }
}

constexpr int64_t kMostElements = int64_t{1} << 40;  // of a tensor

int64_t chunks_of(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

int groups_of(int32_t chunks) { return std::min(chunks, kMostGroups); }

bool known_dtype(int dtype) {
  return dtype == FRWKV_DTYPE_F32 || dtype == FRWKV_DTYPE_F16 || dtype == FRWKV_DTYPE_BF16;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// f(table) for every launch over the tensors, those without elements left out.
template <typename F>
void for_tables(int64_t count, const frwkv_gradient* tensors, F&& f) {
  Table t;
  t.count = t.chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const frwkv_gradient& x = tensors[i];
    if (x.numel == 0) continue;
    const int64_t chunks = chunks_of(x.numel);
    if (t.count == kEntries || t.chunks + chunks > INT32_MAX / 2) {
      f(t);
      t.count = t.chunks = 0;
    }
    t.entry[t.count++] = {x.data,
                          x.out,
                          x.numel,
                          t.chunks,
                          static_cast<uint8_t>(x.dtype),
                          static_cast<uint8_t>(x.out_dtype),
                          aligned16(x.data),
                          aligned16(x.out)};
    t.chunks += static_cast<int32_t>(chunks);
  }
  if (t.count > 0) f(t);
}

int check_tensors(const char* what, int64_t count, const frwkv_gradient* tensors, bool out) {
  if (count < 0 || (count > 0 && tensors == nullptr)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: no list of tensors", what);
  }
  for (int64_t i = 0; i < count; ++i) {
    const frwkv_gradient& x = tensors[i];
    if (x.numel < 0 || x.numel > kMostElements) {
      return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                       "%s: tensor %lld has %lld elements, [0, 2^40] are allowed", what,
                       static_cast<long long>(i), static_cast<long long>(x.numel));
    }
    if (x.numel == 0) continue;
    if (x.data == nullptr || (out && x.out == nullptr)) {
      return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: tensor %lld is null", what,
                       static_cast<long long>(i));
    }
    if (!known_dtype(x.dtype) || (out && !known_dtype(x.out_dtype))) {
      return set_error(FRWKV_ERR_UNSUPPORTED,
                       "%s: tensor %lld must be float32, float16 or bfloat16", what,
                       static_cast<long long>(i));
    }
    if (out && x.data == x.out && x.dtype != x.out_dtype) {
      return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                       "%s: tensor %lld in place has two types", what,
                       static_cast<long long>(i));
    }
  }
  return FRWKV_OK;
}

size_t workspace_of(int64_t count, const frwkv_gradient* tensors) {
  size_t groups = 0;
  for_tables(count, tensors, [&](const Table& t) { groups += groups_of(t.chunks); });
  return 256 + (groups * 8 + 255) / 256 * 256;
}

// factor: null for the norm alone.
void launch_norm(int64_t count, const frwkv_gradient* tensors, double most, double eps,
                 float* norm, float* factor, double* sums, hipStream_t stream) {
  int32_t groups = 0;
  for_tables(count, tensors, [&](const Table& t) {
    const int own = groups_of(t.chunks);
    hipLaunchKernelGGL(squares_kernel, dim3(own), dim3(kThreads), 0, stream, t, sums + groups);
    groups += own;
  });
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(kJoinThreads), 0, stream, sums, groups, most,
                     eps, norm, factor);
}

int begin(const char* what, int64_t count, const frwkv_gradient* tensors, bool out,
          const float* norm, void* workspace, size_t workspace_bytes) {
  const int rc = check_tensors(what, count, tensors, out);
  if (rc != FRWKV_OK) return rc;
  if (!norm) return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: norm is null", what);
  const size_t need = workspace_of(count, tensors);
  if (workspace == nullptr || workspace_bytes < need) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes given, %zu needed",
                     what, workspace == nullptr ? size_t{0} : workspace_bytes, need);
  }
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: workspace must be 256-byte aligned", what);
  }
  return FRWKV_OK;
}

}  // namespace
}  // namespace frwkv

extern "C" {

size_t frwkv_grad_norm_workspace_bytes(int64_t count, const frwkv_gradient* tensors) {
  using namespace frwkv;
  if (check_tensors("frwkv_grad_norm_workspace_bytes", count, tensors, false) != FRWKV_OK) {
    return 0;
  }
  return workspace_of(count, tensors);
}

int frwkv_grad_norm(int64_t count, const frwkv_gradient* tensors, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const int rc = begin("frwkv_grad_norm", count, tensors, false, norm, workspace,
                       workspace_bytes);
  if (rc != FRWKV_OK) return rc;
  launch_norm(count, tensors, 0.0, 0.0, norm, nullptr,
              reinterpret_cast<double*>(static_cast<char*>(workspace) + 256),
              static_cast<hipStream_t>(stream));
  return check_launch("gradient norm");
}

int frwkv_grad_clip(int64_t count, const frwkv_gradient* tensors, double max_norm, double eps,
                    float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_grad_clip";
  const int rc = begin(what, count, tensors, true, norm, workspace, workspace_bytes);
  if (rc != FRWKV_OK) return rc;
  if (!(max_norm >= 0.0) || !std::isfinite(max_norm) || !(eps >= 0.0) || !std::isfinite(eps)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: max_norm and eps must be finite and not negative", what);
  }
  float* factor = static_cast<float*>(workspace);
  const hipStream_t q = static_cast<hipStream_t>(stream);
  launch_norm(count, tensors, max_norm, eps, norm, factor,
              reinterpret_cast<double*>(static_cast<char*>(workspace) + 256), q);
  // A launch's tensors are in place or are not; mixed lists are written as a whole.
  for_tables(count, tensors, [&](const Table& t) {
    bool in_place = true;
    for (int i = 0; i < t.count; ++i) in_place = in_place && t.entry[i].from == t.entry[i].to;
    hipLaunchKernelGGL(scale_kernel, dim3(groups_of(t.chunks)), dim3(kThreads), 0, q, t, factor,
                       in_place);
  });
  return check_launch("gradient clipping");
}

}  // extern "C"
