// The norm of many gradients together, and clipping by it.
//
//   norm = sqrt(sum over all tensors of x^2),  by = min(1, most / (norm + eps)),
//   y = x by  (in place, or to other tensors of types of their own).
// A norm that is not finite leaves by = 1: the gradients stay what they are, and
// the norm tells the caller. by is rounded to 32 bits, as is its product with an element;
// below the normal numbers of 32 bits it keeps 64 and the product is made in them.
//
// Memory bounds both passes: each tensor is read once for the norm and once more
// to be scaled. Tensors are cut into units of kUnit elements, so that a list of small
// tensors and one large one are the same work. Squares are summed in 64 bits: gradients
// beyond 1.8e19 or below 1e-23 have squares that 32 bits do not hold, and the sum
// of many of them loses nothing. Workgroups leave one sum each, added in a fixed order:
// two calls give the same bits. Two forms, by plan_of's rule:
//
// Short lists of few elements stand in the kernels' arguments, and are read through the
// caches. A workgroup takes a run of consecutive chunks and searches the list for the first
// of them. All workgroups that scale add up the sums by themselves, which saves the launch
// that would.
//
// Others are written to the workspace by small kernels that take the list in their
// arguments (nothing is copied from the host, and a captured call keeps its
// list), with the tensor of each unit beside it. Each unit is scaled by a workgroup
// of its own, in the order of memory, which the DRAM answers best: bf16 to fp32, 449M
// elements, 450 us, and 542 in 2048 runs of their own.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "capi_internal.h"
#include "wkv7_device.h"

namespace frwkv {
namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8 * kThreads;  // elements: eight a thread
constexpr int kMany = 4;             // units that are read together
constexpr int kEntries = 112;        // tensors in a launch's arguments: 3.5 KB
constexpr int kMostGroups = 2048;    // workgroups that sum, eight a CU

struct Entry {
  const void* from;
  void* to;
  int64_t numel;
  int32_t first;  // chunk, or unit
  uint8_t dtype, to_dtype;
  bool aligned, to_aligned;  // to 16 bytes
};

struct Entries {
  Entry entry[kEntries];
};

// The whole list as a launch sees it.
struct List {
  int32_t count, chunks;  // or units
  bool in_place;  // all of them
};

// A tensor on its way to the list in the workspace: its data, and its elements with the
// types above them; where it is not written in place, its output beside it.
struct Item {
  uint64_t from, size;
};
constexpr int kTypeBit = 48, kToTypeBit = 52;

template <bool kInPlace>
struct Items {
  static constexpr int kCount = kInPlace ? 240 : 160;  // 3.8 KB of arguments
  Item item[kCount];
  uint64_t to[kInPlace ? 1 : kCount];
};

// The list in the workspace.
struct Places {
  Entry* entry;   // [count]
  int32_t* owner; // [units]  the entry of a unit
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

typedef uint32_t Word2 __attribute__((ext_vector_type(2)));
typedef uint32_t Word4 __attribute__((ext_vector_type(4)));

// kPer consecutive elements.
template <typename T, int kPer>
struct Pack {
  using S = typename IoTraits<T>::storage;
  static constexpr int kBytes = kPer * sizeof(S);
  static_assert(kEntries <= kThreads && (kBytes == 8 || kBytes == 16), "one load, one thread an entry");
  using Word = std::conditional_t<kBytes == 16, Word4, Word2>;
  Word word;
  // kStream: past the caches, for what is not read again soon.
  template <bool kStream>
  __device__ __forceinline__ void load(const void* from, int64_t i) {
    const Word* p = reinterpret_cast<const Word*>(static_cast<const S*>(from) + i);
    word = kStream ? __builtin_nontemporal_load(p) : *p;
  }
  __device__ __forceinline__ void load_unaligned(const void* from, int64_t i, int64_t left) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) put(q, q < left ? static_cast<const S*>(from)[i + q] : S{0});
  }
  __device__ __forceinline__ S get(int e) const {
    if constexpr (sizeof(S) == 4) {
      return __uint_as_float(word[e]);
    } else {
      return static_cast<S>(word[e / 2] >> (16 * (e % 2)));
    }
  }
  // In ascending order: the first half of a word clears the second.
  __device__ __forceinline__ void put(int e, S x) {
    if constexpr (sizeof(S) == 4) {
      word[e] = __float_as_uint(x);
    } else {
      word[e / 2] = e % 2 == 0 ? uint32_t{x} : word[e / 2] | uint32_t{x} << 16;
    }
  }
  __device__ __forceinline__ float at(int e) const { return to_f32<T>(get(e)); }
  __device__ __forceinline__ void set(int e, float x) { put(e, from_f32<T>(x)); }
  template <bool kStream>
  __device__ __forceinline__ void store(void* to, int64_t i) const {
    Word* p = reinterpret_cast<Word*>(static_cast<S*>(to) + i);
    if constexpr (kStream) {
      __builtin_nontemporal_store(word, p);
    } else {
      *p = word;
    }
  }
  __device__ __forceinline__ void store_unaligned(void* to, int64_t i, int64_t left) const {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      if (q < left) static_cast<S*>(to)[i + q] = get(q);
    }
  }
};

// Elements that a lane takes at a time: 16 bytes, and where an fp32 tensor is read or
// written 4 elements, so that a wave's accesses to it are without gaps (bf16 to
// fp32 with 8, whose stores have gaps of 16 bytes: 4.0 TB/s).
template <typename T, typename To>
constexpr int kPerLane = std::is_same_v<T, float> || std::is_same_v<To, float> ? 4 : 8;

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

// Place of a thread's pack j of a chunk.
template <int kPer>
__device__ __forceinline__ int64_t place(int64_t first, int j) {
  return first + (j * kThreads + static_cast<int>(threadIdx.x)) * kPer;
}

template <bool kStream, typename T, int kPer, int kPacks>
__device__ __forceinline__ void load_chunk(const Entry& e, int64_t first,
                                           Pack<T, kPer> (&x)[kPacks]) {
  if (e.aligned && e.numel - first >= kPacks * kThreads * kPer) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) x[j].template load<kStream>(e.from, place<kPer>(first, j));
    return;
  }
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const int64_t i = place<kPer>(first, j);
    if (e.aligned && e.numel - i >= kPer) {
      x[j].template load<kStream>(e.from, i);
    } else {
      x[j].load_unaligned(e.from, i, e.numel - i);
    }
  }
}

// Squares of kEach units of a tensor from `first` on, as far as they go.
template <int kEach, bool kStream>
__device__ __forceinline__ void add_squares(const Entry& e, int64_t first, double (&sum)[4]) {
  with_dtype(e.dtype, [&](auto type) {
    using T = decltype(type);
    constexpr int kPer = kPerLane<T, T>, kPacks = kEach * 8 / kPer;
    Pack<T, kPer> x[kPacks];
    load_chunk<kStream>(e, first, x);
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const double v = x[j].at(q);
        sum[q & 3] = fma(v, v, sum[q & 3]);
      }
    }
  });
}

// kEach units of a tensor, scaled.
template <int kEach, bool kStream, typename Factor>
__device__ __forceinline__ void scale_units(const Entry& e, int64_t first, Factor by) {
  with_dtype(e.dtype, [&](auto type) {
    with_dtype(e.to_dtype, [&](auto to_type) {
      using T = decltype(type);
      using To = decltype(to_type);
      constexpr int kPer = kPerLane<T, To>, kPacks = kEach * 8 / kPer;
      Pack<T, kPer> x[kPacks];
      load_chunk<kStream>(e, first, x);
      const bool whole = e.to_aligned && e.numel - first >= kEach * kUnit;
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        const int64_t i = place<kPer>(first, j);
        Pack<To, kPer> y;
#pragma unroll
        for (int q = 0; q < kPer; ++q) y.set(q, static_cast<float>(x[j].at(q) * by));
        if (whole || (e.to_aligned && e.numel - i >= kPer)) {
          y.template store<kStream>(e.to, i);
        } else {
          y.store_unaligned(e.to, i, e.numel - i);
        }
      }
    });
  });
}

// The entry of a chunk.
__device__ __forceinline__ int entry_of(const Entry* entries, int count, int32_t chunk) {
  int at = 0, left = count;
  while (left > 1) {
    const int half = left / 2;
    if (entries[at + half].first <= chunk) {
      at += half;
      left -= half;
    } else {
      left = half;
    }
  }
  return at;
}

// A workgroup's run of chunks.
struct Run {
  int32_t from, to;
};

__device__ __forceinline__ Run run_of(int32_t chunks) {
  const int64_t g = blockIdx.x, n = gridDim.x;
  return {static_cast<int32_t>(g * chunks / n), static_cast<int32_t>((g + 1) * chunks / n)};
}

// 3.1M fp32 elements of 24 tensors in 5 us, of which the read is 2: launch, list and one
// trip to memory.
template <int kEach>
__global__ __launch_bounds__(kThreads) void run_squares_kernel(Entries entries, List list,
                                                               double* __restrict__ sums) {
  __shared__ double shared[kThreads / 64];
  const Run run = run_of(list.chunks);
  double sum[4] = {};
  int at = entry_of(entries.entry, list.count, run.from);
  for (int32_t c = run.from; c < run.to; ++c) {
    while (at + 1 < list.count && entries.entry[at + 1].first <= c) ++at;
    const Entry e = entries.entry[at];
    add_squares<kEach, false>(e, static_cast<int64_t>(c - e.first) * (kEach * kUnit), sum);
  }
  const double all = workgroup_sum<kThreads>((sum[0] + sum[1]) + (sum[2] + sum[3]), shared);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

// A part of the list to the workspace, and its units' owners. Each workgroup finds the
// tensors' first units for itself: a launch takes 5 us, of which its arguments' way over
// the host's link is most, and fewer of them are what counts.
template <bool kInPlace>
__global__ __launch_bounds__(kThreads) void list_kernel(Items<kInPlace> part, int32_t count,
                                                        int32_t index, int32_t first,
                                                        int32_t units, Places to) {
  static_assert(Items<kInPlace>::kCount <= kThreads, "a thread a tensor");
  __shared__ int32_t firsts[kThreads], waves[kThreads / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  Entry e{};
  int32_t own = 0;
  if (t < count) {
    const uint64_t size = part.item[t].size;
    e.from = reinterpret_cast<const void*>(part.item[t].from);
    e.to = reinterpret_cast<void*>(kInPlace ? part.item[t].from : part.to[kInPlace ? 0 : t]);
    e.numel = static_cast<int64_t>(size & ((uint64_t{1} << kTypeBit) - 1));
    e.dtype = static_cast<uint8_t>(size >> kTypeBit & 3);
    e.to_dtype = static_cast<uint8_t>(size >> kToTypeBit & 3);
    e.aligned = reinterpret_cast<uintptr_t>(e.from) % 16 == 0;
    e.to_aligned = reinterpret_cast<uintptr_t>(e.to) % 16 == 0;
    own = static_cast<int32_t>((e.numel + kUnit - 1) / kUnit);
  }
  int32_t before = own;  // units up to this tensor's end
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int32_t other = __shfl_up(before, off, 64);
    if (lane >= off) before += other;
  }
  if (lane == 63) waves[wave] = before;
  __syncthreads();
  before += first - own;
  for (int w = 0; w < wave; ++w) before += waves[w];
  firsts[t] = before;
  e.first = before;
  if (blockIdx.x == 0 && t < count) to.entry[index + t] = e;
  __syncthreads();
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + t; u < units;
       u += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int32_t unit = first + static_cast<int32_t>(u);
    int at = 0, left = count;
    while (left > 1) {
      const int half = left / 2;
      const bool behind = firsts[at + half] <= unit;
      at += behind ? half : 0;
      left = behind ? left - half : half;
    }
    to.owner[unit] = index + at;
  }
}

// kMany consecutive units at a time, in turns: read together where they are of one tensor.
// Bound by HBM: 449M bf16 elements of 675 tensors in 147 us, 6.1 TB/s (a bare loop over as much
// memory 135 past the caches, kStream, and 150 through them; keeping the last 96 to 224 MB in
// them for the scaling changed the call by less than 2%).
template <bool kStream>
__global__ __launch_bounds__(kThreads) void squares_kernel(Places places, List list,
                                                           double* __restrict__ sums) {
  __shared__ double shared[kThreads / 64];
  double sum[4] = {};
  const int32_t step = static_cast<int32_t>(gridDim.x) * kMany;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kMany; u < list.chunks; u += step) {
    const int32_t last = static_cast<int32_t>(min(u + kMany, static_cast<int64_t>(list.chunks))) - 1;
    int32_t unit = static_cast<int32_t>(u);
    const int32_t at = places.owner[unit];
    if (places.owner[last] == at) {
      const Entry e = places.entry[at];
      add_squares<kMany, kStream>(e, static_cast<int64_t>(unit - e.first) * kUnit, sum);
      continue;
    }
    for (; unit <= last; ++unit) {
      const Entry e = places.entry[places.owner[unit]];
      add_squares<1, kStream>(e, static_cast<int64_t>(unit - e.first) * kUnit, sum);
    }
  }
  const double all = workgroup_sum<kThreads>((sum[0] + sum[1]) + (sum[2] + sum[3]), shared);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

// The sum of all workgroups' sums, the same one for every caller.
template <int kBlock>
__device__ __forceinline__ double total_of(const double* __restrict__ sums, int32_t groups,
                                           double* shared) {
  constexpr int kEach = kMostGroups / kBlock;
  double x[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int32_t g = j * kBlock + static_cast<int32_t>(threadIdx.x);
    x[j] = g < groups ? sums[g] : 0.0;
  }
#pragma unroll
  for (int j = 1; j < kEach; ++j) x[0] += x[j];
  return workgroup_sum<kBlock>(x[0], shared);
}

// 1 where the norm as it is returned, in 32 bits, is not finite.
__device__ __forceinline__ double factor_of(double total, double most, double eps) {
  const double norm = sqrt(total);
  if (!(static_cast<float>(norm) < __builtin_inff())) return 1.0;
  return fmin(1.0, most / (norm + eps));
}

// f(factor) in the bits that hold it.
template <typename F>
__device__ __forceinline__ void with_factor(double by, F&& f) {
  if (by >= 0x1p-126) {
    f(static_cast<float>(by));
  } else {
    f(by);
  }
}

// factor: null for the norm alone.
__global__ __launch_bounds__(kThreads) void norm_kernel(const double* __restrict__ sums,
                                                        int32_t groups, double most, double eps,
                                                        float* norm, double* factor) {
  __shared__ double shared[kThreads / 64];
  const double total = total_of<kThreads>(sums, groups, shared);
  if (threadIdx.x != 0) return;
  *norm = static_cast<float>(sqrt(total));
  if (factor != nullptr) *factor = factor_of(total, most, eps);
}

// From a run's last chunk to its first: what the norm read last is still in the cache.
template <int kEach>
__global__ __launch_bounds__(kThreads) void run_scale_kernel(Entries entries, List list,
                                                             const double* __restrict__ sums,
                                                             int32_t groups, double most,
                                                             double eps,
                                                             float* __restrict__ norm) {
  __shared__ double shared[kThreads / 64];
  const double total = total_of<kThreads>(sums, groups, shared);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(sqrt(total));
  const double factor = factor_of(total, most, eps);
  if (list.in_place && static_cast<float>(factor) == 1.0f) return;
  const Run run = run_of(list.chunks);
  with_factor(factor, [&](auto by) {
    int at = entry_of(entries.entry, list.count, run.to - 1);
    for (int32_t c = run.to - 1; c >= run.from; --c) {
      while (entries.entry[at].first > c) --at;
      const Entry e = entries.entry[at];
      scale_units<kEach, false>(e, static_cast<int64_t>(c - e.first) * (kEach * kUnit), by);
    }
  });
}

// A unit a workgroup, from the last one (and again, beyond what a launch has). Bound by
// HBM: 449M bf16 elements into fp32 in 445 us, 6.0 TB/s; in place 316 us, 5.7 TB/s, and 47 us
// where nothing is to be scaled.
constexpr int kMostScalers = 1 << 22;

template <bool kStream>
__global__ __launch_bounds__(kThreads) void scale_kernel(Places places, List list,
                                                         const double* __restrict__ factor) {
  if (list.in_place && static_cast<float>(*factor) == 1.0f) return;
  with_factor(*factor, [&](auto by) {
    for (int32_t unit = list.chunks - 1 - static_cast<int32_t>(blockIdx.x); unit >= 0;
         unit -= static_cast<int32_t>(gridDim.x)) {
      const Entry e = places.entry[places.owner[unit]];
      scale_units<1, kStream>(e, static_cast<int64_t>(unit - e.first) * kUnit, by);
    }
  });
}

constexpr int64_t kMostElements = int64_t{1} << 40;  // of a tensor

bool known_dtype(int dtype) {
  return dtype == FRWKV_DTYPE_F32 || dtype == FRWKV_DTYPE_F16 || dtype == FRWKV_DTYPE_BF16;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How a list is cut and where it stands.
struct Plan {
  int64_t count;  // tensors with elements
  int64_t units;
  int64_t chunks; // of kMany units each, or of one; in the list's form, of one
  int each;       // units of a chunk; 0: the list stands in the workspace
  bool stream;

  int groups() const {
    const int64_t turns = each == 0 ? (units + kMany - 1) / kMany : chunks;
    return static_cast<int>(std::min<int64_t>(turns, kMostGroups));
  }
  // Workspace: sums, factor, entries, owners.
  size_t sums_bytes() const { return (static_cast<size_t>(groups()) * 8 + 255) / 256 * 256; }
  size_t entry_bytes() const {
    return each != 0 ? 0 : (static_cast<size_t>(count) * sizeof(Entry) + 255) / 256 * 256;
  }
  size_t bytes() const {
    const size_t owners = each != 0 ? 0 : (static_cast<size_t>(units) * 4 + 255) / 256 * 256;
    return 256 + sums_bytes() + entry_bytes() + owners;
  }
};

int64_t chunks_of(int64_t numel, int64_t each) {
  return (numel + each * kUnit - 1) / (each * kUnit);
}

// Most chunks of a list in the arguments: runs of eight, beyond which the order of
// memory makes up for the launches that the other form has more.
constexpr int64_t kMostRuns = 8 * kMostGroups;
// The last-level cache's size: what the list's form reads twice and is larger passes by it.
constexpr int64_t kCacheBytes = int64_t{256} << 20;

Plan plan_of(int64_t count, const frwkv_gradient* tensors) {
  Plan p{0, 0, 0, 1, false};
  int64_t bytes = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t numel = tensors[i].numel;
    if (numel == 0) continue;
    ++p.count;
    p.units += chunks_of(numel, 1);
    p.chunks += chunks_of(numel, kMany);
    bytes += numel * (tensors[i].dtype == FRWKV_DTYPE_F32 ? 4 : 2);
  }
  p.stream = bytes > kCacheBytes;
  if (p.count > kEntries || p.chunks > kMostRuns) {
    p.each = 0;
    p.chunks = p.units;
  } else if (p.units > kMostGroups) {
    p.each = kMany;
  } else {
    p.chunks = p.units;
  }
  return p;
}

// f(items, how many, index of the first, its unit, units) for as many tensors with
// elements as a launch takes.
template <bool kInPlace, typename F>
void for_items(int64_t count, const frwkv_gradient* tensors, F&& f) {
  Items<kInPlace> part;
  int32_t have = 0, done = 0, units = 0, before = 0;
  const auto flush = [&] {
    if (have > 0) f(part, have, done, before, units - before);
    done += have;
    before = units;
    have = 0;
  };
  for (int64_t i = 0; i < count; ++i) {
    const frwkv_gradient& x = tensors[i];
    if (x.numel == 0) continue;
    if (have == Items<kInPlace>::kCount) flush();
    part.item[have] = {reinterpret_cast<uint64_t>(x.data),
                       static_cast<uint64_t>(x.numel) |
                           static_cast<uint64_t>(x.dtype) << kTypeBit |
                           static_cast<uint64_t>(x.out_dtype) << kToTypeBit};
    if constexpr (!kInPlace) part.to[have] = reinterpret_cast<uint64_t>(x.out);
    ++have;
    units += static_cast<int32_t>(chunks_of(x.numel, 1));
  }
  flush();
}

// f(entries) of a list of at most kEntries tensors with elements; chunks are of `each`
// units.
template <typename F>
void with_entries(int64_t count, const frwkv_gradient* tensors, int each, F&& f) {
  Entries part;
  int32_t have = 0, first = 0;
  for (int64_t i = 0; i < count; ++i) {
    const frwkv_gradient& x = tensors[i];
    if (x.numel == 0) continue;
    part.entry[have++] = {x.data,
                          x.out,
                          x.numel,
                          first,
                          static_cast<uint8_t>(x.dtype),
                          static_cast<uint8_t>(x.out_dtype),
                          aligned16(x.data),
                          aligned16(x.out)};
    first += static_cast<int32_t>(chunks_of(x.numel, each));
  }
  f(part);
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

// f(streaming) as a constant.
template <typename F>
void with_stream(bool stream, F&& f) {
  if (stream) {
    f(std::true_type{});
  } else {
    f(std::false_type{});
  }
}

// Launches the norm, with the scaling behind it (scale) or without.
void launch(const Plan& plan, int64_t count, const frwkv_gradient* tensors, bool scale,
            double most, double eps, float* norm, char* workspace, hipStream_t stream) {
  double* factor = scale ? reinterpret_cast<double*>(workspace) : nullptr;
  double* sums = reinterpret_cast<double*>(workspace + 256);
  const int groups = plan.groups();
  List list{static_cast<int32_t>(plan.count), static_cast<int32_t>(plan.chunks), scale};
  for (int64_t i = 0; i < count && list.in_place; ++i) {
    list.in_place = tensors[i].numel == 0 || tensors[i].data == tensors[i].out;
  }
  const auto norm_of = [&] {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, stream, sums, groups, most, eps,
                       norm, factor);
  };
  if (plan.count == 0) return norm_of();
  if (plan.each == 0) {
    char* at = workspace + 256 + plan.sums_bytes();
    const Places places{reinterpret_cast<Entry*>(at),
                        reinterpret_cast<int32_t*>(at + plan.entry_bytes())};
    const auto write = [&](auto in_place) {
      constexpr bool kInPlace = decltype(in_place)::value;
      for_items<kInPlace>(count, tensors, [&](const Items<kInPlace>& part, int32_t have,
                                              int32_t index, int32_t first, int32_t units) {
        const int blocks = std::clamp<int>(units / (4 * kThreads), 1, 256);
        hipLaunchKernelGGL((list_kernel<kInPlace>), dim3(blocks), dim3(kThreads), 0, stream, part,
                           have, index, first, units, places);
      });
    };
    if (list.in_place || !scale) {  // the norm alone writes nothing
      write(std::true_type{});
    } else {
      write(std::false_type{});
    }
    with_stream(plan.stream, [&](auto streaming) {
      constexpr bool kStream = decltype(streaming)::value;
      hipLaunchKernelGGL((squares_kernel<kStream>), dim3(groups), dim3(kThreads), 0, stream,
                         places, list, sums);
      norm_of();
      if (scale) {
        hipLaunchKernelGGL((scale_kernel<kStream>), dim3(std::min(list.chunks, kMostScalers)),
                           dim3(kThreads), 0, stream,
                           places, list, factor);
      }
    });
    return;
  }
  const auto run = [&](auto each) {
    constexpr int kEach = decltype(each)::value;
    with_entries(count, tensors, kEach, [&](const Entries& entries) {
      hipLaunchKernelGGL((run_squares_kernel<kEach>), dim3(groups), dim3(kThreads), 0, stream,
                         entries, list, sums);
      if (scale) {
        hipLaunchKernelGGL((run_scale_kernel<kEach>), dim3(groups), dim3(kThreads), 0, stream,
                           entries, list, sums, groups, most, eps, norm);
      }
    });
  };
  if (plan.each == 1) {
    run(std::integral_constant<int, 1>{});
  } else {
    run(std::integral_constant<int, kMany>{});
  }
  if (!scale) norm_of();
}

int begin(const char* what, int64_t count, const frwkv_gradient* tensors, bool out,
          const float* norm, void* workspace, size_t workspace_bytes, Plan* plan) {
  const int rc = check_tensors(what, count, tensors, out);
  if (rc != FRWKV_OK) return rc;
  *plan = plan_of(count, tensors);
  if (plan->units > INT32_MAX / 2 || plan->count > INT32_MAX / 2) {
    return set_error(FRWKV_ERR_UNSUPPORTED, "%s: too many elements for one call", what);
  }
  if (!norm) return set_error(FRWKV_ERR_INVALID_ARGUMENT, "%s: norm is null", what);
  const size_t need = plan->bytes();
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
  return plan_of(count, tensors).bytes();
}

int frwkv_grad_norm(int64_t count, const frwkv_gradient* tensors, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  Plan plan;
  const int rc = begin("frwkv_grad_norm", count, tensors, false, norm, workspace,
                       workspace_bytes, &plan);
  if (rc != FRWKV_OK) return rc;
  launch(plan, count, tensors, false, 0.0, 0.0, norm, static_cast<char*>(workspace),
         static_cast<hipStream_t>(stream));
  return check_launch("gradient norm");
}

int frwkv_grad_clip(int64_t count, const frwkv_gradient* tensors, double max_norm, double eps,
                    float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  const char* what = "frwkv_grad_clip";
  Plan plan;
  const int rc = begin(what, count, tensors, true, norm, workspace, workspace_bytes, &plan);
  if (rc != FRWKV_OK) return rc;
  if (!(max_norm >= 0.0) || !std::isfinite(max_norm) || !(eps >= 0.0) || !std::isfinite(eps)) {
    return set_error(FRWKV_ERR_INVALID_ARGUMENT,
                     "%s: max_norm and eps must be finite and not negative", what);
  }
  launch(plan, count, tensors, true, max_norm, eps, norm, static_cast<char*>(workspace),
         static_cast<hipStream_t>(stream));
  return check_launch("gradient clipping");
}

}  // extern "C"
