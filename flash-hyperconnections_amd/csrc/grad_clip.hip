// Global norm over many tensors, and scaling by what it allows:
//   norm = (sum |g|^p)^(1/p) for p = 1, 2, max |g| for p = inf;
//   out = g min(1, max_norm / (norm + 1e-6)).
//
// A launch takes up to kTensors tensors, described in its arguments (so there is
// no table to upload and a captured graph keeps its own), and cuts them into
// chunks that its workgroups take in turn.  Each workgroup leaves one partial
// sum; whoever needs the norm adds the partial sums itself, in one fixed order,
// so the result is the same from call to call and the scaling needs no launch
// between it and the sums.
//
// The sums are FP64: squares of FP32 values overflow and underflow FP32 long
// before the norm does, and the matrix of one model holds 10^9 terms.
//
// Bound by HBM traffic: every element is read twice and written once.  The
// scaling walks the chunks from the last to the first, so that it starts with
// what the norm's pass left in the last-level cache.  336 M bf16 elements: 110 us (6.1
// TB/s) and 244 us (5.5 TB/s).
#include <algorithm>

#include "fh_kernels.h"
#include "fh_vec.h"

namespace fh {
namespace {

constexpr int kBlock = 256;
constexpr int kUnroll = 4;
constexpr int64_t kChunk = 2 * kBlock * kUnroll * 16;  // bytes of a chunk
constexpr int kTensors = 96;                            // tensors of a launch: 3.1 KB of its arguments

struct Entry {
  const void* src;
  void* dst;
  int64_t count;
  uint32_t first;  // chunk
  int dtype;
};

struct ClipArgs {
  Entry entries[kTensors];
  int tensors;
  uint32_t chunks;
  double* partial;     // norm: this launch's part; scaling: all of them
  int partials;        // scaling: how many
  int power;           // 1, 2, or 0 for the maximum
  double max_norm;
  float* norm;         // scaling: receives the norm (may be null)
  int inplace;
};

__device__ __forceinline__ double combine(double a, double b, int power) {
  if (power != 0) return a + b;
  return a != a || a > b ? a : b;  // a NaN stays
}

__device__ __forceinline__ double block_combine(double v, int power) {
  __shared__ double area[kBlock / 64];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = combine(v, __shfl_xor(v, d), power);
  if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6] = v;
  __syncthreads();
  v = area[0];
#pragma unroll
  for (int i = 1; i < kBlock / 64; ++i) v = combine(v, area[i], power);
  return v;
}

// The tensor that holds a chunk.
__device__ __forceinline__ int tensor_of(const ClipArgs& a, uint32_t chunk) {
  int low = 0, high = a.tensors - 1;
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (a.entries[mid].first <= chunk) low = mid;
    else high = mid - 1;
  }
  return low;
}

template <typename T, int Power>
__device__ __forceinline__ double chunk_sum(const Entry& e, int64_t begin) {
  using S = typename T::storage;
  constexpr int V = kVec<T>;
  const S* p = static_cast<const S*>(e.src) + begin;
  const int end = static_cast<int>(std::min<int64_t>(e.count - begin, kChunk / static_cast<int64_t>(sizeof(S))));
  double s = 0.0;
  for (int c = static_cast<int>(threadIdx.x) * V; c < end; c += kBlock * V * kUnroll) {
    U32x4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = load_row<T>(p, c + u * (kBlock * V), end);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float f[V];
      to_floats<T>(raw[u], f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = static_cast<double>(f[i]);
        if constexpr (Power == 2) s = __builtin_fma(d, d, s);
        if constexpr (Power == 1) s += __builtin_fabs(d);
        if constexpr (Power == 0) s = combine(s, __builtin_fabs(d), 0);
      }
    }
  }
  return s;
}

template <int Power>
__global__ __launch_bounds__(kBlock) void grad_norm_kernel(ClipArgs a) {
  double s = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const Entry& e = a.entries[tensor_of(a, chunk)];
    const int64_t at = static_cast<int64_t>(chunk - e.first) * kChunk;
    const double part = e.dtype == F32::code    ? chunk_sum<F32, Power>(e, at / 4)
                        : e.dtype == BF16::code ? chunk_sum<BF16, Power>(e, at / 2)
                                                : chunk_sum<F16, Power>(e, at / 2);
    s = combine(s, part, Power);
  }
  s = block_combine(s, Power);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

// The norm from all partial sums, the same in every thread of every workgroup.
__device__ __forceinline__ double total(const ClipArgs& a) {
  double s = 0.0;
  for (int i = threadIdx.x; i < a.partials; i += kBlock) s = combine(s, a.partial[i], a.power);
  s = block_combine(s, a.power);
  return a.power == 2 ? __builtin_sqrt(s) : s;
}

__global__ __launch_bounds__(kBlock) void norm_value_kernel(ClipArgs a) {
  const double norm = total(a);
  if (threadIdx.x == 0) *a.norm = static_cast<float>(norm);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const Entry& e, int64_t begin, float factor) {
  using S = typename T::storage;
  constexpr int V = kVec<T>;
  const S* p = static_cast<const S*>(e.src) + begin;
  S* q = static_cast<S*>(e.dst) + begin;
  const int end = static_cast<int>(std::min<int64_t>(e.count - begin, kChunk / static_cast<int64_t>(sizeof(S))));
  for (int c = static_cast<int>(threadIdx.x) * V; c < end; c += kBlock * V * kUnroll) {
    U32x4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = load_row<T>(p, c + u * (kBlock * V), end);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float f[V];
      to_floats<T>(raw[u], f);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= factor;
      store_row<T>(from_floats<T>(f), q, c + u * (kBlock * V), end);
    }
  }
}

__global__ __launch_bounds__(kBlock) void clip_scale_kernel(ClipArgs a) {
  const double norm = total(a);
  if (a.norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = static_cast<float>(norm);
  const double allowed = a.max_norm / (norm + 1e-6);
  const float factor = allowed > 1.0 ? 1.f : static_cast<float>(allowed);  // NaN stays NaN
  if (a.inplace && factor == 1.f) return;
  for (uint32_t i = blockIdx.x; i < a.chunks; i += gridDim.x) {
    const uint32_t chunk = a.chunks - 1 - i;
    const Entry& e = a.entries[tensor_of(a, chunk)];
    const int64_t at = static_cast<int64_t>(chunk - e.first) * kChunk;
    if (e.dtype == F32::code) chunk_scale<F32>(e, at / 4, factor);
    else if (e.dtype == BF16::code) chunk_scale<BF16>(e, at / 2, factor);
    else chunk_scale<F16>(e, at / 2, factor);
  }
}

int64_t chunks_of(int64_t count, int dtype) {
  const int64_t bytes = count * (dtype == F32::code ? 4 : 2);
  return (bytes + kChunk - 1) / kChunk;
}

// Workgroups of a launch: eight a compute unit fill it.
int64_t blocks_for(int64_t chunks) { return std::min<int64_t>(chunks, 8 * compute_units()); }

// f(args, blocks) for consecutive groups of tensors with elements, each of at
// most kTensors tensors and 2^31 chunks.
template <typename F>
hipError_t in_launches(const ClipList& list, F f) {
  ClipArgs a{};
  const auto flush = [&]() -> hipError_t {
    if (a.tensors == 0) return hipSuccess;
    const hipError_t err = f(a, static_cast<int>(blocks_for(a.chunks)));
    a.tensors = 0;
    a.chunks = 0;
    return err;
  };
  for (int i = 0; i < list.count; ++i) {
    if (list.sizes[i] == 0) continue;
    // A tensor of more than 2^30 chunks (32 TiB) is no tensor of this device.
    const int64_t chunks = chunks_of(list.sizes[i], list.dtypes[i]);
    if (a.tensors == kTensors || a.chunks + chunks > (int64_t{1} << 30)) {
      if (const hipError_t err = flush(); err != hipSuccess) return err;
    }
    a.entries[a.tensors++] = Entry{list.src[i], list.dst != nullptr ? list.dst[i] : nullptr, list.sizes[i], a.chunks,
                                   list.dtypes[i]};
    a.chunks += static_cast<uint32_t>(chunks);
  }
  return flush();
}

}  // namespace

int64_t clip_partials(const ClipList& list) {
  int64_t n = 0;
  (void)in_launches(list, [&](ClipArgs&, int blocks) {
    n += blocks;
    return hipSuccess;
  });
  return n;
}

hipError_t launch_clip(const ClipList& list, int power, double max_norm, bool scale, float* norm, double* partial,
                       hipStream_t stream) {
  int done = 0;
  hipError_t err = in_launches(list, [&](ClipArgs& a, int blocks) {
    a.partial = partial + done;
    done += blocks;
    if (power == 2) grad_norm_kernel<2><<<dim3(blocks), dim3(kBlock), 0, stream>>>(a);
    else if (power == 1) grad_norm_kernel<1><<<dim3(blocks), dim3(kBlock), 0, stream>>>(a);
    else grad_norm_kernel<0><<<dim3(blocks), dim3(kBlock), 0, stream>>>(a);
    return hipGetLastError();
  });
  if (err != hipSuccess) return err;
  if (!scale || done == 0) {
    ClipArgs a{};
    a.partial = partial;
    a.partials = done;
    a.power = power;
    a.norm = norm;
    norm_value_kernel<<<dim3(1), dim3(kBlock), 0, stream>>>(a);
    return hipGetLastError();
  }
  bool first = true;
  return in_launches(list, [&](ClipArgs& a, int blocks) {
    a.partial = partial;
    a.partials = done;
    a.power = power;
    a.max_norm = max_norm;
    a.norm = first ? norm : nullptr;
    a.inplace = list.dst == nullptr;
    if (a.inplace)
      for (int i = 0; i < a.tensors; ++i) a.entries[i].dst = const_cast<void*>(a.entries[i].src);
    first = false;
    clip_scale_kernel<<<dim3(blocks), dim3(kBlock), 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace fh
