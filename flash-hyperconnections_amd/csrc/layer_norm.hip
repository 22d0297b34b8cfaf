// Layer norm over rows of C elements:
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), n = (x - m) r, y = n w + b
// and its gradients, for q = g w:
//   dx = r (q - mean(q) - n mean(q n)),  dw = sum over rows of g n,  db = sum over rows of g.
//
// A row is read once and stays in the registers of the 1, 4, 8 or 16 wavefronts
// that share it, as the raw bits it came as; the variance is a second sum over
// those registers, so rows far off zero lose nothing to cancellation.  All sums
// are FP32.
//
// The parameters' gradients: a workgroup takes rows blockIdx, blockIdx + G, ...
// and every lane keeps the sums of its own columns in registers over them; the
// workgroup's row groups are added through LDS and the G partial rows of [2, C]
// floats by column_sums in a fixed order, so results do not change from call to
// call.
//
// Both directions are bound by HBM traffic: 16384 x 4096 bf16 takes 41 us forward (6.5
// TB/s) and 67 backward (6.0 TB/s); rows of 16384, 2048 of them in FP16, 24 (5.6) and 45,
// where the partial rows of 34 MB count.
#include <algorithm>

#include "fh_kernels.h"
#include "fh_plan.h"
#include "fh_vec.h"

namespace fh {
namespace {

constexpr int kBwdWaves = 8;

// Sum over the WPR wavefronts that share a row, through `area` (WPR floats a row
// group, unused between two calls on different areas).
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* area, int part) {
  v = wave_sum(v);
  if constexpr (WPR == 1) return v;
  if ((threadIdx.x & 63) == 0) area[part] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < WPR; ++i) s += area[i];
  return s;
}

// WPR wavefronts a row, GROUPS rows a workgroup at a time, NC vectors a lane.
template <typename T, bool Whole, int WPR, int GROUPS, int NC>
__global__ __launch_bounds__(64 * WPR * GROUPS) void norm_fwd_kernel(NormArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>;
  __shared__ float area[2][WPR * GROUPS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave / WPR, part = wave % WPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group;
  static_assert(WPR == 1 || GROUPS == 1, "barriers: a workgroup's wavefronts leave together");
  if (row >= a.rows) return;
  const S* x = static_cast<const S*>(a.x) + row * a.x_stride;
  S* y = static_cast<S*>(a.y) + row * a.cols;
  const int first = (part * 64 + lane) * V, cols = static_cast<int>(a.cols);
  U32x4 raw[NC];
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < NC; ++u) raw[u] = load_row<T, Whole>(x, first + u * (64 * WPR * V), cols);
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    float f[V];
    to_floats<T>(raw[u], f);
#pragma unroll
    for (int i = 0; i < V; ++i) sum += f[i];
  }
  const float inv = 1.f / static_cast<float>(a.cols);
  const float mean = row_sum<WPR>(sum, area[0] + group * WPR, part) * inv;
  float square = 0.f;
#pragma unroll
  for (int u = 0; u < NC; ++u) forget(raw[u]);
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int c = first + u * (64 * WPR * V);
    float f[V];
    to_floats<T>(raw[u], f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = c + (Whole ? 0 : i) < cols ? f[i] - mean : 0.f;
      square = __builtin_fmaf(d, d, square);
    }
  }
#pragma unroll
  for (int u = 0; u < NC; ++u) forget(raw[u]);
  const float var = row_sum<WPR>(square, area[1] + group * WPR, part) * inv;
  const float rstd = 1.f / __builtin_sqrtf(var + a.eps);
  if (a.stats != nullptr && part == 0 && lane == 0) {
    a.stats[2 * row] = mean;
    a.stats[2 * row + 1] = rstd;
  }
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int c = first + u * (64 * WPR * V);
    if (c >= cols) break;
    float f[V], w[V], b[V];
    to_floats<T>(raw[u], f);
    load_params<T>(a.weight, a.params_f32, c, cols, 1.f, w);
    load_params<T>(a.bias, a.params_f32, c, cols, 0.f, b);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __builtin_fmaf((f[i] - mean) * rstd, w[i], b[i]);
    store_row<T, Whole>(from_floats<T>(f), y, c, cols);
  }
}

// The same for rows that no workgroup's registers hold: the row is read three times.
template <typename T>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(NormArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, step = 1024 * V;
  __shared__ float area[2][16];
  const int64_t row = blockIdx.x;
  const int part = threadIdx.x >> 6;
  const S* x = static_cast<const S*>(a.x) + row * a.x_stride;
  S* y = static_cast<S*>(a.y) + row * a.cols;
  const int first = static_cast<int>(threadIdx.x) * V, cols = static_cast<int>(a.cols);
  const float inv = 1.f / static_cast<float>(a.cols);
  float sum = 0.f, square = 0.f, f[V], w[V], b[V];
  for (int c = first; c < cols; c += step) {
    to_floats<T>(load_row<T>(x, c, cols), f);
    float s = 0.f;  // a vector at a time: a chain of C / 1024 terms
#pragma unroll
    for (int i = 0; i < V; ++i) s += f[i];
    sum += s;
  }
  const float mean = row_sum<16>(sum, area[0], part) * inv;
  for (int c = first; c < cols; c += step) {
    to_floats<T>(load_row<T>(x, c, cols), f);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = c + i < cols ? f[i] - mean : 0.f;
      s = __builtin_fmaf(d, d, s);
    }
    square += s;
  }
  const float rstd = 1.f / __builtin_sqrtf(row_sum<16>(square, area[1], part) * inv + a.eps);
  if (a.stats != nullptr && threadIdx.x == 0) {
    a.stats[2 * row] = mean;
    a.stats[2 * row + 1] = rstd;
  }
  for (int c = first; c < cols; c += step) {
    to_floats<T>(load_row<T>(x, c, cols), f);
    load_params<T>(a.weight, a.params_f32, c, cols, 1.f, w);
    load_params<T>(a.bias, a.params_f32, c, cols, 0.f, b);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __builtin_fmaf((f[i] - mean) * rstd, w[i], b[i]);
    store_row<T>(from_floats<T>(f), y, c, cols);
  }
}

// dx, and with Params the workgroup's row of `partial` ([G, 2, C]: dw, db).  Eight
// wavefronts, whose registers hold the sums of up to four vectors of 16-bit columns a
// lane and the next row, which is loaded while this one is summed (the row groups
// wait for one another at every row).
template <typename T, bool Whole, int WPR, int NC, bool Params>
__global__ __launch_bounds__(64 * kBwdWaves) void norm_bwd_kernel(NormArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, GROUPS = kBwdWaves / WPR;
  constexpr int kWidth = 64 * WPR * V;  // columns of one vector of every lane of a row group
  __shared__ float2 area[2][kBwdWaves];
  __shared__ __attribute__((aligned(16))) float sums[Params ? GROUPS * 2 * kWidth : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave / WPR, part = wave % WPR;
  const int first = (part * 64 + lane) * V, cols = static_cast<int>(a.cols);
  const float inv = 1.f / static_cast<float>(cols);
  float w[NC][V], dw[Params ? NC : 1][V], db[Params ? NC : 1][V];
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    load_params<T>(a.weight, a.params_f32, first + u * kWidth, cols, 1.f, w[u]);
    if constexpr (Params) {
#pragma unroll
      for (int i = 0; i < V; ++i) dw[u][i] = db[u][i] = 0.f;
    }
  }
  // Rows blockIdx + G group, then G GROUPS further each turn; every group makes the
  // same number of turns.  Past the last row a group loads that row again and
  // neither adds nor stores.
  const int64_t stride = static_cast<int64_t>(gridDim.x) * GROUPS;
  const int turns = static_cast<int>((a.rows - blockIdx.x + stride - 1) / stride);
  int64_t row = blockIdx.x + static_cast<int64_t>(gridDim.x) * group;
  U32x4 xr[NC], gr[NC];
  float mean, rstd;
  const auto fetch = [&](int64_t r) {
    const int64_t at = r < a.rows ? r : a.rows - 1;
    const S* x = static_cast<const S*>(a.x) + at * a.x_stride;
    const S* g = static_cast<const S*>(a.grad) + at * a.grad_stride;
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      xr[u] = load_row<T, Whole>(x, first + u * kWidth, cols);
      gr[u] = load_row<T, Whole>(g, first + u * kWidth, cols);
    }
    mean = a.stats[2 * at];
    rstd = a.stats[2 * at + 1];
  };
  fetch(row);
  for (int t = 0; t < turns; ++t, row += stride) {
    const bool live = row < a.rows;
    U32x4 xc[NC], gc[NC];
#pragma unroll
    for (int u = 0; u < NC; ++u) xc[u] = xr[u], gc[u] = gr[u];
    const float m = mean, r = rstd;
    if (t + 1 < turns) fetch(row + stride);
    float s1 = 0.f, s2 = 0.f;
    if (live) {
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        float xf[V], gf[V];
        to_floats<T>(xc[u], xf);
        to_floats<T>(gc[u], gf);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // Past the row's end g and so q are 0.
          const float n = (xf[i] - m) * r, q = gf[i] * w[u][i];
          s1 += q;
          s2 = __builtin_fmaf(q, n, s2);
          if constexpr (Params) {
            dw[u][i] = __builtin_fmaf(gf[i], n, dw[u][i]);
            db[u][i] += gf[i];
          }
        }
        // One vector's values at a time.
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      forget(xc[u]);
      forget(gc[u]);
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if constexpr (WPR > 1) {
      // Two areas in turn: a wavefront writes one again after a barrier that follows
      // every read of it.
      if (lane == 0) area[t & 1][wave] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        const float2 v = area[t & 1][group * WPR + i];
        s1 += v.x;
        s2 += v.y;
      }
    }
    if (live) {
      const float c1 = s1 * inv, c2 = s2 * inv;
      S* dx = static_cast<S*>(a.y) + row * a.cols;
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        float xf[V], gf[V];
        to_floats<T>(xc[u], xf);
        to_floats<T>(gc[u], gf);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float n = (xf[i] - m) * r, q = gf[i] * w[u][i];
          xf[i] = r * (__builtin_fmaf(-n, c2, q) - c1);
        }
        store_row<T, Whole>(from_floats<T>(xf), dx, first + u * kWidth, cols);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if constexpr (Params) {
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      // The groups' sums of this vector's columns, added in order 0, 1, ....
      float* own = sums + group * 2 * kWidth + first;
      if (u > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        *reinterpret_cast<float4*>(own + i) = make_float4(dw[u][i], dw[u][i + 1], dw[u][i + 2], dw[u][i + 3]);
        *reinterpret_cast<float4*>(own + kWidth + i) = make_float4(db[u][i], db[u][i + 1], db[u][i + 2], db[u][i + 3]);
      }
      __syncthreads();
      for (int j = threadIdx.x; j < 2 * kWidth; j += 64 * kBwdWaves) {
        float s = sums[j];
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) s += sums[k * 2 * kWidth + j];
        const int c = j % kWidth + u * kWidth;
        if (c < cols) out[j / kWidth * a.cols + c] = s;
      }
    }
  }
}

// dx of rows that no workgroup's registers hold.
template <typename T>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(NormArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, step = 1024 * V;
  __shared__ float area[2][16];
  const int64_t row = blockIdx.x;
  const int part = threadIdx.x >> 6;
  const S* x = static_cast<const S*>(a.x) + row * a.x_stride;
  const S* g = static_cast<const S*>(a.grad) + row * a.grad_stride;
  S* dx = static_cast<S*>(a.y) + row * a.cols;
  const int first = static_cast<int>(threadIdx.x) * V, cols = static_cast<int>(a.cols);
  const float inv = 1.f / static_cast<float>(a.cols);
  const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
  float s1 = 0.f, s2 = 0.f, xf[V], gf[V], w[V];
  for (int c = first; c < cols; c += step) {
    to_floats<T>(load_row<T>(x, c, cols), xf);
    to_floats<T>(load_row<T>(g, c, cols), gf);
    load_params<T>(a.weight, a.params_f32, c, cols, 1.f, w);
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float q = gf[i] * w[i];
      t1 += q;
      t2 = __builtin_fmaf(q, (xf[i] - mean) * rstd, t2);
    }
    s1 += t1;
    s2 += t2;
  }
  const float c1 = row_sum<16>(s1, area[0], part) * inv;
  const float c2 = row_sum<16>(s2, area[1], part) * inv;
  for (int c = first; c < cols; c += step) {
    to_floats<T>(load_row<T>(x, c, cols), xf);
    to_floats<T>(load_row<T>(g, c, cols), gf);
    load_params<T>(a.weight, a.params_f32, c, cols, 1.f, w);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float n = (xf[i] - mean) * rstd, q = gf[i] * w[i];
      xf[i] = rstd * (__builtin_fmaf(-n, c2, q) - c1);
    }
    store_row<T>(from_floats<T>(xf), dx, c, cols);
  }
}

// The workgroup's row of `partial` for such rows: 1024 columns at rows blockIdx.y, + gridDim.y, ....
template <typename T>
__global__ __launch_bounds__(1024) void norm_params_long_kernel(NormArgs a) {
  using S = typename T::storage;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float x = to_f32<T>(static_cast<const S*>(a.x)[row * a.x_stride + c]);
    const float g = to_f32<T>(static_cast<const S*>(a.grad)[row * a.grad_stride + c]);
    dw = __builtin_fmaf(g, (x - a.stats[2 * row]) * a.stats[2 * row + 1], dw);
    db += g;
  }
  float* out = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
  out[c] = dw;
  out[a.cols + c] = db;
}

// Column sums of `partial` [count, width] from column `begin` on: sixteen wavefronts take
// every sixteenth row, their sums are added in order.  Columns below `split` go to
// `first`, the others to `second`.
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* partial, int count, int64_t width,
                                                           int64_t begin, int64_t split, void* first, void* second,
                                                           int dtype) {
  __shared__ float area[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = begin + static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float s = 0.f;
  if (c < width)
#pragma unroll 8
    for (int k = wave; k < count; k += 16) s += partial[k * width + c];
  area[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= width) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += area[k][lane];
  void* out = c < split ? first : second;
  const int64_t at = c < split ? c : c - split;
  if (out == nullptr) return;
  if (dtype == F32::code) store_elem<F32>(out, at, s);
  if (dtype == BF16::code) store_elem<BF16>(out, at, s);
  if (dtype == F16::code) store_elem<F16>(out, at, s);
}

// launch(args, workgroups) for as many rows at a time as workgroups of `threads` threads and
// `groups` rows may be in one launch, up to the first that fails.
template <typename T, typename Launch>
hipError_t in_row_ranges(const NormArgs& a, int groups, int threads, Launch launch) {
  return in_slices(a.rows, most_groups(threads) * groups, [&](int64_t first, int64_t count) {
    using S = typename T::storage;
    NormArgs part = a;
    part.x = static_cast<const S*>(a.x) + first * a.x_stride;
    if (a.grad != nullptr) part.grad = static_cast<const S*>(a.grad) + first * a.grad_stride;
    part.y = static_cast<S*>(a.y) + first * a.cols;
    if (a.stats != nullptr) part.stats = a.stats + 2 * first;
    part.rows = count;
    launch(part, dim3(static_cast<uint32_t>((count + groups - 1) / groups)));
    return hipGetLastError();
  });
}

template <typename T, int WPR, int GROUPS, int NC>
hipError_t fwd(const NormArgs& a, hipStream_t stream) {
  constexpr int threads = 64 * WPR * GROUPS;
  return in_row_ranges<T>(a, GROUPS, threads, [&](const NormArgs& part, dim3 grid) {
    if (a.cols % kVec<T> == 0) {
      norm_fwd_kernel<T, true, WPR, GROUPS, NC><<<grid, dim3(threads), 0, stream>>>(part);
    } else {
      norm_fwd_kernel<T, false, WPR, GROUPS, NC><<<grid, dim3(threads), 0, stream>>>(part);
    }
  });
}

template <typename T, bool Whole, int WPR, int NC>
hipError_t bwd_rows(const NormArgs& a, int blocks, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(blocks)), block(64 * kBwdWaves);
  if (a.partial != nullptr) {
    norm_bwd_kernel<T, Whole, WPR, NC, true><<<grid, block, 0, stream>>>(a);
  } else {
    norm_bwd_kernel<T, Whole, WPR, NC, false><<<grid, block, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T, int WPR, int NC>
hipError_t bwd(const NormArgs& a, int blocks, hipStream_t stream) {
  return a.cols % kVec<T> == 0 ? bwd_rows<T, true, WPR, NC>(a, blocks, stream)
                               : bwd_rows<T, false, WPR, NC>(a, blocks, stream);
}

constexpr int64_t kMostVectors = 4096;    // of a forward row in registers
constexpr int64_t kMostBackward = 16384;  // columns of a backward row in registers

int64_t vectors(int dtype, int64_t cols) {
  const int v = dtype == F32::code ? 4 : 8;
  return (cols + v - 1) / v;
}

}  // namespace

hipError_t launch_column_sums(const float* partial, int count, int64_t width, int64_t split, void* first,
                              void* second, int dtype, hipStream_t stream) {
  return in_slices(width, most_groups(1024) * 64, [&](int64_t begin, int64_t columns) {
    column_sums_kernel<<<dim3(static_cast<uint32_t>((columns + 63) / 64)), dim3(1024), 0, stream>>>(
        partial, count, width, begin, split, first, second, dtype);
    return hipGetLastError();
  });
}

int norm_blocks(int dtype, int64_t rows, int64_t cols) {
  if (cols > kMostBackward) return static_cast<int>(std::min<int64_t>(rows, 64));
  return static_cast<int>(std::min<int64_t>(rows, compute_units()));
}

hipError_t launch_norm(const NormArgs& a, int dtype, hipStream_t stream) {
  const int64_t nv = vectors(dtype, a.cols);
  return with_type(dtype, [&](auto t) -> hipError_t {
    using T = decltype(t);
    if (nv > kMostVectors) {
      return in_row_ranges<T>(a, 1, 1024, [&](const NormArgs& part, dim3 grid) {
        norm_fwd_long_kernel<T><<<grid, dim3(1024), 0, stream>>>(part);
      });
    }
    if (nv <= 64) return fwd<T, 1, 4, 1>(a, stream);
    if (nv <= 128) return fwd<T, 1, 4, 2>(a, stream);
    // Few rows: four wavefronts to each, for the time that one row takes (64 x 4096 bf16: 7.7 -> 4.4 us).
    if (nv <= 512 && a.rows <= 2 * compute_units())
      return nv <= 256 ? fwd<T, 4, 1, 1>(a, stream) : fwd<T, 4, 1, 2>(a, stream);
    if (nv <= 256) return fwd<T, 1, 4, 4>(a, stream);
    if (nv <= 512) return fwd<T, 1, 4, 8>(a, stream);
    if (nv <= 1024) return fwd<T, 4, 1, 4>(a, stream);
    if (nv <= 2048) return fwd<T, 4, 1, 8>(a, stream);
    return fwd<T, 8, 1, 8>(a, stream);
  });
}

hipError_t launch_norm_backward(const NormArgs& a, void* dweight, void* dbias, int param_dtype, int dtype,
                                hipStream_t stream) {
  const int64_t nv = vectors(dtype, a.cols);
  const int blocks = norm_blocks(dtype, a.rows, a.cols);
  hipError_t err = with_type(dtype, [&](auto t) -> hipError_t {
    using T = decltype(t);
    if (a.cols > kMostBackward) {
      const hipError_t err = in_row_ranges<T>(a, 1, 1024, [&](const NormArgs& part, dim3 grid) {
        norm_bwd_long_kernel<T><<<grid, dim3(1024), 0, stream>>>(part);
      });
      if (err != hipSuccess) return err;
      if (a.partial != nullptr)
        norm_params_long_kernel<T><<<dim3(static_cast<uint32_t>((a.cols + 1023) / 1024), blocks), dim3(1024), 0,
                                     stream>>>(a);
      return hipGetLastError();
    }
    if (nv <= 64) return bwd<T, 1, 1>(a, blocks, stream);
    if (nv <= 128) return bwd<T, 1, 2>(a, blocks, stream);
    if (nv <= 256) return bwd<T, 1, 4>(a, blocks, stream);
    if (nv <= 512) return bwd<T, 2, 4>(a, blocks, stream);
    if (nv <= 1024) return bwd<T, 4, 4>(a, blocks, stream);
    if (nv <= 2048) return bwd<T, 8, 4>(a, blocks, stream);
    if constexpr (T::code == F32::code) return bwd<T, 8, 8>(a, blocks, stream);
    return hipErrorInvalidValue;  // 16384 columns are 2048 vectors of a 16-bit type
  });
  if (err != hipSuccess || a.partial == nullptr) return err;
  return launch_column_sums(a.partial, blocks, 2 * a.cols, a.cols, dweight, dbias, param_dtype, stream);
}

}  // namespace fh
