// Matrix products of the linear layer in 128 x 128 tiles, where tiles of 256 are too
// few to fill the card, and the joining of sums in several slices.
//
// Such products are short: what costs is the time from one step's loads to the next.
// So a compute unit holds one workgroup, of eight wavefronts with 32 x 64 results each,
// whose four buffers keep three steps of 64 on their way (two workgroups with one step
// each on its way took twice as long a step).  The wavefronts meet once a step.
#include <algorithm>
#include <type_traits>

#include "linear_tiles.h"

namespace fh {
namespace {

constexpr int kTile = 128, kRing = 4;
constexpr int kBuffer = kTile * kStep * 2;  // bytes of one operand's step

// k = 32 half .. + 31 of the step in buffer R; y: [2 kk + tile].
template <int R, bool ACols, bool BCols>
__device__ __forceinline__ void read_half(const Finder<ACols, kTile>& fa, const Finder<BCols, kTile>& fb, int half,
                                          U32x4 (&x)[2], U32x4 (&y)[4]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    x[kk] = fa.read(R * kBuffer, 0, 2 * half + kk);
    y[2 * kk] = fb.read(R * kBuffer, 0, 2 * half + kk);
    y[2 * kk + 1] = fb.read(R * kBuffer, 1, 2 * half + kk);
  }
}

// B's rows as the instruction's rows: a lane then holds four neighbouring n of one m.
template <typename E>
__device__ __forceinline__ void multiply(Floats16 (&acc)[2], U32x4 x, U32x4 y0, U32x4 y1) {
  acc[0] = mfma32<E>(y0, x, acc[0]);
  acc[1] = mfma32<E>(y1, x, acc[1]);
}

// The step in buffer R.  x0 and y0 hold its first half, and after it the next one's.
template <int R, typename T, bool ACols, bool BCols>
__device__ __forceinline__ void step(Feeder<ACols, kTile>& a, Feeder<BCols, kTile>& b,
                                     const Finder<ACols, kTile>& fa, const Finder<BCols, kTile>& fb,
                                     Floats16 (&acc)[2], U32x4 (&x0)[2], U32x4 (&x1)[2], U32x4 (&y0)[4],
                                     U32x4 (&y1)[4]) {
  read_half<R>(fa, fb, 1, x1, y1);
  multiply<T>(acc, x0[0], y0[0], y0[1]);
  multiply<T>(acc, x0[1], y0[2], y0[3]);
  __builtin_amdgcn_sched_barrier(0);
  // This step's buffer has been read, and the next one's loads are there once only the
  // four of each of the two steps behind it are on their way.
  wait_lds();
  wait_loads<8>();
  meet();
  read_half<(R + 1) % kRing>(fa, fb, 0, x0, y0);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    a.stage(u, R * kBuffer);
    b.stage(u, R * kBuffer);
    multiply<T>(acc, x1[u], y1[2 * u], y1[2 * u + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  a.advance();
  b.advance();
}

template <typename T, bool ACols, bool BCols>
__global__ __launch_bounds__(512) void product_kernel(ProductArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * kRing * kBuffer];  // A's ring, B's ring
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * kTile, n0 = tile.n * kTile, slice = blockIdx.y;
  const Steps<kStep> steps(p, slice);
  const int count = steps.end - steps.begin;
  Feeder<ACols, kTile> a;
  Feeder<BCols, kTile> b;
  a.init(p.a, p.lda, m0, p.m, p.k, steps.begin, lds_address(lds), lane, wave);
  b.init(p.b, p.ldb, n0, p.n, p.k, steps.begin, lds_address(lds) + kRing * kBuffer, lane, wave);
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 64;
  const Finder<ACols, kTile> fa(lds_address(lds), wm, lane);
  const Finder<BCols, kTile> fb(lds_address(lds) + kRing * kBuffer, wn, lane);
  Floats16 acc[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
  if (count > 0) {
#pragma unroll
    for (int s = 0; s < kRing; ++s) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        a.stage(u, s * kBuffer);
        b.stage(u, s * kBuffer);
      }
      a.advance();
      b.advance();
    }
    wait_loads<4 * (kRing - 1)>();
    meet();
    U32x4 x0[2], x1[2], y0[4], y1[4];
    read_half<0>(fa, fb, 0, x0, y0);
    // Loads and reads go on past the last step, of zeros.
    for (int s = 0; s < count; s += 4) {
      step<0, T>(a, b, fa, fb, acc, x0, x1, y0, y1);
      if (s + 1 < count) step<1, T>(a, b, fa, fb, acc, x0, x1, y0, y1);
      if (s + 2 < count) step<2, T>(a, b, fa, fb, acc, x0, x1, y0, y1);
      if (s + 3 < count) step<3, T>(a, b, fa, fb, acc, x0, x1, y0, y1);
    }
  }
  wait_loads<0>();
  __syncthreads();  // the buffers have been read: each wavefront takes 8 KB of them
  char* area = lds + wave * 8192;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      park(area, lane & 31, 8 * j + 2 * q + (lane >> 5),
           Floats4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]});
  finish_parked<T, 32>(p, slice, area, m0 + wm, n0 + wn, lane);
}

// Sums of one step, at most 64 terms: two workgroups a compute unit, one storing while
// the other loads.
template <typename T, bool ACols, bool BCols>
__global__ __launch_bounds__(512, 4) void outer_product_kernel(ProductArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[8 * 8192];  // A's and B's step, then the results
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * kTile, n0 = tile.n * kTile;
  Feeder<ACols, kTile> a;
  Feeder<BCols, kTile> b;
  a.init(p.a, p.lda, m0, p.m, p.k, 0, lds_address(lds), lane, wave);
  b.init(p.b, p.ldb, n0, p.n, p.k, 0, lds_address(lds) + kBuffer, lane, wave);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    a.stage(u, 0);
    b.stage(u, 0);
  }
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 64;
  const Finder<ACols, kTile> fa(lds_address(lds), wm, lane);
  const Finder<BCols, kTile> fb(lds_address(lds) + kBuffer, wn, lane);
  Floats16 acc[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
  wait_loads<0>();
  meet();
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (16 * kk >= p.k) break;
    multiply<T>(acc, fa.read(0, 0, kk), fb.read(0, 0, kk), fb.read(0, 1, kk));
  }
  wait_lds();
  meet();
  char* area = lds + wave * 8192;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      park(area, lane & 31, 8 * j + 2 * q + (lane >> 5),
           Floats4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]});
  finish_parked<T, 32>(p, 0, area, m0 + wm, n0 + wn, lane);
}

// Adds the slices in order and finishes.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(ProductArgs p) {
  const int across = (p.n + 7) / 8, slices = p.slices;
  const int64_t total = static_cast<int64_t>(p.m) * across, size = static_cast<int64_t>(p.m) * p.n;
  p.slices = 1;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < total;
       q += static_cast<int64_t>(gridDim.x) * 256) {
    const int row = static_cast<int>(q / across), col = static_cast<int>(q % across) * 8;
    float sum[8] = {}, v[8];
    const float* from = p.partial + static_cast<int64_t>(row) * p.n + col;
    for (int s = 0; s < slices; ++s, from += size) {
      load_eight(from, p.n - col, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
    finish_eight<T>(p, 0, row, col, sum);
  }
}

template <typename T>
hipError_t run(const ProductArgs& p, bool a_cols, bool b_cols, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.tiles_m * p.tiles_n), static_cast<uint32_t>(p.slices)), block(512);
  if (p.k <= kStep && p.slices == 1) {
    if (!a_cols && !b_cols) outer_product_kernel<T, false, false><<<grid, block, 0, stream>>>(p);
    if (!a_cols && b_cols) outer_product_kernel<T, false, true><<<grid, block, 0, stream>>>(p);
    if (a_cols && b_cols) outer_product_kernel<T, true, true><<<grid, block, 0, stream>>>(p);
    return hipGetLastError();
  }
  if (!a_cols && !b_cols) product_kernel<T, false, false><<<grid, block, 0, stream>>>(p);
  if (!a_cols && b_cols) product_kernel<T, false, true><<<grid, block, 0, stream>>>(p);
  if (a_cols && b_cols) product_kernel<T, true, true><<<grid, block, 0, stream>>>(p);
  if (a_cols && !b_cols) return hipErrorInvalidValue;  // no such product
  return hipGetLastError();
}

template <typename T>
hipError_t join(const ProductArgs& p, hipStream_t stream) {
  const int64_t groups = static_cast<int64_t>(p.m) * ((p.n + 7) / 8);
  join_kernel<T><<<dim3(static_cast<uint32_t>(std::min<int64_t>((groups + 255) / 256, 4096))), dim3(256), 0,
                   stream>>>(p);
  return hipGetLastError();
}

void set_tiles(ProductArgs& p, int side) {
  p.side = side;
  p.tiles_m = (p.m + side - 1) / side;
  p.tiles_n = (p.n + side - 1) / side;
}

}  // namespace

void plan_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols) {
  const bool f32 = dtype == F32::code;
  if (!f32 && plan_narrow_product(p, a_cols, b_cols)) return;
  if (!f32 && p.k <= kStep) {
    set_tiles(p, kTile);
    p.slices = 1;
    return;
  }
  const int64_t units = compute_units();
  const auto rounds = [&](int64_t groups) { return static_cast<double>((groups + units - 1) / units); };
  // Microseconds, measured: a workgroup of a tile of 256 takes 5 and 1.15 a step of 64, one of a tile
  // of 128 takes 3 and 0.8 (FP32: 1.0 a step of 32); slices cost a launch and their sums' way to
  // memory and back.
  set_tiles(p, kTile);
  const int64_t steps = f32 ? (p.k + 31) / 32 : (p.k + 63) / 64;
  const double step = f32 ? 1.0 : 0.8;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  const double results = static_cast<double>(p.m) * p.n;
  double best = 0.0;
  for (int64_t s = 1; s <= 16 && s <= std::max<int64_t>(1, steps / 4); ++s) {
    const double us = rounds(tiles * s) * (3.0 + step * static_cast<double>((steps + s - 1) / s)) +
                      (s > 1 ? 4.0 + results * 1e-6 * static_cast<double>(s + 1) : 0.0);
    if (s == 1 || us < best) {
      best = us;
      p.slices = static_cast<int>(s);
    }
  }
  if (f32) return;
  ProductArgs wide = p;
  set_tiles(wide, 256);
  wide.slices = 1;
  if (rounds(static_cast<int64_t>(wide.tiles_m) * wide.tiles_n) * (5.0 + 1.15 * static_cast<double>(steps)) < best)
    p = wide;
}

hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream) {
  hipError_t err;
  if (dtype == F32::code) {
    err = launch_f32_product(p, a_cols, b_cols, stream);
  } else if (p.side == 256) {
    err = launch_wide_product(p, dtype, a_cols, b_cols, stream);
  } else if (p.side == kTile) {
    err = with_half_type(dtype, [&](auto t) { return run<decltype(t)>(p, a_cols, b_cols, stream); });
  } else {
    err = launch_narrow_product(p, dtype, a_cols, b_cols, stream);
  }
  if (err != hipSuccess || p.slices == 1) return err;
  return with_type(dtype, [&](auto t) { return join<decltype(t)>(p, stream); });
}

}  // namespace fh
