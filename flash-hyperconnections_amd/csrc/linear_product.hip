// Matrix products of the linear layer in tiles of 128 or 256 rows by 128 columns, where
// tiles of 256 x 256 are too few to fill the card, and the joining of sums in several
// slices.
//
// A compute unit holds one workgroup of eight wavefronts, whose buffers keep two or
// three steps of 64 on their way.  The wavefronts meet once a step.  The smaller tile asks
// the L2 for 32 KB a step of 1 M multiply-adds: 14 TB/s over 1024 x 4096 x 4096 in 37 us.
#include <algorithm>
#include <type_traits>

#include "linear_tiles.h"

namespace fh {
namespace {

constexpr int kTile = 128;
constexpr int kBuffer = kTile * kStep * 2;  // bytes of one operand's step of 128 rows

// A tile of 128 or 256 rows by 128 columns: 32 Tall x 64 results a wavefront, and the
// steps that its LDS holds.
template <int Tall>
struct Shape {
  static constexpr int kRows = kTile * Tall, kRing = Tall == 1 ? 4 : 3;
  static constexpr int kA = kRows * kStep * 2, kB = kBuffer;    // bytes of an operand's step
  static constexpr int kLoads = 2 * Tall + 2;                   // of a wavefront's in a step
};

// k = 32 half .. + 31 of the step in buffer R; x: [Tall kk + tile], y: [2 kk + tile].
template <int R, int Tall, bool ACols, bool BCols>
__device__ __forceinline__ void read_half(const Finder<ACols, kTile * Tall>& fa, const Finder<BCols, kTile>& fb,
                                          int half, U32x4 (&x)[2 * Tall], U32x4 (&y)[4]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
    for (int i = 0; i < Tall; ++i) x[Tall * kk + i] = fa.read(R * Shape<Tall>::kA, i, 2 * half + kk);
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
template <int R, typename T, int Tall, bool ACols, bool BCols>
__device__ __forceinline__ void step(Feeder<ACols, kTile * Tall>& a, Feeder<BCols, kTile>& b,
                                     const Finder<ACols, kTile * Tall>& fa, const Finder<BCols, kTile>& fb,
                                     Floats16 (&acc)[Tall][2], U32x4 (&x0)[2 * Tall], U32x4 (&x1)[2 * Tall],
                                     U32x4 (&y0)[4], U32x4 (&y1)[4]) {
  constexpr int kRing = Shape<Tall>::kRing;
  read_half<R, Tall>(fa, fb, 1, x1, y1);
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int i = 0; i < Tall; ++i) multiply<T>(acc[i], x0[Tall * kk + i], y0[2 * kk], y0[2 * kk + 1]);
  __builtin_amdgcn_sched_barrier(0);
  // This step's buffer has been read, and the next one's loads are there once only those
  // of the steps behind it are on their way.
  wait_lds();
  wait_loads<(kRing - 2) * Shape<Tall>::kLoads>();
  meet();
  read_half<(R + 1) % kRing, Tall>(fa, fb, 0, x0, y0);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int i = 0; i < Tall; ++i) {
      a.stage(Tall * u + i, R * Shape<Tall>::kA);
      if (i == 0) b.stage(u, R * kBuffer);
      multiply<T>(acc[i], x1[Tall * u + i], y1[2 * u], y1[2 * u + 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  a.advance();
  b.advance();
}

template <typename T, int Tall, bool ACols, bool BCols>
__global__ __launch_bounds__(512, 2) void product_kernel(ProductArgs p) {
  using S = Shape<Tall>;
  constexpr int kRing = S::kRing;
  __shared__ __attribute__((aligned(1024))) char lds[kRing * (S::kA + S::kB)];  // A's ring, B's ring
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * S::kRows, n0 = tile.n * kTile, slice = blockIdx.y;
  const Steps<kStep> steps(p, slice);
  const int count = steps.end - steps.begin;
  Feeder<ACols, kTile * Tall> a;
  Feeder<BCols, kTile> b;
  a.init(p.a, p.lda, m0, p.m, p.k, steps.begin, lds_address(lds), lane, wave);
  b.init(p.b, p.ldb, n0, p.n, p.k, steps.begin, lds_address(lds) + kRing * S::kA, lane, wave);
  const int wm = (wave >> 1) * 32 * Tall, wn = (wave & 1) * 64;
  const Finder<ACols, kTile * Tall> fa(lds_address(lds), wm, lane);
  const Finder<BCols, kTile> fb(lds_address(lds) + kRing * S::kA, wn, lane);
  Floats16 acc[Tall][2];
#pragma unroll
  for (int i = 0; i < Tall; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  if (count > 0) {
#pragma unroll
    for (int s = 0; s < kRing; ++s) {
#pragma unroll
      for (int u = 0; u < 2 * Tall; ++u) a.stage(u, s * S::kA);
#pragma unroll
      for (int u = 0; u < 2; ++u) b.stage(u, s * kBuffer);
      a.advance();
      b.advance();
    }
    wait_loads<S::kLoads * (kRing - 1)>();
    meet();
    U32x4 x0[2 * Tall], x1[2 * Tall], y0[4], y1[4];
    read_half<0, Tall>(fa, fb, 0, x0, y0);
    // Loads and reads go on past the last step, of zeros.
    for (int s = 0; s < count; s += kRing) {
      step<0, T, Tall>(a, b, fa, fb, acc, x0, x1, y0, y1);
      if (s + 1 < count) step<1, T, Tall>(a, b, fa, fb, acc, x0, x1, y0, y1);
      if (s + 2 < count) step<2, T, Tall>(a, b, fa, fb, acc, x0, x1, y0, y1);
      if constexpr (kRing == 4) {
        if (s + 3 < count) step<3, T, Tall>(a, b, fa, fb, acc, x0, x1, y0, y1);
      }
    }
  }
  wait_loads<0>();
  __syncthreads();  // the buffers have been read: each wavefront takes a part of them
  char* area = lds + wave * 8192 * Tall;
#pragma unroll
  for (int i = 0; i < Tall; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const Floats16& v = acc[i][j];
        park(area, 32 * i + (lane & 31), 8 * j + 2 * q + (lane >> 5),
             Floats4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
      }
  finish_parked<T, 32 * Tall>(p, slice, area, m0 + wm, n0 + wn, lane);
}

// Sums of one step, at most 64 terms: two workgroups a compute unit, one storing while
// the other loads.  Bound by the stores: 16384 x 16 x 16384 bf16 (537 MB) takes 124 to
// 137 us; tiles of 256 x 256 took 157 to 166, the 128 x 128 tiles with a ring 179.
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

// sum += Count slices `size` apart, in order, all on their way at once.
template <int Count>
__device__ __forceinline__ void add_slices(const float*& from, int64_t size, int left, float (&sum)[8]) {
  float v[Count][8];
#pragma unroll
  for (int u = 0; u < Count; ++u, from += size) load_some(from, left, v[u]);
#pragma unroll
  for (int u = 0; u < Count; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += v[u][e];
}

// Adds the slices in order and finishes.  Bound by the loads' latency: 12 slices of 16 x
// 16384 sums take 5.3 us, and took 7.9 with each waited for; 8 of 64 x 4096 take 4.1 and
// took 5.1.  (Workgroups of one wavefront and of four take the same time.)
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(ProductArgs p) {
  const int across = (p.n + 7) / 8, slices = p.slices;
  const int64_t total = static_cast<int64_t>(p.m) * across, size = static_cast<int64_t>(p.m) * p.n;
  p.slices = 1;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < total;
       q += static_cast<int64_t>(gridDim.x) * 256) {
    const int row = static_cast<int>(q / across), col = static_cast<int>(q % across) * 8;
    float sum[8] = {};
    const float* from = p.partial + static_cast<int64_t>(row) * p.n + col;
    const int left = p.n - col;
    for (int s = 8; s <= slices; s += 8) add_slices<8>(from, size, left, sum);
    if (slices & 4) add_slices<4>(from, size, left, sum);
    if (slices & 2) add_slices<2>(from, size, left, sum);
    if (slices & 1) add_slices<1>(from, size, left, sum);
    finish_some<T>(p, 0, row, col, sum);
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
  if (p.side_m == kTile) {
    if (!a_cols && !b_cols) product_kernel<T, 1, false, false><<<grid, block, 0, stream>>>(p);
    if (!a_cols && b_cols) product_kernel<T, 1, false, true><<<grid, block, 0, stream>>>(p);
    if (a_cols && b_cols) product_kernel<T, 1, true, true><<<grid, block, 0, stream>>>(p);
  } else {
    if (!a_cols && !b_cols) product_kernel<T, 2, false, false><<<grid, block, 0, stream>>>(p);
    if (!a_cols && b_cols) product_kernel<T, 2, false, true><<<grid, block, 0, stream>>>(p);
    if (a_cols && b_cols) product_kernel<T, 2, true, true><<<grid, block, 0, stream>>>(p);
  }
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

void set_tiles(ProductArgs& p, int rows, int cols) {
  p.side_m = rows;
  p.side_n = cols;
  p.tiles_m = (p.m + rows - 1) / rows;
  p.tiles_n = (p.n + cols - 1) / cols;
}

}  // namespace

void plan_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols) {
  const bool f32 = dtype == F32::code;
  if (plan_narrow_product(p, dtype, a_cols, b_cols)) return;
  if (p.k <= (f32 ? 32 : kStep)) {
    set_tiles(p, kTile, kTile);
    p.slices = 1;
    return;
  }
  const int64_t units = compute_units();
  const auto rounds = [&](int64_t groups) { return static_cast<double>((groups + units - 1) / units); };
  // Microseconds of a workgroup: fixed, and a step of 64 (FP32: 32) with one workgroup on the
  // card and what a full card adds.  Slices cost a launch and their sums' way to memory and
  // back.  Fitted to 128 .. 4096 x 4096 x 4096, 2048 x 1024 x 4096, 64 x 16384 x 4096 and
  // 3000 x 700 x 5000 in each tile and 1 to 16 slices.  The times it gives are up to 13% off
  // (40% at 3000 x 700 x 5000, whose operands are laid out first); of sixteen shapes swept,
  // fourteen had the chosen form among those timed, each within 1 us of the fastest.  For
  // instance 1024 x 4096 x 4096 bf16: 39 us in 128 x 128 (chosen), 48 in 256 x 128, 54 in
  // 256 x 256 at their best slices; FP32 2048 x 4096 x 4096: 405 and 352 (chosen).
  struct Cost {
    int rows, cols;
    double fixed, step, shared;
  };
  constexpr Cost kF32[] = {{kTile, kTile, 4.2, 1.27, 0.3}, {2 * kTile, kTile, 7.0, 2.1, 0.55}};
  constexpr Cost kHalf[] = {
      {kTile, kTile, 4.2, 0.33, 0.2}, {2 * kTile, kTile, 7.0, 0.56, 0.34}, {256, 256, 10.0, 1.0, 0.55}};
  const int64_t steps = f32 ? (p.k + 31) / 32 : (p.k + 63) / 64;
  const double results = static_cast<double>(p.m) * p.n;
  double best = -1.0;
  ProductArgs chosen = p;
  const auto consider = [&](const Cost& c) {
    set_tiles(p, c.rows, c.cols);
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    for (int64_t s = 1; s <= 16 && s <= std::max<int64_t>(1, steps / 4); ++s) {
      const double full = std::min(1.0, static_cast<double>(tiles * s) / static_cast<double>(units));
      const double us =
          rounds(tiles * s) * (c.fixed + (c.step + c.shared * full) * static_cast<double>((steps + s - 1) / s)) +
          (s > 1 ? 3.5 + 1.3e-6 * results * static_cast<double>(s) : 0.0);
      if (best < 0.0 || us < best) {
        best = us;
        p.slices = static_cast<int>(s);
        chosen = p;
      }
    }
  };
  if (f32) {
    for (const Cost& c : kF32) consider(c);
  } else {
    for (const Cost& c : kHalf) consider(c);
  }
  p = chosen;
}

hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream) {
  hipError_t err;
  if (p.side_n < kTile) {
    err = launch_narrow_product(p, dtype, a_cols, b_cols, stream);
  } else if (dtype == F32::code) {
    err = launch_f32_product(p, a_cols, b_cols, stream);
  } else if (p.side_n == 256) {
    err = launch_wide_product(p, dtype, a_cols, b_cols, stream);
  } else {
    err = with_half_type(dtype, [&](auto t) { return run<decltype(t)>(p, a_cols, b_cols, stream); });
  }
  if (err != hipSuccess || p.slices == 1) return err;
  return with_type(dtype, [&](auto t) { return join<decltype(t)>(p, stream); });
}

}  // namespace fh
