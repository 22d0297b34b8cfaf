// FP32 matrix products of the linear layer in tiles of 128 or 256 rows by 128 columns,
// on the bf16 matrix instructions: sixteen times the rate of the FP32 ones.
//
// A value is the exact sum of three bf16 parts of eight bits each, cut off rather than
// rounded, so that nothing overflows.  Six of the nine products of parts make an FP32
// product to about 2^-23; the leading ones and the five smaller ones have accumulators
// of their own, so that the small terms are not rounded to the large sums' last bits.
//
// The parts are formed on the way from global memory to LDS: the operands are read as
// they are, four bytes an element at any alignment, and half as many panels go through
// LDS as if each product of parts read its own.
//
// A step of 32 of the sum's terms takes a wavefront of the smaller tile 24 matrix
// instructions and 150 others, 1.3 to 1.6 us; the larger tile's does twice the products for
// 1.6 times the splitting in 2.1 to 2.7 us.  2048 x 4096 x 4096 took 405 us in the one and
// 352 in the other, and takes 337 (204 TFLOP/s) since results leave in whole lines.  Smaller
// products stay well below that: in the three of 1500 x 1027 x 771, 63 to 108 tiles in 2 to
// 4 slices, a compute unit has one workgroup of 11 to 13 steps, and the matrix cores are busy
// 36 to 38% of the time.  What of splitting, LDS writes, barriers and the joins of slices
// takes the rest was not separated.
#include <algorithm>

#include "linear_parts.h"

namespace fh {
namespace {

constexpr int kTile = 128, kDepth = 32, kThreads = 512;
template <int Side>
constexpr int kPanel = Side * kDepth * 2;  // bytes of one part of one operand's step

typedef short S16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
using LdsShorts = __attribute__((address_space(3))) S16x4;
using LdsBytes = __attribute__((address_space(3))) char;

__device__ __forceinline__ int swap_of(int k) { return 2 * (((k & 3) << 1) | ((k >> 3) & 1)); }

// One operand's way from memory to LDS.  In rows: Side rows of 32, 16-byte chunk c of
// row r at place c ^ ((r >> 3) & 3); a thread takes four terms of every 64th row.  In
// columns: 32 rows of Side, chunk c of row k at place c ^ swap_of(k); a thread takes four
// columns of every few rows.
template <bool Cols, int Side>
struct Mover {
  static constexpr int kPasses = Side / 64;
  const float* at[kPasses];
  int64_t step;
  int k[kPasses], left;  // this thread's first terms; the sum's terms from here on
  int columns;           // in columns: valid ones of this thread's four
  uint32_t to[kPasses];
  bool inside;           // every row (column) of the tile is valid
  float v[kPasses][4];

  __device__ __forceinline__ void init(const float* data, int64_t ld, int first, int count, int t0, int k_all,
                                       uint32_t lds) {
    const int t = threadIdx.x;
    inside = first + Side <= count;
    left = k_all - t0 * kDepth;
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
      if constexpr (Cols) {
        const int row = t / (Side / 4) + 2048 / Side * u, col = t % (Side / 4) * 4;
        k[u] = row;
        columns = count - first - col;
        at[u] = data + (static_cast<int64_t>(t0) * kDepth + row) * ld + first + col;
        to[u] = lds + row * (2 * Side) + (((col >> 3) ^ swap_of(row)) << 4) + (col & 4) * 2;
      } else {
        const int row = t / 8 + 64 * u, term = t % 8 * 4;
        k[u] = term;
        at[u] = data + static_cast<int64_t>(first + row < count ? first + row : count - 1) * ld + t0 * kDepth + term;
        to[u] = lds + row * (2 * kDepth) + (((term >> 3) ^ ((row >> 3) & 3)) << 4) + (term & 4) * 2;
      }
    }
    step = Cols ? kDepth * ld : kDepth;
  }
  // Begins this step's loads, zeros past the sum's end and the last column.
  __device__ __forceinline__ void fetch() {
    if (left >= kDepth && (!Cols || inside)) {
#pragma unroll
      for (int u = 0; u < kPasses; ++u) __builtin_memcpy(v[u], at[u], 16);
    } else {
#pragma unroll
      for (int u = 0; u < kPasses; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool valid = Cols ? k[u] < left && i < columns : k[u] + i < left;
          v[u][i] = valid ? at[u][i] : 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) at[u] += step;
    left -= kDepth;
  }
  // Their parts, to LDS `offset` bytes on.
  __device__ __forceinline__ void put(int offset) {
    uint2 part[kPasses][3];
    float odd = 0.f;
#pragma unroll
    for (int u = 0; u < kPasses; ++u) split(v[u], part[u], odd);
    if (__builtin_expect(__any(odd != odd), 0)) {
#pragma unroll
      for (int u = 0; u < kPasses; ++u) split_exactly(v[u], part[u]);
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u)
#pragma unroll
      for (int i = 0; i < 3; ++i)
        *(__attribute__((address_space(3))) U32x2*)(reinterpret_cast<LdsBytes*>(to[u]) + offset + i * kPanel<Side>) =
            U32x2{part[u][i].x, part[u][i].y};
  }
};

// Where a lane finds its 8 elements k = 16 kk + 8 (lane / 32) + 0..7 of row (column)
// first + 32 i + lane % 32.
template <bool Cols, int Side>
struct Finder {
  uint32_t at;
  __device__ __forceinline__ Finder(uint32_t lds, int first, int lane) {
    if constexpr (Cols) {
      const int i = lane & 15, g = lane >> 4;
      const int k = 8 * (g >> 1) + (i >> 2), c = (first >> 4) + (g & 1);
      at = lds + k * (2 * Side) + ((c ^ (swap_of(k) >> 1)) << 5) + (((i & 3) >> 1) << 4) + ((i & 1) << 3);
    } else {
      const int r = lane & 31;
      at = lds + (first + r) * (2 * kDepth) + (((lane >> 5) ^ ((r >> 3) & 3)) << 4);
    }
  }
  __device__ __forceinline__ U32x4 read(int offset, int i, int kk) const {
    U32x4 w;
    if constexpr (Cols) {
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (i << 6)) + offset + kk * 16 * 2 * Side;
      const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)p);
      const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)(p + 4 * 2 * Side));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      w = U32x4{l.x, l.y, h.x, h.y};
    } else {
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (kk << 5)) + offset + i * 32 * 2 * kDepth;
      w = *(__attribute__((address_space(3))) U32x4*)p;
    }
    return w;
  }
};

// One step from the buffer at `offset`: large += a0 b0, small += the five next products.
template <int Tall, bool ACols, bool BCols>
__device__ __forceinline__ void multiply(const Finder<ACols, kTile * Tall>& fa, const Finder<BCols, kTile>& fb,
                                         int offset, Floats16 (&large)[Tall][2], Floats16 (&small)[Tall][2]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    U32x4 y[2][3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      y[0][i] = fb.read(offset + i * kPanel<kTile>, 0, kk);
      y[1][i] = fb.read(offset + i * kPanel<kTile>, 1, kk);
    }
#pragma unroll
    for (int t = 0; t < Tall; ++t) {
      U32x4 x[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) x[i] = fa.read(offset + i * kPanel<kTile * Tall>, t, kk);
      // B's rows as the instruction's rows: a lane then holds four neighbouring n of one m.
      const auto add = [&](int a, int b, Floats16(&acc)[2]) {
        acc[0] = mfma32<BF16>(y[0][b], x[a], acc[0]);
        acc[1] = mfma32<BF16>(y[1][b], x[a], acc[1]);
      };
      add(2, 0, small[t]);
      add(0, 0, large[t]);
      add(0, 2, small[t]);
      add(1, 1, small[t]);
      add(1, 0, small[t]);
      add(0, 1, small[t]);
    }
  }
}

template <int Tall, bool ACols, bool BCols, Finish F>
__global__ __launch_bounds__(kThreads, 2) void f32_product_kernel(ArgsOf<F> p) {
  if (!fit<F, ACols>(p)) return;
  constexpr int kBuffer = 3 * (kPanel<kTile * Tall> + kPanel<kTile>);
  __shared__ __attribute__((aligned(1024))) char lds[2 * kBuffer];  // [buffer][A's parts, B's parts]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [tile, slice] = piece_of<BCols>(p);
  const int m0 = tile.m * kTile * Tall, n0 = tile.n * kTile;
  const Steps<kDepth> steps(p, slice);
  const int count = steps.end - steps.begin;
  const uint32_t lds_a = lds_address(lds), lds_b = lds_a + 3 * kPanel<kTile * Tall>;
  Mover<ACols, kTile * Tall> a;
  Mover<BCols, kTile> b;
  a.init(static_cast<const float*>(p.a), p.lda, m0, p.m, steps.begin, p.k, lds_a);
  b.init(static_cast<const float*>(p.b), p.ldb, n0, p.n, steps.begin, p.k, lds_b);
  const int wm = (wave >> 1) * 32 * Tall, wn = (wave & 1) * 64;
  const Finder<ACols, kTile * Tall> fa(lds_a, wm, lane);
  const Finder<BCols, kTile> fb(lds_b, wn, lane);
  Floats16 large[Tall][2], small[Tall][2];
#pragma unroll
  for (int t = 0; t < Tall; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) large[t][j][e] = small[t][j][e] = 0.f;
  a.fetch();
  b.fetch();
  a.put(0);
  b.put(0);
  if (count > 1) {
    a.fetch();
    b.fetch();
  }
  __syncthreads();
  for (int s = 0; s < count; ++s) {
    const int offset = (s & 1) * kBuffer, other = kBuffer - offset;
    multiply<Tall>(fa, fb, offset, large, small);
    if (s + 1 < count) {
      a.put(other);
      b.put(other);
      if (s + 2 < count) {
        a.fetch();
        b.fetch();
      }
    }
    __syncthreads();
  }
  char* area = lds + wave * 8192 * Tall;
#pragma unroll
  for (int t = 0; t < Tall; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        Floats4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = large[t][j][4 * q + e] + small[t][j][4 * q + e];
        park(area, 32 * t + (lane & 31), 8 * j + 2 * q + (lane >> 5), v);
      }
  finish_parked<F32, F, 32 * Tall>(p, slice, area, m0 + wm, n0 + wn, lane);
}

// Sums of one step, at most 32 terms: one buffer, so that two workgroups share a compute
// unit and one stores while the other loads.  Bound by the stores: dx of 16384 x 4096 into
// 1 to 32 takes 56 to 63 us (268 MB), in the kernel above 79 to 85.
template <bool ACols, bool BCols, Finish F>
__global__ __launch_bounds__(kThreads, 4) void f32_outer_kernel(ArgsOf<F> p) {
  if (!fit<F, ACols>(p)) return;
  constexpr int kParked = 8 * 8192;  // 32 x 64 sums of each wavefront
  static_assert(6 * kPanel<kTile> <= kParked, "the parts fit where the sums go");
  __shared__ __attribute__((aligned(1024))) char lds[kParked];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * kTile, n0 = tile.n * kTile;
  const uint32_t lds_a = lds_address(lds), lds_b = lds_a + 3 * kPanel<kTile>;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 64;
  {
    Mover<ACols, kTile> a;
    Mover<BCols, kTile> b;
    a.init(static_cast<const float*>(p.a), p.lda, m0, p.m, 0, p.k, lds_a);
    b.init(static_cast<const float*>(p.b), p.ldb, n0, p.n, 0, p.k, lds_b);
    a.fetch();
    b.fetch();
    a.put(0);
    b.put(0);
  }
  __syncthreads();
  Floats16 large[1][2], small[1][2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) large[0][j][e] = small[0][j][e] = 0.f;
  multiply<1>(Finder<ACols, kTile>(lds_a, wm, lane), Finder<BCols, kTile>(lds_b, wn, lane), 0, large, small);
  __syncthreads();
  char* area = lds + wave * 8192;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      Floats4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = large[0][j][4 * q + e] + small[0][j][4 * q + e];
      park(area, lane & 31, 8 * j + 2 * q + (lane >> 5), v);
    }
  finish_parked<F32, F, 32>(p, 0, area, m0 + wm, n0 + wn, lane);
}

}  // namespace

hipError_t launch_f32_product(const ProductArgs& p, bool a_cols, bool b_cols, Finish finish, const LossParts* loss, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.tiles_m * p.tiles_n), static_cast<uint32_t>(p.slices)), block(kThreads);
  return with_layout(a_cols, b_cols, finish, [&](auto a, auto b, auto f) {
    if (p.side_m == kTile && p.k <= kDepth && p.slices == 1)
      f32_outer_kernel<a.value, b.value, f.value><<<dim3(grid.x), block, 0, stream>>>(args_of<f.value>(p, loss));
    else if (p.side_m == kTile)
      f32_product_kernel<1, a.value, b.value, f.value><<<grid, block, 0, stream>>>(args_of<f.value>(p, loss));
    else
      f32_product_kernel<2, a.value, b.value, f.value><<<grid, block, 0, stream>>>(args_of<f.value>(p, loss));
    return hipGetLastError();
  });
}

}  // namespace fh
