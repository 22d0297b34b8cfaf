// Matrix products of the linear layer in 256 x 256 tiles, for sums large enough to
// fill the card with them.
//
// Eight wavefronts of 128 x 64 results each, on 32 x 32 x 16 instructions (half as many
// to issue as 16 x 16 x 32, for the same work): a wavefront reads 24 KB of LDS for 1 M
// multiply-adds (64 x 64 results of a 128 x 128 tile's wavefront need a third more).
// The sum runs in steps of 64 through two buffers, filled by loads that go to LDS
// directly, in whole cache lines (steps of 32 in four buffers asked the L2 for half
// lines and took a tenth longer).  A step has four phases of eight matrix instructions;
// every two of them go with reads of the phase to come or with a load, so that LDS and
// the loads work beside the matrix cores.  Before the last phase the wavefronts meet:
// by then this step's buffer has been read, and the next one's loads are there.
#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace fh {
namespace {

constexpr int kSide = 256, kDepth = 64;
constexpr int kBuffer = kSide * kDepth * 2;  // bytes of one operand's step

__device__ __forceinline__ int swap_of(int k) { return 2 * (((k & 3) << 1) | ((k >> 3) & 1)); }

// One operand's way into LDS.  In rows: 256 rows of 64 elements, 16-byte chunk c of
// row r at place c ^ ((r >> 1) & 7).  In columns: 64 rows of 256, chunk c of row k at
// place c ^ swap_of(k).  Both spread every wavefront's reads over all banks.  Each
// wavefront has four loads a step, whose resources move with the steps: a full step
// costs a few scalar instructions.
template <bool Cols>
struct Feeder {
  uint64_t base[4];    // of the loads
  uint32_t bytes[4];   // of their resources in a full step: the last valid row's end
  int64_t step;        // bytes from one step in k to the next
  int32_t voff[2];     // of the even and the odd loads
  int at_k;            // the first k of this lane's chunk in load 0
  int left;            // elements of the sum from here on

  __device__ __forceinline__ void init(const uint16_t* data, int64_t ld, int first, int count, int lane, int wave) {
    const int32_t row = static_cast<int32_t>(2 * ld);
    if constexpr (Cols) {
      step = 2 * kDepth * ld;
      at_k = wave * 8 + (lane >> 5);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = (lane & 31) ^ swap_of(at_k + 2 * u);
        voff[u] = first + 8 * c < count ? ((lane >> 5) + 2 * u) * row + 16 * c : kOutOfRange;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        base[u] = reinterpret_cast<uint64_t>(data + first + (wave * 8 + (u & 2) * 2) * ld);
        bytes[u] = 0x7FFFFFFFu;
      }
    } else {
      step = 2 * kDepth;
      at_k = 8 * ((lane & 7) ^ (lane >> 4));
#pragma unroll
      for (int u = 0; u < 2; ++u) voff[u] = (lane >> 3) * row + 2 * (at_k ^ (32 * u));
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int from = first + wave * 32 + 8 * u, more = count - from < 8 ? count - from : 8;
        base[u] = reinterpret_cast<uint64_t>(data + from * ld);
        bytes[u] = more > 0 ? (more - 1) * row + 2 * kDepth : 0;
      }
    }
  }
  // Moves to step t of a sum of k elements, `offset` bytes further on.
  __device__ __forceinline__ void go(int64_t offset, int t, int k) {
#pragma unroll
    for (int u = 0; u < 4; ++u) base[u] += offset + t * step;
    left = k - t * kDepth;
  }
  // Loads load u of this step to LDS address `lds`, zero past the sum's end and the last row.
  __device__ __forceinline__ void stage(int u, uint32_t lds) const {
    U32x4 rs{static_cast<uint32_t>(base[u]), static_cast<uint32_t>(base[u] >> 32) & 0xFFFFu, bytes[u], 0x00020000u};
    if (__builtin_expect(left >= kDepth, 1)) {
      lds_load16(rs, lds, voff[u & 1], 0);
    } else {
      if (!Cols) rs[2] = bytes[u] > 0 ? bytes[u] - 2 * (kDepth - left) : 0;
      const int k = Cols ? at_k + 2 * u : at_k ^ (32 * (u & 1));
      lds_load16(rs, lds, k < left ? voff[u & 1] : kOutOfRange, 0);
    }
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int u = 0; u < 4; ++u) base[u] += step;
    left -= kDepth;
  }
};

typedef short S16x4 __attribute__((ext_vector_type(4)));
using LdsShorts = __attribute__((address_space(3))) S16x4;
using LdsBytes = __attribute__((address_space(3))) char;

// Where a lane finds its part of an operand: 8 elements k = 16 kk + 8 (lane / 32) + 0..7
// of row (column) first + 32 i + lane % 32, `first` a multiple of 64.
template <bool Cols>
struct Finder {
  uint32_t at;
  __device__ __forceinline__ Finder(uint32_t lds, int first, int lane) {
    if constexpr (Cols) {
      const int i = lane & 15, g = lane >> 4;
      const int k = 8 * (g >> 1) + (i >> 2), c = (first >> 4) + (g & 1);
      at = lds + k * (2 * kSide) + ((c ^ (swap_of(k) >> 1)) << 5) + (((i & 3) >> 1) << 4) + ((i & 1) << 3);
    } else {
      const int r = lane & 31;
      at = lds + (first + r) * (2 * kDepth) + (((lane >> 5) ^ ((r >> 1) & 7)) << 4);
    }
  }
  template <int Buffer>
  __device__ __forceinline__ U32x4 read(int i, int kk) const {
    U32x4 w;
    if constexpr (Cols) {
      uint32_t at = this->at;
      asm volatile("" : "+v"(at));  // formed anew for each read rather than kept in a register for each place
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (i << 6)) + Buffer * kBuffer + kk * 16 * 2 * kSide;
      const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)p);
      const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)(p + 4 * 2 * kSide));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      w = U32x4{l.x, l.y, h.x, h.y};
    } else {
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (kk << 5)) + Buffer * kBuffer + i * 32 * 2 * kDepth;
      w = *(__attribute__((address_space(3))) U32x4*)p;
    }
    return w;
  }
};

__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// An operand's steps of a slice: the next one to load.
template <typename T, bool Cols>
struct Feed {
  Feeder<Cols> f, start;
  Steps<T, kDepth> steps;
  int next;
  uint32_t lds;

  __device__ __forceinline__ void place(const ProductArgs& p, bool of_a) {
    int64_t oa, ob;
    int t;
    steps.place(p, next, t, oa, ob);
    f = start;
    f.go(of_a ? oa : ob, t, p.k);
  }
  __device__ __forceinline__ void stage(int u, int buffer) const { f.stage(u, lds + buffer * kBuffer + u * 1024); }
  __device__ __forceinline__ void advance(const ProductArgs& p, bool of_a) {
    ++next;
    f.advance();
    if constexpr (T::code == F32::code) {  // the next pair of planes begins
      if (f.left <= 0 && next < steps.end) place(p, of_a);
    }
  }
};

// Two matrix instructions: B's rows go in as their rows, so that a lane holds four
// neighbouring n of one m.
template <typename E>
__device__ __forceinline__ void two(Floats16 (&acc)[2], U32x4 x, U32x4 y0, U32x4 y1) {
  acc[0] = mfma32<E>(y0, x, acc[0]);
  acc[1] = mfma32<E>(y1, x, acc[1]);
}

template <int Buffer, bool Cols>
__device__ __forceinline__ void read_two(const Finder<Cols>& f, int i, int kk, U32x4* to) {
  to[0] = f.template read<Buffer>(i, kk);
  to[1] = f.template read<Buffer>(i + 1, kk);
}

// Step s, in buffer B.  x0 and y hold A's rows 0..63 and B's rows of k = 0..31 of it
// ([2 (k / 16) + tile]), and after it those of the next step.  (Registers are passed
// by reference: captured ones went to memory.)
template <int B, typename T, bool ACols, bool BCols>
__device__ __forceinline__ void step(const ProductArgs& p, Feed<T, ACols>& a, Feed<T, BCols>& b,
                                     const Finder<ACols>& fa, const Finder<BCols>& fb, int s, int count,
                                     Floats16 (&acc)[4][2], U32x4 (&x0)[4], U32x4 (&x1)[4], U32x4 (&y)[4],
                                     U32x4 (&z)[4]) {
  using E = std::conditional_t<T::code == F16::code, F16, BF16>;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) read_two<B>(fa, 2, i, x1 + 2 * i);
    if (s + 1 < count) b.stage(i, B ^ 1);
    two<E>(acc[i & 1], x0[i], y[i & 2], y[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (s + 1 < count) b.advance(p, false);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) {
      read_two<B>(fa, 0, 2 + i, x0 + 2 * i);
      read_two<B>(fb, 0, 2 + i, z + 2 * i);
    }
    two<E>(acc[2 + (i & 1)], x1[i], y[i & 2], y[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) read_two<B>(fa, 2, 2 + i, x1 + 2 * i);
    two<E>(acc[i & 1], x0[i], z[i & 2], z[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  wait_lds();
  wait_vm<0>();
  meet();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2 && s + 1 < count) {
      read_two<B ^ 1>(fa, 0, i, x0 + 2 * i);
      read_two<B ^ 1>(fb, 0, i, y + 2 * i);
    }
    if (s + 2 < count) a.stage(i, B);
    two<E>(acc[2 + (i & 1)], x1[i], z[i & 2], z[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (s + 2 < count) a.advance(p, true);
}

template <typename T, bool ACols, bool BCols>
__global__ __launch_bounds__(512, 2) void wide_product_kernel(ProductArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * kBuffer];  // A, A, B, B
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * kSide, n0 = tile.n * kSide, slice = blockIdx.y;
  const Steps<T, kDepth> steps(p, slice);
  const int count = steps.end - steps.begin;
  Feed<T, ACols> a{{}, {}, steps, steps.begin, lds_address(lds) + wave * 4096};
  Feed<T, BCols> b{{}, {}, steps, steps.begin, lds_address(lds) + 2 * kBuffer + wave * 4096};
  a.start.init(p.a, p.lda, m0, p.m, lane, wave);
  b.start.init(p.b, p.ldb, n0, p.n, lane, wave);
  const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
  const Finder<ACols> fa(lds_address(lds), wm, lane);
  const Finder<BCols> fb(lds_address(lds) + 2 * kBuffer, wn, lane);
  Floats16 acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  U32x4 x0[4], x1[4], y[4], z[4];
  if (count > 0) {
    a.place(p, true);
    b.place(p, false);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      a.stage(u, 0);
      b.stage(u, 0);
    }
    a.advance(p, true);
    b.advance(p, false);
    wait_vm<0>();
    meet();
    if (count > 1) {
#pragma unroll
      for (int u = 0; u < 4; ++u) a.stage(u, 1);
      a.advance(p, true);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      read_two<0>(fa, 0, i, x0 + 2 * i);
      read_two<0>(fb, 0, i, y + 2 * i);
    }
    for (int s = 0; s < count; s += 2) {
      step<0>(p, a, b, fa, fb, s, count, acc, x0, x1, y, z);
      if (s + 1 < count) step<1>(p, a, b, fa, fb, s + 1, count, acc, x0, x1, y, z);
    }
  }
  __syncthreads();  // the buffers have been read: each wavefront takes 16 KB of them
  char* area = lds + wave * 16384;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const Floats16& v = acc[2 * half + i][j];
          park(area, 32 * i + (lane & 31), 8 * j + 2 * q + (lane >> 5),
               Floats4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
        }
    finish_parked<T>(p, slice, area, m0 + wm + 64 * half, n0 + wn, lane);
  }
}

template <typename T>
hipError_t run(const ProductArgs& p, bool a_cols, bool b_cols, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.tiles_m * p.tiles_n), static_cast<uint32_t>(p.slices)), block(512);
  if (!a_cols && !b_cols) wide_product_kernel<T, false, false><<<grid, block, 0, stream>>>(p);
  if (!a_cols && b_cols) wide_product_kernel<T, false, true><<<grid, block, 0, stream>>>(p);
  if (a_cols && b_cols) wide_product_kernel<T, true, true><<<grid, block, 0, stream>>>(p);
  if (a_cols && !b_cols) return hipErrorInvalidValue;  // no such product
  return hipGetLastError();
}

}  // namespace

hipError_t launch_wide_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream) {
  return with_type(dtype, [&](auto t) { return run<decltype(t)>(p, a_cols, b_cols, stream); });
}

}  // namespace fh
