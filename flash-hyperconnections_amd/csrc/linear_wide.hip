// Matrix products of the linear layer in 256 x 256 tiles, for sums large enough to
// fill the card with them.
//
// Eight wavefronts of 128 x 64 results each, on 32 x 32 x 16 instructions (half as many
// to issue as 16 x 16 x 32, for the same work): a wavefront reads 24 KB of LDS for 0.5 M
// multiply-adds (64 x 64 results of a 128 x 128 tile's wavefront need a third more).
// The sum runs in steps of 64 through two buffers, filled by loads that go to LDS
// directly, in whole cache lines (steps of 32 in four buffers asked the L2 for half
// lines and took a tenth longer).  A step has four phases of eight matrix instructions;
// every two of them go with reads of the phase to come or with a load, so that LDS and
// the loads work beside the matrix cores.  Before the last phase the wavefronts meet:
// by then this step's buffer has been read, and the next one's loads are there.
//
// 16384 x 4096 x 16384 bf16 (2.2 TFLOP) takes 1.93 ms forward with gelu and a saved sum,
// 1.71 for dx and 1.68 for dW; the matrix cores are busy 64, 68 and 81% of the time, at a
// clock of 1.6 to 1.8 GHz: on operands of zeros the three take 1.26, 1.55 and 1.33 ms.
#include <algorithm>
#include <type_traits>

#include "linear_tiles.h"

namespace fh {
namespace {

constexpr int kSide = 256;
constexpr int kBuffer = kSide * kStep * 2;  // bytes of one operand's step

// Two matrix instructions: B's rows go in as their rows, so that a lane holds four
// neighbouring n of one m.
template <typename E>
__device__ __forceinline__ void two(Floats16 (&acc)[2], U32x4 x, U32x4 y0, U32x4 y1) {
  acc[0] = mfma32<E>(y0, x, acc[0]);
  acc[1] = mfma32<E>(y1, x, acc[1]);
}

template <int Buffer, bool Cols>
__device__ __forceinline__ void read_two(const Finder<Cols, kSide>& f, int i, int kk, U32x4* to) {
  to[0] = f.read(Buffer * kBuffer, i, kk);
  to[1] = f.read(Buffer * kBuffer, i + 1, kk);
}

// A step in buffer B.  x0 and y hold A's rows 0..63 and B's rows of k = 0..31 of it
// ([2 (k / 16) + tile]), and after it those of the next step.  (Registers are passed
// by reference: captured ones went to memory.)
template <int B, typename T, bool ACols, bool BCols>
__device__ __forceinline__ void step(Feeder<ACols, kSide>& a, Feeder<BCols, kSide>& b,
                                     const Finder<ACols, kSide>& fa, const Finder<BCols, kSide>& fb,
                                     Floats16 (&acc)[4][2], U32x4 (&x0)[4], U32x4 (&x1)[4], U32x4 (&y)[4],
                                     U32x4 (&z)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) read_two<B>(fa, 2, i, x1 + 2 * i);
    b.stage(i, (B ^ 1) * kBuffer);
    two<T>(acc[i & 1], x0[i], y[i & 2], y[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  b.advance();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) {
      read_two<B>(fa, 0, 2 + i, x0 + 2 * i);
      read_two<B>(fb, 0, 2 + i, z + 2 * i);
    }
    two<T>(acc[2 + (i & 1)], x1[i], y[i & 2], y[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) read_two<B>(fa, 2, 2 + i, x1 + 2 * i);
    two<T>(acc[i & 1], x0[i], z[i & 2], z[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  wait_lds();
  wait_vm<0>();
  meet();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < 2) {
      read_two<B ^ 1>(fa, 0, i, x0 + 2 * i);
      read_two<B ^ 1>(fb, 0, i, y + 2 * i);
    }
    a.stage(i, B * kBuffer);
    two<T>(acc[2 + (i & 1)], x1[i], z[i & 2], z[(i & 2) + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  a.advance();
}

template <typename T, bool ACols, bool BCols, Finish F>
__global__ __launch_bounds__(512, 2) void wide_product_kernel(ArgsOf<F> p) {
  if (!fit<F, ACols>(p)) return;
  __shared__ __attribute__((aligned(1024))) char lds[4 * kBuffer];  // A, A, B, B
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto [tile, slice] = piece_of<BCols>(p);
  const int m0 = tile.m * kSide, n0 = tile.n * kSide;
  const Steps<kStep> steps(p, slice);
  const int count = steps.end - steps.begin;
  Feeder<ACols, kSide> a;
  Feeder<BCols, kSide> b;
  a.init(p.a, p.lda, m0, p.m, p.k, steps.begin, lds_address(lds), lane, wave);
  b.init(p.b, p.ldb, n0, p.n, p.k, steps.begin, lds_address(lds) + 2 * kBuffer, lane, wave);
  const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
  const Finder<ACols, kSide> fa(lds_address(lds), wm, lane);
  const Finder<BCols, kSide> fb(lds_address(lds) + 2 * kBuffer, wn, lane);
  Floats16 acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  U32x4 x0[4], x1[4], y[4], z[4];
  if (count > 0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      a.stage(u, 0);
      b.stage(u, 0);
    }
    a.advance();
    b.advance();
    wait_vm<0>();
    meet();
#pragma unroll
    for (int u = 0; u < 4; ++u) a.stage(u, kBuffer);
    a.advance();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      read_two<0>(fa, 0, i, x0 + 2 * i);
      read_two<0>(fb, 0, i, y + 2 * i);
    }
    // Loads and reads go on past the last step, of zeros.
    for (int s = 0; s < count; s += 2) {
      step<0, T>(a, b, fa, fb, acc, x0, x1, y, z);
      if (s + 1 < count) step<1, T>(a, b, fa, fb, acc, x0, x1, y, z);
    }
  }
  wait_vm<0>();
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
    finish_parked<T, F, 64>(p, slice, area, m0 + wm + 64 * half, n0 + wn, lane);
  }
}

}  // namespace

hipError_t launch_wide_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish,
                               const LossParts* loss, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.tiles_m * p.tiles_n), static_cast<uint32_t>(p.slices)), block(512);
  return with_half_type(dtype, [&](auto t) {
    return with_layout(a_cols, b_cols, finish, [&](auto a, auto b, auto f) {
      wide_product_kernel<decltype(t), a.value, b.value, f.value><<<grid, block, 0, stream>>>(args_of<f.value>(p, loss));
      return hipGetLastError();
    });
  });
}

}  // namespace fh
