// Matrix products of the linear layer in 256 x 256 tiles, for sums large enough to
// fill the card with them.
//
// Eight wavefronts of 128 x 64 results each: a wavefront reads 24 KB of LDS for 1 M
// multiply-adds, three quarters of the time that its matrix instructions take (64 x 64
// results of a 128 x 128 tile's wavefront read for as long as they compute).  The sum
// runs in steps of 64 through two buffers, filled by loads that go to LDS directly.
// A step has four phases of 16 matrix instructions, and each phase reads the next
// one's operands, so that LDS works beside the matrix cores; before the last phase
// the wavefronts meet, for by then this step's buffer has been read (it takes the
// loads of the step after the next) and the next step's has been filled.
#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace fh {
namespace {

constexpr int kSide = 256, kDepth = 64;
constexpr int kBuffer = kSide * kDepth * 2;  // bytes of one operand's step

__device__ __forceinline__ int swap_of(int k) { return 2 * ((k & 3) | (((k >> 3) & 1) << 2)); }

// One operand's way into LDS.  In rows: 256 rows of 64 elements, 16-byte chunk c of
// row r at place c ^ (r & 7).  In columns: 64 rows of 256, chunk c of row k at place
// c ^ swap_of(k).  Both spread every wavefront's reads over all banks.
//
// A wavefront's four loads differ by a scalar: registers are short here, so a load has
// its own resource and the lanes' offsets are common (in columns to loads 0, 2 and
// 1, 3, whose chunks change places differently).
template <bool Cols>
struct WidePanel {
  const char* base;  // of this wavefront's load 0
  int64_t step;      // bytes from one step in k to the next
  int32_t next;      // and from one load to the next (in columns to the next but one)
  int32_t voff[Cols ? 2 : 1];
  int at_k;          // the first k of this lane's chunk in load 0 (in columns 2 more each load)
  int rows;          // in rows: those left from load 0 on

  __device__ __forceinline__ void init(const uint16_t* data, int64_t ld, int first, int count, int lane, int wave) {
    if constexpr (Cols) {
      base = reinterpret_cast<const char*>(data + first + wave * 8 * ld);
      step = 2 * kDepth * ld;
      next = static_cast<int32_t>(8 * ld);
      at_k = wave * 8 + (lane >> 5);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = (lane & 31) ^ swap_of(at_k + 2 * u);
        voff[u] = first + 8 * c < count ? static_cast<int32_t>(2 * (((lane >> 5) + 2 * u) * ld + 8 * c)) : kOutOfRange;
      }
    } else {
      base = reinterpret_cast<const char*>(data + (first + wave * 32) * ld);
      step = 2 * kDepth;
      next = static_cast<int32_t>(16 * ld);
      at_k = 8 * ((lane & 7) ^ (lane >> 3));
      voff[0] = static_cast<int32_t>(2 * ((lane >> 3) * ld + at_k));
      rows = count - first - wave * 32;
    }
  }
  // Loads the elements from k0 = 64 tile on, zero past the sum's end `k` and the last
  // row, to LDS address `lds`.
  __device__ __forceinline__ void stage(int64_t offset, int tile, int k, uint32_t lds, int wave) const {
    const char* from = base + offset + tile * step;
    const int left = k - tile * kDepth;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      int32_t at, records;
      if constexpr (Cols) {
        at = at_k + 2 * u < left ? voff[u & 1] : kOutOfRange;
        records = 0x7FFFFFFF;
      } else {
        // The last valid row's last valid element of this step ends the resource.
        const int more = rows - 8 * u < 8 ? rows - 8 * u : 8;
        at = at_k < left ? voff[0] : kOutOfRange;
        records = more > 0 ? (more - 1) * (next >> 3) + 2 * (left < kDepth ? left : kDepth) : 0;
      }
      U32x4 rs = rsrc_words(from + static_cast<int64_t>(next) * (Cols ? u >> 1 : u));
      rs[2] = static_cast<uint32_t>(records);
      lds_load16(rs, lds + (wave * 4 + u) * 1024, at, 0);
    }
  }
};

typedef short S16x4 __attribute__((ext_vector_type(4)));
using LdsShorts = __attribute__((address_space(3))) S16x4;
using LdsBytes = __attribute__((address_space(3))) char;

// Where a lane finds its part of an operand: 8 elements k = 32 kk + 8 (lane / 16) + 0..7
// of row (column) first + 16 i + lane % 16, `first` a multiple of 64.
template <bool Cols>
struct Finder {
  uint32_t at;
  __device__ __forceinline__ Finder(uint32_t lds, int first, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (Cols) {
      const int k = 8 * g + (i >> 2);
      at = lds + k * (2 * kSide) + (((first >> 4) ^ (swap_of(k) >> 1)) << 5) + (((i & 3) >> 1) << 4) + ((i & 1) << 3);
    } else {
      at = lds + (first + i) * (2 * kDepth) + ((g ^ (i & 7)) << 4);
    }
  }
  template <int Buffer>
  __device__ __forceinline__ U32x4 read(int i, int kk) const {
    U32x4 w;
    uint32_t at = this->at;
    if constexpr (Cols) asm volatile("" : "+v"(at));  // formed anew for each read rather than kept in a register for each place
    if constexpr (Cols) {
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (i << 5)) + Buffer * kBuffer + kk * 32 * 2 * kSide;
      const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)p);
      const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)(p + 4 * 2 * kSide));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      w = U32x4{l.x, l.y, h.x, h.y};
    } else {
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (kk << 6)) + Buffer * kBuffer + i * 16 * 2 * kDepth;
      w = *(__attribute__((address_space(3))) U32x4*)p;
    }
    return w;
  }
};

// Rows 64 Half .. + 63 of the wavefront's 128: B's rows go in as the instruction's rows,
// so that a lane holds four neighbouring n of one m.
template <typename E, int Half>
__device__ __forceinline__ void multiply(Floats4 (&acc)[8][4], const U32x4 (&x)[4], const U32x4 (&y)[4]) {
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[Half * 4 + i][j] = mfma16<E>(y[j], x[i], acc[Half * 4 + i][j]);
  __builtin_amdgcn_s_setprio(0);
}

template <int Buffer, int First, bool Cols>
__device__ __forceinline__ void read_four(const Finder<Cols>& f, int kk, U32x4 (&to)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i] = f.template read<Buffer>(First + i, kk);
}

// One LDS read of the next phase beside each few matrix instructions of this one.
template <int Reads>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < Reads; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x8, 16 / Reads, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, bool ACols, bool BCols>
struct Work {
  const ProductArgs& p;
  const Steps<T> steps;
  int count, wave;
  uint32_t lds;
  WidePanel<ACols> a;
  WidePanel<BCols> b;

  __device__ __forceinline__ void stage(int s, int buffer) const {
    int64_t oa, ob;
    int t;
    steps.place(p, steps.begin + s, t, oa, ob);
    a.stage(oa, t, p.k, lds + buffer * kBuffer, wave);
    b.stage(ob, t, p.k, lds + (2 + buffer) * kBuffer, wave);
  }
};

// Step s, in buffer B; x[0] and y[0] hold its first operands, and the next one's after it.
// (Registers are passed by reference: captured ones went to memory.)
template <int B, typename T, bool ACols, bool BCols>
__device__ __forceinline__ void step(const Work<T, ACols, BCols>& w, const Finder<ACols>& fa, const Finder<BCols>& fb,
                                     int s, Floats4 (&acc)[8][4], U32x4 (&x0)[4], U32x4 (&x1)[4], U32x4 (&y0)[4],
                                     U32x4 (&y1)[4]) {
  using E = std::conditional_t<T::code == F16::code, F16, BF16>;
  constexpr int ra = ACols ? 8 : 4, rab = ra + (BCols ? 8 : 4);
  read_four<B, 4>(fa, 0, x1);
  multiply<E, 0>(acc, x0, y0);
  interleave<ra>();
  read_four<B, 0>(fa, 1, x0);
  read_four<B, 0>(fb, 1, y1);
  multiply<E, 1>(acc, x1, y0);
  interleave<rab>();
  read_four<B, 4>(fa, 1, x1);
  multiply<E, 0>(acc, x0, y1);
  interleave<ra>();
  // This buffer has been read; the next one's loads are a step old.
  wait_lds();
  wait_vm<0>();
  meet();
  if (s + 2 < w.count) w.stage(s + 2, B);
  __builtin_amdgcn_sched_barrier(0);
  if (s + 1 < w.count) {
    read_four<B ^ 1, 0>(fa, 0, x0);
    read_four<B ^ 1, 0>(fb, 0, y0);
  }
  multiply<E, 1>(acc, x1, y1);
  interleave<rab>();
}

template <typename T, bool ACols, bool BCols>
__global__ __launch_bounds__(512, 2) void wide_product_kernel(ProductArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * kBuffer];  // A, A, B, B
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * kSide, n0 = tile.n * kSide, slice = blockIdx.y;
  Work<T, ACols, BCols> w{p, Steps<T>(p, slice), 0, wave, lds_address(lds)};
  w.count = w.steps.end - w.steps.begin;
  w.a.init(p.a, p.lda, m0, p.m, lane, wave);
  w.b.init(p.b, p.ldb, n0, p.n, lane, wave);
  const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
  const Finder<ACols> fa(w.lds, wm, lane);
  const Finder<BCols> fb(w.lds + 2 * kBuffer, wn, lane);
  Floats4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = Floats4{0.f, 0.f, 0.f, 0.f};
  U32x4 x0[4], x1[4], y0[4], y1[4];  // A's rows in halves of 64, B's 64
  if (w.count > 0) {
    w.stage(0, 0);
    if (w.count > 1) {
      w.stage(1, 1);
      wait_vm<8>();
    } else {
      wait_vm<0>();
    }
    meet();
    read_four<0, 0>(fa, 0, x0);
    read_four<0, 0>(fb, 0, y0);
    for (int s = 0; s < w.count; s += 2) {
      step<0>(w, fa, fb, s, acc, x0, x1, y0, y1);
      if (s + 1 < w.count) step<1>(w, fa, fb, s + 1, acc, x0, x1, y0, y1);
    }
  }
  __syncthreads();  // the buffers have been read: each wavefront takes 16 KB of them
  finish_block<T>(p, slice, acc, lds + wave * 16384, m0 + wm, n0 + wn, lane);
  finish_block<T>(p, slice, acc + 4, lds + wave * 16384, m0 + wm + 64, n0 + wn, lane);
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
