// Matrix products of the linear layer, in 128 x 128 tiles on the matrix cores.
#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace fh {
namespace {

typedef short S16x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 128, kDepth = 64;
constexpr int kPanel = kTile * kDepth;  // elements of one operand's tile

// Exchange of 16-byte chunks along an LDS row of a tile in columns, by the row k.
__device__ __forceinline__ int swap_of(int k) { return 2 * ((k & 3) | (((k >> 3) & 1) << 2)); }

// One operand's way through LDS.  In rows: 128 rows of 64 elements, chunk c of row
// r at place c ^ (r & 7).  In columns: 64 rows of 128 elements, chunk c of row k at
// place c ^ swap_of(k).
template <bool Cols>
struct Panel {
  U32x4 rsrc;
  int32_t voff[4];   // of the wavefront's four loads
  int at_k[4];       // the first k of each lane's chunk, in the tile
  int64_t step;      // bytes from one tile in k to the next
  const char* base;

  __device__ __forceinline__ void init(const uint16_t* data, int64_t ld, int first, int count, int lane, int wave) {
    base = reinterpret_cast<const char*>(data + (Cols ? static_cast<int64_t>(first) : first * ld));
    step = 2 * (Cols ? kDepth * ld : kDepth);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (Cols) {
        const int k = (wave * 4 + u) * 4 + (lane >> 4), c = (lane & 15) ^ swap_of(k);
        voff[u] = first + 8 * c < count ? static_cast<int32_t>(2 * (k * ld + 8 * c)) : kOutOfRange;
        at_k[u] = k;
      } else {
        const int r = (wave * 4 + u) * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
        const int row = first + r < count ? r : count - 1 - first;
        voff[u] = static_cast<int32_t>(2 * (row * ld + 8 * c));
        at_k[u] = 8 * c;
      }
    }
  }
  // Loads the tile from k0 on into `lds`; k is the sum's length.
  __device__ __forceinline__ void stage(int64_t offset, int tile, int k, uint32_t lds, int wave) const {
    const U32x4 rs = rsrc_words(base + offset + tile * step);
    const int left = k - tile * kDepth;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      lds_load16(rs, lds + (wave * 4 + u) * 1024, at_k[u] < left ? voff[u] : kOutOfRange, 0);
  }
};

// Lane's 8 elements k = 32 kk + 8 (lane / 16) + 0..7 of row (column) first + lane % 16.
template <bool Cols>
__device__ __forceinline__ U32x4 fragment(const uint16_t* tile, int first, int kk, int lane) {
  U32x4 w;
  if constexpr (Cols) {
    const int i = lane & 15, k = kk * 32 + 8 * (lane >> 4) + (i >> 2);
    const int col = first + 4 * (i & 3);
    const uint16_t* p = tile + k * kTile + (((col >> 3) ^ swap_of(k)) << 3) + (col & 7);
    using Lds = __attribute__((address_space(3))) S16x4;
    const S16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)p);
    const S16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p + 4 * kTile));
    __builtin_memcpy(&w, &lo, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&w) + 8, &hi, 8);
  } else {
    const int r = first + (lane & 15), c = kk * 4 + (lane >> 4);
    w = *reinterpret_cast<const U32x4*>(tile + r * kDepth + ((c ^ (r & 7)) << 3));
  }
  return w;
}

template <typename T, bool ACols, bool BCols>
__global__ __launch_bounds__(256) void product_kernel(ProductArgs p) {
  using E = std::conditional_t<T::code == F16::code, F16, BF16>;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[2][2][kPanel];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile tile = tile_of(p, blockIdx.x);
  const int m0 = tile.m * kTile, n0 = tile.n * kTile, slice = blockIdx.y;
  Panel<ACols> a;
  Panel<BCols> b;
  a.init(p.a, p.lda, m0, p.m, lane, wave);
  b.init(p.b, p.ldb, n0, p.n, lane, wave);
  const Steps<T, kDepth> steps(p, slice);
  const auto stage = [&](int step, int buffer) {
    int64_t oa, ob;
    int t;
    steps.place(p, step, t, oa, ob);
    a.stage(oa, t, p.k, lds_address(lds[buffer][0]), wave);
    b.stage(ob, t, p.k, lds_address(lds[buffer][1]), wave);
  };
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  Floats4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = Floats4{0.f, 0.f, 0.f, 0.f};
  if (steps.begin < steps.end) stage(steps.begin, 0);
  for (int s = steps.begin; s < steps.end; ++s) {
    const int buffer = (s - steps.begin) & 1;
    wait_vm<0>();
    __syncthreads();  // the tile is there, and the other buffer has been read
    if (s + 1 < steps.end) stage(s + 1, buffer ^ 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      U32x4 fa[4], fb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fa[i] = fragment<ACols>(lds[buffer][0], wm + 16 * i, kk, lane);
        fb[i] = fragment<BCols>(lds[buffer][1], wn + 16 * i, kk, lane);
      }
      // B's rows as the instruction's rows: a lane then holds four neighbouring n of one m.
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma16<E>(fb[j], fa[i], acc[i][j]);
    }
  }
  __syncthreads();  // the buffers have been read: each wavefront takes 16 KB of them
  char* area = reinterpret_cast<char*>(lds) + wave * 16384;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) park(area, 16 * i + (lane & 15), 4 * j + (lane >> 4), acc[i][j]);
  finish_parked<T>(p, slice, area, m0 + wm, n0 + wn, lane);
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
  const dim3 grid(static_cast<uint32_t>(p.tiles_m * p.tiles_n), static_cast<uint32_t>(p.slices)), block(256);
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

void plan_product(ProductArgs& p, int dtype) {
  const int64_t steps = static_cast<int64_t>((p.k + kDepth - 1) / kDepth) * (dtype == F32::code ? 6 : 1);
  const int64_t units = compute_units();
  // Tiles of 256 once they keep nearly all compute units at work to the end.
  set_tiles(p, 256);
  p.slices = 1;
  const int64_t wide = static_cast<int64_t>(p.tiles_m) * p.tiles_n, rounds = (wide + units - 1) / units;
  if (wide * 10 >= rounds * units * 8 && p.m > 128 && p.n > 128) return;
  set_tiles(p, kTile);
  // Slices of at least eight steps until two workgroups a compute unit have work.
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  p.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2 * units / tiles, steps / 8)));
}

hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream) {
  if (p.side == 256) return launch_wide_product(p, dtype, a_cols, b_cols, stream);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const hipError_t err = run<T>(p, a_cols, b_cols, stream);
    return err != hipSuccess || p.slices == 1 ? err : join<T>(p, stream);
  });
}

}  // namespace fh
