// Matrix products of the linear layer, in 128 x 128 tiles on the matrix cores.
#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace fh {
namespace {

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));
typedef short S16x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 128, kDepth = 64;
constexpr int kPanel = kTile * kDepth;  // elements of one operand's tile

template <typename E>
__device__ __forceinline__ Floats4 mfma(U32x4 a, U32x4 b, Floats4 c) {
  if constexpr (E::code == F16::code) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(F16x8, a), __builtin_bit_cast(F16x8, b), c, 0, 0,
                                                  0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0,
                                                   0, 0);
  }
}

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
  const int tile = blockIdx.x, slice = blockIdx.y;
  const int m0 = tile / p.tiles_n * kTile, n0 = tile % p.tiles_n * kTile;
  Panel<ACols> a;
  Panel<BCols> b;
  a.init(p.a, p.lda, m0, p.m, lane, wave);
  b.init(p.b, p.ldb, n0, p.n, lane, wave);
  // FP32: products of planes, the smallest first; those of 2^-24 and below are left out.
  const int pairs = T::code == F32::code ? 6 : 1;
  const int depth = (p.k + kDepth - 1) / kDepth, steps = depth * pairs;
  const int begin = static_cast<int>(static_cast<int64_t>(steps) * slice / p.slices);
  const int end = static_cast<int>(static_cast<int64_t>(steps) * (slice + 1) / p.slices);
  const auto stage = [&](int step, int buffer) {
    int64_t oa = 0, ob = 0;
    int t = step;
    if constexpr (T::code == F32::code) {
      const int pair = step / depth;
      t -= pair * depth;
      const int pa = (0x210100 >> (20 - 4 * pair)) & 15, pb = (0x012010 >> (20 - 4 * pair)) & 15;
      oa = 2 * pa * p.plane_a;
      ob = 2 * pb * p.plane_b;
    }
    a.stage(oa, t, p.k, lds_address(lds[buffer][0]), wave);
    b.stage(ob, t, p.k, lds_address(lds[buffer][1]), wave);
  };
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  Floats4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = Floats4{0.f, 0.f, 0.f, 0.f};
  if (begin < end) stage(begin, 0);
  for (int s = begin; s < end; ++s) {
    const int buffer = (s - begin) & 1;
    wait_vm<0>();
    __syncthreads();  // the tile is there, and the other buffer has been read
    if (s + 1 < end) stage(s + 1, buffer ^ 1);
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
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma<E>(fb[j], fa[i], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = m0 + wm + 16 * i + (lane & 15), col = n0 + wn + 16 * j + 4 * (lane >> 4);
      if (row >= p.m || col >= p.n) continue;
      if (p.slices > 1) {
        float* to = p.partial + (static_cast<int64_t>(slice) * p.m + row) * p.n + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.n) to[e] = acc[i][j][e];
      } else {
        const float sum[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        finish_four<T>(p, row, col, sum);
      }
    }
}

// Adds the slices in order and finishes.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(ProductArgs p) {
  const int quads = (p.n + 3) / 4;
  const int64_t total = static_cast<int64_t>(p.m) * quads;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < total;
       q += static_cast<int64_t>(gridDim.x) * 256) {
    const int row = static_cast<int>(q / quads), col = static_cast<int>(q % quads) * 4;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const float* from = p.partial + static_cast<int64_t>(row) * p.n + col;
    for (int s = 0; s < p.slices; ++s, from += static_cast<int64_t>(p.m) * p.n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.n) sum[e] += from[e];
    finish_four<T>(p, row, col, sum);
  }
}

template <typename T>
hipError_t run(const ProductArgs& p, bool a_cols, bool b_cols, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.tiles_m * p.tiles_n), static_cast<uint32_t>(p.slices)), block(256);
  if (!a_cols && !b_cols) product_kernel<T, false, false><<<grid, block, 0, stream>>>(p);
  if (!a_cols && b_cols) product_kernel<T, false, true><<<grid, block, 0, stream>>>(p);
  if (a_cols && b_cols) product_kernel<T, true, true><<<grid, block, 0, stream>>>(p);
  if (a_cols && !b_cols) return hipErrorInvalidValue;  // no such product
  if (const hipError_t err = hipGetLastError(); err != hipSuccess || p.slices == 1) return err;
  const int64_t quads = static_cast<int64_t>(p.m) * ((p.n + 3) / 4);
  join_kernel<T><<<dim3(static_cast<uint32_t>(std::min<int64_t>((quads + 255) / 256, 4096))), block, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace

void plan_product(ProductArgs& p, int dtype) {
  p.tiles_m = (p.m + kTile - 1) / kTile;
  p.tiles_n = (p.n + kTile - 1) / kTile;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  const int64_t steps = static_cast<int64_t>((p.k + kDepth - 1) / kDepth) * (dtype == F32::code ? 6 : 1);
  // Slices of at least eight steps until two workgroups a compute unit have work.
  p.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2 * compute_units() / tiles, steps / 8)));
}

hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream) {
  return with_type(dtype, [&](auto t) { return run<decltype(t)>(p, a_cols, b_cols, stream); });
}

}  // namespace fh
