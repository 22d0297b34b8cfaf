// Pieces shared by the kernels of the linear layer: activations, the epilogue of
// a product and the description of a product.
#pragma once

#include <type_traits>

#include "fh_kernels.h"
#include "fh_vec.h"
#include "flash_hypercons.h"

namespace fh {

typedef float Floats4 __attribute__((ext_vector_type(4)));

// D[m][n] = sum over k of A[m][k] B[n][k] and what follows it.  An operand is in
// rows (k contiguous, rows ld elements apart) or in columns (m or n contiguous, a
// row for each k).  16-bit operands have 16-byte aligned rows of whole 16-byte
// vectors; FP32 ones any rows.
struct ProductArgs {
  const void *a, *b;
  int64_t lda, ldb;
  int m, n, k;
  int tiles_m, tiles_n;
  int side_m, side_n;    // of a tile
  int slices;            // of the sum over k
  float* partial;        // [slices, m, n] where there are several
  const void* bias;      // [n] or null, FP32 or the output's type
  int bias_f32;
  const void* residual;  // [m, n], rows ldr apart, or null
  int64_t ldr;
  int act;
  void* saved;           // receives the sum with its bias, or null
  void* out;             // [m, n] contiguous
};

// What the backward needs of the sum z = x W^T + b: FP32 for FP32 results, and
// FP16 for 16-bit ones, whatever they are.  Every activation's slope is 0 or 1 to
// its last bit beyond +-65504, where values are clamped, and FP16's 11 bits keep
// the slope's error well below that of rounding dz: with gelu and normal z the
// weight's gradient is off by 0.00233 with z exact or in FP16, by 0.00241 in bf16.
// A positive z below FP16's smallest value, 2^-24, is kept as that value: relu's slope
// is 1 for every positive sum, and the other slopes change by less than 2^-24 there.
template <typename T>
using Saved = std::conditional_t<T::code == F32::code, F32, F16>;

__device__ __forceinline__ float clamp_saved(float z) {
  if (z > 0.f) return __builtin_amdgcn_fmed3f(z, 0x1p-24f, 65504.f);
  return z < -65504.f ? -65504.f : z;  // and a NaN
}

// Phi(z) and the normal density at z, by formula 7.1.26 of Abramowitz and Stegun's
// handbook: Phi is off by 7e-8 at most, about the rounding of 1 + erf in FP32.  Far out on
// the negative side that is no longer small beside gelu itself: relative to it the formula
// errs by 5e-4 at z = -4, where gelu is -1e-4, by 4e-3 at -6 (-6e-9) and 4e-2 at -13, where
// 1 + erf in FP32 has lost every digit from -5.5 on.  The exponential it needs is the
// density's as well.  A gelu adds 74 us to 16384 x 4096 x 16384 bf16 so, and 169 with
// the library's erff.
struct Normal {
  float phi, density;
};
__device__ __forceinline__ Normal normal_of(float z) {
  const float x = __builtin_fabsf(z);
  const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);  // exp(-z^2 / 2)
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.23164189f, x, 1.f));  // 0.3275911 / sqrt(2)
  float s = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  s = __builtin_fmaf(s, t, 1.421413741f);
  s = __builtin_fmaf(s, t, -0.284496736f);
  s = __builtin_fmaf(s, t, 0.254829592f);
  const float tail = 0.5f * (s * t) * e;  // Phi(-|z|)
  return {z < 0.f ? tail : 1.f - tail, 0.39894228040143268f * e};
}

// 1 / (1 + exp(-v)), by the hardware's exp2 and reciprocal (one unit in the last place
// each) for 16-bit results.
template <typename T>
__device__ __forceinline__ float logistic(float v) {
  if constexpr (T::code == F32::code) return 1.f / (1.f + expf(-v));
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

// act(z) of a vector; relu keeps a NaN.
template <typename T, int V>
__device__ __forceinline__ void activate(float (&v)[V], int act) {
  switch (act) {
    case FH_ACT_RELU:
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = v[k] < 0.f ? 0.f : v[k];
      break;
    case FH_ACT_GELU:
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if constexpr (T::code == F32::code) v[k] *= 0.5f * (1.f + erff(v[k] * 0.70710678118654752f));
        else v[k] *= normal_of(v[k]).phi;
      }
      break;
    case FH_ACT_GELU_TANH:
      // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), without the difference of near values.
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] *= logistic<T>(1.5957691216057308f * __builtin_fmaf(0.044715f * v[k] * v[k], v[k], v[k]));
      break;
    case FH_ACT_SILU:
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] *= logistic<T>(v[k]);
      break;
    default: break;
  }
}

// f times act'(z), of a vector.
template <typename T, int V>
__device__ __forceinline__ void slope_times(const float (&z)[V], int act, float (&f)[V]) {
  switch (act) {
    case FH_ACT_RELU:
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = z[i] > 0.f ? f[i] : 0.f;
      break;
    case FH_ACT_GELU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (T::code == F32::code) {
          f[i] *= 0.5f * (1.f + erff(z[i] * 0.70710678118654752f)) +
                  z[i] * (0.39894228040143268f * expf(-0.5f * z[i] * z[i]));
        } else {
          const Normal n = normal_of(z[i]);
          f[i] *= __builtin_fmaf(z[i], n.density, n.phi);
        }
      }
      break;
    case FH_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = logistic<T>(1.5957691216057308f * __builtin_fmaf(0.044715f * z[i] * z[i], z[i], z[i]));
        const float du2 = 1.5957691216057308f * __builtin_fmaf(0.134145f * z[i], z[i], 1.f);
        // q (1 - q) is 0 where exp has left its range, whatever z du2 is.
        const float curve = q * (1.f - q);
        f[i] *= curve > 0.f ? __builtin_fmaf(z[i] * du2, curve, q) : q;
      }
      break;
    case FH_ACT_SILU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = logistic<T>(z[i]), curve = q * (1.f - q);
        f[i] *= curve > 0.f ? __builtin_fmaf(z[i], curve, q) : q;
      }
      break;
    default: break;
  }
}

// Elements 0 .. count - 1 of V, count at least 1.
template <typename S, int V>
__device__ __forceinline__ void load_some(const S* from, int count, S (&e)[V]) {
  if (count >= V) {
    __builtin_memcpy(e, from, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = i < count ? from[i] : S{};
  }
}
// Nontemporal unless they are read again soon, as partial sums are.
template <bool Soon = false, typename S, int V>
__device__ __forceinline__ void store_some(const S (&e)[V], S* to, int count) {
  if (Soon && count >= V) {
    __builtin_memcpy(to, e, sizeof(e));
  } else if (count >= V) {
    U32x4 w[sizeof(e) / 16];
    __builtin_memcpy(w, e, sizeof(e));
#pragma unroll
    for (size_t i = 0; i < sizeof(e) / 16; ++i) store16(w[i], to + i * (16 / sizeof(S)));
  } else {
#pragma unroll
    for (int i = 0; i < V - 1; ++i)
      if (i < count) to[i] = e[i];
  }
}

// Values rounded to the storage type.
template <typename T, int V>
__device__ __forceinline__ void round_some(const float (&f)[V], typename T::storage (&e)[V]) {
  if constexpr (T::code == F32::code) {
    __builtin_memcpy(e, f, sizeof(e));
  } else {
    static_assert(V == 8, "16 bytes");
    const U32x4 w{round_pair<T>(f[0], f[1]), round_pair<T>(f[2], f[3]), round_pair<T>(f[4], f[5]),
                  round_pair<T>(f[6], f[7])};
    __builtin_memcpy(e, &w, sizeof(e));
  }
}

// V neighbouring results (row i, columns j .. j + V - 1) on their way out: bias,
// activation, residual; or into the slice's partial sums.
template <typename T, int V>
__device__ __forceinline__ void finish_some(const ProductArgs& p, int slice, int i, int j, float (&v)[V]) {
  using S = typename T::storage;
  using Z = Saved<T>;
  if (i >= p.m || j >= p.n) return;
  const int64_t at = static_cast<int64_t>(i) * p.n + j;
  const int left = p.n - j;
  if (p.slices > 1) {
    store_some<true>(v, p.partial + static_cast<int64_t>(slice) * p.m * p.n + at, left);
    return;
  }
  if (p.bias != nullptr) {
    float b[V];
    if (p.bias_f32) {
      load_some(static_cast<const float*>(p.bias) + j, left, b);
    } else {
      S e[V];
      load_some(static_cast<const S*>(p.bias) + j, left, e);
#pragma unroll
      for (int k = 0; k < V; ++k) b[k] = to_f32<T>(e[k]);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] += b[k];
  }
  if (p.saved != nullptr) {
    float z[V];
    typename Z::storage e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = T::code == F32::code ? v[k] : clamp_saved(v[k]);
    round_some<Z>(z, e);
    store_some(e, static_cast<typename Z::storage*>(p.saved) + at, left);
  }
  if (p.act != FH_ACT_NONE) activate<T>(v, p.act);
  S e[V];
  if (p.residual != nullptr) {
    load_some(static_cast<const S*>(p.residual) + static_cast<int64_t>(i) * p.ldr + j, left, e);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] += to_f32<T>(e[k]);
  }
  round_some<T>(v, e);
  store_some(e, static_cast<S*>(p.out) + at, left);
}

// Rows x 64 results of a wavefront on their way out through 256 bytes a row of its own
// LDS, so that eight lanes (FP32: sixteen) store 64 neighbouring columns of a row, 16 bytes
// each.  16-byte chunk c of row r is at place c ^ (r & 15), which spreads reads and writes
// over the banks.  (FP32 in two stores of 16
// bytes a lane, each instruction over every other 16 bytes, took 107 us for dx of
// 16384 x 4096 into 16, where this takes 85 in the same kernel.)
__device__ __forceinline__ void park(char* area, int r, int c, Floats4 v) {
  *reinterpret_cast<Floats4*>(area + r * 256 + ((c ^ (r & 15)) << 4)) = v;
}
template <typename T, int Rows>
__device__ __forceinline__ void finish_parked(const ProductArgs& p, int slice, const char* area, int row, int col,
                                              int lane) {
  asm volatile("" ::: "memory");  // one wavefront's LDS accesses run in order
  if constexpr (T::code == F32::code) {
#pragma unroll 2
    for (int it = 0; it < Rows / 4; ++it) {
      const int r = 4 * it + (lane >> 4), c = lane & 15;
      float v[4];
      __builtin_memcpy(v, area + r * 256 + ((c ^ (r & 15)) << 4), 16);
      finish_some<T>(p, slice, row + r, col + 4 * c, v);
    }
  } else {
#pragma unroll 2
    for (int it = 0; it < Rows / 8; ++it) {
      const int r = 8 * it + (lane >> 3), c = 2 * (lane & 7);
      float v[8];
      __builtin_memcpy(v, area + r * 256 + ((c ^ (r & 15)) << 4), 16);
      __builtin_memcpy(v + 4, area + r * 256 + (((c + 1) ^ (r & 15)) << 4), 16);
      finish_some<T>(p, slice, row + r, col + 8 * (lane & 7), v);
    }
  }
  asm volatile("" ::: "memory");
}

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));

template <typename E>
__device__ __forceinline__ Floats4 mfma16(U32x4 a, U32x4 b, Floats4 c) {
  if constexpr (E::code == F16::code) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(F16x8, a), __builtin_bit_cast(F16x8, b), c, 0, 0,
                                                  0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0,
                                                   0, 0);
  }
}

typedef float Floats16 __attribute__((ext_vector_type(16)));

template <typename E>
__device__ __forceinline__ Floats16 mfma32(U32x4 a, U32x4 b, Floats16 c) {
  if constexpr (E::code == F16::code) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(F16x8, a), __builtin_bit_cast(F16x8, b), c, 0, 0,
                                                  0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0,
                                                   0, 0);
  }
}

// The tile of a workgroup.  Workgroups go to the eight dies in turn; each die takes
// one eighth of the tiles in a row, eight tiles of m for each n, so that what runs on
// it at a time shares operands in its L2.
struct Tile {
  int m, n;
};
__device__ __forceinline__ Tile tile_of(const ProductArgs& p, int block) {
  const int tiles = p.tiles_m * p.tiles_n, die = block & 7, each = tiles >> 3, more = tiles & 7;
  const int at = die * each + (die < more ? die : more) + (block >> 3);
  const int band = 8 * p.tiles_n, first = at / band * 8;
  const int high = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
  const int in = at - first * p.tiles_n;
  return {first + in % high, in / high};
}

// The steps of Depth in k that a slice of a sum takes.
template <int Depth>
struct Steps {
  int begin, end;
  __device__ __forceinline__ Steps(const ProductArgs& p, int slice) {
    const int64_t steps = (p.k + Depth - 1) / Depth;
    begin = static_cast<int>(steps * slice / p.slices);
    end = static_cast<int>(steps * (slice + 1) / p.slices);
  }
};

// s_waitcnt vmcnt(N) for N up to 63.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt immediate");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

constexpr int64_t kMostStride = int64_t{1} << 22;  // elements: 256 rows of a 16-bit tile within 2^31 bytes

// Sets tiles and slices of a product; a sum in several slices needs slices * m * n
// floats.  `dtype` is the operands' and the output's.
void plan_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols);
// The same for a product with at most 32 rows or columns, and in FP32 whole aligned
// vectors; false for others.
bool plan_narrow_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols);
hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream);
hipError_t launch_f32_product(const ProductArgs& p, bool a_cols, bool b_cols, hipStream_t stream);
hipError_t launch_narrow_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream);
// 16-bit types.
hipError_t launch_wide_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream);

}  // namespace fh
