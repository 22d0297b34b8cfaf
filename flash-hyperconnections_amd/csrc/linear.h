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
// row for each k).  FP32 operands come as three bf16 planes, `plane` elements
// apart, whose sum they are.
struct ProductArgs {
  const uint16_t *a, *b;
  int64_t lda, ldb;
  int64_t plane_a, plane_b;
  int m, n, k;
  int tiles_m, tiles_n;
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
// the slope's error well below that of rounding dz (bf16 would add a third to the
// error of the weight's gradient).
template <typename T>
using Saved = std::conditional_t<T::code == F32::code, F32, F16>;

__device__ __forceinline__ float clamp_saved(float z) { return z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z; }

// act(z); relu keeps a NaN.
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case FH_ACT_RELU: return z < 0.f ? 0.f : z;
    case FH_ACT_GELU: return z * (0.5f * (1.f + erff(z * 0.70710678118654752f)));
    case FH_ACT_GELU_TANH: {
      // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), without the difference of near values.
      const float u2 = 1.5957691216057308f * __builtin_fmaf(0.044715f * z * z, z, z);
      return z / (1.f + expf(-u2));
    }
    case FH_ACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}

// act'(z).
__device__ __forceinline__ float slope(float z, int act) {
  switch (act) {
    case FH_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case FH_ACT_GELU:
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * (0.39894228040143268f * expf(-0.5f * z * z));
    case FH_ACT_GELU_TANH: {
      const float u2 = 1.5957691216057308f * __builtin_fmaf(0.044715f * z * z, z, z);
      const float q = 1.f / (1.f + expf(-u2));
      const float du2 = 1.5957691216057308f * __builtin_fmaf(0.134145f * z, z, 1.f);
      // q (1 - q) is 0 where exp has left its range, whatever z du2 is.
      const float curve = q * (1.f - q);
      return curve > 0.f ? __builtin_fmaf(z * du2, curve, q) : q;
    }
    case FH_ACT_SILU: {
      const float q = 1.f / (1.f + expf(-z)), curve = q * (1.f - q);
      return curve > 0.f ? __builtin_fmaf(z, curve, q) : q;
    }
    default: return 1.f;
  }
}

// Four neighbouring results (row i, columns j .. j + 3) on their way out.
template <typename T>
__device__ __forceinline__ void finish_four(const ProductArgs& p, int i, int j, const float (&sum)[4]) {
  using S = typename T::storage;
  using Z = typename Saved<T>::storage;
  const int64_t at = static_cast<int64_t>(i) * p.n + j;
  const int left = p.n - j;
  S r[4] = {};
  if (p.residual != nullptr) {
    const S* from = static_cast<const S*>(p.residual) + static_cast<int64_t>(i) * p.ldr + j;
    if (left >= 4) {
      __builtin_memcpy(r, from, sizeof(r));
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < left) r[e] = from[e];
    }
  }
  S y[4];
  Z z[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float v = sum[e];
    if (p.bias != nullptr) v += e < left ? load_param<T>(p.bias, p.bias_f32, j + e) : 0.f;
    z[e] = T::code == F32::code ? static_cast<Z>(v) : static_cast<Z>(clamp_saved(v));
    v = activate(v, p.act);
    if (p.residual != nullptr) v += to_f32<T>(r[e]);
    y[e] = from_f32<T>(v);
  }
  S* out = static_cast<S*>(p.out) + at;
  Z* saved = static_cast<Z*>(p.saved) + at;
  if (left >= 4) {
    __builtin_memcpy(out, y, sizeof(y));
    if (p.saved != nullptr) __builtin_memcpy(saved, z, sizeof(z));
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) {
        out[e] = y[e];
        if (p.saved != nullptr) saved[e] = z[e];
      }
  }
}

// Sets tiles and slices of a product; a sum in several slices needs slices * m * n
// floats.  `dtype` is the output's; FP32 runs on bf16 planes.
void plan_product(ProductArgs& p, int dtype);
hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream);

}  // namespace fh
