// Pieces shared by the kernels of the linear layer: activations, the epilogue of
// a product and the description of a product.
#pragma once

#include <type_traits>

#include "fh_kernels.h"
#include "fh_vec.h"
#include "flash_hypercons.h"
#include "workspace.h"

namespace fh {

typedef float Floats4 __attribute__((ext_vector_type(4)));

// What becomes of a product's results: the linear layer's epilogue; the softmax
// statistics of logits, which are not kept; these and the logits' exponentials; the logits'
// gradients; or a sum that goes on from another product's and is scaled at its end.
enum class Finish { kLinear, kStats, kExp, kSlope, kSum };
// The narrow kernel leaves these to the join, in two slices at least: finishing them itself, it kept a frame in scratch
// memory.
constexpr bool joined_if_narrow(Finish f, bool f32) { return f == Finish::kSlope && f32; }
// Those that go by whole rows of 64 logits.
constexpr bool of_logits(Finish f) { return f == Finish::kStats || f == Finish::kExp || f == Finish::kSlope; }

// What the others need beside the product.  Their rows are the first *live ones from
// row0 on (of the sum where A is in columns), as many as there are targets.
struct LossParts {
  const int* live;
  int row0;
  const int* label;      // [rows] targets, negative where out of range
  int col0;              // the vocabulary's entry of column 0
  float2* stats;         // kStats, kExp: [columns / 64, rows] maximum and sum of exponentials, groups stats_ld apart
  int64_t stats_ld;
  float *chosen, *rest;  // kStats, kExp: [rows] logits of the targets, and the sums of their 64 without them
  const float4* row;     // kSlope: [rows] the logarithm of the row's sum, the factor of its gradient, and p - 1 of its target
  int parts;             // kSlope: 2 for dz in two parts, in rows next to each other
  int64_t ld;            // kExp, kSlope: rows of out, whole vectors, zero past n
  float* sums;           // kSum: [m, n] of the sum so far
  int first, last;       // kSum: whether sums is not read, or not written but scaled into out
  const float* scale;    // kSum
  const int* index;      // kSum: [rows] rows of out, or null
  int groups, units;     // kSum, A in rows: workgroups launched and compute units, or 0 where slices stay as planned
};

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
  int paired;            // 16 bits, 128 x 128: two workgroups a compute unit
  float* partial;        // [slices, m, n] where there are several
  const void* bias;      // [n] or null, FP32 or the output's type
  int bias_f32;
  const void* residual;  // [m, n], rows ldr apart, or null
  int64_t ldr;
  int act;
  void* saved;           // receives the sum with its bias, or null
  void* out;             // [m, n] contiguous
};
struct LossProductArgs : ProductArgs {
  LossParts loss;
};
// What a kernel with this finish is given.
template <Finish F>
using ArgsOf = std::conditional_t<F == Finish::kLinear, ProductArgs, LossProductArgs>;
template <Finish F>
ArgsOf<F> args_of(const ProductArgs& p, const LossParts* loss) {
  ArgsOf<F> args{};
  static_cast<ProductArgs&>(args) = p;
  if constexpr (F != Finish::kLinear) args.loss = *loss;
  return args;
}

// Fits a product's rows, or its sum where A is in columns, to what is live.
template <Finish F, bool ACols>
__device__ __forceinline__ void fit_live(ArgsOf<F>& p) {
  if constexpr (F != Finish::kLinear) {
    const int more = *p.loss.live - p.loss.row0, live = more > 0 ? more : 0;
    int& rows = ACols ? p.k : p.m;
    rows = live < rows ? live : rows;
  }
}
// The same and its tiles; false for a workgroup past them.  A sum of fewer rows than it was planned for goes in
// more slices, as far as workgroups were launched, for no compute unit to be without (4096 x 2048 rows of which
// 1640 have a target, 32768 words: dx 325 -> 212 us).
template <Finish F, bool ACols>
__device__ __forceinline__ bool fit(ArgsOf<F>& p) {
  if constexpr (F != Finish::kLinear && !ACols) {
    const int planned = p.tiles_m;
    fit_live<F, ACols>(p);
    p.tiles_m = (p.m + p.side_m - 1) / p.side_m;
    const int tiles = p.tiles_m * p.tiles_n;
    if constexpr (F == Finish::kSum) {
      if (p.loss.groups != 0 && p.tiles_m < planned && tiles > 0) {
        const int most = p.loss.groups < p.loss.units ? p.loss.groups : p.loss.units;
        const int slices = most / tiles < 16 ? most / tiles : 16;
        p.slices = slices > p.slices ? slices : p.slices;
      }
    }
    if constexpr (F == Finish::kSum) return blockIdx.x + gridDim.x * blockIdx.y < static_cast<uint32_t>(tiles * p.slices);
    return blockIdx.x < static_cast<uint32_t>(tiles);
  } else {
    fit_live<F, ACols>(p);
    if constexpr (F == Finish::kSum) return p.k > 0 || p.loss.first || p.loss.last;  // or nothing is added
    return true;
  }
}

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

template <typename T, int V>
__device__ __forceinline__ void add_bias(const ProductArgs& p, int j, int left, float (&v)[V]) {
  using S = typename T::storage;
  if (p.bias == nullptr) return;
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

constexpr float kLog2e = 1.4426950408889634f;

// A value of the lane that the quad's permutation or the mirror of 8 or 16 lanes gives.
template <int Control>
__device__ __forceinline__ float from_lane(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), Control, 0xF, 0xF, true));
}
// f over the values of Lanes neighbouring lanes, the same bits in each.
template <int Lanes, typename F>
__device__ __forceinline__ float over_lanes(float v, F f) {
  v = f(v, from_lane<0xB1>(v));
  v = f(v, from_lane<0x4E>(v));
  if constexpr (Lanes >= 8) v = f(v, from_lane<0x141>(v));
  if constexpr (Lanes >= 16) v = f(v, from_lane<0x140>(v));
  return v;
}

// What a finish needs of a row.  It is loaded for all of a wavefront's rows at once: a load
// waited for in each of eight turns took a quarter of a short sum's time.
template <Finish F>
struct RowOf {
  __device__ __forceinline__ void load(const ArgsOf<F>&, int) {}
};
template <>
struct RowOf<Finish::kStats> {
  int label;
  __device__ __forceinline__ void load(const LossProductArgs& p, int i) { label = i < p.m ? p.loss.label[i] - p.loss.col0 : 0; }
};
template <>
struct RowOf<Finish::kExp> : RowOf<Finish::kStats> {};
template <>
struct RowOf<Finish::kSlope> {
  int label;
  float lse, factor, hit;
  __device__ __forceinline__ void load(const LossProductArgs& p, int i) {
    label = 0;
    lse = factor = hit = 0.f;
    if (i < p.m) {
      const float4 row = p.loss.row[i];
      label = p.loss.label[i] - p.loss.col0;
      lse = row.x;
      factor = row.y;
      hit = row.z;
    }
  }
};

// exp(v - from).  For results of 16 bits by the hardware's exp2, whose argument's rounding is
// worth 2^-23 of |v - from|.  (One multiply-add instead of the difference overflows where both
// are the type's lowest value.)
template <typename T>
__device__ __forceinline__ float exp_from(float v, float from) {
  if constexpr (T::code == F32::code) return expf(v - from);
  return __builtin_amdgcn_exp2f((v - from) * kLog2e);
}

// Exponentials are kept in FP16 beside 16-bit operands, times 2^15: they lie in 0 .. 1, keep 11
// bits down to 2^-29 and are zero below 2^-40, where bf16 would keep 8.
constexpr float kKept = 32768.f;

// Logits of Lanes V neighbouring columns of row i, V a lane: their maximum m and the sum
// of exp(z - m), as far as columns are valid, and the target's logit; for kExp the
// exponentials too.  -inf alone gives m = -inf and a sum of zero; a NaN or +inf makes the sum
// NaN.
template <typename T, Finish F, int Lanes, int V>
__device__ __forceinline__ void stats_some(const LossProductArgs& p, const RowOf<F>& of, int i, int j,
                                           float (&v)[V]) {
  if (i >= p.m) return;  // the same in all of these lanes
  const int left = p.n - j;
  if (left > 0) add_bias<T>(p, j, left, v);
  const float none = -__builtin_inff();
  if (left < V) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k < left ? v[k] : none;
  }
  float m = v[0];
#pragma unroll
  for (int k = 1; k < V; ++k) m = __builtin_fmaxf(m, v[k]);
  m = over_lanes<Lanes>(m, [](float a, float b) { return __builtin_fmaxf(a, b); });
  const float from = m == none ? 0.f : m;
  const int at = of.label - j;
  if (at >= 0 && at < V && at < left) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k == at) p.loss.chosen[i] = v[k];
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    v[k] = exp_from<T>(v[k], from);
    s += v[k];
  }
  const int inside = of.label - (j & ~63);
  if (inside >= 0 && inside < 64) {  // the same in all of these lanes
    float rest = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) rest += k == at ? 0.f : v[k];
    rest = over_lanes<Lanes>(rest, [](float a, float b) { return a + b; });
    if (j % 64 == 0) p.loss.rest[i] = rest;
  }
  if (F == Finish::kExp && j < p.loss.ld) {
    using Z = Saved<T>;
    auto* to = static_cast<typename Z::storage*>(p.out) + static_cast<int64_t>(i) * p.loss.ld + j;
    if constexpr (T::code == F32::code) {
      __builtin_memcpy(to, v, sizeof(v));
    } else {
      typename Z::storage e[V];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] *= kKept;
      round_some<Z>(v, e);
      store_some(e, to, V);
    }
  }
  s = over_lanes<Lanes>(s, [](float a, float b) { return a + b; });
  if (j % 64 == 0 && left > 0) p.loss.stats[static_cast<int64_t>(j / 64) * p.loss.stats_ld + i] = make_float2(m, s);
}

// Logits on their way to the gradients of z: (exp(z - lse) - [target]) times the row's
// factor, rounded to the storage type, which the products that follow take.  (Root mean
// square 0.0017 of a term in bf16, beside as much for their results' own rounding.  Of few rows
// one term makes most of a result, which may then be off by 2^-9: those come in two parts.)
template <typename T, int V>
__device__ __forceinline__ void slope_some(const LossProductArgs& p, const RowOf<Finish::kSlope>& of, int i, int j,
                                           float (&v)[V]) {
  using S = typename T::storage;
  if (i >= p.m || j >= p.loss.ld) return;
  const int left = p.n - j, at = of.label - j;
  if (left > 0) add_bias<T>(p, j, left, v);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = exp_from<T>(v[k], of.lse);
  if (at >= 0 && at < V) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k == at ? of.hit : v[k];
  }
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] *= of.factor;
  if (left < V) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k < left ? v[k] : 0.f;
  }
  S e[V];
  round_some<T>(v, e);
  S* to = static_cast<S*>(p.out) + static_cast<int64_t>(i) * p.loss.parts * p.loss.ld + j;
  __builtin_memcpy(to, e, sizeof(e));
  if (T::code != F32::code && p.loss.parts == 2) {
    // What the first part leaves out, in the next row.
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] -= to_f32<T>(e[k]);
    round_some<T>(v, e);
    __builtin_memcpy(to + p.loss.ld, e, sizeof(e));
  }
}

// V results of a sum on their way into the sum so far, or at its end scaled and out.
template <typename T, int V>
__device__ __forceinline__ void sum_some(const LossProductArgs& p, int i, int j, float (&v)[V]) {
  using S = typename T::storage;
  const int64_t at = static_cast<int64_t>(i) * p.n + j;
  const int left = p.n - j;
  if (!p.loss.first) {
    float before[V];
    load_some(p.loss.sums + at, left, before);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] += before[k];
  }
  if (!p.loss.last) {
    store_some<true>(v, p.loss.sums + at, left);
    return;
  }
  const float scale = *p.loss.scale;
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] *= scale;
  S e[V];
  round_some<T>(v, e);
  const int64_t row = p.loss.index != nullptr ? p.loss.index[i] : i;
  store_some(e, static_cast<S*>(p.out) + row * p.n + j, left);
}

// V neighbouring results (row i, columns j .. j + V - 1) into the slice's partial sums.
template <int V>
__device__ __forceinline__ void keep_some(const ProductArgs& p, int slice, int i, int j, const float (&v)[V]) {
  if (i < p.m && j < p.n)
    store_some<true>(v, p.partial + (static_cast<int64_t>(slice) * p.m + i) * p.n + j, p.n - j);
}

// The same on their way out: bias, activation, residual; or into the slice's partial sums, but
// for finishes of logits, which are whole sums here.  Lanes neighbouring lanes have the results
// beside these.
template <typename T, Finish F, int Lanes, int V>
__device__ __forceinline__ void finish_some(const ArgsOf<F>& p, const RowOf<F>& of, int slice, int i, int j,
                                            float (&v)[V]) {
  using S = typename T::storage;
  using Z = Saved<T>;
  if constexpr (F == Finish::kSlope) {
    slope_some<T>(p, of, i, j, v);
    return;
  } else if constexpr (of_logits(F)) {
    stats_some<T, F, Lanes>(p, of, i, j, v);
    return;
  }
  if (i >= p.m || j >= p.n) return;
  if (p.slices > 1) {
    keep_some(p, slice, i, j, v);
    return;
  }
  const int64_t at = static_cast<int64_t>(i) * p.n + j;
  const int left = p.n - j;
  if constexpr (F == Finish::kSum) {
    sum_some<T>(p, i, j, v);
    return;
  }
  add_bias<T>(p, j, left, v);
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
template <typename T, Finish F, int Rows>
__device__ __forceinline__ void finish_parked(const ArgsOf<F>& p, int slice, const char* area, int row, int col,
                                              int lane) {
  if constexpr (F == Finish::kSum && T::code != F32::code) {
    // FP32 sums in whole lines, sixteen lanes to a row, four rows' loads on their way at a time.
    if (p.slices == 1 && !p.loss.last) {
      asm volatile("" ::: "memory");
      const int c = lane & 15, j = col + 4 * c, left = p.n - j;
#pragma unroll 1
      for (int it = 0; it < Rows / 4; it += 4) {
        float before[4][4] = {};
        int64_t at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = row + 4 * (it + u) + (lane >> 4);
          at[u] = i < p.m && left > 0 ? static_cast<int64_t>(i) * p.n + j : -1;
          if (!p.loss.first && at[u] >= 0) load_some(p.loss.sums + at[u], left, before[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = 4 * (it + u) + (lane >> 4);
          float v[4];
          __builtin_memcpy(v, area + r * 256 + ((c ^ (r & 15)) << 4), 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] += before[u][k];
          if (at[u] >= 0) store_some(v, p.loss.sums + at[u], left);
        }
      }
      asm volatile("" ::: "memory");
      return;
    }
  }
  constexpr int down = T::code == F32::code ? 4 : 8, turns = Rows / down;  // rows at a time
  const int first = T::code == F32::code ? lane >> 4 : lane >> 3;
  if constexpr (of_logits(F)) {
    if (p.slices > 1) {
      asm volatile("" ::: "memory");
#pragma unroll 2
      for (int it = 0; it < Rows / 4; ++it) {
        const int r = 4 * it + (lane >> 4), c = lane & 15;
        float v[4];
        __builtin_memcpy(v, area + r * 256 + ((c ^ (r & 15)) << 4), 16);
        keep_some(p, slice, row + r, col + 4 * c, v);
      }
      asm volatile("" ::: "memory");
      return;
    }
  }
  RowOf<F> of[turns];
#pragma unroll
  for (int it = 0; it < turns; ++it) of[it].load(p, row + first + down * it);
  asm volatile("" ::: "memory");  // one wavefront's LDS accesses run in order
  const auto turn = [&](int it) {
    const int r = down * it + first;
    if constexpr (T::code == F32::code) {
      const int c = lane & 15;
      float v[4];
      __builtin_memcpy(v, area + r * 256 + ((c ^ (r & 15)) << 4), 16);
      finish_some<T, F, 16>(p, of[it], slice, row + r, col + 4 * c, v);
    } else {
      const int c = 2 * (lane & 7);
      float v[8];
      __builtin_memcpy(v, area + r * 256 + ((c ^ (r & 15)) << 4), 16);
      __builtin_memcpy(v + 4, area + r * 256 + (((c + 1) ^ (r & 15)) << 4), 16);
      finish_some<T, F, 8>(p, of[it], slice, row + r, col + 8 * (lane & 7), v);
    }
  };
  if constexpr (of_logits(F)) {
#pragma unroll
    for (int it = 0; it < turns; ++it) turn(it);
  } else {
#pragma unroll 2
    for (int it = 0; it < turns; ++it) turn(it);
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

// The same with the sum's slices.  With B in columns each die takes one eighth of the slices' tiles, those of a
// slice in a row, so that most dies read a part of the operands that no other does, and whole rows of it: the 256
// bytes that a tile has of each lie in few of an L2's channels (dx of 200 x 1024 into 50001 words, 16 slices: 60
// -> 42 us).  In rows the other way is 6% faster (64 x 16384 x 4096).
struct Piece {
  Tile tile;
  int slice;
};
template <bool BCols>
__device__ __forceinline__ Piece piece_of(const ProductArgs& p) {
  if (!BCols || p.slices == 1) return {tile_of(p, blockIdx.x), static_cast<int>(blockIdx.y)};
  const int tiles = p.tiles_m * p.tiles_n, all = tiles * p.slices;
  const int block = blockIdx.x + gridDim.x * blockIdx.y, die = block & 7, each = all >> 3, more = all & 7;
  const int at = die * each + (die < more ? die : more) + (block >> 3);
  const int slice = at / tiles, in = at % tiles;
  return {{in % p.tiles_m, in / p.tiles_m}, slice};
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
void plan_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish = Finish::kLinear);
// The same for a product with at most 32 rows or columns, and in FP32 whole aligned
// vectors; false for others.  Not for kExp, whose products have many rows.
bool plan_narrow_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish);
// `loss` is null for Finish::kLinear.
hipError_t launch_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, hipStream_t stream,
                          Finish finish = Finish::kLinear, const LossParts* loss = nullptr);
hipError_t launch_f32_product(const ProductArgs& p, bool a_cols, bool b_cols, Finish finish, const LossParts* loss,
                              hipStream_t stream);
hipError_t launch_narrow_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish,
                                 const LossParts* loss, hipStream_t stream);
// 16-bit types.
hipError_t launch_wide_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish,
                               const LossParts* loss, hipStream_t stream);

// Calls f with the operands' layouts and the finish as types, where there is such a product:
// of rows by rows (logits and their gradients too), rows by columns, columns by columns.
template <bool B>
using Flag = std::integral_constant<bool, B>;
template <Finish F>
using FinishType = std::integral_constant<Finish, F>;
template <typename Call>
hipError_t with_layout(bool a_cols, bool b_cols, Finish finish, Call call) {
  if (!a_cols && !b_cols) {
    if (finish == Finish::kLinear) return call(Flag<false>{}, Flag<false>{}, FinishType<Finish::kLinear>{});
    if (finish == Finish::kStats) return call(Flag<false>{}, Flag<false>{}, FinishType<Finish::kStats>{});
    if (finish == Finish::kExp) return call(Flag<false>{}, Flag<false>{}, FinishType<Finish::kExp>{});
    if (finish == Finish::kSlope) return call(Flag<false>{}, Flag<false>{}, FinishType<Finish::kSlope>{});
  } else if (b_cols) {
    if (finish == Finish::kLinear && !a_cols) return call(Flag<false>{}, Flag<true>{}, FinishType<Finish::kLinear>{});
    if (finish == Finish::kLinear) return call(Flag<true>{}, Flag<true>{}, FinishType<Finish::kLinear>{});
    if (finish == Finish::kSum && !a_cols) return call(Flag<false>{}, Flag<true>{}, FinishType<Finish::kSum>{});
    if (finish == Finish::kSum) return call(Flag<true>{}, Flag<true>{}, FinishType<Finish::kSum>{});
  }
  return hipErrorInvalidValue;  // no such product
}

// An operand as the products read it.
struct Laid {
  const void* data;
  int64_t ld;
};

// `data` [rows, cols] as it is where the products read it so, or laid out anew in the workspace.
hipError_t lay_out(const void* data, int64_t stride, int64_t rows, int64_t cols, int dtype, Workspace& ws, Laid& got,
                   hipStream_t stream);

}  // namespace fh
