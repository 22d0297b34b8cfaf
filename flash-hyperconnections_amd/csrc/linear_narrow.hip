// Matrix products of the linear layer where one operand has at most 32 rows: a few
// tokens through a large weight, or many tokens into a few outputs.  They read the
// other operand once, at the rate that HBM gives; the matrix cores are idle for most
// of it.
//
// A wavefront streams strips of the long operand, 64 rows and 64 of the sum's terms at
// a time, through three buffers of its own, so that it meets nobody and two strips are
// on their way while it works on one: 64 KB a compute unit, what it takes to keep HBM
// busy.  Where the long operand is in rows the four wavefronts of a workgroup take
// every fourth strip of the same rows and add their sums at the end; in columns they
// take neighbouring 64 columns each.
//
// Taken up to 32 rows, one strip's worth of the short operand.  1 x 4096 x 16384 bf16 takes
// 22 us (6.0 TB/s) in one launch, in 128 x 128 tiles 22 and 4 for the join; 16384 x 16384
// into 16 takes 94 us (5.7 TB/s), 102 to 106 before in those tiles.
//
// FP32 operands stream in strips of as many bytes, 32 of the sum's terms, and are split
// into bf16 parts on their way from LDS; they have to be whole aligned vectors, and go
// through the tiles otherwise.  Calls, in the tiles before: 1 x 4096 x 16384 takes 46 us
// forward (104) and 66 for dx (106), 1 x 4096 x 4096 20 (33) and 27 (33); dW of 16384 x
// 4096 into 16 takes 70 to 72 (107).
#include <algorithm>
#include <type_traits>

#include "linear_parts.h"

namespace fh {
namespace {

constexpr int kRing = 3, kLong = 64, kShort = 32, kLine = 128;  // bytes of a row of a strip
constexpr int kLongBytes = kLong * kLine, kShortBytes = kShort * kLine;
template <typename T>
constexpr int kDepth = kLine / static_cast<int>(sizeof(typename T::storage));  // of the sum's terms in a strip
constexpr int kSlot = kLongBytes + kShortBytes;  // a strip of both operands
constexpr int kLoads = kSlot / 1024;             // of a strip

typedef short S16x4 __attribute__((ext_vector_type(4)));
using LdsShorts = __attribute__((address_space(3))) S16x4;
using LdsBytes = __attribute__((address_space(3))) char;

// Span rows (columns) of an operand, E bytes an element.  In rows: Span rows of 128 bytes,
// 16-byte chunk c of row r at place c ^ ((r >> 1) & 7).  In columns, a row for each k: 16
// bits, 64 rows, chunk c of row k at place c ^ swap_of(k); FP32, 32 rows, of 64 columns
// likewise and of 32 with row k at place slot_of(k).
template <int E, bool Cols, int Span>
struct Strip {
  static constexpr int kDepth = kLine / E, kVec = 16 / E;
  static constexpr int kCount = Span / 8;                      // loads
  static constexpr int kRows = Cols ? 1024 / (Span * E) : 8;   // rows of memory in each
  const char* base;
  int64_t step;
  int32_t row, voff[2];
  int rows, at_k;

  __device__ __forceinline__ static int swap_of(int k) {
    if constexpr (E == 4) return Span == 64 ? ((k >> 2) & 1) << 3 : 0;
    return Span == 64 ? (((k >> 1) & 1) << 2) | (((k >> 3) & 1) << 1) : ((k >> 3) & 1) << 1;
  }
  __device__ __forceinline__ static int slot_of(int k) { return E == 4 && Span == 32 ? k ^ ((k >> 2) & 1) : k; }
  __device__ __forceinline__ void init(const void* operand, int64_t ld, int first, int count, int lane) {
    base = static_cast<const char*>(operand) + E * (Cols ? static_cast<int64_t>(first) : first * ld);
    row = static_cast<int32_t>(E * ld);
    step = Cols ? kDepth * static_cast<int64_t>(row) : kLine;
    rows = count - first;
    if constexpr (Cols) {
      constexpr int across = Span / kVec;  // chunks of a row
      at_k = slot_of(lane / across);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = (lane % across) ^ swap_of(at_k + u * kRows);
        voff[u] = first + kVec * c < count ? at_k * row + 16 * c : kOutOfRange;
      }
    } else {
      at_k = kVec * ((lane & 7) ^ (lane >> 4));
#pragma unroll
      for (int u = 0; u < 2; ++u) voff[u] = (lane >> 3) * row + E * (at_k ^ (4 * kVec * u));
    }
  }
  // Loads the strip of step t, zero past the sum's end and the last row.
  __device__ __forceinline__ void stage(int t, int k, uint32_t lds) const {
    const char* from = base + t * step;
    const int left = k - t * kDepth;
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      U32x4 rs = rsrc_words(from + static_cast<int64_t>(u * kRows) * row);
      int at;
      if constexpr (Cols) {
        at = at_k + u * kRows;
      } else {
        // The last valid row's last chunk of this step ends the resource.
        const int more = rows - 8 * u < 8 ? rows - 8 * u : 8;
        rs[2] = more > 0 ? (more - 1) * row + E * (left < kDepth ? (left + kVec - 1) & -kVec : kDepth) : 0;
        at = at_k ^ (4 * kVec * (u & 1));
      }
      lds_load16(rs, lds + u * 1024, at < left ? voff[u & 1] : kOutOfRange, 0);
    }
  }
  // 16 bits: elements k = 16 kk + 8 (lane / 32) + 0..7 of row (column) 32 i + lane % 32.
  __device__ __forceinline__ static U32x4 read(uint32_t lds, int i, int kk, int lane) {
    static_assert(E == 2, "16-bit elements");
    U32x4 w;
    if constexpr (Cols) {
      const int j = lane & 15, g = lane >> 4, k = 8 * (g >> 1) + (j >> 2);
      const int c = (i << 2) + ((g & 1) << 1) + ((j & 3) >> 1);
      auto* p = reinterpret_cast<LdsBytes*>(lds + k * (2 * Span) + ((c ^ swap_of(k)) << 4) + ((j & 1) << 3)) +
                kk * 16 * 2 * Span;
      const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)p);
      const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)(p + 4 * 2 * Span));
      // Rows k + 4 change places like rows k where the exchange goes by k >> 3 and k >> 1.
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      w = U32x4{l.x, l.y, h.x, h.y};
    } else {
      w = chunk(lds, 32 * i + (lane & 31), 2 * kk + (lane >> 5));
    }
    return w;
  }
  // FP32: elements k = 16 kk + 8 (e / 4) + 4 (lane / 32) + e % 4, e = 0..7, of the same.  Any
  // order of the terms does that both operands have, and in rows this one reads as 16 bits do.
  __device__ __forceinline__ static void read_floats(uint32_t lds, int i, int kk, int lane, float (&v)[8]) {
    static_assert(E == 4, "FP32 elements");
    const int r = 32 * i + (lane & 31), h = lane >> 5;
    if constexpr (Cols) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = 16 * kk + 8 * (e >> 2) + 4 * h + (e & 3);
        const uint32_t at = lds + slot_of(k) * (E * Span) + (((r >> 2) ^ swap_of(k)) << 4) + (r & 3) * 4;
        v[e] = *(__attribute__((address_space(3))) float*)reinterpret_cast<LdsBytes*>(at);
      }
    } else {
      const U32x4 lo = chunk(lds, r, 4 * kk + h), hi = chunk(lds, r, 4 * kk + 2 + h);
      __builtin_memcpy(v, &lo, 16);
      __builtin_memcpy(v + 4, &hi, 16);
    }
  }

 private:
  __device__ __forceinline__ static U32x4 chunk(uint32_t lds, int r, int c) {
    return *(__attribute__((address_space(3))) U32x4*)reinterpret_cast<LdsBytes*>(lds + r * kLine +
                                                                                 ((c ^ ((r >> 1) & 7)) << 4));
  }
};

// The three parts of 8 values each of a lane's three fragments.
__device__ __forceinline__ void split_three(const float (&v)[3][8], U32x4 (&w)[3][3]) {
  uint2 part[3][2][3];
  float odd = 0.f;
  float quad[3][2][4];
  __builtin_memcpy(quad, v, sizeof(quad));
#pragma unroll
  for (int f = 0; f < 3; ++f)
#pragma unroll
    for (int q = 0; q < 2; ++q) split(quad[f][q], part[f][q], odd);
  if (__builtin_expect(__any(odd != odd), 0)) {
#pragma unroll
    for (int f = 0; f < 3; ++f)
#pragma unroll
      for (int q = 0; q < 2; ++q) split_exactly(quad[f][q], part[f][q]);
  }
#pragma unroll
  for (int f = 0; f < 3; ++f)
#pragma unroll
    for (int i = 0; i < 3; ++i)
      w[f][i] = U32x4{part[f][0][i].x, part[f][0][i].y, part[f][1][i].x, part[f][1][i].y};
}

// LongA: A is the long operand.
template <typename T, bool LongA, bool LongCols, bool ShortCols, Finish F>
__global__ __launch_bounds__(256) void narrow_product_kernel(ArgsOf<F> p) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * kRing * kSlot];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slice = blockIdx.y;
  // Each die takes neighbouring tiles: in columns one tile's 512 bytes of a row lie in two
  // of an L2's sixteen channels.
  const Tile tile = tile_of(p, blockIdx.x);
  fit_live<F, LongA ? LongCols : ShortCols>(p);
  const int first = (tile.m + tile.n) * (LongCols ? 4 * kLong : kLong) + (LongCols ? wave * kLong : 0);
  constexpr bool f32 = T::code == F32::code;
  constexpr int E = f32 ? 4 : 2;
  const Steps<kDepth<T>> steps(p, slice);
  // In rows a wavefront takes every fourth strip.
  const int begin = steps.begin + (LongCols ? 0 : wave), by = LongCols ? 1 : 4;
  const int count = steps.end > begin ? (steps.end - begin + by - 1) / by : 0;
  Strip<E, LongCols, kLong> l;
  Strip<E, ShortCols, kShort> s;
  l.init(LongA ? p.a : p.b, LongA ? p.lda : p.ldb, first, LongA ? p.m : p.n, lane);
  s.init(LongA ? p.b : p.a, LongA ? p.ldb : p.lda, 0, LongA ? p.n : p.m, lane);
  const uint32_t ring = lds_address(lds) + wave * kRing * kSlot;
  const auto stage = [&](int i) {
    const uint32_t to = ring + i % kRing * kSlot;
    l.stage(begin + i * by, p.k, to);
    s.stage(begin + i * by, p.k, to + kLongBytes);
  };
  Floats16 acc[2], small[2];  // FP32: the leading products of parts, and the five next ones
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = small[i][e] = 0.f;
  if (first < (LongA ? p.m : p.n)) {
    for (int i = 0; i < kRing && i < count; ++i) stage(i);
    for (int i = 0; i < count; ++i) {
      // Strip i is there once only the loads of the strips behind it are on their way.
      if (i + 2 < count) wait_loads<2 * kLoads>();
      else if (i + 1 < count) wait_loads<kLoads>();
      else wait_loads<0>();
      asm volatile("" ::: "memory");
      const uint32_t at = ring + i % kRing * kSlot;
      if constexpr (f32) {
        float v[2][3][8];  // [kk][the long operand's two fragments, the short one's]
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          l.read_floats(at, 0, kk, lane, v[kk][0]);
          l.read_floats(at, 1, kk, lane, v[kk][1]);
          s.read_floats(at + kLongBytes, 0, kk, lane, v[kk][2]);
        }
        wait_lds();
        asm volatile("" ::: "memory");
        if (i + kRing < count) stage(i + kRing);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          U32x4 w[3][3];
          split_three(v[kk], w);
          const auto add = [&](int a, int b, Floats16(&to)[2]) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              to[j] = LongA ? mfma32<BF16>(w[2][b], w[j][a], to[j]) : mfma32<BF16>(w[j][a], w[2][b], to[j]);
          };
          add(2, 0, small);
          add(0, 0, acc);
          add(0, 2, small);
          add(1, 1, small);
          add(1, 0, small);
          add(0, 1, small);
        }
      } else {
        U32x4 x[2][4], y[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          x[0][kk] = l.read(at, 0, kk, lane);
          x[1][kk] = l.read(at, 1, kk, lane);
          y[kk] = s.read(at + kLongBytes, 0, kk, lane);
        }
        wait_lds();
        asm volatile("" ::: "memory");
        if (i + kRing < count) stage(i + kRing);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            // The operand whose rows are the results' columns first: a lane holds four neighbouring ones.
            acc[j] = LongA ? mfma32<T>(y[kk], x[j][kk], acc[j]) : mfma32<T>(x[j][kk], y[kk], acc[j]);
      }
    }
  }
  if constexpr (f32) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][e] += small[j][e];
  }
  // [m][n] of a wavefront's sums in its own part of the ring: 64 x 32 or 32 x 64.
  constexpr int across = LongA ? kShort : kLong, down = LongA ? kLong : kShort;
  wait_lds();
  float* area = reinterpret_cast<float*>(lds + wave * kRing * kSlot);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = (LongA ? 32 * j : 0) + (lane & 31), n = (LongA ? 0 : 32 * j) + 8 * q + 4 * (lane >> 5);
      const int c = (n >> 2) ^ (m & 7);  // 16-byte chunks of a row change places by the row
      *reinterpret_cast<Floats4*>(area + m * across + 4 * c) =
          Floats4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    }
  const auto get = [&](const float* from, int m, int n, float (&v)[8]) {
    __builtin_memcpy(v, from + m * across + 4 * ((n >> 2) ^ (m & 7)), 16);
    __builtin_memcpy(v + 4, from + m * across + 4 * (((n >> 2) + 1) ^ (m & 7)), 16);
  };
  constexpr int groups = across / 8;
  if constexpr (LongCols) {
    asm volatile("" ::: "memory");
#pragma unroll 1
    for (int i = lane; i < groups * down; i += 64) {
      const int m = i / groups, n = i % groups * 8;
      float v[8];
      get(area, m, n, v);
      const int row = (LongA ? first : 0) + m, col = (LongA ? 0 : first) + n;
      if constexpr (joined_if_narrow(F, f32)) {
        keep_some(p, slice, row, col, v);
      } else {
        RowOf<F> of;
        of.load(p, row);
        finish_some<T, F, groups>(p, of, slice, row, col, v);
      }
    }
  } else {
    const int m = threadIdx.x / groups, n = threadIdx.x % groups * 8;
    __syncthreads();
    static_assert(groups * down == 256, "one group of results a thread");
    float v[8], w[8];
    get(reinterpret_cast<const float*>(lds), m, n, v);
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      get(reinterpret_cast<const float*>(lds + k * kRing * kSlot), m, n, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e];
    }
    const int i = (LongA ? first : 0) + m, j = (LongA ? 0 : first) + n;
    if constexpr (joined_if_narrow(F, f32)) {
      keep_some(p, slice, i, j, v);
    } else if (of_logits(F) && p.slices > 1) {
      keep_some(p, slice, i, j, v);
    } else {
      RowOf<F> of;
      of.load(p, i);
      finish_some<T, F, groups>(p, of, slice, i, j, v);
    }
  }
}

}  // namespace

bool plan_narrow_product(ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish) {
  if (p.m > kShort && p.n > kShort) return false;
  const bool f32 = dtype == F32::code;
  if (f32) {
    // Whole 16-byte vectors; 16-bit operands come so.
    const auto whole = [&](const void* data, int64_t ld, int count) {
      return reinterpret_cast<uintptr_t>(data) % 16 == 0 && ld % 4 == 0 && ld < kMostStride && count % 4 == 0;
    };
    if (!whole(p.a, p.lda, a_cols ? p.m : p.k) || !whole(p.b, p.ldb, b_cols ? p.n : p.k)) return false;
  }
  const bool long_a = p.m > p.n, cols = long_a ? a_cols : b_cols;
  p.side_m = p.side_n = kShort;
  p.tiles_m = p.tiles_n = 1;
  const int side = cols ? 4 * kLong : kLong;
  int& tiles = long_a ? p.tiles_m : p.tiles_n;
  tiles = ((long_a ? p.m : p.n) + side - 1) / side;
  const int depth = f32 ? kDepth<F32> : kDepth<F16>;
  const int64_t steps = (p.k + depth - 1) / depth;
  // Slices of at least four strips a wavefront until every compute unit has a workgroup; in
  // columns of 16 bits three for each (dW of 16384 x 16384 into 16: 149 us with 4 slices, 90
  // with 12); FP32 one (dx of 1 x 4096 x 16384: 69 us, with three 83).
  // A sum of the loss in whole rounds of the compute units only: FP32 gradients of 12 x 3456 into 122688 take 1095 us
  // with 18 slices of 14 tiles, 1325 with 19; bf16 of 1 x 3456 487 and 500.
  const int64_t groups = compute_units() * (cols && !f32 ? 3 : 1);
  const int64_t most = finish == Finish::kSum ? groups / tiles : (groups + tiles - 1) / tiles;
  p.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, steps / (cols ? 4 : 16))));
  return true;
}

hipError_t launch_narrow_product(const ProductArgs& p, int dtype, bool a_cols, bool b_cols, Finish finish,
                                 const LossParts* loss, hipStream_t stream) {
  const bool long_a = p.m > p.n;
  const dim3 grid(static_cast<uint32_t>(long_a ? p.tiles_m : p.tiles_n), static_cast<uint32_t>(p.slices)), block(256);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_layout(a_cols, b_cols, finish, [&](auto a, auto b, auto f) {
      if constexpr (f.value == Finish::kExp) {
        return hipErrorInvalidValue;  // planned in tiles
      } else {
        if (long_a) narrow_product_kernel<T, true, a.value, b.value, f.value><<<grid, block, 0, stream>>>(args_of<f.value>(p, loss));
        else narrow_product_kernel<T, false, b.value, a.value, f.value><<<grid, block, 0, stream>>>(args_of<f.value>(p, loss));
        return hipGetLastError();
      }
    });
  });
}

}  // namespace fh
