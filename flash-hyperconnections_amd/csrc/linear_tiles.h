// How the operands of a product in tiles go through LDS.
#pragma once

#include "linear.h"

namespace fh {
namespace {

constexpr int kStep = 64;  // of the sum's terms

__device__ __forceinline__ int swap_of(int k) { return 2 * (((k & 3) << 1) | ((k >> 3) & 1)); }

// One operand's way into LDS, Side of its rows (columns) and 64 of the sum's terms a
// step.  In rows: Side rows of 64 elements, 16-byte chunk c of row r at place
// c ^ ((r >> 1) & 7).  In columns: 64 rows of Side, chunk c of row k at place
// c ^ swap_of(k).  Both spread every wavefront's reads over all banks.
//
// Each of eight wavefronts has kLoads loads a step, whose resources move with the steps.
// Nothing here branches: a lane past the sum's end, in its last step or beyond it,
// loads from out of range, which gives zeros.
template <bool Cols, int Side>
struct Feeder {
  static constexpr int kLoads = Side / 64;
  static constexpr int kRows = Cols ? 512 / Side : 8;  // rows of memory in a load
  U32x4 rsrc[kLoads];
  int64_t step;     // bytes from one step in k to the next
  int32_t voff[2];  // of the even and the odd loads
  int at_k;         // the first k of this lane's chunk in load 0
  int left;         // elements of the sum from here on
  uint32_t lds;     // where this wavefront's loads go in the first buffer

  // Side rows (columns) from `first` on, of `count`; the sum has k terms, and `begin` steps of it are left out.
  __device__ __forceinline__ void init(const void* operand, int64_t ld, int first, int count, int k, int begin,
                                       uint32_t to, int lane, int wave) {
    const auto* data = static_cast<const uint16_t*>(operand);
    lds = to + wave * kLoads * 1024;
    const int32_t row = static_cast<int32_t>(2 * ld);
    if constexpr (Cols) {
      constexpr int across = Side / 8;  // chunks of a row
      step = 2 * kStep * ld;
      at_k = wave * 8 + lane / across;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = (lane % across) ^ swap_of(at_k + u * kRows);
        voff[u] = first + 8 * c < count ? lane / across * row + 16 * c : kOutOfRange;
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u) rsrc[u] = rsrc_words(data + first + (wave * 8 + u * kRows) * ld);
    } else {
      step = 2 * kStep;
      at_k = 8 * ((lane & 7) ^ (lane >> 4));
#pragma unroll
      for (int u = 0; u < 2; ++u) voff[u] = (lane >> 3) * row + 2 * (at_k ^ (32 * u));
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        // The last valid row's end in this step ends the resource (its chunks are whole).
        const int from = first + (wave * kLoads + u) * 8, more = count - from < 8 ? count - from : 8;
        rsrc[u] = rsrc_words(data + from * ld);
        rsrc[u][2] = more > 0 ? (more - 1) * row + 2 * (k < kStep ? (k + 7) & ~7 : kStep) : 0;
      }
    }
    left = k;
    advance(begin);
  }
  // Loads load u of this step into the buffer `offset` bytes on, zero past the sum's end and the last row.
  __device__ __forceinline__ void stage(int u, int offset) const {
    const int k = Cols ? at_k + u * kRows : at_k ^ (32 * (u & 1));
    lds_load16(rsrc[u], lds + offset + u * 1024, k < left ? voff[u & 1] : kOutOfRange, 0);
  }
  __device__ __forceinline__ void advance(int64_t steps = 1) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const uint64_t base = (static_cast<uint64_t>(rsrc[u][1]) << 32 | rsrc[u][0]) + steps * step;
      rsrc[u][0] = static_cast<uint32_t>(base);
      rsrc[u][1] = static_cast<uint32_t>(base >> 32);
    }
    left -= static_cast<int>(steps) * kStep;
  }
};

typedef short S16x4 __attribute__((ext_vector_type(4)));
using LdsShorts = __attribute__((address_space(3))) S16x4;
using LdsBytes = __attribute__((address_space(3))) char;

// Where a lane finds its part of an operand: 8 elements k = 16 kk + 8 (lane / 32) + 0..7
// of row (column) first + 32 i + lane % 32, `first` a multiple of
// 32 (of 64 for more than one i).
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
      at = lds + (first + r) * (2 * kStep) + (((lane >> 5) ^ ((r >> 1) & 7)) << 4);
    }
  }
  // `offset`: of the buffer, in bytes.
  __device__ __forceinline__ U32x4 read(int offset, int i, int kk) const {
    U32x4 w;
    if constexpr (Cols) {
      uint32_t at = this->at;
      asm volatile("" : "+v"(at));  // formed anew for each read rather than kept in a register for each place
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (i << 6)) + offset + kk * 16 * 2 * Side;
      const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)p);
      const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts*)(p + 4 * 2 * Side));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      w = U32x4{l.x, l.y, h.x, h.y};
    } else {
      auto* p = reinterpret_cast<LdsBytes*>(at ^ (kk << 5)) + offset + i * 32 * 2 * kStep;
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

}  // namespace
}  // namespace fh
