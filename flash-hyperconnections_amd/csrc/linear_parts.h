// FP32 values as sums of three bf16 parts.
#pragma once

#include "linear.h"

namespace fh {
namespace {

// Four values' parts, two values to a dword.  An infinity or NaN goes into the last
// part, which meets only the other operand's first, beside a one in the first part:
// inf x (second or third part 0) would be NaN, where inf x b is an infinity.
__device__ __forceinline__ void split_exactly(const float (&v)[4], uint2 (&part)[3]) {
  uint32_t w[4][3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bits = __float_as_uint(v[i]);
    const float r = v[i] - __uint_as_float(bits & 0xFFFF0000u);
    w[i][0] = bits & 0xFFFF0000u;
    w[i][1] = __float_as_uint(r) & 0xFFFF0000u;
    w[i][2] = __float_as_uint(r - __uint_as_float(w[i][1]));
    if (!finite_f32(v[i])) {
      w[i][0] = 0x3F800000u | (bits & 0x80000000u);
      w[i][1] = 0;
      w[i][2] = v[i] != v[i] ? 0x7FC00000u : bits;
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
    part[k] = make_uint2((w[0][k] >> 16) | (w[1][k] & 0xFFFF0000u), (w[2][k] >> 16) | (w[3][k] & 0xFFFF0000u));
}

// The same where all values are finite; `odd` becomes NaN where one is not.
__device__ __forceinline__ void split(const float (&v)[4], uint2 (&part)[3], float& odd) {
  uint32_t m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = v[i] - __uint_as_float(__float_as_uint(v[i]) & 0xFFFF0000u);
    m[i] = __float_as_uint(r);
    const float s = r - __uint_as_float(m[i] & 0xFFFF0000u);
    l[i] = __float_as_uint(s);
    odd += s;
  }
  // The top halves of two dwords in one.
  const auto tops = [](uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); };
  part[0] = make_uint2(tops(__float_as_uint(v[0]), __float_as_uint(v[1])),
                       tops(__float_as_uint(v[2]), __float_as_uint(v[3])));
  part[1] = make_uint2(tops(m[0], m[1]), tops(m[2], m[3]));
  part[2] = make_uint2(tops(l[0], l[1]), tops(l[2], l[3]));
}

}  // namespace
}  // namespace fh
