// What the kernels of int4 products share: their arguments, and the format's arithmetic.
//
// A weight is s (q - z): q a whole number of 4 bits, s and z those of its group of 2^shift * 32 columns. Codes
// lie in blocks of 32 elements of 16 bytes; byte b of each 4 bytes holds element b of eight in its low half and
// element b + 4 in its high half, so that masked halves are bytes of four neighbours.
#pragma once

#include "mxfp4_product.h"

namespace mps {

struct Int4Args : ProductArgs {
  const void *scales;
  const uint8_t *zeros;  // nullptr: 8
  int32_t scale_type, groups, shift;  // groups a row; blocks a group, as a power of two
};

// Scale and zero of a weight's row `row` (of all experts') and group.
__device__ inline float int4_scale(const Int4Args &a, int64_t row, int32_t group) {
  return load_as_float(a.scales, a.scale_type, row * a.groups + group);
}
__device__ inline float int4_zero(const Int4Args &a, int64_t row, int32_t group) {
  return a.zeros ? (float)(a.zeros[row * a.groups + group] & 31) : 8.0f;
}

// Eight codes less their zero, exactly, in 16 bits.
template <int XT>
__device__ inline u32x4 int4_values(uint32_t codes, float zero) {
  const uint32_t lo = codes & 0x0f0f0f0fu, hi = codes >> 4 & 0x0f0f0f0fu;
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? lo : hi;
    const float a = (float)(w >> (16 * (i % 2)) & 255) - zero, b = (float)(w >> (16 * (i % 2) + 8) & 255) - zero;
    v[i] = pack2(a, b, XT);
  }
  return v;
}

template <int XT>
__device__ inline f32x4 mfma16(u32x4 x, u32x4 w, f32x4 c) {
  if constexpr (XT == MPS_TYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
}

}  // namespace mps
