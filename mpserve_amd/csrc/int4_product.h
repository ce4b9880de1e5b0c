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
  const void *sums;                   // many rows: x's sums, `sums_row` bytes a row of x
  int64_t sums_row;
};

// Scale and zero of a weight's row `row` (of all experts') and group.
__device__ inline float int4_scale(const Int4Args &a, int64_t row, int32_t group) {
  return load_as_float(a.scales, a.scale_type, row * a.groups + group);
}
__device__ inline float int4_zero(const Int4Args &a, int64_t row, int32_t group) {
  return a.zeros ? (float)(a.zeros[row * a.groups + group] & 31) : 8.0f;
}

// Eight codes as they are, 0 to 15, in 16 bits, exactly: a byte below 16 is an FP8 (e4m3) number too, 2^-9 times its
// value, which the conversions multiply by 2^9. Three masks and shifts and four conversions for eight values.
template <int XT>
__device__ inline u32x4 int4_codes(uint32_t codes) {
  const uint32_t lo = codes & 0x0f0f0f0fu, hi = codes >> 4 & 0x0f0f0f0fu;
  u32x4 v;
  if constexpr (XT == MPS_TYPE_BF16) {
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true));
  } else {
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true));
  }
  return v;
}

// Eight codes less their zero, exactly, in 16 bits: three times the instructions.
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

// 16 bytes a lane from memory to LDS, lane after lane from `to` (alike for all lanes) on. By an instruction of its own, since behind the
// compiler's the next read of LDS waits for all such loads; the kernels wait for theirs by count.
__device__ inline uint32_t lds_address(const uint8_t *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p; }
__device__ inline void copy16_apart(const uint8_t *from, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(__builtin_amdgcn_readfirstlane(to)), "v"(from) : "memory");
}

// An address that is alike for all lanes, in scalar registers.
__device__ inline const uint8_t *scalar(const uint8_t *p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const uint8_t *>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 |
                                           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v));
}

// The same from `base`, alike for all lanes, and a lane's bytes behind it, which take one register. The base may come from a vector
// instruction, behind which a load has to keep five instructions' distance: the compiler does not see that this is one.
__device__ inline void copy16_apart(const uint8_t *base, uint32_t from, uint32_t to) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(__builtin_amdgcn_readfirstlane(to)), "v"(from), "s"(scalar(base)) : "memory");
}

// Eight ones: x times these is the sum of x.
template <int XT>
__device__ inline u32x4 int4_ones() {
  constexpr uint32_t two = XT == MPS_TYPE_BF16 ? 0x3f803f80u : 0x3c003c00u;
  return u32x4{two, two, two, two};
}

__device__ inline float scale_value(uint32_t bits, int32_t type) {
  return type == MPS_TYPE_BF16 ? Elem<MPS_TYPE_BF16>::get((uint16_t)bits) : Elem<MPS_TYPE_F16>::get((uint16_t)bits);
}

template <int XT>
__device__ inline f32x4 mfma16(u32x4 x, u32x4 w, f32x4 c) {
  if constexpr (XT == MPS_TYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
}

// A period is 16 blocks. Groups of at least 128 have at most four of a row's scales in one (kFew), finer ones up to
// sixteen; a row's scales and zeros are read a period ahead in windows of that many, at any alignment, which
// near a row's end begin earlier: `window_start`, alike for all rows.
template <bool kFew>
struct Window {
  static constexpr int kEntries = kFew ? 4 : 16, kBytes = kFew ? 16 : 48;  // of LDS, a row: scales, then zeros
  uint32_t scales[kEntries / 2], zeros[kEntries / 4];
};
template <bool kFew>
__device__ inline int32_t window_start(const Int4Args &a, int32_t period) {
  return max(0, min((16 * period) >> a.shift, a.groups - Window<kFew>::kEntries));
}
// A row that has fewer in all has them in its window from the start (load_all). The loads have no branches among them, behind which the
// compiler would wait for all that are under way. Without zeros, others' bytes stand in for them.
__device__ inline const uint8_t *zeros_or_any(const Int4Args &a) { return a.zeros ? a.zeros : static_cast<const uint8_t *>(a.scales); }
template <bool kFew>
__device__ inline void load_window(const Int4Args &a, int64_t row, int32_t start, Window<kFew> &w) {
  __builtin_memcpy(w.scales, static_cast<const uint16_t *>(a.scales) + row * a.groups + start, sizeof(w.scales));
  __builtin_memcpy(w.zeros, zeros_or_any(a) + row * a.groups + start, sizeof(w.zeros));
}
template <bool kFew>
__device__ inline void load_all(const Int4Args &a, int64_t row, Window<kFew> &w) {
  constexpr int kEntries = Window<kFew>::kEntries;
  const uint16_t *const s = static_cast<const uint16_t *>(a.scales) + row * a.groups;
  const uint8_t *const z = zeros_or_any(a) + row * a.groups;
  uint32_t e[kEntries], f[kEntries];
#pragma unroll
  for (int i = 0; i < kEntries; ++i) e[i] = s[min(i, a.groups - 1)], f[i] = z[min(i, a.groups - 1)];
#pragma unroll
  for (int i = 0; i < kEntries / 2; ++i) w.scales[i] = e[2 * i] | e[2 * i + 1] << 16;
#pragma unroll
  for (int i = 0; i < kEntries / 4; ++i) w.zeros[i] = f[4 * i] | f[4 * i + 1] << 8 | f[4 * i + 2] << 16 | f[4 * i + 3] << 24;
}
template <bool kFew>
__device__ inline void put_window(const Int4Args &a, const Window<kFew> &w, uint8_t *lds) {
  constexpr int kEntries = Window<kFew>::kEntries;
  uint32_t *const to = reinterpret_cast<uint32_t *>(lds);
#pragma unroll
  for (int i = 0; i < kEntries / 2; ++i) to[i] = w.scales[i];
#pragma unroll
  for (int i = 0; i < kEntries / 4; ++i) to[kEntries / 2 + i] = a.zeros ? w.zeros[i] & 0x1f1f1f1fu : 0x08080808u;
}
template <bool kFew>
__device__ inline void read_window(const Int4Args &a, const uint8_t *row, int32_t entry, float &scale, float &zero) {
  scale = scale_value(*reinterpret_cast<const uint16_t *>(row + 2 * entry), a.scale_type);
  zero = (float)row[2 * Window<kFew>::kEntries + entry];
}

// Few rows (int4_rows.hip): x is 16-bit rows of whole 16-byte pieces.
Prediction predict_int4_rows(const Int4Args &a, int32_t cus);
void launch_int4_rows(const Int4Args &a, int32_t x_type, int choice, hipStream_t stream);

// Many rows (int4_tile.hip): x is 16-bit rows of whole blocks at 16-byte addresses, with its sums over spans of a group or, of a larger
// one, 128 columns. A sum is three BF16 numbers, the first eight bits (and sign), the next eight and the rest. A row has first, second, third and
// first again of each span; then the second ones by themselves; zeros past the last span, to a multiple of 16.
Prediction predict_int4_tiles(const Int4Args &a, int32_t cus);
void launch_int4_tiles(const Int4Args &a, int32_t x_type, int choice, hipStream_t stream);
inline int32_t sums_shift(const Int4Args &a) { return a.shift < 2 ? a.shift : 2; }
inline int32_t sums_spans(const Int4Args &a) { return (int32_t)(((int64_t)a.row_blocks + (1 << sums_shift(a)) - 1) >> sums_shift(a)); }
inline int64_t sums_row_bytes(const Int4Args &a) { return (int64_t)(sums_spans(a) + 15) / 16 * 160; }

}  // namespace mps
