// What the product kernels share: their arguments, and which expert a tile of rows belongs to.
#pragma once

#include "mxfp4_common.h"

namespace mps {

struct ProductArgs {
  const void *x;
  const uint8_t *x_scales;
  int64_t x_stride;  // elements (16-bit x) from row to row
  const uint8_t *w, *w_scales;
  const void *bias;
  void *out;
  const int32_t *offsets, *order;  // experts only
  int32_t rows, x_rows, n, row_blocks, k;
  int32_t experts, top, gather;
  int32_t bias_type, out_type;
};

// The expert and the rows of tile `tile`, where every expert's rows are cut into tiles of `size`
// rows and the rows past the last expert's into more tiles, as those of expert `experts`.
// All lanes get the same answer, and the compiler knows it (lanes are read, not shuffled), so that it stays in
// scalar registers; {-1, 0, 0} past the last tile.
struct Tile {
  int32_t expert, first, end;
};
__device__ inline Tile find_tile(const int32_t *offsets, int32_t experts, int32_t rows, int32_t size, int32_t tile) {
  const int lane = threadIdx.x & 63;
  int32_t before = 0;
  for (int32_t e0 = 0; e0 <= experts; e0 += 64) {
    const int32_t e = e0 + lane;
    int32_t first = 0, end = 0;
    if (e <= experts) {
      first = min(max(offsets[e], 0), rows);  // bad offsets give bad sums, never bad addresses
      end = e < experts ? max(first, min(offsets[e + 1], rows)) : rows;
    }
    const int32_t tiles = (end - first + size - 1) / size;
    int32_t upto = tiles;
    for (int d = 1; d < 64; d *= 2) {
      const int32_t v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const uint64_t hit = __ballot(before + upto > tile);
    if (hit) {
      const int at = __ffsll((unsigned long long)hit) - 1;
      const int32_t here = __builtin_amdgcn_readlane(tiles, at), in = tile - before - (__builtin_amdgcn_readlane(upto, at) - here);
      if ((uint32_t)in >= (uint32_t)here) break;  // bad offsets whose tiles add up to 2^31 and more
      const int32_t f = __builtin_amdgcn_readlane(first, at) + in * size;
      return {e0 + at, f, min(f + size, __builtin_amdgcn_readlane(end, at))};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0};
}

// How many of these tiles there are.
__device__ inline int32_t count_tiles(const int32_t *offsets, int32_t experts, int32_t rows, int32_t size) {
  const int lane = threadIdx.x & 63;
  int32_t tiles = 0;
  for (int32_t e = lane; e <= experts; e += 64) {
    const int32_t first = min(max(offsets[e], 0), rows), end = e < experts ? max(first, min(offsets[e + 1], rows)) : rows;
    tiles += (end - first + size - 1) / size;
  }
  for (int d = 32; d > 0; d /= 2) tiles += __shfl_xor(tiles, d);
  return __builtin_amdgcn_readfirstlane(tiles);
}

// Eight elements of a 16-bit row from `col` on, at any alignment, as bits; zeros past column k.
__device__ inline u32x4 load_row8(const uint16_t *row, int64_t col, int64_t k) {
  if (col + 8 <= k) return *reinterpret_cast<const u32x4_any *>(row + col);
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col + i < k) v[i / 2] |= (uint32_t)row[col + i] << (16 * (i % 2));
  return v;
}

// Eight codes' values in BF16, scaled: exact but for scales 253 and 254, where 2^128 and more are infinite.
__device__ inline bf16x8 widen(uint32_t codes, float scale) {
  u32x4 v;
  v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return __builtin_bit_cast(bf16x8, v);
}

// A quarter of eight codes' values in BF16, exact for every scale (1.5 * 2^127 down to 2^-130, of which BF16 still has
// the last bit). Where `widen` could overflow, x meets it four times: no product is infinite that need not be,
// and a zero of x stays one. That takes four times the matrix instructions and more, so the kernels go on as
// if nothing could overflow, note whether a scale was 2^65 or more, which no weight in use has, and if so
// make the sums again this way.
__device__ inline bf16x8 widen_quarter(uint32_t codes, uint32_t s) {
  const float scale = __uint_as_float(s == 255 ? 0x7fc00000u : s > 2 ? (s - 2) << 23 : 0x00100000u << s);
  const f32x2 f[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3)};
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i].x * scale) >> 16 | (__float_as_uint(f[i].y * scale) & 0xffff0000u);
  return __builtin_bit_cast(bf16x8, v);
}

// Has bits of kLargeScale if one of 16 scale bytes is 192 or more.
constexpr uint32_t kLargeScale = 0x80808080u;
__device__ inline uint32_t large_scales(u32x4 s) {
  return (s[0] & s[0] << 1) | (s[1] & s[1] << 1) | (s[2] & s[2] << 1) | (s[3] & s[3] << 1);
}

// The codes' values in FP16, without a scale.
__device__ inline f16x8 widen_f16(uint32_t codes) {
  u32x4 v;
  v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 0));
  v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 1));
  v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 2));
  v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 3));
  return __builtin_bit_cast(f16x8, v);
}

__device__ inline void copy16(const uint8_t *from, uint8_t *lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// 16 scale bytes of a row from block `b` on, and zeros (2^-127, which takes any product to zero or
// leaves a zero x as it is) past the row's last block. Rows start at any address. The load comes
// apart from what is done to it, so that nothing waits for it where it is issued: near a row's
// end it takes the last 16 bytes, which move_scales then moves down.
__device__ inline u32x4 load_scales(const uint8_t *row, int32_t b, int32_t blocks) {
  u32x4 v = {0, 0, 0, 0};
  if (blocks >= 16) {
    __builtin_memcpy(&v, row + min(b, blocks - 16), 16);
  } else {
#pragma unroll 1
    for (int i = 0; i < blocks; ++i) v[i / 4] |= (uint32_t)row[i] << (8 * (i % 4));
  }
  return v;
}
__device__ inline u32x4 move_scales(u32x4 v, int32_t b, int32_t blocks) {
  if (blocks < 16 || b + 16 <= blocks) return v;
  const int32_t past = b + 16 - blocks;
  return past < 16 ? __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, v) >> (8 * past)) : u32x4{0, 0, 0, 0};
}

// Two values as 16-bit ones.
__device__ inline uint32_t pack2(float lo, float hi, int32_t type) {
  if (type == MPS_TYPE_BF16) return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
}

// Four neighbouring columns of a row of the output, at any alignment; those past the last are left out.
__device__ inline void store4(const ProductArgs &a, int64_t row, int32_t col, f32x4 v) {
  const int64_t at = row * a.n + col;
  if (col + 4 > a.n) {
    for (int j = 0; j < 4; ++j)
      if (col + j < a.n) store_as(a.out, a.out_type, at + j, v[j]);
  } else if (a.out_type == MPS_TYPE_F32) {
    *reinterpret_cast<u32x4_any *>(static_cast<float *>(a.out) + at) = __builtin_bit_cast(u32x4, v);
  } else {
    typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
    *reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(a.out) + at) = u32x2_any{pack2(v[0], v[1], a.out_type), pack2(v[2], v[3], a.out_type)};
  }
}

// Eight of them.
__device__ inline void store8(const ProductArgs &a, int64_t row, int32_t col, f32x4 v, f32x4 w) {
  if (col + 8 > a.n || a.out_type == MPS_TYPE_F32) {
    store4(a, row, col, v);
    store4(a, row, col + 4, w);
  } else {
    *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(a.out) + row * a.n + col) =
        u32x4{pack2(v[0], v[1], a.out_type), pack2(v[2], v[3], a.out_type), pack2(w[0], w[1], a.out_type), pack2(w[2], w[3], a.out_type)};
  }
}

// The biases of four neighbouring columns; zeros past the last column.
__device__ inline f32x4 load_bias4(const ProductArgs &a, int32_t expert, int32_t col) {
  f32x4 v = {0, 0, 0, 0};
  for (int j = 0; j < 4; ++j)
    if (col + j < a.n) v[j] = load_as_float(a.bias, a.bias_type, (int64_t)expert * a.n + col + j);
  return v;
}

constexpr int32_t kMaxProductK = 1 << 24;  // offsets inside a tile fit 32 bits

// Tiles of `size` rows: m ranges that are not empty have at most (rows + m (size - 1)) / size, which
// does not need the offsets.
inline int64_t product_tiles(const ProductArgs &a, int64_t size) {
  const int64_t ranges = a.offsets ? (a.experts < a.rows ? a.experts + 1 : a.rows) : 1;
  return (a.rows + ranges * (size - 1)) / size;
}

// As many as there will be: experts' loads are unknown here, so pairs are taken to be spread evenly
// at random; a range ends in the middle of a tile.
inline double expected_tiles(const ProductArgs &a, int64_t size) {
  if (!a.offsets) return (double)((a.rows + size - 1) / size);
  const double met = a.experts * (1.0 - __builtin_exp(-(double)a.rows / a.experts));
  const double tiles = (double)a.rows / size + 0.5 * met;
  return tiles > met ? tiles : met;
}

// The share of these tiles that have rows in their first half only: an expert's last tile is one or not, but
// where experts have less than half a tile each, all are.
inline double expected_halves(const ProductArgs &a, int64_t size) {
  if (!a.offsets || a.rows == 0) return 0;
  const double met = a.experts * (1.0 - __builtin_exp(-(double)a.rows / a.experts)), fill = a.rows / met / (double)size;
  const double share = fill <= 0.4 ? 1.0 : fill >= 0.6 ? 0.5 : 1.0 - 2.5 * (fill - 0.4);
  return share * met / expected_tiles(a, size);
}

constexpr double kMostWorkItems = 4294967295.0;  // of a grid, in one direction

// The current device's CUs; asked once a device (mxfp4_product.hip).
int32_t compute_units();

// One of a kernel's shapes (-1: none fits a grid), and the microseconds that it is predicted to take (the launch and the first
// loads, alike for all, are left out).
struct Prediction {
  int choice;
  double us;
};

// Few rows (mxfp4_rows.hip). x is MXFP4, or 16-bit rows of whole 16-byte pieces.
Prediction predict_rows(const ProductArgs &a, int32_t x_type, int32_t cus);
void launch_rows(const ProductArgs &a, int32_t x_type, int choice, hipStream_t stream);
inline bool piece_rows(const void *x, int64_t stride, int64_t k) { return aligned16(x) && stride % 8 == 0 && k % 8 == 0; }

// Many rows (mxfp4_tile.hip). x is MXFP4, or 16-bit rows of whole blocks at 16-byte addresses.
Prediction predict_tiles(const ProductArgs &a, int32_t x_type, int32_t cus);
void launch_tiles(const ProductArgs &a, int32_t x_type, int choice, hipStream_t stream);
inline bool block_rows(const void *x, int64_t stride, int64_t k) { return aligned16(x) && stride % 8 == 0 && k % 32 == 0; }
inline int64_t packed_width(int64_t k) { return (k + 31) / 32 * 32; }

}  // namespace mps
