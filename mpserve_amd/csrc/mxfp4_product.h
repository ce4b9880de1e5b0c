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
  int32_t planes;   // BF16 rows that are added up to one row of x
  int64_t x_plane;  // elements from one to the next
};

// The expert and the rows of tile `tile`, where every expert's rows are cut into tiles of `size`
// rows and the rows past the last expert's into more tiles, as those of expert `experts`.
// All lanes get the same answer; {-1, 0, 0} past the last tile.
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
      const int32_t in = tile - before - (__shfl(upto, at) - __shfl(tiles, at));
      const int32_t f = __shfl(first, at) + in * size;
      return {e0 + at, f, min(f + size, __shfl(end, at))};
    }
    before += __shfl(upto, 63);
  }
  return {-1, 0, 0};
}

// Eight elements of a 16-bit row from `col` on, as bits; zeros past column k.
__device__ inline u32x4 load_row8(const uint16_t *row, int64_t col, int64_t k, bool whole) {
  if (whole && col + 8 <= k) return *reinterpret_cast<const u32x4 *>(row + col);
  u32x4 v = {0, 0, 0, 0};
  for (int i = 0; i < 8; ++i)
    if (col + i < k) v[i / 2] |= (uint32_t)row[col + i] << (16 * (i % 2));
  return v;
}

// FP16 as a sum of two BF16: hi takes the first eight significant bits, lo the other three exactly.
__device__ inline void split_f16(u32x4 v, bf16x8 &hi, bf16x8 &lo) {
  for (int i = 0; i < 8; ++i) {
    const float f = Elem<MPS_TYPE_F16>::get((uint16_t)(v[i / 2] >> (16 * (i % 2))));
    hi[i] = (__bf16)f;
    lo[i] = (__bf16)(f - (float)hi[i]);
  }
}

constexpr int32_t kMaxProductK = 1 << 24;  // offsets inside a tile fit 32 bits

// Rows in tiles of `size`: an upper bound that does not need the offsets.
inline int64_t product_tiles(const ProductArgs &a, int64_t size) {
  return (a.rows + size - 1) / size + (a.offsets ? a.experts : 0);
}

// Many rows (mxfp4_tile.hip). x is MXFP4, or BF16 in rows of whole 128-byte pieces at 16-byte
// addresses; `planes` of them, x_plane elements apart, add up to a row of x.
void launch_tiles(const ProductArgs &a, int32_t x_type, hipStream_t stream);
inline bool tile_rows(const void *x, int64_t stride, int64_t k) { return aligned16(x) && stride % 8 == 0 && k % 64 == 0; }
// Writes x[rows, a.k] as such rows, a.x_plane elements wide, with zeros past column k.
void launch_pack(const void *x, int32_t x_type, int64_t rows, int64_t stride, const ProductArgs &a, void *out,
                 hipStream_t stream);
inline int64_t packed_width(int64_t k) { return (k + 63) / 64 * 64; }

}  // namespace mps
