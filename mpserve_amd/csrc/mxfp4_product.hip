// Products with MXFP4 weights: y[t, n] = sum over k of x[t, k] * w[n, k], plus a bias.
//
// x is BF16, FP16 or MXFP4; w is MXFP4; sums are FP32 in the matrix cores and are rounded once, to
// the output's type. With 16-bit x the weights' values are written out as BF16, which holds each
// exactly (two significant bits and the exponent of the scale), and FP16 x as a BF16 sum
// hi + lo, also exact: eight significant bits each, and FP16 has eleven.
//
// For experts, rows of x belong to experts by ranges (offsets) and each expert has weights of
// its own; rows may be gathered from a token's row by the sorted order.
#include "mxfp4_common.h"

namespace mps {
namespace {

struct Args {
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

__device__ inline void split_f16(u32x4 v, bf16x8 &hi, bf16x8 &lo) {
  for (int i = 0; i < 8; ++i) {
    const float f = Elem<MPS_TYPE_F16>::get((uint16_t)(v[i / 2] >> (16 * (i % 2))));
    hi[i] = (__bf16)f;
    lo[i] = (__bf16)(f - (float)hi[i]);
  }
}

// Few rows: a workgroup takes 16 weight rows and kTiles * 16 rows of x, and its waves take the
// blocks of k in turn and add up their sums through LDS. A lane's 16 bytes of codes are one block
// of one weight row.
constexpr int kWaves = 4;

template <int kX, int kTiles>
__global__ __launch_bounds__(kWaves * 64) void mxfp4_few_rows_kernel(Args a) {
  __shared__ float sums[kWaves][kTiles * 4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  Tile tile = {0, (int32_t)blockIdx.y * kTiles * 16, 0};
  tile.end = min(a.rows, tile.first + kTiles * 16);
  if (a.offsets) tile = find_tile(a.offsets, a.experts, a.rows, kTiles * 16, blockIdx.y);
  if (tile.expert < 0) return;
  const int32_t n0 = blockIdx.x * 16;
  f32x4 acc[kTiles] = {};
  if (tile.expert < max(a.experts, 1)) {
    const int64_t wrow = (int64_t)tile.expert * a.n + min(n0 + r, a.n - 1);
    const uint8_t *w = a.w + wrow * a.row_blocks * 16, *ws = a.w_scales + wrow * a.row_blocks;
    int64_t xrow[kTiles];
    bool there[kTiles];
    for (int t = 0; t < kTiles; ++t) {
      const int32_t row = tile.first + t * 16 + r;
      there[t] = row < tile.end;
      xrow[t] = there[t] ? (a.gather ? min((uint32_t)a.order[row] / (uint32_t)a.top, (uint32_t)a.x_rows - 1) : row) : 0;
    }
    const bool whole = kX != MPS_TYPE_MXFP4 && aligned16(a.x) && a.x_stride % 8 == 0;
    for (int32_t b0 = wave * 4; b0 < a.row_blocks; b0 += kWaves * 4) {
      const int32_t b = b0 + g;
      const bool in = b < a.row_blocks;
      i32x4 c = {0, 0, 0, 0};
      uint32_t s = 127;
      if (in) {
        c = *reinterpret_cast<const i32x4 *>(w + (int64_t)b * 16);
        s = ws[b];
      }
      if constexpr (kX == MPS_TYPE_MXFP4) {
        const i32x8 wa = {c[0], c[1], c[2], c[3], 0, 0, 0, 0};
        for (int t = 0; t < kTiles; ++t) {
          i32x4 xc = {0, 0, 0, 0};
          uint32_t xs = 127;
          if (in && there[t]) {
            const int64_t at = xrow[t] * a.row_blocks + b;
            xc = reinterpret_cast<const i32x4 *>(a.x)[at];
            xs = a.x_scales[at];
          }
          const i32x8 xb = {xc[0], xc[1], xc[2], xc[3], 0, 0, 0, 0};
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc[t], 4, 4, 0, s, 0, xs);
        }
      } else {
        const float scale = mx_scale(s);
        for (int j = 0; j < 4; ++j) {
          u32x4 wv;
          wv[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], scale, 0));
          wv[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], scale, 1));
          wv[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], scale, 2));
          wv[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], scale, 3));
          const bf16x8 wa = __builtin_bit_cast(bf16x8, wv);
          for (int t = 0; t < kTiles; ++t) {
            u32x4 v = {0, 0, 0, 0};
            if (in && there[t])
              v = load_row8(static_cast<const uint16_t *>(a.x) + xrow[t] * a.x_stride, (int64_t)b * kMxBlock + 8 * j, a.k, whole);
            if constexpr (kX == MPS_TYPE_BF16) {
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa, __builtin_bit_cast(bf16x8, v), acc[t], 0, 0, 0);
            } else {
              bf16x8 hi, lo;
              split_f16(v, hi, lo);
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa, hi, acc[t], 0, 0, 0);
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa, lo, acc[t], 0, 0, 0);
            }
          }
        }
      }
    }
  }
  for (int t = 0; t < kTiles; ++t)
    for (int i = 0; i < 4; ++i) sums[wave][t * 4 + i][lane] = acc[t][i];
  __syncthreads();
  // A lane has output row first + 16 t + r, columns n0 + 4 g + i. The waves share the tiles.
  for (int t = wave; t < kTiles; t += kWaves) {
    const int32_t row = tile.first + t * 16 + r;
    if (row >= tile.end) continue;
    for (int i = 0; i < 4; ++i) {
      const int32_t n = n0 + 4 * g + i;
      if (n >= a.n) continue;
      float y = 0;
      for (int w = 0; w < kWaves; ++w) y += sums[w][t * 4 + i][lane];
      if (a.bias && tile.expert < max(a.experts, 1))
        y += load_as_float(a.bias, a.bias_type, (int64_t)tile.expert * a.n + n);
      store_as(a.out, a.out_type, (int64_t)row * a.n + n, y);
    }
  }
}

template <int kX>
void launch(const Args &a, hipStream_t stream) {
  constexpr int kTiles = 4;
  const int64_t tiles = (a.rows + kTiles * 16 - 1) / (kTiles * 16) + (a.offsets ? a.experts : 0);
  const dim3 grid((unsigned)((a.n + 15) / 16), (unsigned)tiles);
  hipLaunchKernelGGL((mxfp4_few_rows_kernel<kX, kTiles>), grid, dim3(kWaves * 64), 0, stream, a);
}

int check(const mps_mxfp4_product *p) {
  if (!p) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product is NULL");
  if (p->x_type != MPS_TYPE_BF16 && p->x_type != MPS_TYPE_F16 && p->x_type != MPS_TYPE_MXFP4)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: x must be BF16, FP16 or MXFP4");
  if (!is_float_type(p->out_type) || (p->bias && !is_float_type(p->bias_type)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: unknown output or bias type");
  if (p->rows < 0 || p->n < 0 || p->k < 0 || p->experts < 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: negative size");
  if (p->rows > INT32_MAX - 1024 || p->n > INT32_MAX - 1024 || p->k > INT32_MAX - 1024)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: a size is over 2^31 - 1025");
  if (p->experts > MPS_MAX_EXPERTS)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: %lld experts are over %d", (long long)p->experts, MPS_MAX_EXPERTS);
  if (p->rows == 0 || p->n == 0) return MPS_OK;
  if (!p->out) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: null pointer");
  if (p->k > 0 && (!p->x || !p->w || !p->w_scales || (p->x_type == MPS_TYPE_MXFP4 && !p->x_scales)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: null pointer");
  if (!aligned16(p->w) || (p->x_type == MPS_TYPE_MXFP4 && !aligned16(p->x)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: codes must be 16-byte aligned");
  if (p->x_type != MPS_TYPE_MXFP4 && p->x_stride < 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: negative row stride");
  if (p->experts > 0 && !p->offsets) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: experts need offsets");
  if (p->gather && (p->experts == 0 || !p->order || p->top <= 0))
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: a gather needs experts, the sorted order and top > 0");
  return MPS_OK;
}

}  // namespace
}  // namespace mps

using namespace mps;

extern "C" {

int mps_mxfp4_product_workspace(const mps_mxfp4_product *p, int64_t *bytes) {
  last_error().clear();
  const int rc = check(p);
  if (rc != MPS_OK) return rc;
  if (!bytes) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: null pointer");
  *bytes = 0;
  return MPS_OK;
}

int mps_mxfp4_multiply(const mps_mxfp4_product *p, void *workspace, int64_t workspace_bytes, void *stream) {
  last_error().clear();
  const int rc = check(p);
  if (rc != MPS_OK || p->rows == 0 || p->n == 0) return rc;
  Args a = {};
  a.x = p->x, a.x_scales = p->x_scales, a.x_stride = p->x_stride;
  a.w = p->w, a.w_scales = p->w_scales, a.bias = p->bias, a.out = p->out;
  a.offsets = p->experts > 0 ? p->offsets : nullptr, a.order = p->order;
  a.rows = (int32_t)p->rows, a.x_rows = (int32_t)(p->gather ? p->rows / p->top : p->rows), a.n = (int32_t)p->n, a.k = (int32_t)p->k, a.row_blocks = (int32_t)mx_blocks(p->k);
  a.experts = (int32_t)p->experts, a.top = (int32_t)p->top, a.gather = p->gather;
  a.bias_type = p->bias_type, a.out_type = p->out_type;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p->x_type == MPS_TYPE_MXFP4)
    launch<MPS_TYPE_MXFP4>(a, s);
  else if (p->x_type == MPS_TYPE_BF16)
    launch<MPS_TYPE_BF16>(a, s);
  else
    launch<MPS_TYPE_F16>(a, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
