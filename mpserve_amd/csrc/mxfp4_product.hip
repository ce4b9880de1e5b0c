// Products with MXFP4 weights: y[t, n] = sum over k of x[t, k] * w[n, k], plus a bias.
//
// x is BF16, FP16 or MXFP4; w is MXFP4; sums are FP32 in the matrix cores and are rounded once, to
// the output's type. With 16-bit x the weights' values are written out as BF16, which holds each
// exactly (two significant bits and the exponent of the scale), and FP16 x as a BF16 sum
// hi + lo, also exact: eight significant bits each, and FP16 has eleven.
//
// For experts, rows of x belong to experts by ranges (offsets) and each expert has weights of
// its own; rows may be gathered from a token's row by the sorted order.
#include "mxfp4_product.h"

namespace mps {
namespace {

// Few rows: a workgroup takes 16 weight rows and kTiles * 16 rows of x, and its waves take the
// blocks of k in turn and add up their sums through LDS. A lane's 16 bytes of codes are one block
// of one weight row.
constexpr int kWaves = 4;

template <int kX, int kTiles>
__global__ __launch_bounds__(kWaves * 64) void mxfp4_few_rows_kernel(ProductArgs a) {
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
void launch(const ProductArgs &a, hipStream_t stream) {
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
  if (p->rows > INT32_MAX - 1024 || p->n > INT32_MAX - 1024)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: a size is over 2^31 - 1025");
  if (p->k > kMaxProductK) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: k is over %d", kMaxProductK);
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

// Which kernel takes a product, and what it needs.
struct Way {
  bool tiles;         // mxfp4_tile.hip; else few rows
  bool packed;        // x is packed into the workspace first
  int32_t planes;     // BF16 rows a row of x becomes
  int64_t x_rows, workspace;
};
Way way_of(const mps_mxfp4_product *p) {
  Way w = {};
  w.x_rows = p->gather ? p->rows / p->top : p->rows;
  w.planes = p->x_type == MPS_TYPE_F16 ? 2 : 1;
  w.tiles = p->rows > 64 * (p->experts > 0 ? p->experts : 1);
  w.packed = w.tiles && (p->x_type == MPS_TYPE_F16 || (p->x_type == MPS_TYPE_BF16 && !tile_rows(p->x, p->x_stride, p->k)));
  if (w.packed) w.workspace = w.x_rows * w.planes * packed_width(p->k) * 2;
  return w;
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
  *bytes = p->rows > 0 && p->n > 0 ? way_of(p).workspace : 0;
  return MPS_OK;
}

int mps_mxfp4_multiply(const mps_mxfp4_product *p, void *workspace, int64_t workspace_bytes, void *stream) {
  last_error().clear();
  const int rc = check(p);
  if (rc != MPS_OK || p->rows == 0 || p->n == 0) return rc;
  const Way way = way_of(p);
  if (way.workspace > 0 && (!workspace || workspace_bytes < way.workspace || !aligned16(workspace)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: %lld bytes of workspace are needed, 16-byte aligned",
                (long long)way.workspace);
  ProductArgs a = {};
  a.x = p->x, a.x_scales = p->x_scales, a.x_stride = p->x_stride;
  a.w = p->w, a.w_scales = p->w_scales, a.bias = p->bias, a.out = p->out;
  a.offsets = p->experts > 0 ? p->offsets : nullptr, a.order = p->order;
  a.rows = (int32_t)p->rows, a.x_rows = (int32_t)way.x_rows, a.planes = 1, a.n = (int32_t)p->n, a.k = (int32_t)p->k, a.row_blocks = (int32_t)mx_blocks(p->k);
  a.experts = (int32_t)p->experts, a.top = (int32_t)p->top, a.gather = p->gather;
  a.bias_type = p->bias_type, a.out_type = p->out_type;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (way.packed) {
    a.x_stride = way.planes * packed_width(p->k), a.x_plane = packed_width(p->k), a.planes = way.planes;
    launch_pack(p->x, p->x_type, way.x_rows, p->x_stride, a, workspace, s);
    a.x = workspace;
  }
  if (way.tiles)
    launch_tiles(a, p->x_type, s);
  else if (p->x_type == MPS_TYPE_MXFP4)
    launch<MPS_TYPE_MXFP4>(a, s);
  else if (p->x_type == MPS_TYPE_BF16)
    launch<MPS_TYPE_BF16>(a, s);
  else
    launch<MPS_TYPE_F16>(a, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
