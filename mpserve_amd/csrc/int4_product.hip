// Products with int4 weights: y[t, n] = sum over k of x[t, k] * s (q - z)[n, k], plus a bias.
//
// q - z is exact in 16 bits, so that matrix instructions multiply it by x exactly; a group's sum gets its scale in
// FP32, and the sum of the groups is rounded once, to the output's type.
#include "int4_product.h"

namespace mps {
namespace {

// A wave a 16 x 16 tile, from memory: lane 16 g + r has piece g of a block of k, of row r of x and of the weight.
template <int XT>
__global__ __launch_bounds__(64) void int4_simple_kernel(Int4Args a) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  Tile tile = {0, (int32_t)blockIdx.y * 16, 0};
  tile.end = min(a.rows, tile.first + 16);
  if (a.offsets) tile = find_tile(a.offsets, a.experts, a.rows, 16, blockIdx.y);
  if (tile.expert < 0) return;
  const bool none = tile.expert >= max(a.experts, 1);
  const int32_t n0 = blockIdx.x * 16;
  int32_t from = min(tile.first + r, tile.end - 1);
  if (a.gather) from = min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1);
  const uint16_t *const x = static_cast<const uint16_t *>(a.x) + from * a.x_stride;
  const int64_t w_row = (int64_t)(none ? 0 : tile.expert) * a.n + min(n0 + r, a.n - 1);
  const uint8_t *const w = a.w + w_row * a.row_blocks * 16;
  f32x4 sum = {0, 0, 0, 0};
  for (int32_t b0 = 0; b0 < (none ? 0 : a.row_blocks); b0 += 1 << a.shift) {
    const int32_t group = b0 >> a.shift;
    const float scale = int4_scale(a, w_row, group), zero = int4_zero(a, w_row, group);
    f32x4 part = {0, 0, 0, 0};
    for (int32_t b = b0; b < min(a.row_blocks, b0 + (1 << a.shift)); ++b) {
      const u32x4 xv = load_row8(x, (int64_t)b * 32 + g * 8, a.k);
      const uint32_t codes = *reinterpret_cast<const uint32_t *>(w + (int64_t)b * 16 + g * 4);
      part = mfma16<XT>(xv, int4_values<XT>(codes, zero), part);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(scale, part[i], sum[i]);
  }
  const int32_t col = n0 + r;
  if (col >= a.n) return;
  const float bias = a.bias && !none ? load_as_float(a.bias, a.bias_type, (int64_t)tile.expert * a.n + col) : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int32_t row = tile.first + 4 * g + i;
    if (row < tile.end) store_as(a.out, a.out_type, (int64_t)row * a.n + col, sum[i] + bias);
  }
}

int check(const mps_int4_product *p) {
  if (!p) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product is NULL");
  if (p->x_type != MPS_TYPE_BF16 && p->x_type != MPS_TYPE_F16)
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: x must be BF16 or FP16");
  if (p->scale_type != MPS_TYPE_BF16 && p->scale_type != MPS_TYPE_F16)
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: scales must be BF16 or FP16");
  if (!is_float_type(p->out_type) || (p->bias && !is_float_type(p->bias_type)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: unknown output or bias type");
  if (p->rows < 0 || p->n < 0 || p->k < 0 || p->experts < 0 || p->x_stride < 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: negative size");
  if (p->rows > INT32_MAX - 1024 || p->n > INT32_MAX - 1024)
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: a size is over 2^31 - 1025");
  if (p->k > kMaxProductK) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: k is over %d", kMaxProductK);
  if (p->group < 32 || p->group > (1 << 30) || (p->group & (p->group - 1)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: the group must be a power of two from 32 to 2^30");
  if (p->experts > MPS_MAX_EXPERTS)
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: %lld experts are over %d", (long long)p->experts, MPS_MAX_EXPERTS);
  if (p->rows == 0 || p->n == 0) return MPS_OK;
  if (!p->out || (p->k > 0 && (!p->x || !p->w || !p->scales))) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: null pointer");
  if (!aligned16(p->w)) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: codes must be 16-byte aligned");
  if (p->experts > 0 && !p->offsets) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: experts need offsets");
  if (p->gather && (p->experts == 0 || !p->order || p->top <= 0))
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: a gather needs experts, the sorted order and top > 0");
  if (p->gather && p->rows % p->top != 0)  // x has rows / top rows: there has to be one
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: a gather's %lld rows are no multiple of top (%lld)", (long long)p->rows, (long long)p->top);
  return MPS_OK;
}

}  // namespace
}  // namespace mps

using namespace mps;

extern "C" {

int mps_int4_product_workspace(const mps_int4_product *p, int64_t *bytes) {
  last_error().clear();
  const int rc = check(p);
  if (rc != MPS_OK) return rc;
  if (!bytes) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: null pointer");
  *bytes = 0;
  return MPS_OK;
}

int mps_int4_multiply(const mps_int4_product *p, void *workspace, int64_t workspace_bytes, void *stream) {
  last_error().clear();
  const int rc = check(p);
  if (rc != MPS_OK || p->rows == 0 || p->n == 0) return rc;
  Int4Args a = {};
  a.x = p->x, a.x_stride = p->x_stride, a.w = p->w, a.bias = p->bias, a.out = p->out;
  a.offsets = p->experts > 0 ? p->offsets : nullptr, a.order = p->order;
  a.rows = (int32_t)p->rows, a.x_rows = (int32_t)(p->gather ? p->rows / p->top : p->rows);
  a.n = (int32_t)p->n, a.k = (int32_t)p->k, a.row_blocks = (int32_t)mx_blocks(p->k);
  a.experts = (int32_t)p->experts, a.top = (int32_t)p->top, a.gather = p->gather;
  a.bias_type = p->bias_type, a.out_type = p->out_type;
  a.scales = p->scales, a.zeros = p->zeros, a.scale_type = p->scale_type;
  a.groups = (int32_t)((p->k + p->group - 1) / p->group);
  while ((int64_t)32 << a.shift < p->group) ++a.shift;
  const int64_t tiles = product_tiles(a, 16);
  const dim3 grid((unsigned)((a.n + 15) / 16), (unsigned)tiles);
  if (tiles > 65535) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: too many rows");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p->x_type == MPS_TYPE_BF16)
    hipLaunchKernelGGL(int4_simple_kernel<MPS_TYPE_BF16>, grid, dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL(int4_simple_kernel<MPS_TYPE_F16>, grid, dim3(64), 0, s, a);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
