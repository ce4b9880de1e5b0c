// Products with MXFP4 weights: y[t, n] = sum over k of x[t, k] * w[n, k], plus a bias.
//
// x is BF16, FP16 or MXFP4; w is MXFP4; sums are FP32 in the matrix cores and are rounded once, to
// the output's type. Products are exact: beside BF16 x the weights' values are widened to BF16, which holds
// each (two significant bits and the exponent of the scale; near 2^127 a quarter of it), beside FP16 x
// the codes' to FP16, a block's sum getting its scale in FP32, and MXFP4 x is multiplied as it is.
//
// For experts, rows of x belong to experts by ranges (offsets) and each expert has weights of
// its own; rows may be gathered from a token's row by the sorted order.
#include <atomic>

#include "mxfp4_product.h"

namespace mps {
namespace {

// x[rows, k] as rows of whole blocks, `width` elements wide, with zeros past column k; eight
// elements a work-item.
__global__ __launch_bounds__(256) void mxfp4_pack_kernel(const uint16_t *__restrict__ x, int64_t rows, int64_t stride,
                                                         int32_t k, int32_t width, uint16_t *__restrict__ out) {
  const uint32_t pieces = (uint32_t)width / 8;
  for (int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x; unit < rows * pieces; unit += (int64_t)gridDim.x * 256) {
    const int64_t row = unit / pieces;
    const int32_t col = (int32_t)(unit - row * pieces) * 8;
    *reinterpret_cast<u32x4 *>(out + row * width + col) = load_row8(x + row * stride, col, k);
  }
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
  // x has rows / top rows, of which the kernels take none past the last: there has to be one.
  if (p->gather && p->rows % p->top != 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: a gather's %lld rows are no multiple of top (%lld)", (long long)p->rows, (long long)p->top);
  // The kernels find MXFP4 rows by an offset from their tile's first one.
  if (p->gather && p->x_type == MPS_TYPE_MXFP4)
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: a gather needs 16-bit x");
  return MPS_OK;
}

}  // namespace

int32_t compute_units() {
  constexpr int kDevices = 64;
  static std::atomic<int32_t> known[kDevices];
  int device = 0, cus = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= kDevices) return 256;
  if (const int32_t k = known[device].load(std::memory_order_relaxed)) return k;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus < 1) return 256;
  known[device].store(cus, std::memory_order_relaxed);
  return cus;
}

namespace {

// Which kernel takes a product, and what it needs.
struct Way {
  ProductArgs args;
  bool tiles;  // mxfp4_tile.hip, else mxfp4_rows.hip: the one predicted to be done earlier
  int choice;
  bool packed;  // x is packed into the workspace first
  int64_t workspace;
};
Way way_of(const mps_mxfp4_product *p) {
  Way w = {};
  ProductArgs &a = w.args;
  a.x = p->x, a.x_scales = p->x_scales, a.x_stride = p->x_stride;
  a.w = p->w, a.w_scales = p->w_scales, a.bias = p->bias, a.out = p->out;
  a.offsets = p->experts > 0 ? p->offsets : nullptr, a.order = p->order;
  a.rows = (int32_t)p->rows, a.x_rows = (int32_t)(p->gather ? p->rows / p->top : p->rows);
  a.n = (int32_t)p->n, a.k = (int32_t)p->k, a.row_blocks = (int32_t)mx_blocks(p->k);
  a.experts = (int32_t)p->experts, a.top = (int32_t)p->top, a.gather = p->gather;
  a.bias_type = p->bias_type, a.out_type = p->out_type;
  const int32_t cus = compute_units();
  const Prediction rows = predict_rows(a, p->x_type, cus), tiles = predict_tiles(a, p->x_type, cus);
  w.tiles = tiles.choice >= 0 && (rows.choice < 0 || tiles.us < rows.us);
  w.choice = w.tiles ? tiles.choice : rows.choice;
  w.packed = p->x_type != MPS_TYPE_MXFP4 && p->k > 0 &&
             !(w.tiles ? block_rows(p->x, p->x_stride, p->k) : piece_rows(p->x, p->x_stride, p->k));
  if (w.packed) w.workspace = a.x_rows * packed_width(p->k) * 2;
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
  if (way.choice < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: %lld x %lld outputs are too many", (long long)p->rows, (long long)p->n);
  if (way.workspace > 0 && (!workspace || workspace_bytes < way.workspace || !aligned16(workspace)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4 product: %lld bytes of workspace are needed, 16-byte aligned",
                (long long)way.workspace);
  ProductArgs a = way.args;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (way.packed) {
    const int32_t width = (int32_t)packed_width(p->k);
    const dim3 grid(workgroups(((int64_t)a.x_rows * (width / 8) + 255) / 256));
    hipLaunchKernelGGL(mxfp4_pack_kernel, grid, dim3(256), 0, s, static_cast<const uint16_t *>(p->x), (int64_t)a.x_rows,
                       p->x_stride, a.k, width, static_cast<uint16_t *>(workspace));
    a.x = workspace, a.x_stride = width, a.k = width;
  }
  if (way.tiles)
    launch_tiles(a, p->x_type, way.choice, s);
  else
    launch_rows(a, p->x_type, way.choice, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
