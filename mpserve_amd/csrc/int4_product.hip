// Products with int4 weights: y[t, n] = sum over k of x[t, k] * s (q - z)[n, k], plus a bias.
//
// Both q and q - z are exact in 16 bits, so that matrix instructions multiply them by x exactly; a group's sum gets its scale in
// FP32, and the sum of the groups is rounded once, to the output's type. Few rows are bound by the weights' bytes and go to the
// kernel that streams them, many by the matrix cores and go to tiles; the one with the smaller predicted time is taken (4096 -> 14336,
// groups of 128, microseconds: 32 rows 14.6 and 31; 48 rows 14336 -> 4096 23 and 90; 4096 rows 1155 and, by the card, 470 to 510).
#include "int4_product.h"

namespace mps {
namespace {

// x[rows, k] as rows of whole blocks, `width` elements wide, with zeros past column k; eight elements a work-item.
__global__ __launch_bounds__(256) void int4_pack_kernel(const uint16_t *__restrict__ x, int64_t rows, int64_t stride, int32_t k, int32_t width,
                                                        uint16_t *__restrict__ out) {
  const uint32_t pieces = (uint32_t)width / 8;
  for (int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x; unit < rows * pieces; unit += (int64_t)gridDim.x * 256) {
    const int64_t row = unit / pieces;
    const int32_t col = (int32_t)(unit - row * pieces) * 8;
    *reinterpret_cast<u32x4 *>(out + row * width + col) = load_row8(x + row * stride, col, k);
  }
}

// The sums of x over spans of 32 << shift columns, at most 128, in FP32 by a tree, as three BF16 numbers; and x packed, if asked for. A wave takes
// 512 columns of a row, eight a lane.
template <int XT>
__global__ __launch_bounds__(256) void int4_sums_kernel(const uint16_t *__restrict__ x, int64_t rows, int64_t stride, int32_t k, int32_t spans,
                                                        int32_t shift, uint8_t *__restrict__ sums, int64_t sums_row, int32_t width,
                                                        uint16_t *__restrict__ packed) {
  const int lane = threadIdx.x & 63, in_span = 4 << shift;  // lanes a span
  const int32_t padded = (spans + 15) / 16 * 16, pieces = (padded << shift) / 16;
  const int64_t units = rows * pieces;
  for (int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += (int64_t)gridDim.x * 4) {
    const int64_t row = unit / pieces;
    const int32_t piece = (int32_t)(unit - row * pieces), col = piece * 512 + lane * 8, span = piece * (16 >> shift) + lane / in_span;
    float sum = 0;
    if (col < width) {
      const u32x4 v = load_row8(x + row * stride, col, k);
      if (packed) *reinterpret_cast<u32x4 *>(packed + row * width + col) = v;
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[2 * i] = Elem<XT>::get((uint16_t)v[i]), f[2 * i + 1] = Elem<XT>::get((uint16_t)(v[i] >> 16));
      sum = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
    }
    for (int d = 1; d < in_span; d *= 2) sum += __shfl_xor(sum, d);
    if (lane % in_span == 0) {
      uint32_t p[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        p[i] = Elem<MPS_TYPE_BF16>::put(sum);
        sum -= Elem<MPS_TYPE_BF16>::get((uint16_t)p[i]);
      }
      uint8_t *const to = sums + row * sums_row;
      *reinterpret_cast<uint64_t *>(to + span * 8) = (uint64_t)(p[2] | p[0] << 16) << 32 | (p[0] | p[1] << 16);
      *reinterpret_cast<uint16_t *>(to + padded * 8 + span * 2) = (uint16_t)p[1];
    }
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

// Which kernel takes a product, and what it needs.
struct Way {
  Int4Args args;
  bool tiles;  // int4_tile.hip, else int4_rows.hip: the one predicted to be done earlier
  int choice;
  bool packed;  // x is packed into the workspace first
  int64_t packed_bytes, workspace;  // the packed x, then its sums
};
Way way_of(const mps_int4_product *p) {
  Way w = {};
  Int4Args &a = w.args;
  a.x = p->x, a.x_stride = p->x_stride, a.w = p->w, a.bias = p->bias, a.out = p->out;
  a.offsets = p->experts > 0 ? p->offsets : nullptr, a.order = p->order;
  a.rows = (int32_t)p->rows, a.x_rows = (int32_t)(p->gather ? p->rows / p->top : p->rows);
  a.n = (int32_t)p->n, a.k = (int32_t)p->k, a.row_blocks = (int32_t)mx_blocks(p->k);
  a.experts = (int32_t)p->experts, a.top = (int32_t)p->top, a.gather = p->gather;
  a.bias_type = p->bias_type, a.out_type = p->out_type;
  a.scales = p->scales, a.zeros = p->zeros, a.scale_type = p->scale_type;
  a.groups = (int32_t)((p->k + p->group - 1) / p->group);
  while ((int64_t)32 << a.shift < p->group) ++a.shift;
  const int32_t cus = compute_units();
  const Prediction rows = predict_int4_rows(a, cus), tiles = predict_int4_tiles(a, cus);
  w.tiles = tiles.choice >= 0 && (rows.choice < 0 || tiles.us < rows.us);
  w.choice = w.tiles ? tiles.choice : rows.choice;
  w.packed = p->k > 0 && !(w.tiles ? block_rows(p->x, p->x_stride, p->k) : piece_rows(p->x, p->x_stride, p->k));
  if (w.packed) w.packed_bytes = a.x_rows * packed_width(p->k) * 2;
  if (w.tiles) a.sums_row = sums_row_bytes(a);
  w.workspace = w.packed_bytes + a.x_rows * a.sums_row;
  return w;
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
  *bytes = p->rows > 0 && p->n > 0 ? way_of(p).workspace : 0;
  return MPS_OK;
}

int mps_int4_multiply(const mps_int4_product *p, void *workspace, int64_t workspace_bytes, void *stream) {
  last_error().clear();
  const int rc = check(p);
  if (rc != MPS_OK || p->rows == 0 || p->n == 0) return rc;
  const Way way = way_of(p);
  if (way.choice < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: %lld x %lld outputs are too many", (long long)p->rows, (long long)p->n);
  if (way.workspace > 0 && (!workspace || workspace_bytes < way.workspace || !aligned16(workspace)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "int4 product: %lld bytes of workspace are needed, 16-byte aligned", (long long)way.workspace);
  Int4Args a = way.args;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int32_t width = (int32_t)packed_width(p->k), k = a.k;
  uint16_t *const packed = way.packed ? static_cast<uint16_t *>(workspace) : nullptr;
  const uint16_t *const x = static_cast<const uint16_t *>(p->x);
  if (way.tiles && k > 0) {
    uint8_t *const sums = static_cast<uint8_t *>(workspace) + way.packed_bytes;
    const int32_t shift = sums_shift(a), spans = sums_spans(a);
    const dim3 grid(workgroups(((int64_t)a.x_rows * (((spans + 15) / 16) << shift) + 3) / 4));
    if (p->x_type == MPS_TYPE_BF16)
      hipLaunchKernelGGL(int4_sums_kernel<MPS_TYPE_BF16>, grid, dim3(256), 0, s, x, (int64_t)a.x_rows, p->x_stride, k, spans, shift, sums,
                         a.sums_row, width, packed);
    else
      hipLaunchKernelGGL(int4_sums_kernel<MPS_TYPE_F16>, grid, dim3(256), 0, s, x, (int64_t)a.x_rows, p->x_stride, k, spans, shift, sums,
                         a.sums_row, width, packed);
    a.sums = sums;
  } else if (way.packed) {
    const dim3 grid(workgroups(((int64_t)a.x_rows * (width / 8) + 255) / 256));
    hipLaunchKernelGGL(int4_pack_kernel, grid, dim3(256), 0, s, x, (int64_t)a.x_rows, p->x_stride, k, width, packed);
  }
  if (way.packed) a.x = workspace, a.x_stride = width, a.k = width;
  if (way.tiles)
    launch_int4_tiles(a, p->x_type, way.choice, s);
  else
    launch_int4_rows(a, p->x_type, way.choice, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
