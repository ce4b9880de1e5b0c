// MXFP4 quantization and its inverse (the format: mxfp4_common.h).
//
// Quantization of a block x[0..31]:
//   s = max(0, exponent byte of max|x| as FP32 - 2), that is floor(log2 max|x|) - 2, biased by
//       127 and at least 0: the largest element lands in [4, 8) and codes reach 6;
//   code = x / 2^(s - 127) rounded to the nearest code, ties to the even one, above 6 to 6; the
//       sign is kept, -0 included. Scaling by a power of two is exact, so this is the only
//       rounding.
// A block with an infinity or a NaN has s = 255 and zero codes: it reads back as NaN.
//
// Both are bound by memory: 2 + 17/32 bytes an element for BF16. Four lanes share a block, eight
// elements each, so a wave reads 1 KiB (BF16) and writes 256 bytes of codes at a time; the
// block's maximum takes two steps across the four lanes.
#include "mxfp4_common.h"

namespace mps {
namespace {

constexpr int kThreads = 256;

__device__ inline uint32_t quad_max(uint32_t v) {
  const uint32_t a = __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);  // lanes 1, 0, 3, 2
  v = v > a ? v : a;
  const uint32_t b = __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);  // lanes 2, 3, 0, 1
  return v > b ? v : b;
}

// Eight elements of a row from column `col` on, at any alignment; zeros past column k.
template <int T>
__device__ inline void load8(const typename Elem<T>::raw *row, int64_t col, int64_t k, uint32_t (&v)[T == MPS_TYPE_F32 ? 8 : 4]) {
  if (col + 8 <= k) {
    constexpr int n = T == MPS_TYPE_F32 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const u32x4 q = reinterpret_cast<const u32x4_any *>(row + col)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = q[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      typename Elem<T>::raw e = 0;
      if (col + i < k) e = row[col + i];
      if constexpr (T == MPS_TYPE_F32)
        v[i] = __float_as_uint(e);
      else
        v[i / 2] = i % 2 ? v[i / 2] | (uint32_t)e << 16 : e;
    }
  }
}

// kFlat: blocks lie one after the other in x, so no row is needed.
template <int T, bool kFlat>
__global__ __launch_bounds__(kThreads) void mxfp4_quantize_kernel(const typename Elem<T>::raw *__restrict__ x,
                                                                  uint32_t blocks, uint32_t row_blocks, int64_t k,
                                                                  int64_t stride, uint32_t *__restrict__ codes,
                                                                  uint8_t *__restrict__ scales) {
  for (uint64_t unit = (uint64_t)blockIdx.x * kThreads + threadIdx.x; unit < (uint64_t)blocks * 4;  // whole blocks, so whole quads
       unit += (uint64_t)gridDim.x * kThreads) {
    const uint32_t block = (uint32_t)(unit >> 2), part = (uint32_t)unit & 3;
    uint32_t row = 0, in_row = block;
    if (!kFlat) row = block / row_blocks, in_row = block - row * row_blocks;
    uint32_t v[T == MPS_TYPE_F32 ? 8 : 4];
    load8<T>(x + (int64_t)row * stride, (int64_t)in_row * kMxBlock + part * 8, kFlat ? INT64_MAX : k, v);

    uint32_t s;
    if constexpr (T == MPS_TYPE_F32) {
      uint32_t m = 0;
      for (int i = 0; i < 8; ++i) m = max(m, v[i] & 0x7fffffffu);
      s = quad_max(m) >> 23;
    } else {
      // Magnitudes order as their bits do, NaN above infinity.
      u16x2 m = {0, 0};
      for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
      const uint32_t top = quad_max(max((uint32_t)m.x, (uint32_t)m.y));
      if constexpr (T == MPS_TYPE_BF16)
        s = top >> 7;
      else
        s = __float_as_uint(Elem<T>::get((uint16_t)top)) >> 23;
    }
    const bool finite = s != 255;
    s = finite ? (s > 2 ? s - 2 : 0) : 255;

    const float scale = mx_scale(s);
    uint32_t c = 0;
    if constexpr (T == MPS_TYPE_F32) {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[0]), __uint_as_float(v[1]), scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[2]), __uint_as_float(v[3]), scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[4]), __uint_as_float(v[5]), scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[6]), __uint_as_float(v[7]), scale, 3);
    } else if constexpr (T == MPS_TYPE_BF16) {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[0]), scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[1]), scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[2]), scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, v[3]), scale, 3);
    } else {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[0]), scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[1]), scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[2]), scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, v[3]), scale, 3);
    }
    codes[unit] = finite ? c : 0;
    if (part == 0) scales[block] = (uint8_t)s;
  }
}

// Eight elements a lane: 4 bytes of codes in, 16 (or 32) out.
template <int T, bool kFlat>
__global__ __launch_bounds__(kThreads) void mxfp4_dequantize_kernel(const uint32_t *__restrict__ codes,
                                                                    const uint8_t *__restrict__ scales,
                                                                    uint32_t blocks, uint32_t row_blocks, int64_t k,
                                                                    typename Elem<T>::raw *__restrict__ out) {
  for (uint64_t unit = (uint64_t)blockIdx.x * kThreads + threadIdx.x; unit < (uint64_t)blocks * 4;
       unit += (uint64_t)gridDim.x * kThreads) {
    const uint32_t block = (uint32_t)(unit >> 2), part = (uint32_t)unit & 3;
    const uint32_t c = codes[unit];
    const float scale = mx_scale(scales[block]);
    uint32_t v[T == MPS_TYPE_F32 ? 8 : 4];
    if constexpr (T == MPS_TYPE_F32) {
      const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
      const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
      const float f[8] = {a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
      for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(f[i]);
    } else if constexpr (T == MPS_TYPE_BF16) {
      v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
      v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
      v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
      v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
    } else {
      v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0));
      v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1));
      v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2));
      v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3));
    }
    uint32_t row = 0, in_row = block;
    if (!kFlat) row = block / row_blocks, in_row = block - row * row_blocks;
    const int64_t col = (int64_t)in_row * kMxBlock + part * 8;
    typename Elem<T>::raw *o = out + (int64_t)row * k + col;
    if (kFlat || col + 8 <= k) {
      constexpr int n = T == MPS_TYPE_F32 ? 2 : 1;
#pragma unroll
      for (int i = 0; i < n; ++i) reinterpret_cast<u32x4_any *>(o)[i] = u32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < k) {
          if constexpr (T == MPS_TYPE_F32)
            o[i] = __uint_as_float(v[i]);
          else
            o[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
        }
    }
  }
}

int check_shape(const char *what, int32_t type, int64_t rows, int64_t k, const void *values, const void *codes,
                const void *scales) {
  if (!is_float_type(type)) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", what, (int)type);
  if (rows < 0 || k < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (rows == 0 || k == 0) return MPS_OK;
  if (!values || !codes || !scales) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (rows >= (int64_t)UINT32_MAX / mx_blocks(k))
    return fail(MPS_ERR_INVALID_ARGUMENT, "%s: %lld rows of %lld elements are over 2^32 blocks", what, (long long)rows,
                (long long)k);
  if ((reinterpret_cast<uintptr_t>(codes) & 3) != 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "%s: codes must be 4-byte aligned", what);
  return MPS_OK;
}

template <int T>
void launch_quantize(const void *x, int64_t rows, int64_t k, int64_t stride, uint8_t *codes, uint8_t *scales,
                     hipStream_t stream) {
  typedef typename Elem<T>::raw raw;
  const uint32_t row_blocks = (uint32_t)mx_blocks(k), blocks = (uint32_t)rows * row_blocks;
  const dim3 grid(workgroups(((int64_t)blocks * 4 + kThreads - 1) / kThreads));
  if (k % kMxBlock == 0 && (rows == 1 || stride == k))
    hipLaunchKernelGGL((mxfp4_quantize_kernel<T, true>), grid, dim3(kThreads), 0, stream, static_cast<const raw *>(x),
                       blocks, row_blocks, k, stride, reinterpret_cast<uint32_t *>(codes), scales);
  else
    hipLaunchKernelGGL((mxfp4_quantize_kernel<T, false>), grid, dim3(kThreads), 0, stream,
                       static_cast<const raw *>(x), blocks, row_blocks, k, stride,
                       reinterpret_cast<uint32_t *>(codes), scales);
}

template <int T>
void launch_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t k, void *out,
                       hipStream_t stream) {
  typedef typename Elem<T>::raw raw;
  const uint32_t row_blocks = (uint32_t)mx_blocks(k), blocks = (uint32_t)rows * row_blocks;
  const dim3 grid(workgroups(((int64_t)blocks * 4 + kThreads - 1) / kThreads));
  if (k % kMxBlock == 0)
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<T, true>), grid, dim3(kThreads), 0, stream,
                       reinterpret_cast<const uint32_t *>(codes), scales, blocks, row_blocks, k,
                       static_cast<raw *>(out));
  else
    hipLaunchKernelGGL((mxfp4_dequantize_kernel<T, false>), grid, dim3(kThreads), 0, stream,
                       reinterpret_cast<const uint32_t *>(codes), scales, blocks, row_blocks, k,
                       static_cast<raw *>(out));
}

}  // namespace
}  // namespace mps

using namespace mps;

extern "C" {

int mps_mxfp4_quantize(const void *x, int32_t type, int64_t rows, int64_t k, int64_t row_stride, uint8_t *codes,
                       uint8_t *scales, void *stream) {
  last_error().clear();
  const int rc = check_shape("mxfp4_quantize", type, rows, k, x, codes, scales);
  if (rc != MPS_OK || rows == 0 || k == 0) return rc;
  if (row_stride < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "mxfp4_quantize: negative row stride");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (type == MPS_TYPE_BF16)
    launch_quantize<MPS_TYPE_BF16>(x, rows, k, row_stride, codes, scales, s);
  else if (type == MPS_TYPE_F16)
    launch_quantize<MPS_TYPE_F16>(x, rows, k, row_stride, codes, scales, s);
  else
    launch_quantize<MPS_TYPE_F32>(x, rows, k, row_stride, codes, scales, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_mxfp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t k, void *out, int32_t type,
                         void *stream) {
  last_error().clear();
  const int rc = check_shape("mxfp4_dequantize", type, rows, k, out, codes, scales);
  if (rc != MPS_OK || rows == 0 || k == 0) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (type == MPS_TYPE_BF16)
    launch_dequantize<MPS_TYPE_BF16>(codes, scales, rows, k, out, s);
  else if (type == MPS_TYPE_F16)
    launch_dequantize<MPS_TYPE_F16>(codes, scales, rows, k, out, s);
  else
    launch_dequantize<MPS_TYPE_F32>(codes, scales, rows, k, out, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
