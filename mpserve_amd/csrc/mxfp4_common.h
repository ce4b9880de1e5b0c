// What the MXFP4 and expert kernels share: element types, vectors, and the format's arithmetic.
//
// MXFP4: 32 consecutive elements of a row share a scale 2^(s - 127), s a byte (255: the whole
// block is NaN), and each has a code of 4 bits: sign, two bits of exponent, one of mantissa
// (0, 0.5, 1, 1.5, 2, 3, 4, 6). A row of k elements has ceil(k / 32) blocks: as many scale
// bytes, and 16 bytes of codes each, the earlier element in a byte's low half.
#pragma once

#include "mps_common.h"

namespace mps {

constexpr int kMxBlock = 32;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16-byte accesses take any alignment
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// A grid holds fewer than 2^32 work-items: kernels over elements or rows get at most this many
// workgroups (of 256) and go on where the grid ends.
constexpr int64_t kMostWorkgroups = 1 << 22;
inline unsigned workgroups(int64_t wanted) { return (unsigned)(wanted < kMostWorkgroups ? wanted : kMostWorkgroups); }

inline int64_t mx_blocks(int64_t k) { return (k + kMxBlock - 1) / kMxBlock; }
__host__ __device__ inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool is_float_type(int32_t t) { return t == MPS_TYPE_BF16 || t == MPS_TYPE_F16 || t == MPS_TYPE_F32; }
inline int64_t type_bytes(int32_t t) { return t == MPS_TYPE_F32 ? 4 : 2; }

// The scale conversions take: only the exponent's bits count, so byte 0 is 2^-127 though its
// bits are those of 0.0, and byte 255 makes every result NaN.
__device__ inline float mx_scale(uint32_t s) { return __uint_as_float(s << 23); }

// The scale itself, for FP32 arithmetic.
__device__ inline float mx_scale_value(uint32_t s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23);
}

template <int T>
struct Elem;
template <>
struct Elem<MPS_TYPE_BF16> {
  typedef uint16_t raw;
  static __device__ float get(raw v) { return __uint_as_float((uint32_t)v << 16); }
  // Round to nearest even; a NaN stays one.
  static __device__ raw put(float f) { return __builtin_bit_cast(raw, (__bf16)f); }
};
template <>
struct Elem<MPS_TYPE_F16> {
  typedef uint16_t raw;
  static __device__ float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ raw put(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
};
template <>
struct Elem<MPS_TYPE_F32> {
  typedef float raw;
  static __device__ float get(raw v) { return v; }
  static __device__ raw put(float f) { return f; }
};

// One value of a type known only at run time (biases, routing weights: uniform branches).
__device__ inline float load_as_float(const void *p, int32_t type, int64_t i) {
  if (type == MPS_TYPE_F32) return static_cast<const float *>(p)[i];
  const uint16_t v = static_cast<const uint16_t *>(p)[i];
  return type == MPS_TYPE_BF16 ? Elem<MPS_TYPE_BF16>::get(v) : Elem<MPS_TYPE_F16>::get(v);
}
__device__ inline void store_as(void *p, int32_t type, int64_t i, float f) {
  if (type == MPS_TYPE_F32)
    static_cast<float *>(p)[i] = f;
  else
    static_cast<uint16_t *>(p)[i] = type == MPS_TYPE_BF16 ? Elem<MPS_TYPE_BF16>::put(f) : Elem<MPS_TYPE_F16>::put(f);
}

}  // namespace mps
