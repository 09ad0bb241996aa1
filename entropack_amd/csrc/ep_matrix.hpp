// What the matrix products share: fragment types of the matrix-core instructions, output kinds, element conversions.
#pragma once

#include "ep_common.hpp"

namespace ep {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

enum : int { kOutBF16 = 0, kOutF16 = 1, kOutF32 = 2 };

__device__ __forceinline__ uint32_t bf16_bits_of(float v) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const float2v two = {v, 0.0f};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2)) & 0xFFFFu;
}

__device__ __forceinline__ void store_out(void* y, int kind, int64_t at, float v) {
  if (kind == kOutBF16) reinterpret_cast<uint16_t*>(y)[at] = static_cast<uint16_t>(bf16_bits_of(v));
  else if (kind == kOutF16) reinterpret_cast<_Float16*>(y)[at] = static_cast<_Float16>(v);
  else reinterpret_cast<float*>(y)[at] = v;
}

__device__ __forceinline__ float load_bias(const void* bias, int kind, int n) {
  if (kind == kOutBF16) return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(bias)[n]) << 16);
  if (kind == kOutF16) return static_cast<float>(reinterpret_cast<const _Float16*>(bias)[n]);
  return reinterpret_cast<const float*>(bias)[n];
}

}  // namespace ep
