// Vector types and 16-bit conversions shared by the row and decoding kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sa {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Bf16 {
  // The two values of a dword, and two floats rounded to nearest even into one.
  __device__ static inline float lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
  __device__ static inline float hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
  __device__ static inline uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
  }
  __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

struct Fp16 {
  __device__ static inline float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
  __device__ static inline float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
  __device__ static inline uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  }
  __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// Signed byte i of a dword as a float.
__device__ inline float byte_float(uint32_t w, int i) { return (float)((int32_t)(w << (24 - 8 * i)) >> 24); }

}  // namespace
}  // namespace sa
