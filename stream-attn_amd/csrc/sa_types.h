// Vector types and 16-bit conversions shared by the row and decoding kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "seqattn_hip.h"

namespace sa {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
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
  // e4m3 bytes 2 kHalf and 2 kHalf + 1 of a dword, times 2^e as a float.
  template <bool kHalf>
  __device__ static inline uint32_t e4m3_pair(uint32_t w, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, kHalf));
  }
  // The four values of two dwords over 2^e to e4m3, to nearest even; at most 448.
  __device__ static inline uint32_t to_e4m3(uint32_t a, uint32_t b, float power) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const s16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(s16x2{0, 0}, __builtin_bit_cast(bf16x2, a), power, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, __builtin_bit_cast(bf16x2, b), power, true));
  }
  static constexpr uint32_t kInfinity = 0x7f80u;
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
  template <bool kHalf>
  __device__ static inline uint32_t e4m3_pair(uint32_t w, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, kHalf));
  }
  __device__ static inline uint32_t to_e4m3(uint32_t a, uint32_t b, float power) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const s16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(s16x2{0, 0}, __builtin_bit_cast(f16x2, a), power, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, __builtin_bit_cast(f16x2, b), power, true));
  }
  static constexpr uint32_t kInfinity = 0x7c00u;
  __device__ static inline f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// Signed byte i of a dword as a float.
__device__ inline float byte_float(uint32_t w, int i) { return (float)((int32_t)(w << (24 - 8 * i)) >> 24); }

// e4m3 bytes 2 kHalf and 2 kHalf + 1 of a dword as floats.
template <bool kHalf>
__device__ inline f32x2 e4m3_floats(uint32_t w) {
  return __builtin_amdgcn_cvt_pk_f32_fp8((int)w, kHalf);
}

// Four floats of at most 448 to e4m3, to nearest even (NaN stays NaN).
__device__ inline uint32_t e4m3_pack(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

// The value of an E8M0 scale: 2^(byte - 127), NaN for 255.
__device__ inline float e8m0_value(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}

}  // namespace

// What pages hold: rows of the operands' type, INT8 with an fp16 scale per row
// and head, e4m3 with an E8M0 scale per block of rows and head.
enum PageKind { kRowPages = SA_PAGES_ROWS, kInt8Pages = SA_PAGES_INT8, kE4m3Pages = SA_PAGES_E4M3 };

// log2 of a block's rows, -1 where blocks of that many cannot be: a power of two
// from 16 on that divides a page.
inline int32_t block_log2(int32_t block_tokens, int32_t page_tokens) {
  if (block_tokens < 16 || (block_tokens & (block_tokens - 1)) || page_tokens % block_tokens) return -1;
  return __builtin_ctz(block_tokens);
}

}  // namespace sa
