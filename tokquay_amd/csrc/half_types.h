// The 16-bit element types of the chunk kernels: what differs between bf16 and fp16.
#pragma once

#include "tq_internal.h"

namespace tq {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOnes = 0x3f803f80u;  // 1, 1
  static constexpr uint32_t kExponent = 0x7f80u;  // all ones: an infinity or a NaN
  // log2 units that a weight of the running maximum lies above 1, and that one may lie above that: 2^(kLift + kSlack + 1) is finite.
  static constexpr float kLift = 0.f, kSlack = 8.f;
  static __device__ __forceinline__ float load(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
  // C/D: column lane % 16, rows 4 (lane / 16) + 0..3. A: row, B: column lane % 16, depth 8 (lane / 16) + 0..7.
  static __device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
};

struct Fp16 {
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOnes = 0x3c003c00u;
  static constexpr uint32_t kExponent = 0x7c00u;
  static constexpr float kLift = 7.f, kSlack = 7.f;
  static __device__ __forceinline__ float load(uint16_t bits) { return (float)__builtin_bit_cast(_Float16, bits); }
  static __device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
};

// Two floats rounded to nearest into one 32-bit word, a in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename T::x2));
}

}  // namespace
}  // namespace tq
