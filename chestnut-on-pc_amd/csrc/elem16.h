// The 16-bit element types of the token-cache kernels (f16 and bf16): vector types,
// conversions, the matrix products, and the division by a launch constant.
#pragma once

#include "common.h"

namespace ck {

typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

// The element-type codes of include/chestnut.h.
constexpr int DT_F16 = 1, DT_BF16 = 4, DT_E4M3 = 5;

template <typename T>
struct Elem;
template <>
struct Elem<half_t> {
  typedef half2_t v2;
  typedef half4_t v4;
  typedef half8_t v8;
  // the largest value that a rounding to four significant bits leaves finite
  static constexpr float top = 61440.0f;
  // exponent field of two packed values, and its lowest bit: (u & EXP) + LOW has a
  // half's top bit set where that half is an infinity or a NaN
  static constexpr unsigned EXP = 0x7C007C00u, LOW = 0x04000400u;
  // softmax weights, up to 2^8 before this, are kept 2^LIFT times as large: the type's top is not
  // far, its bottom is (many keys at 2^-25 of the strongest one's weight still count)
  static constexpr float LIFT = 7.0f;
  static __device__ __forceinline__ float16_t mfma32(v8 a, v8 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4_t mfma16(v8 a, v8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 a, float c) {   // c + a[0] + a[1]
    return __builtin_amdgcn_fdot2(a, v2{(half_t)1.0f, (half_t)1.0f}, c, false);
  }
};
template <>
struct Elem<bf16_t> {
  typedef bf16x2_t v2;
  typedef bf16x4_t v4;
  typedef bf16x8_t v8;
  static constexpr float top = 3.19014718988379809496913694467282698e38f;   // 1.875 * 2^127
  static constexpr unsigned EXP = 0x7F807F80u, LOW = 0x00800080u;
  static constexpr float LIFT = 0.0f;
  static __device__ __forceinline__ float16_t mfma32(v8 a, v8 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4_t mfma16(v8 a, v8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 a, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(a, v2{(bf16_t)1.0f, (bf16_t)1.0f}, c, false);
  }
};

// Two floats rounded to nearest even (one v_cvt_pk instruction).
template <typename T>
__device__ __forceinline__ typename Elem<T>::v2 pack2(float a, float b) {
  return __builtin_convertvector(float2_t{a, b}, typename Elem<T>::v2);
}

// n / d for n, d < 2^16: umulhi(n, m) with m = ceil(2^32 / d) is exact there
// (d = 1 has no such m and is passed as 0).
inline unsigned div_magic(unsigned d) { return d == 1 ? 0u : (unsigned)((0x100000000ull + d - 1) / d); }
__device__ __forceinline__ unsigned div_by(unsigned n, unsigned m) { return m ? __umulhi(n, m) : n; }

}  // namespace ck
