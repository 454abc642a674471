// The 4-bit weight format (include/rwkv_w4.h) in registers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "w4_launch.hpp"

namespace rwkv_w4 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf_bits(uint32_t b) { return __builtin_bit_cast(float, b << 16); }

// The eight weights of a word, without their group's scale, divided by kShrink,
// as bf16 (exact: the conversion's factor is a power of two). A product's sums
// are taken of these and multiplied by kShrink at the end, so that a sum
// overflows only where the result or a partial sum of it does.
constexpr float kShrink = 8.f;
__device__ __forceinline__ bf16x8 weights8(uint32_t w) {
  constexpr float k = 1.f / kShrink;
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, k, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, k, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, k, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, k, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// kParts bf16 vectors that add up to eight activations: one for bf16, three for
// fp32 (8 significant bits each, cut off and not rounded, so that the largest
// numbers do not overflow). An infinity is wholly in the first, a NaN in all.
template <int kParts>
struct Parts {
  bf16x8 p[kParts];
};
__device__ __forceinline__ Parts<3> split(const float (&x)[8]) {
  Parts<3> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x[e]) & 0xffff0000u);
    const float rest = x[e] == hi ? 0.f : x[e] - hi;
    const float mid = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, rest) & 0xffff0000u);
    const float v[3] = {hi, mid, rest - mid};
#pragma unroll
    for (int i = 0; i < 3; ++i)
      r.p[i][e] = __builtin_bit_cast(__bf16, static_cast<uint16_t>(__builtin_bit_cast(uint32_t, v[i]) >> 16));
  }
  return r;
}

// the scales of an output's inputs 128 k .., as floats
template <int kGroup>
__device__ __forceinline__ void load_scales(const void* scales, int64_t at, float (&s)[kInputs / kGroup]) {
  constexpr int n = kInputs / kGroup;
  const uint16_t* const p = static_cast<const uint16_t*>(scales) + at * n;
  if constexpr (n == 1) {
    s[0] = bf_bits(*p);
  } else if constexpr (n == 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    s[0] = bf_bits(w & 0xffffu);
    s[1] = bf_bits(w >> 16);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    s[0] = bf_bits(w.x & 0xffffu);
    s[1] = bf_bits(w.x >> 16);
    s[2] = bf_bits(w.y & 0xffffu);
    s[3] = bf_bits(w.y >> 16);
  }
}

}  // namespace rwkv_w4
