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
// are taken of these and multiplied by kShrink at the end. A group's sum, which
// its scale has yet to make small, is at most 128 * 6 / 1024 of the largest
// activation and so never overflows. At the other end the products are exact
// (multiples of 2^-133 2^-11), and a scaled sum is rounded to a multiple of 2^-149:
// 2^-139 in the result. (A factor of 8 lost two activations of 3e38 at a scale of
// 0.01 to infinity.)
constexpr float kShrink = 1024.f;
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

// The scales of an output's inputs 128 k .. as they are stored, and one of them as
// a float. They are loaded apart from their use: a conversion where the load stands
// waits there, before the loads after it are on their way.
template <int kGroup>
struct Scales {
  static constexpr int kCount = kInputs / kGroup, kWords = (kCount + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ float operator[](int i) const {
    return __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};
template <int kGroup>
__device__ __forceinline__ Scales<kGroup> load_scales(const void* scales, int64_t at) {
  Scales<kGroup> s;
  const uint16_t* const p = static_cast<const uint16_t*>(scales) + at * Scales<kGroup>::kCount;
  if constexpr (kGroup == 128) {
    s.w[0] = *p;
  } else if constexpr (kGroup == 64) {
    s.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    s.w[0] = w.x;
    s.w[1] = w.y;
  }
  return s;
}

}  // namespace rwkv_w4
