// Dropout whose mask is drawn where it is used (include/rwkv_dropout.h), with the
// addition to a residual in the same pass; its backward is the same kernel.
//
// A thread draws one Philox4x32-10 block, eight 16-bit numbers, for eight consecutive
// elements: sixteen bits decide as well as 32 do (p is a multiple of 2^-16, and what
// is kept is scaled by the probability in use), for half the multiplications.
//
// Memory bounds it: 16384 x 4096 bf16 with a residual 73 us, 5.5 TB/s (part of it from the
// last level's cache; a copy from memory reaches 4.96); without one 48, 5.6; 8192 x 768
// bf16 onto an fp32 residual 12 us, 5.2. Small calls are a launch (127 x 768: 2.4 us).
#include <algorithm>

#include "dropout_launch.hpp"

namespace rwkv_drop {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256, kEach = 8;

struct Words {
  uint32_t w[4];
};
__device__ __forceinline__ Words philox(uint64_t q, uint32_t site, uint32_t step, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(q), c1 = static_cast<uint32_t>(q >> 32), c2 = site, c3 = step;
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

template <bool BF>
__device__ __forceinline__ float load_one(const void* base, int64_t i) {
  if constexpr (BF) return static_cast<float>(static_cast<const __bf16*>(base)[i]);
  else return static_cast<const float*>(base)[i];
}
template <bool BF>
__device__ __forceinline__ void load_eight(const void* base, int64_t i, float (&v)[kEach]) {
  if constexpr (BF) {
    const bf16x8 p = *reinterpret_cast<const bf16x8*>(static_cast<const __bf16*>(base) + i);
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = static_cast<float>(p[e]);
  } else {
    const f32x4* const p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + i);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  }
}
template <bool BF>
__device__ __forceinline__ void store_eight(void* base, int64_t i, const float (&v)[kEach]) {
  if constexpr (BF) {
    bf16x8 p;
#pragma unroll
    for (int e = 0; e < kEach; ++e) p[e] = static_cast<__bf16>(v[e]);
    *reinterpret_cast<bf16x8*>(static_cast<__bf16*>(base) + i) = p;
  } else {
    f32x4* const p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + i);
    p[0] = f32x4{v[0], v[1], v[2], v[3]};
    p[1] = f32x4{v[4], v[5], v[6], v[7]};
  }
}

// kWhole: all operands begin on a 16-byte boundary, and so does every eight of them.
template <bool BF, bool OBF, bool kAdd, bool kWhole>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const Call c) {
  const uint64_t seed = static_cast<uint64_t>(c.rng[0]);
  const uint32_t step = static_cast<uint32_t>(c.rng[1]);
  const float scale = c.threshold ? 65536.f / static_cast<float>(c.threshold) : 0.f;
  const int64_t groups = (c.n + kEach - 1) / kEach;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; q < groups; q += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t i = q * kEach;
    const bool full = kWhole && i + kEach <= c.n;
    float x[kEach], r[kEach];
    if (full) {
      load_eight<BF>(c.x, i, x);
      if constexpr (kAdd) load_eight<OBF>(c.residual, i, r);
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        x[e] = i + e < c.n ? load_one<BF>(c.x, i + e) : 0.f;
        if constexpr (kAdd) r[e] = i + e < c.n ? load_one<OBF>(c.residual, i + e) : 0.f;
      }
    }
    const Words u = philox(static_cast<uint64_t>(q), c.site, step, seed);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const uint32_t number = e % 2 ? u.w[e / 2] >> 16 : u.w[e / 2] & 0xffffu;
      x[e] = number < c.threshold ? x[e] * scale : 0.f;
      if constexpr (kAdd) x[e] += r[e];
    }
    if (full) {
      store_eight<OBF>(c.out, i, x);
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (i + e < c.n) {
          if constexpr (OBF) static_cast<__bf16*>(c.out)[i + e] = static_cast<__bf16>(x[e]);
          else static_cast<float*>(c.out)[i + e] = x[e];
        }
    }
  }
}

constexpr int64_t kMostBlocks = 1 << 22;   // a launch has fewer than 2^32 threads; beyond, a thread takes several eights

template <bool BF, bool OBF, bool kAdd>
void launch(const Call& c, hipStream_t s) {
  const uintptr_t places = reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.residual) | reinterpret_cast<uintptr_t>(c.out);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((c.n + kThreads * kEach - 1) / (kThreads * kEach), kMostBlocks)));
  if ((places & 15) == 0) hipLaunchKernelGGL((dropout_kernel<BF, OBF, kAdd, true>), grid, dim3(kThreads), 0, s, c);
  else hipLaunchKernelGGL((dropout_kernel<BF, OBF, kAdd, false>), grid, dim3(kThreads), 0, s, c);
}
template <bool BF, bool OBF>
void launch(const Call& c, hipStream_t s) {
  if (c.residual) launch<BF, OBF, true>(c, s);
  else launch<BF, OBF, false>(c, s);
}

}  // namespace

hipError_t launch(const Call& c, hipStream_t s) {
  if (c.bf16) c.out_bf16 ? launch<true, true>(c, s) : launch<true, false>(c, s);
  else c.out_bf16 ? launch<false, true>(c, s) : launch<false, false>(c, s);
  return hipGetLastError();
}

}  // namespace rwkv_drop
