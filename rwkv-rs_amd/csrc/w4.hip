// Products with 4-bit weights, and quantising and restoring them
// (include/rwkv_w4.h).
//
// linear: y[m, n] = sum over groups G of s[n, G] * sum over k in G of x[m, k] v[n, k].
// The values v are small bf16 numbers, so the inner sums are matrix
// instructions on bf16 operands whose products are exact; a group's sum is
// multiplied by its scale in fp32 and added to the total. (Weights times scale
// rounded to bf16 would be one operation less for each four products and 2^-9
// off each.) An fp32 activation is three bf16 parts that hold all of it.
//
// The weights' bytes bound it for up to 8 rows of a wide matrix: few_kernel, 1 x 4096
// x 16384 (34 MB) 8.6 us, 8 x 4096 x 65536 28 us (4.8 TB/s, what a copy reaches). More
// rows, up to 64, wait for their activations, which every workgroup reads: 12 x 10240 x
// 2560 11.0 us (1.3 TB/s of weights), 64 x 4096 x 16384 17.1 (2.1). Many rows are
// matrix products: tile_kernel, 512 x 2048 x 8192 22.9 us (750 TFLOP/s), 2048 x 4096 x
// 4096 62 to 69 us (1105 to 1000; groups of 64), a library product of bf16 matrices of
// 8192^3 1130 to 1400.
#include <algorithm>
#include <iterator>

#include "w4_device.hpp"

namespace rwkv_w4 {
namespace {

constexpr int kWave = 64;

// Rows of inputs that are no multiple of eight begin anywhere; the hardware takes
// such addresses in one access.
struct __attribute__((packed, aligned(2))) Half8 {
  bf16x8 v;
};
struct __attribute__((packed, aligned(4))) Float8 {
  float v[8];
};

// Elements i .. i + 7 of a row of n in its type, those past its end zero (kWhole:
// there are none).
template <bool BF>
struct Eight {
  std::conditional_t<BF, bf16x8, float[8]> v;
};
template <bool BF, bool kWhole>
__device__ __forceinline__ Eight<BF> load8(const void* row, int64_t i, int64_t n) {
  using T = std::conditional_t<BF, __bf16, float>;
  const T* const p = static_cast<const T*>(row) + i;
  Eight<BF> x;
  if (kWhole || i + 8 <= n) {
    if constexpr (BF) {
      x.v = reinterpret_cast<const Half8*>(p)->v;
    } else {
      const Float8 w = *reinterpret_cast<const Float8*>(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) x.v[e] = w.v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x.v[e] = T(0.f);
      if (i + e < n) x.v[e] = p[e];
    }
  }
  return x;
}

template <bool BF>
__device__ __forceinline__ void store8(void* row, int64_t i, int64_t n, const float (&v)[8]) {
  if (i + 8 <= n) {
    if constexpr (BF) {
      Half8 w;
#pragma unroll
      for (int e = 0; e < 8; ++e) w.v[e] = static_cast<__bf16>(v[e]);
      *reinterpret_cast<Half8*>(static_cast<uint16_t*>(row) + i) = w;
    } else {
      Float8 w;
#pragma unroll
      for (int e = 0; e < 8; ++e) w.v[e] = v[e];
      *reinterpret_cast<Float8*>(static_cast<float*>(row) + i) = w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (i + e >= n) return;
      if constexpr (BF) static_cast<__bf16*>(row)[i + e] = static_cast<__bf16>(v[e]);
      else static_cast<float*>(row)[i + e] = v[e];
    }
  }
}

__device__ __forceinline__ char* row_at(void* base, int64_t row, int64_t n, bool bf) {
  return static_cast<char*>(base) + row * n * (bf ? 2 : 4);
}

// ---------------------------------------------------------- quantise, restore
// A wave takes a block of 16 outputs and 128 inputs, lane l the output l % 16
// at the inputs 32 j + 8 (l / 16) .. + 7 of each j, which are its 16 bytes of
// the packed block; four lanes hold 32 consecutive inputs of an output. HBM bounds
// both: 65536 x 768 fp32 quantised and restored 93 us for 453 MB (4.9 TB/s).
constexpr int kBlockWaves = 4;

// Eight weights' codes: the nearest magnitude to |w| / s, ties to the even
// mantissa, as the hardware's conversion rounds the quotient. The quotient is the
// correctly rounded one (a product with the rounded reciprocal, corrected by its
// residual, which is exact), and that is on a midpoint m only where w / s is: m s
// has at most eleven significant bits, so another w is at least a unit in its own
// last place away from it, and its quotient more than half of one in m's. Numbers
// near the ends of fp32's range are moved to its middle first. What rounds to zero
// has no sign. By comparisons with the seven midpoints it was twice the
// instructions: 65536 x 768 bf16 42 us, so 29.
struct Scale {
  float shift, s, inverse;
  __device__ __forceinline__ explicit Scale(float scale) {
    shift = scale < 0x1p-64f ? 0x1p100f : scale > 0x1p64f ? 0x1p-100f : 1.f;
    s = scale * shift;
    inverse = 1.f / s;
  }
  __device__ __forceinline__ float quotient(float w) const {
    w *= shift;
    const float q = w * inverse;
    return fmaf(fmaf(-q, s, w), inverse, q);
  }
};
__device__ __forceinline__ uint32_t codes_of(const float (&w)[8], const Scale& s) {
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, s.quotient(w[0]), s.quotient(w[1]), 1.f, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, s.quotient(w[2]), s.quotient(w[3]), 1.f, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, s.quotient(w[4]), s.quotient(w[5]), 1.f, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, s.quotient(w[6]), s.quotient(w[7]), 1.f, 3);
  const uint32_t some = (word & 0x77777777u) + 0x77777777u;   // bit 3 of each code whose magnitude is not 0
  return word & (some | 0x77777777u);
}

constexpr uint32_t kMaxScale = 0x7e2a;   // the largest bf16 number six times which is an fp32 number

template <bool BF, int kGroup>
__global__ __launch_bounds__(kBlockWaves* kWave) void quantize_kernel(const WeightCall c) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint32_t ib = static_cast<uint32_t>(blocks_in(c.in)), blocks = static_cast<uint32_t>(blocks_out(c.out)) * ib;
  const uint32_t first = blockIdx.x * kBlockWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t i = first; i < blocks; i += gridDim.x * kBlockWaves) {
    const uint32_t out = i / ib;
    const int64_t b = i, n = out, k = i - out * ib, row = n * kRows + r;
    Eight<BF> x[4];
    float w[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = load8<BF, false>(row_at(c.weight, min(row, c.out - 1), c.in, BF), k * kInputs + 32 * j + 8 * g, c.in);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[j][e] = row < c.out ? static_cast<float>(x[j].v[e]) : 0.f;
    // the largest magnitude as an integer: infinities and NaN are above all numbers
    uint32_t top[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top[j] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top[j] = max(top[j], __builtin_bit_cast(uint32_t, w[j][e]) & 0x7fffffffu);
    }
    constexpr int kGroups = kInputs / kGroup, kSteps = kGroup / 32;
    uint16_t scale[kGroups];
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      uint32_t t = top[q * kSteps];
#pragma unroll
      for (int j = 1; j < kSteps; ++j) t = max(t, top[q * kSteps + j]);
      t = max(t, static_cast<uint32_t>(__shfl_xor(static_cast<int>(t), 16)));
      t = max(t, static_cast<uint32_t>(__shfl_xor(static_cast<int>(t), 32)));
      const float s = __builtin_bit_cast(float, t) * (1.f / 6.f);
      const uint32_t rounded = __builtin_bit_cast(uint16_t, static_cast<__bf16>(s));
      scale[q] = static_cast<uint16_t>(t >= 0x7f800000u ? 0x7fc0u : min(rounded, kMaxScale));
    }
    u32x4 word;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float s = bf_bits(scale[j / kSteps]);
      word[j] = 0;
      const uint32_t codes = codes_of(w[j], Scale(s));
      if (s > 0.f) word[j] = codes;   // not 0, and not NaN
    }
    reinterpret_cast<u32x4*>(c.packed)[b * kWave + lane] = word;
    if (g == 0)
#pragma unroll
      for (int q = 0; q < kGroups; ++q) static_cast<uint16_t*>(c.scales)[(b * kRows + r) * kGroups + q] = scale[q];
  }
}

template <bool BF, int kGroup>
__global__ __launch_bounds__(kBlockWaves* kWave) void dequantize_kernel(const WeightCall c) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const uint32_t ib = static_cast<uint32_t>(blocks_in(c.in)), blocks = static_cast<uint32_t>(blocks_out(c.out)) * ib;
  const uint32_t first = blockIdx.x * kBlockWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t i = first; i < blocks; i += gridDim.x * kBlockWaves) {
    const uint32_t out = i / ib;
    const int64_t b = i, n = out, k = i - out * ib, row = n * kRows + r;
    if (row >= c.out) continue;
    const u32x4 word = reinterpret_cast<const u32x4*>(c.packed)[b * kWave + lane];
    const Scales<kGroup> s = load_scales<kGroup>(c.scales, b * kRows + r);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 v = weights8(word[j]);
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = kShrink * static_cast<float>(v[e]) * s[32 * j / kGroup];
      store8<BF>(row_at(c.weight, row, c.in, BF), k * kInputs + 32 * j + 8 * g, c.in, w);
    }
  }
}

// --------------------------------------------------------------------- linear
// v_mfma_f32_16x16x32_bf16: lane l holds A[row l % 16] and B[column l % 16] at
// k = 8 (l / 16) .. + 7, the result D[row 4 (l / 16) + r][column l % 16].
template <bool BF>
__device__ __forceinline__ auto parts(const Eight<BF>& x) {
  if constexpr (BF) return Parts<1>{{x.v}};
  else return split(x.v);
}

template <int kParts>
__device__ __forceinline__ f32x4 multiply(const Parts<kParts>& x, const bf16x8& w, f32x4 sum) {
#pragma unroll
  for (int i = kParts - 1; i >= 0; --i) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], w, sum, 0, 0, 0);
  return sum;
}

__device__ __forceinline__ float rounded(float v) { return static_cast<float>(static_cast<__bf16>(v)); }
__device__ __forceinline__ float squared_relu(float v) {
  v = rounded(v);
  return v > 0.f ? v * v : v == v ? 0.f : v;   // NaN stays
}
template <bool BF>
__device__ __forceinline__ void store_y(const LinearCall& c, int64_t row, int64_t col, float v) {
  if (row >= c.rows || col >= c.out) return;
  v *= kShrink;
  if constexpr (BF) {
    if (c.finish == kAddTo) static_cast<float*>(c.y)[row * c.out + col] += rounded(v);
    else static_cast<__bf16*>(c.y)[row * c.out + col] = static_cast<__bf16>(c.finish == kSquaredRelu ? squared_relu(v) : v);
  } else {
    static_cast<float*>(c.y)[row * c.out + col] = v;
  }
}

// eight outputs of a row, from the sums before the last multiplication
template <bool BF>
__device__ __forceinline__ void store_y8(const LinearCall& c, int64_t row, int64_t col, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= kShrink;
  if constexpr (BF) {
    if (c.finish == kAddTo) {
      void* const to = row_at(c.y, row, c.out, false);
      const Eight<false> x = load8<false, false>(to, col, c.out);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = x.v[e] + rounded(v[e]);
      store8<false>(to, col, c.out, v);
      return;
    }
    if (c.finish == kSquaredRelu) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = squared_relu(v[e]);
    }
  }
  store8<BF>(row_at(c.y, row, c.out, BF), col, c.out, v);
}

// Few rows. A workgroup forms 16 NT outputs of up to 16 MT rows; its waves split
// the inputs in blocks of 128 (one 16-byte load of weights a lane and 16 outputs,
// four matrix instructions a tile) and add up through LDS in wave order. A wave
// has kDepth blocks' loads in flight: what the weights' stream needs is bytes in
// flight on every compute unit, from many waves, or several tiles or blocks a wave.
// us, 1 row, (NT, waves, depth): 4096 x 16384 one tile at a time 11.4, (1, 8, 4)
// 12.8, (4, 8, 1) 11.1, (2, 16, 1) 8.9; 768 x 65536, 8 rows, (1, 8, 4) 17.0, (2,
// 16, 1) 11.5, (4, 8, 2) 9.5; 4096 x 4096 (1, 8, 4) 5.2, (1, 16, 2) 4.7; 16384 x
// 4096 one tile at a time 23.9, (1, 16, 2) 11.4, (2, 16, 1) 14.
template <bool BF, bool kWhole, int kGroup, int MT, int NT, int kWaves, int kDepth>
__global__ __launch_bounds__(kWaves* kWave) void few_kernel(const LinearCall c) {
  __shared__ float part[kWaves][MT * NT * 256];
  constexpr int kParts = BF ? 1 : 3, kSteps = kGroup / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = lane & 15, g = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * NT, ib = blocks_in(c.in), ob = blocks_out(c.out);
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * 16 * MT;
  const void* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = row_at(const_cast<void*>(c.x), min(row0 + 16 * m + t, c.rows - 1), c.in, BF);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int64_t k0 = wave; k0 < ib; k0 += kWaves * kDepth) {
    u32x4 word[kDepth][NT];
    Scales<kGroup> s[kDepth][NT];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int64_t k = k0 + d * kWaves;
      if (k < ib) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int64_t b = min(n0 + n, ob - 1) * ib + k;   // past the end: the last outputs, not stored
          word[d][n] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(c.packed) + b * kWave + lane);
          s[d][n] = load_scales<kGroup>(c.scales, b * kRows + t);
        }
      }
    }
    Eight<BF> xs[kDepth][MT][4];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int64_t k = k0 + d * kWaves;
      if (k < ib) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) xs[d][m][j] = load8<BF, kWhole>(x[m], k * kInputs + 32 * j + 8 * g, c.in);
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (k0 + d * kWaves < ib) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f32x4 sum[NT];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Parts<kParts> a = parts<BF>(xs[d][m][j]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              sum[n] = multiply(a, weights8(word[d][n][j]), j % kSteps == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sum[n]);
              if (j % kSteps == kSteps - 1) acc[m][n] += sum[n] * s[d][n][32 * j / kGroup];
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4*>(&part[wave][(m * NT + n) * 256 + 4 * lane]) = acc[m][n];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * NT * 256; i += kWaves * kWave) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += part[w][i];
    const int l = (i >> 2) & 63, m = i / (NT * 256), n = i / 256 % NT;
    store_y<BF>(c, row0 + 16 * m + 4 * (l >> 4) + (i & 3), (n0 + n) * kRows + (l & 15), v);
  }
}

// Between a wave's writes to its part of LDS and its lanes' reads of each other's,
// and before that part is written again. The LDS takes a wave's accesses in order;
// this keeps the compiler's order.
__device__ __forceinline__ void wave_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Many rows. A workgroup forms 16 MT rows by 64 NT outputs of `share` blocks of
// inputs, its four waves 16 NT outputs each; where the inputs are shared among
// workgroups, join_kernel adds up what they leave. The rows' activations of 128
// inputs go through LDS in the order in which the waves' matrix instructions read
// them: piece (row 16 m + t, inputs 32 j + 8 g ..) of 16 bytes at place 16 g + (t ^
// spread(g, j)) of 64 for (m, j). With few_kernel's way of reading activations 512 x
// 2048 x 8192 took 124 us.
//
// Loads are two blocks ahead, in registers of their own for odd and even blocks, as
// they come from memory: activations are asked for once LDS has the ones before,
// weights once the products have. A condition around a load, a conversion at it or a
// copy of what it brings made the compiler wait for all of them in each block: 512 x
// 2048 x 8192 fp32 81 us, then 50; 512 x 8192 x 2048 40, then 32. The last blocks ask
// for the last one again instead. (4, 4) tiles have registers for one block ahead.
// A tile's sums are added to the total while the next tile's products run, which
// hides the wait for them (128 x 4096 x 4096 15.3, then 13.0; 512 x 2048 x 8192 in
// groups of 32 29.8, then 27.2), and results are stored by way of LDS, eight outputs
// a lane (512 x 2048 x 8192 26.4, then 25.0; 2048 x 4096 x 4096 71.5, then 67.4).
// What is left there is the loop: 1.15 us a block of (4, 2) tiles on two workgroups a
// compute unit, of which the matrix units are busy for 45%, as in a large library
// product.
constexpr int kTileWaves = 4, kTileThreads = kTileWaves * kWave;
// Eight neighbouring threads bring pieces (g, j) of one row with all g and two j:
// their places are to differ modulo 8 (128 bytes a cycle). A read takes 16 lanes a
// cycle, places 0 to 3 and 12 to 15 of a g and 4 to 11 of the next or the other way
// round: g and g + 1 are to agree in whether bits 2 and 3 of it differ. (4 g + j gave
// two-way conflicts in both, half of the LDS's busy cycles.)
__device__ __forceinline__ int spread(int g, int j) { return 2 * g + (j & 1) + (j >> 1) * 8; }
template <bool BF, bool kWhole, int kGroup, int MT, int NT>
__global__ __launch_bounds__(kTileThreads, 2) void tile_kernel(const LinearCall c, const int64_t share) {
  constexpr int kParts = BF ? 1 : 3, kSteps = kGroup / 32, kGroups = kInputs / kGroup, kPiecesOfRow = kInputs / 8;
  constexpr int kLoads = 16 * MT * kPiecesOfRow / kTileThreads;   // pieces a thread brings
  constexpr int kAhead = MT * NT > 8 ? 1 : 2;
  constexpr int kPitch = 16 * NT + 4;   // of a wave's 16 rows of results: the four that a store writes apart in banks
  using Blocks = bf16x8[2][kParts][MT * 4 * kWave];
  using Results = float[kTileWaves][16 * kPitch];
  __shared__ __attribute__((aligned(16))) char lds[std::max(sizeof(Blocks), sizeof(Results))];
  Blocks& xs = *reinterpret_cast<Blocks*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = lane & 15, g = lane >> 4;
  const int64_t ib = blocks_in(c.in), ob = blocks_out(c.out);
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * 16 * MT;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) * kTileWaves + wave) * NT;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  Eight<BF> bring[kAhead][kLoads];
  u32x4 word[kAhead][NT];
  Scales<kGroup> s[kAhead][NT];
  const int piece = tid % kPiecesOfRow;
  auto load_w = [&](int d, int64_t k) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t b = min(n0 + n, ob - 1) * ib + k;   // past the end: the last outputs, not stored
      word[d][n] = reinterpret_cast<const u32x4*>(c.packed)[b * kWave + lane];
      s[d][n] = load_scales<kGroup>(c.scales, b * kRows + t);
    }
  };
  auto load_x = [&](int d, int64_t k) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int64_t row = min(row0 + tid / kPiecesOfRow + i * (kTileThreads / kPiecesOfRow), c.rows - 1);
      bring[d][i] = load8<BF, kWhole>(row_at(const_cast<void*>(c.x), row, c.in, BF), k * kInputs + 8 * piece, c.in);
    }
  };
  const int64_t first = blockIdx.z * share, k1 = min(first + share, ib);
#pragma unroll
  for (int d = 0; d < kAhead; ++d) {
    load_x(d, min(first + d, k1 - 1));
    load_w(d, min(first + d, k1 - 1));
    __builtin_amdgcn_sched_barrier(0);
  }
  auto step = [&](int d, int buffer, int64_t k) {
    bf16x8(*const at)[MT * 4 * kWave] = xs[buffer];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = tid / kPiecesOfRow + i * (kTileThreads / kPiecesOfRow), j = piece >> 2, q = piece & 3;
      const int place = (row / 16 * 4 + j) * kWave + 16 * q + ((row & 15) ^ spread(q, j));
      const Parts<kParts> x = parts<BF>(bring[d][i]);
#pragma unroll
      for (int p = 0; p < kParts; ++p) at[p][place] = x.p[p];
    }
    __syncthreads();   // the block before is read: its place is written only after the next of these
    load_x(d, min(k + kAhead, k1 - 1));
    __builtin_amdgcn_sched_barrier(0);
    Parts<kParts> a[kSteps][MT];
    f32x4 before[MT];   // the sums of the tiles and group before, not yet in acc
#pragma unroll
    for (int i = 0; i < kGroups * NT; ++i) {
      const int q = i / NT, n = i % NT;
      if (n == 0) {
#pragma unroll
        for (int e = 0; e < kSteps; ++e)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int p = 0; p < kParts; ++p)
              a[e][m].p[p] = at[p][(m * 4 + q * kSteps + e) * kWave + 16 * g + (t ^ spread(g, q * kSteps + e))];
      }
      f32x4 sum[MT];
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        const bf16x8 v = weights8(word[d][n][q * kSteps + e]);
#pragma unroll
        for (int m = 0; m < MT; ++m) sum[m] = multiply(a[e][m], v, e == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sum[m]);
      }
      if (i > 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][(i - 1) % NT] += before[m] * s[d][(i - 1) % NT][(i - 1) / NT];
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) before[m] = sum[m];
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][NT - 1] += before[m] * s[d][NT - 1][kGroups - 1];
    load_w(d, min(k + kAhead, k1 - 1));
    __builtin_amdgcn_sched_barrier(0);
  };
  int64_t k = first;
  if constexpr (kAhead == 1) {
    for (int buffer = 0; k < k1; ++k, buffer ^= 1) step(0, buffer, k);
  } else {
    for (; k + 1 < k1; k += 2) {
      step(0, 0, k);
      step(1, 1, k + 1);
    }
    if (k < k1) step(0, 0, k);
  }
  // 16 rows of the wave's results at a time go through LDS to be stored in pieces of
  // eight outputs
  const bool shared = gridDim.z > 1;
  float* const out = (*reinterpret_cast<Results*>(lds))[wave];
  __syncthreads();   // all have read the last block
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) out[(4 * g + r) * kPitch + 16 * n + t] = acc[m][n][r];
    wave_exchange();
#pragma unroll
    for (int i = lane; i < 32 * NT; i += kWave) {
      const int at = i % (2 * NT) * 8;
      const int64_t row = row0 + 16 * m + i / (2 * NT), col = n0 * kRows + at;
      if (row >= c.rows || col >= c.out) continue;
      const f32x4* const from = reinterpret_cast<const f32x4*>(out + i / (2 * NT) * kPitch + at);
      const f32x4 lo = from[0], hi = from[1];
      float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if (shared) store8<false>(c.partial + (blockIdx.z * c.rows + row) * c.out, col, c.out, v);
      else store_y8<BF>(c, row, col, v);
    }
    wave_exchange();
  }
}

// The parts that tile_kernel's workgroups left of each output, in order.
template <bool BF>
__global__ __launch_bounds__(256) void join_kernel(const LinearCall c, const int splits) {
  const int64_t n = c.rows * c.out, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
#pragma unroll 4
  for (int z = 0; z < splits; ++z) v += c.partial[z * n + i];
  v *= kShrink;
  if constexpr (BF) static_cast<__bf16*>(c.y)[i] = static_cast<__bf16>(v);
  else static_cast<float*>(c.y)[i] = v;
}

// ----------------------------------------------------------------- dispatch
template <typename F>
hipError_t by_group(int group, F&& f) {
  if (group == 32) f(std::integral_constant<int, 32>());
  else if (group == 64) f(std::integral_constant<int, 64>());
  else f(std::integral_constant<int, 128>());
  return hipGetLastError();
}
template <typename F>
hipError_t by_type(bool bf16, int group, F&& f) {
  return by_group(group, [&](auto g) { bf16 ? f(std::true_type(), g) : f(std::false_type(), g); });
}

// a block of weights a wave; beyond what a launch holds, several
dim3 block_grid(const WeightCall& c) {
  const int64_t blocks = blocks_out(c.out) * blocks_in(c.in);
  return dim3(static_cast<unsigned>(std::min<int64_t>((blocks + kBlockWaves - 1) / kBlockWaves, 1 << 20)));
}

}  // namespace

hipError_t launch_quantize(const WeightCall& c, hipStream_t stream) {
  return by_type(c.bf16, c.group, [&](auto bf, auto group) {
    hipLaunchKernelGGL((quantize_kernel<bf(), group()>), block_grid(c), dim3(kBlockWaves * kWave), 0,
                       stream, c);
  });
}

hipError_t launch_dequantize(const WeightCall& c, hipStream_t stream) {
  return by_type(c.bf16, c.group, [&](auto bf, auto group) {
    hipLaunchKernelGGL((dequantize_kernel<bf(), group()>), block_grid(c), dim3(kBlockWaves * kWave), 0,
                       stream, c);
  });
}

namespace {

template <bool BF, bool kWhole, int kGroup, int MT, int NT, int kWaves, int kDepth>
void few(const LinearCall& c, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((blocks_out(c.out) + NT - 1) / NT),
                  static_cast<unsigned>((c.rows + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((few_kernel<BF, kWhole, kGroup, MT, NT, kWaves, kDepth>), grid, dim3(kWaves * kWave), 0, s, c);
}
// Up to 16 rows run on few_kernel; more on it or on tile_kernel's tiles of 16 MT rows
// and 64 NT outputs, with the inputs of each shared among several workgroups or not,
// whichever a linear model of the time, in ns, holds to be fastest. A block of inputs
// (few_kernel: a wave's) takes `block` and `each` for every workgroup that a compute
// unit has of the launch; shared inputs a launch more and the parts' way through
// memory. The numbers are fitted to 7100 timings of 17 to 2048 rows by 768 x 768 to
// 4096 x 16384 and 768 x 65536 (rms 9% bf16, 8% fp32; few_kernel's 7 to 11%); the
// tiles picked are on average 0.9% (bf16) and 1.4% (fp32) slower than the fastest that
// was timed, bf16 tiles of (2, 4) and (4, 1) among them. kFewLaunch is 1000 lower than
// its fit, for the second launch and the workspace that few_kernel does not ask the
// host for. us, model's pick / one tile of (4, 4), fp32 (4, 2), for all, shared among
// up to 512 workgroups: 256 x 2048 x 8192 15 / 26, 64 x 2560 x 10240 12 / 19, 512 x
// 2048 x 8192 fp32 50 / 70; few_kernel / tiles: 17 x 768 x 768 2.9 / 4.6, 17 x 2048 x
// 8192 5.5 / 9.2, 64 x 2048 x 2048 9.7 / 7.4.
struct Tile {
  int MT, NT;
  int64_t block, each;
};
constexpr Tile kBf16Tiles[] = {{2, 1, 89, 153}, {2, 2, 136, 259}, {4, 2, 86, 537}, {4, 4, 536, 701}};
constexpr Tile kF32Tiles[] = {{2, 1, 232, 470}, {2, 2, 252, 698}, {2, 4, 373, 1016}};
// few_kernel's `each` is for 16 MT rows; fewer, which are fewer lines to read, take
// (rows + 20) / (16 MT + 20) of it.
constexpr Tile kBf16Few[] = {{2, 1, 0, 1860}, {2, 2, 960, 1280}, {4, 1, 210, 3390}};
constexpr Tile kF32Few[] = {{2, 1, 2080, 1920}, {2, 2, 3350, 1700}, {4, 1, 340, 7850}};
constexpr int64_t kFewRows = 16, kFewMost = 64, kFewWaves = 8;
constexpr int64_t kUnits = 256, kFewLaunch = 1000, kLaunch = 4000, kJoin = 2000, kJoinBytesPerNs = 2400, kMaxSplits = 64;
struct Plan {
  bool few;
  int MT, NT, splits;
  int64_t share;   // blocks of inputs of a workgroup
};
int few_columns(int64_t rows, int64_t ob) {   // few_kernel's NT
  if (rows > 32) return 1;
  if (rows > 16) return ob >= 512 ? 2 : 1;
  return ob >= 2048 ? 4 : ob >= 512 ? 2 : 1;
}
int64_t blocks_ns(const Tile& t, int64_t groups, int64_t blocks) {
  const int64_t all = groups <= 4 * kUnits ? (groups + kUnits - 1) / kUnits * t.each : groups * t.each / kUnits;
  return blocks * (t.block + all);
}
Plan plan(int64_t rows, int64_t out, int64_t in, bool bf16, bool may_share) {
  const int64_t ob = blocks_out(out), ib = blocks_in(in);
  const int NT = few_columns(rows, ob);
  Plan best{true, rows <= 16 ? 1 : rows <= 32 ? 2 : 4, NT, 1, ib};
  if (rows <= kFewRows) return best;
  int64_t least = INT64_MAX;
  if (rows <= kFewMost) {
    Tile t = (bf16 ? kBf16Few : kF32Few)[rows > 32 ? 2 : NT - 1];
    t.each = t.each * (rows + 20) / (16 * t.MT + 20);
    least = kFewLaunch + blocks_ns(t, (ob + NT - 1) / NT, (ib + kFewWaves - 1) / kFewWaves);
  }
  auto consider = [&](const Tile& t, int64_t count, int64_t splits) {
    const int64_t share = (ib + splits - 1) / splits;
    splits = (ib + share - 1) / share;
    int64_t ns = kLaunch + blocks_ns(t, count * splits, share);
    if (splits > 1) ns += kJoin + splits * rows * out * 4 / kJoinBytesPerNs;
    if (ns >= least) return;
    least = ns;
    best = Plan{false, t.MT, t.NT, static_cast<int>(splits), share};
  };
  const Tile* const tiles = bf16 ? kBf16Tiles : kF32Tiles;
  const int n = bf16 ? std::size(kBf16Tiles) : std::size(kF32Tiles);
  for (int i = 0; i < n; ++i) {
    const Tile& t = tiles[i];
    const int64_t count = (rows + 16 * t.MT - 1) / (16 * t.MT) * ((ob + 4 * t.NT - 1) / (4 * t.NT));
    consider(t, count, 1);
    if (!may_share) continue;
    for (int64_t units = kUnits; units <= 4 * kUnits; units += kUnits)   // one to four workgroups a compute unit
      if (const int64_t splits = std::min({units / count, ib, kMaxSplits}); splits > 1) consider(t, count, splits);
  }
  return best;
}

template <bool BF, bool kWhole, int kGroup, int MT, int NT>
void tiles(const LinearCall& c, const Plan& t, hipStream_t s) {
  constexpr int cols = kTileWaves * NT;
  const dim3 grid(static_cast<unsigned>((blocks_out(c.out) + cols - 1) / cols),
                  static_cast<unsigned>((c.rows + 16 * MT - 1) / (16 * MT)), t.splits);
  hipLaunchKernelGGL((tile_kernel<BF, kWhole, kGroup, MT, NT>), grid, dim3(kTileThreads), 0, s, c, t.share);
  if (t.splits > 1)
    hipLaunchKernelGGL(join_kernel<BF>, dim3(static_cast<unsigned>((c.rows * c.out + 255) / 256)), dim3(256), 0, s, c,
                       t.splits);
}

template <bool BF, bool kWhole, int kGroup>
void linear(const LinearCall& c, hipStream_t s) {
  const Plan t = plan(c.rows, c.out, c.in, BF, c.partial != nullptr);
  if (t.few) {
    if (t.MT == 4) return few<BF, kWhole, kGroup, 4, 1, 8, 1>(c, s);
    if (t.MT == 2) {
      if (t.NT == 2) return few<BF, kWhole, kGroup, 2, 2, 8, 1>(c, s);
      return few<BF, kWhole, kGroup, 2, 1, 8, BF ? 2 : 1>(c, s);
    }
    if (t.NT == 4) return few<BF, kWhole, kGroup, 1, 4, 8, BF ? 2 : 1>(c, s);
    if (t.NT == 2) return few<BF, kWhole, kGroup, 1, 2, BF ? 16 : 8, 1>(c, s);
    return few<BF, kWhole, kGroup, 1, 1, 16, BF ? 2 : 1>(c, s);
  }
  if constexpr (BF) {
    if (t.NT == 4) return tiles<BF, kWhole, kGroup, 4, 4>(c, t, s);
    if (t.MT == 4) return tiles<BF, kWhole, kGroup, 4, 2>(c, t, s);
  } else {
    if (t.NT == 4) return tiles<BF, kWhole, kGroup, 2, 4>(c, t, s);
  }
  if (t.NT == 2) return tiles<BF, kWhole, kGroup, 2, 2>(c, t, s);
  tiles<BF, kWhole, kGroup, 2, 1>(c, t, s);
}

}  // namespace

int64_t workspace_bytes(int64_t rows, int64_t out, int64_t in, bool bf16) {
  const int splits = plan(rows, out, in, bf16, true).splits;
  return splits == 1 ? 0 : splits * rows * out * 4;
}

hipError_t launch_linear(const LinearCall& c, hipStream_t stream) {
  return by_type(c.bf16, c.group, [&](auto bf, auto group) {
    if (c.in % kInputs == 0) linear<bf(), true, group()>(c, stream);
    else linear<bf(), false, group()>(c, stream);
  });
}

}  // namespace rwkv_w4
