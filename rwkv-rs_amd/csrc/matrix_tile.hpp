// A tile of a matrix product of 16-bit operands on the matrix cores, sums in
// fp32, for the kernels that do something else with the sums than store them.
//
// out[p, q] = sum_k P[p, k] Q[q, k] for kP values of p and kQ of q. Each operand
// lies in memory either by rows (P[p, k .. k + 7] consecutive) or by steps (P[p ..
// p + 7, k] consecutive), so that a matrix and its transpose are read from where
// they are: rows go to the matrix instructions as they are, steps by the LDS loads
// that transpose 4 x 16 elements.
//
// A workgroup of kWavesP x kWavesQ waves brings kStep steps of both operands at a
// time to LDS (16 bytes a lane, without a stop in registers), kStages - 1 of them
// ahead of the products, behind one barrier each. Instruction 16x16x32: lane l has
// element l % 16 of p or q and the steps 8 (l / 16) .. + 7; of the sums, lane l has
// q = l % 16 and p = 4 (l / 16) .. + 3.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rwkv_tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32;              // steps of k a stage
constexpr int kStepBytes = kStep * 2;
constexpr int kPieces = kStepBytes / 16;

template <bool kHalf>   // fp16 operands, or bf16
__device__ __forceinline__ f32x4 multiply(s16x8 p, s16x8 q, f32x4 c) {
  if constexpr (kHalf)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}

// 16 bytes from each lane's address to consecutive places from `to` on.
__device__ __forceinline__ void bring(const char* from, char* to) {
  typedef const void __attribute__((address_space(1))) * Global;
  typedef void __attribute__((address_space(3))) * Local;
  __builtin_amdgcn_global_load_lds((Global)(uintptr_t)from, (Local)to, 16, 0, 0);
}

// An operand of a tile: element (i, k) at base + i * pitch + 2 k (rows) or base + k *
// pitch + 2 i (steps). `items` and `steps`: how many there are from the tile's first
// on. Beyond them the last one is read again: rows that nobody stores, or steps
// whose other operand is zero. In the steps' form i is read in eights, and the pitch
// covers the last eight whole.
struct Operand {
  const char* base;
  int64_t pitch;
  int64_t items, steps;
};

enum Layout { kRows, kSteps };
// Where the 16-byte pieces of a row lie, so that the lanes of a read touch different
// banks. kSpread: tile i's lane m reads row 64 (i / 4) + 16 (m / 4) + 4 (i % 4) + m %
// 4 instead of 16 i + m, which leaves a lane with 16 consecutive p.
template <bool kSpread>
__device__ __forceinline__ int row_swizzle(int row) { return (-(row >> (kSpread ? 4 : 2))) & 3; }
__device__ __forceinline__ int step_swizzle(int k) { return (k & 3) | ((k >> 1) & 4); }

// How a workgroup's lanes bring an operand of kItems to LDS and read it back.
template <Layout kLayout, int kItems, int kWaves, bool kSpread>
struct Side {
  static constexpr int kBytes = kItems * kStepBytes;
  static constexpr int kLoads = kBytes / (kWaves * 1024);   // a wave's instructions a stage
  static_assert(kBytes % (kWaves * 1024) == 0);
  static_assert(kLayout == kRows || kItems >= 128);         // a step's pieces are swapped within sixteen
  static constexpr int kPerStep = kItems / 8;               // pieces of a step (steps' form)
  uint32_t at[kLoads];     // byte offset of a lane's piece from the stage's first element
  const char* base;
  int64_t pitch, steps;

  // the step (steps' form) or row that load j of this lane brings
  __device__ __forceinline__ int line(int j, int wave, int lane) const {
    const int place = (j * kWaves + wave) * 64 + lane;
    return kLayout == kRows ? place / kPieces : place / kPerStep;
  }
  // bytes from the line's first element on
  __device__ __forceinline__ int within(int j, int wave, int lane) const {
    const int place = (j * kWaves + wave) * 64 + lane, l = line(j, wave, lane);
    if constexpr (kLayout == kRows) return 16 * ((place % kPieces) ^ row_swizzle<kSpread>(l));
    const int c = place % kPerStep;
    return 16 * (c ^ (2 * step_swizzle(l)));
  }
  __device__ __forceinline__ void init(const Operand& o, int wave, int lane) {
    base = o.base;
    pitch = o.pitch;
    steps = o.steps;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int l = line(j, wave, lane);
      if constexpr (kLayout == kRows) {
        at[j] = static_cast<uint32_t>(min(static_cast<int64_t>(l), o.items - 1) * pitch) + within(j, wave, lane);
      } else {
        const int last = static_cast<int>(min(o.items - 1, static_cast<int64_t>(kItems - 1)) / 8 * 16);
        at[j] = static_cast<uint32_t>(l * pitch) + min(within(j, wave, lane), last);
      }
    }
  }
  // steps k .. k + kStep - 1 of the operand's array at `offset` bytes from the first one
  __device__ __forceinline__ void load(char* lds, int64_t offset, int64_t k, int wave, int lane) const {
    if constexpr (kLayout == kRows) {
      const char* from = base + offset + 2 * k;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) bring(from + at[j], lds + (j * kWaves + wave) * 1024);
    } else {
      const char* from = base + offset + k * pitch;
      if (k + kStep <= steps) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) bring(from + at[j], lds + (j * kWaves + wave) * 1024);
      } else {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const int64_t beyond = max(k + line(j, wave, lane) - (steps - 1), static_cast<int64_t>(0));
          bring(from + at[j] - beyond * pitch, lds + (j * kWaves + wave) * 1024);
        }
      }
    }
  }
  // what lane (m, g) of a wave whose items begin at `first` gives to tile i's instruction
  __device__ __forceinline__ s16x8 read(const char* lds, int first, int i, int m, int g) const {
    if constexpr (kLayout == kRows) {
      const int row = first + (kSpread ? 64 * (i / 4) + 16 * (m >> 2) + 4 * (i % 4) + (m & 3) : 16 * i + m);
      return *reinterpret_cast<const s16x8*>(lds + row * kStepBytes + 16 * (g ^ row_swizzle<kSpread>(row)));
    } else {
      typedef __attribute__((address_space(3))) s16x4* Local;
      const int k = 8 * g + (m >> 2);          // and k + 4, whose pieces lie alike
      const int piece = (first / 8 + 2 * i + ((m & 3) >> 1)) ^ (2 * step_swizzle(k));
      const char* from = lds + k * (kItems * 2) + 16 * piece + 8 * (m & 1);
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Local)(from));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Local)(from + 4 * kItems * 2));
      return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
};

// kPlanes 1: bf16 operands. 2: each operand is two fp16 arrays, the second (`plane`
// bytes behind the first) holding what rounding took from the first: the product is
// hi hi + hi lo + lo hi.
template <Layout kLayoutP, Layout kLayoutQ, int kP, int kQ, int kWavesP, int kWavesQ, bool kSpread, int kPlanes>
struct Tile {
  static constexpr int kWaves = kWavesP * kWavesQ, kThreads = 64 * kWaves;
  static constexpr int kStages = 3;
  static constexpr int kWaveP = kP / kWavesP, kWaveQ = kQ / kWavesQ;
  static constexpr int kTilesP = kWaveP / 16, kTilesQ = kWaveQ / 16;
  static_assert(!kSpread || kWaveP % 64 == 0);
  using SideP = Side<kLayoutP, kP, kWaves, kSpread>;
  using SideQ = Side<kLayoutQ, kQ, kWaves, false>;
  static constexpr int kStageBytes = SideP::kBytes + SideQ::kBytes;
  static constexpr int kLdsBytes = kStages * kStageBytes;
  static constexpr int kLoads = SideP::kLoads + SideQ::kLoads;
  static constexpr int kParts = kPlanes == 1 ? 1 : 3;

  f32x4 acc[kTilesP][kTilesQ];

  // Sums over the steps [k0, k1), whole stages. The workgroup may use `lds` again
  // once all of its waves have come back.
  __device__ __forceinline__ void sum(char* lds, const Operand& p, const Operand& q, int64_t plane_p, int64_t plane_q,
                                      int64_t k0, int64_t k1) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int wave_p = wave % kWavesP * kWaveP, wave_q = wave / kWavesP * kWaveQ;
#pragma unroll
    for (int i = 0; i < kTilesP; ++i)
#pragma unroll
      for (int j = 0; j < kTilesQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    SideP sp;
    SideQ sq;
    sp.init(p, wave, lane);
    sq.init(q, wave, lane);
    int64_t k = k0;      // the next stage's steps
    int part = 0;        // and which product of planes it belongs to
    auto load = [&](int stage) {
      char* const at = lds + stage * kStageBytes;
      sp.load(at, kPlanes > 1 && part == 2 ? plane_p : 0, k, wave, lane);
      sq.load(at + SideP::kBytes, kPlanes > 1 && part == 1 ? plane_q : 0, k, wave, lane);
      // past the last stage, that one is brought again, so that a wait always finds as
      // many loads behind it
      if (k + kStep < k1) {
        k += kStep;
      } else if (part + 1 < kParts) {
        ++part;
        k = k0;
      }
    };
    const int64_t stages = (k1 - k0) / kStep * kParts;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load(s);
    int now = 0, next = kStages - 1;
    for (int64_t s = 0; s < stages; ++s) {
      // this wave's loads of stage s are here, and behind the barrier everyone's; and
      // everyone has read the stage that is overwritten next
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * kLoads) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      load(next);
      const char* const at = lds + now * kStageBytes;
      s16x8 b[kTilesQ];
#pragma unroll
      for (int j = 0; j < kTilesQ; ++j) b[j] = sq.read(at + SideP::kBytes, wave_q, j, m, g);
#pragma unroll
      for (int i = 0; i < kTilesP; ++i) {
        const s16x8 a = sp.read(at, wave_p, i, m, g);
#pragma unroll
        for (int j = 0; j < kTilesQ; ++j) acc[i][j] = multiply<(kPlanes > 1)>(a, b[j], acc[i][j]);
      }
      now = now == kStages - 1 ? 0 : now + 1;
      next = next == kStages - 1 ? 0 : next + 1;
    }
    // the loads that were brought for no product, and everyone's reads
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
};

}  // namespace rwkv_tile
