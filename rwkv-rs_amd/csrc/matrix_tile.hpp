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
// time to LDS (16 bytes a lane, without a stop in registers), a stage or two ahead of
// the products, behind one barrier each. Instruction 16x16x32: lane l has
// element l % 16 of p or q and the steps 8 (l / 16) .. + 7; of the sums, lane l has
// q = l % 16 and p = 4 (l / 16) .. + 3.
//
// Why so: 256 x 256 sums on eight waves of 256 registers a lane (128 of them sums) and five
// slots of 32 KiB, all of LDS, for 64 steps of the operands. A stage is 512 instructions,
// 0.86 us at the dense peak; it takes 1.1 to 1.2, and over 4096 channels 1.4, where the
// matrix cores draw the power that there is and the clock falls (1.49 PFLOP/s; products
// from registers alone sustain 1.98). Stages of 32 steps, whose rows are half cache lines,
// were bound by the L2's requests: 2048 x 4096 x 65536 1104 us for 839. Two loops were
// slower: instructions of 32 x 32 x 16 (1.4 PFLOP/s from registers) and four waves of 128 x
// 128 (registers spill; 3 to 5%).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace rwkv_tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;              // steps of k a stage: whole cache lines of an operand that lies by rows

template <bool kFp16>   // or bf16
__device__ __forceinline__ f32x4 multiply(s16x8 p, s16x8 q, f32x4 c) {
  if constexpr (kFp16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}

__device__ __forceinline__ s16x8 half_to_bf16(s16x8 v) {
  const f16x8 h = __builtin_bit_cast(f16x8, v);
  bf16x8 b;
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = static_cast<__bf16>(static_cast<float>(h[e]));
  return __builtin_bit_cast(s16x8, b);
}

// 16 bytes from each lane's offset to consecutive places from `to` on. A buffer load:
// the compiler takes a global one to LDS for one that LDS may answer too, and waits for
// every LDS read behind it.
typedef __amdgpu_buffer_rsrc_t Buffer;
// A value that is the same in all lanes, where the compiler cannot see that it is.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return static_cast<int64_t>(uniform(static_cast<int>(v >> 32))) << 32 | static_cast<uint32_t>(uniform(static_cast<int>(v)));
}
__device__ __forceinline__ Buffer buffer(const char* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, -1, 0x00020000);
}
__device__ __forceinline__ void bring(Buffer from, uint32_t offset, int shift, char* to) {
  typedef void __attribute__((address_space(3))) * Local;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Local)to, 16, offset, shift, 0, 0);
}

// An operand of a tile: element (i, k) at base + i * pitch + 2 k (rows) or base + k *
// pitch + 2 i (steps). `items` and `steps`: how many there are from the tile's first
// on. Beyond them the last one is read again: rows that nobody stores, or steps
// whose other operand is zero. In the steps' form i is read in eights, and the pitch
// covers the last eight whole.
struct Operand {
  const char* base;
  int64_t pitch;
  int items, steps;
};

enum Layout { kRows, kSteps };
// Where the 16-byte pieces of a row lie, so that the lanes of a read touch different
// banks. kSpread: tile i's lane m reads row 32 (i / 2) + 8 (m / 4) + 4 (i % 2) + m %
// 4 instead of 16 i + m, which leaves a lane with 8 consecutive p of two tiles.
template <bool kSpread>
__device__ __forceinline__ int row_swizzle(int row) { return ((-(row >> (kSpread ? 3 : 2))) & 3) + 2 * (row & 2); }
__device__ __forceinline__ int step_swizzle(int k) { return (k & 3) | ((k >> 1) & 4); }

// How a workgroup's lanes bring an operand of kItems to LDS and read it back: kSize bytes
// an element, kSteps of them a stage.
template <Layout kLayout, int kItems, int kWaves, bool kSpread, int kSteps = kStep, int kSize = 2>
struct Side {
  static constexpr int kBytes = kItems * kSteps * kSize;
  static constexpr int kLoads = kBytes / (kWaves * 1024);   // a wave's instructions a stage
  static_assert(kBytes % (kWaves * 1024) == 0);
  static_assert(kLayout == kRows || kItems * kSize >= 256); // a step's pieces are swapped within sixteen
  static constexpr int kRowBytes = kSteps * kSize, kPieces = kRowBytes / 16;   // of a row (rows' form)
  static constexpr int kPerStep = kItems * kSize / 16;      // pieces of a step (steps' form)
  uint32_t at[kLoads];     // byte offset of a lane's piece from the stage's first element
  const char* base;
  int64_t pitch;
  int items, steps;
  bool ended;              // the places are of the last stage, which is not whole

  // the step (steps' form) or row that load j of this lane brings
  __device__ __forceinline__ int line(int j, int wave, int lane) const {
    const int place = (j * kWaves + wave) * 64 + lane;
    return kLayout == kRows ? place / kPieces : place / kPerStep;
  }
  // where a line's pieces lie in LDS: swapped, so that the lanes of a read touch different banks
  __device__ __forceinline__ static int swap(int line) {
    if constexpr (kLayout == kRows) return kPieces == 8 ? row_swizzle<kSpread>(line) : row_swizzle<kSpread>(line) & 3;
    else return kSize == 2 ? 2 * step_swizzle(line) : 4 * ((line >> 3) & 3);
  }
  // bytes from the line's first element on
  __device__ __forceinline__ int within(int j, int wave, int lane) const {
    const int place = (j * kWaves + wave) * 64 + lane;
    return 16 * (place % (kLayout == kRows ? kPieces : kPerStep) ^ swap(line(j, wave, lane)));
  }
  // Places of a stage from step k on, of which `steps` are left from k = 0; a whole stage's
  // do not depend on k.
  __device__ __forceinline__ void set(int k, int wave, int lane) {
    const int last = max(steps - 1 - k, 0);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int l = line(j, wave, lane), bytes = within(j, wave, lane);
      if constexpr (kLayout == kRows) {
        at[j] = static_cast<uint32_t>(min(l, items - 1) * pitch) + (kSize == 4 ? min(bytes, last / 4 * 16) : bytes);
      } else {
        at[j] = static_cast<uint32_t>(min(l, last) * pitch) + min(bytes, min(items - 1, kItems - 1) / (16 / kSize) * 16);
      }
    }
  }
  __device__ __forceinline__ void init(const Operand& o, int wave, int lane) {
    base = reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(o.base)));
    pitch = o.pitch;
    items = uniform(o.items);
    steps = uniform(o.steps);
    ended = false;
    set(0, wave, lane);
  }
  // Before the loads of the stage from step k on. Rows of 16-bit elements are whole stages.
  __device__ __forceinline__ void turn(int k, int wave, int lane) {
    if constexpr (kLayout == Layout::kSteps || kSize == 4) {
      const bool end = k + kSteps > steps;
      if (end || ended) {
        set(k, wave, lane);
        ended = end;
      }
    }
  }
  // The buffer of the steps k .. k + kStep - 1 of the operand's array at `offset` bytes
  // from the first one, and its load j.
  __device__ __forceinline__ Buffer stage(int64_t offset, int k) const {
    return buffer(base + offset + (kLayout == kRows ? kSize * k : min(k, steps - 1) * pitch));
  }
  __device__ __forceinline__ void load(int j, char* lds, Buffer from, int wave) const {
    bring(from, at[j], 0, lds + (j * kWaves + wave) * 1024);
  }
  // Of a lane (m, g) of a wave whose items begin at `first`: what read() of the steps' form
  // begins with. Tile i's place is this with 32 i in exclusive or.
  __device__ __forceinline__ static uint32_t lane_at(int first, int m, int g) {
    if constexpr (kLayout == kRows) return 0;
    const int k = 8 * g + (m >> 2);
    return k * (kItems * 2) + 16 * ((first / 8 + ((m & 3) >> 1)) ^ swap(k)) + 8 * (m & 1);
  }
  // what that lane gives to tile i's instruction over half a stage's steps
  __device__ __forceinline__ s16x8 read(const char* lds, uint32_t at_lane, int half, int first, int i, int m, int g) const {
    static_assert(kSize == 2);
    if constexpr (kLayout == kRows) {
      const int row = first + (kSpread ? 32 * (i / 2) + 8 * (m >> 2) + 4 * (i % 2) + (m & 3) : 16 * i + m);
      return *reinterpret_cast<const s16x8*>(lds + row * kRowBytes + 16 * ((4 * half + g) ^ swap(row)));
    } else {
      typedef __attribute__((address_space(3))) s16x4* Local;
      const char* const from = lds + (at_lane ^ (32 * i)) + 32 * half * (kItems * 2);   // and four steps on, whose pieces lie alike
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Local)(from));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Local)(from + 4 * kItems * 2));
      return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // the same of fp32 elements
  __device__ __forceinline__ void read(const char* lds, int first, int i, int m, int g, float (&v)[8]) const {
    static_assert(kSize == 4 && kSteps == 32);
    if constexpr (kLayout == kRows) {
      const int row = first + (kSpread ? 32 * (i / 2) + 8 * (m >> 2) + 4 * (i % 2) + (m & 3) : 16 * i + m);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 p = *reinterpret_cast<const f32x4*>(lds + row * kRowBytes + 16 * ((2 * g + h) ^ swap(row)));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = p[e];
      }
    } else {
      const char* const from = lds + 16 * ((first / 4 + 4 * i + (m >> 2)) ^ swap(8 * g)) + 4 * (m & 3);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float*>(from + (8 * g + e) * (kItems * kSize));
    }
  }
};

// What the operands are: kBf16; kHalf, both fp16; kHalfQ, P bf16 and Q fp16, which is
// rounded to bf16 on its way to the products; kHalves, each two fp16 arrays, the second
// (`plane` bytes behind the first) holding what rounding took from the first: the
// product is hi hi + hi lo + lo hi; kThirds, each three bf16 arrays that add up to an
// fp32 number: the six products down to 2^-16 of the first.
enum Kind { kBf16, kHalf, kHalfQ, kHalves, kThirds };
constexpr int kThirdsParts = 6;
__device__ __forceinline__ int third_p(int part) { return part == 2 || part == 3 ? 1 : part == 5 ? 2 : 0; }
__device__ __forceinline__ int third_q(int part) { return part == 1 || part == 3 ? 1 : part == 4 ? 2 : 0; }

// LDS holds three stages of one operand and two of the other (kDeepP: three of P). The
// loop's barrier lies kTail groups of products before a stage's end, when all of the
// stage has been read: behind it the next stage's first reads and the loads that
// overwrite this one are issued under the products that are left. With kLead, LDS holds
// one stage more than that of both: for small tiles, whose products take less time than a
// load.
template <Layout kLayoutP, Layout kLayoutQ, int kP, int kQ, int kWavesP, int kWavesQ, bool kSpread, bool kDeepP, Kind kKind,
          int kLead = 0>
struct Tile {
  static constexpr int kWaves = kWavesP * kWavesQ, kItemsQ = kQ, kAcross = kWavesP;
  static constexpr int kWaveP = kP / kWavesP, kWaveQ = kQ / kWavesQ;
  static constexpr int kTilesP = kWaveP / 16, kTilesQ = kWaveQ / 16;
  static_assert(!kSpread || kWaveP % 32 == 0);
  using SideP = Side<kLayoutP, kP, kWaves, kSpread>;
  using SideQ = Side<kLayoutQ, kQ, kWaves, false>;
  static constexpr int kSlotsP = kLead ? kLead + 1 : kDeepP ? 3 : 2, kSlotsQ = kLead ? kLead + 1 : kDeepP ? 2 : 3;
  static constexpr int kPlaceQ = kSlotsP * SideP::kBytes;
  static constexpr int kLdsBytes = kPlaceQ + kSlotsQ * SideQ::kBytes;
  static constexpr int kDeepLoads = kDeepP ? SideP::kLoads : SideQ::kLoads;
  // a wave's loads behind those of the stage that is waited for
  static constexpr int kBehind = kLead ? (kLead - 1) * (SideP::kLoads + SideQ::kLoads) : kDeepLoads;
  static_assert(kBehind < 64);
  static constexpr int kParts = kKind == kHalves ? 3 : kKind == kThirds ? kThirdsParts : 1;
  static constexpr int kTail = kTilesP / 2, kBody = 2 * kTilesP - kTail;   // groups of kTilesQ products
  static constexpr int kHeldP = 2;

  f32x4 acc[kTilesP][kTilesQ];

  // The next stage of an operand to be brought: its first step, which product of planes
  // it belongs to, and its slot. Past the last stage that one is brought again, so that
  // a wait always finds as many loads behind it.
  template <int kSlots>
  struct Next {
    int k, part, slot;
    __device__ __forceinline__ void advance(int k0, int k1) {
      slot = slot == kSlots - 1 ? 0 : slot + 1;
      if (k + kStep < k1) {
        k += kStep;
      } else if (part + 1 < kParts) {
        ++part;
        k = k0;
      }
    }
  };
  // What a wave has of a stage before its products begin, and of the stage before it:
  // the factors of the products that are left there.
  struct Held {
    s16x8 q[kTilesQ], p[kHeldP];
    s16x8 last_q[kTilesQ], last_p[kTail];
  };
  struct Place {
    SideP p;
    SideQ q;
    int64_t plane_p, plane_q;
    int wave, lane;
    uint32_t at_p, at_q;
    __device__ __forceinline__ Buffer from(const Next<kSlotsP>& n) const {
      return p.stage(kKind == kHalves ? (n.part == 2 ? plane_p : 0) : kKind == kThirds ? third_p(n.part) * plane_p : 0, n.k);
    }
    __device__ __forceinline__ Buffer from(const Next<kSlotsQ>& n, int) const {
      return q.stage(kKind == kHalves ? (n.part == 1 ? plane_q : 0) : kKind == kThirds ? third_q(n.part) * plane_q : 0, n.k);
    }
    __device__ __forceinline__ s16x8 read_p(const char* lds, uint32_t at, int half, int i) const {
      return p.read(lds, at, half, wave % kWavesP * kWaveP, i, lane & 15, lane >> 4);
    }
    __device__ __forceinline__ s16x8 read_q(const char* lds, uint32_t at, int half, int j) const {
      return q.read(lds, at, half, wave / kWavesP * kWaveQ, j, lane & 15, lane >> 4);
    }
  };
  __device__ __forceinline__ static void bring_p(int n, char* lds, const Place& a, Buffer from, const Next<kSlotsP>& next) {
    a.p.load(n, lds + next.slot * SideP::kBytes, from, a.wave);
  }
  __device__ __forceinline__ static void bring_q(int n, char* lds, const Place& a, Buffer from, const Next<kSlotsQ>& next) {
    a.q.load(n, lds + kPlaceQ + next.slot * SideQ::kBytes, from, a.wave);
  }
  __device__ __forceinline__ void products(int i, s16x8 p, const s16x8 (&q)[kTilesQ]) {
#pragma unroll
    for (int j = 0; j < kTilesQ; ++j) acc[i][j] = multiply<(kKind == kHalf || kKind == kHalves)>(p, q[j], acc[i][j]);
  }

  // From one barrier to the next: the products that are left of the stage before, and
  // this one's but for the last kTail groups. `to_p`, `to_q` are where the loads go and
  // `p`, `q` what is read, apart from one another, which is said here for the compiler:
  // it otherwise waits for all loads before a transposing read. Left to itself it also
  // puts each read right before its products and waits there; the groups fix the order,
  // with reads two groups ahead or more and none in the last.
  template <bool kFirst>
  __device__ __forceinline__ void step(char* __restrict to_p, char* __restrict to_q, const char* __restrict p,
                                       const char* __restrict q, Held& held, const Place& a, const Next<kSlotsP>& next_p,
                                       const Next<kSlotsQ>& next_q) {
    constexpr int kHolds = kTilesQ + kHeldP, kHoldsPerGroup = (kHolds + kTail - 1) / kTail;
    constexpr int kReads = 2 * kTilesP - kHeldP + kTilesQ, kReadsPerGroup = (kReads + kBody - 3) / (kBody - 2);
    constexpr int kNear = kDeepP ? SideQ::kLoads : SideP::kLoads;       // of the operand with two slots: first
    constexpr int kNearPerGroup = (kNear + kTail - 1) / kTail, kDeepPerGroup = (kDeepLoads + kBody - 1) / kBody;
    const Buffer from_p = a.from(next_p), from_q = a.from(next_q, 0);
    // Unknown anew for each stage, or the compiler keeps every tile's place in a register of
    // its own through the loop, of which there are none left.
    uint32_t at_p = a.at_p, at_q = a.at_q;
    if constexpr (kLayoutP == kSteps) asm volatile("" : "+v"(at_p));
    if constexpr (kLayoutQ == kSteps) asm volatile("" : "+v"(at_q));
    auto load_near = [&](int n) {
      if (n >= kNear) return;
      if constexpr (kDeepP) a.q.load(n, to_q, from_q, a.wave);
      else a.p.load(n, to_p, from_p, a.wave);
    };
    auto load_deep = [&](int n) {
      if (n >= kDeepLoads) return;
      if constexpr (kDeepP) a.p.load(n, to_p, from_p, a.wave);
      else a.q.load(n, to_q, from_q, a.wave);
    };
#pragma unroll
    for (int i = 0; i < kTail; ++i) {
#pragma unroll
      for (int n = i * kNearPerGroup; n < (i + 1) * kNearPerGroup; ++n) load_near(n);
#pragma unroll
      for (int n = i * kHoldsPerGroup; n < (i + 1) * kHoldsPerGroup; ++n) {
        if (n < kTilesQ) held.q[n] = a.read_q(q, at_q, 0, n);
        else if (n < kHolds) held.p[n - kTilesQ] = a.read_p(p, at_p, 0, n - kTilesQ);
      }
      if constexpr (!kFirst) products(kTilesP - kTail + i, held.last_p[i], held.last_q);
      if constexpr (kKind == kHalfQ) {
        // two groups behind the reads; what the tail cannot hold, before the products
#pragma unroll
        for (int n = (i - 2) * kHoldsPerGroup; n < (i == kTail - 1 ? kTilesQ : (i - 1) * kHoldsPerGroup); ++n)
          if (n >= 0 && n < kTilesQ) held.q[n] = half_to_bf16(held.q[n]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    s16x8 at[2][kTilesP];
#pragma unroll
    for (int i = 0; i < kHeldP; ++i) at[0][i] = held.p[i];
#pragma unroll
    for (int i = 0; i < kBody; ++i) {
#pragma unroll
      for (int n = i * kDeepPerGroup; n < (i + 1) * kDeepPerGroup; ++n) load_deep(n);
#pragma unroll
      for (int n = i * kReadsPerGroup; n < (i + 1) * kReadsPerGroup; ++n) {
        if (n < kTilesP - kHeldP) at[0][n + kHeldP] = a.read_p(p, at_p, 0, n + kHeldP);
        else if (n < kTilesP - kHeldP + kTilesQ) held.last_q[n - (kTilesP - kHeldP)] = a.read_q(q, at_q, 1, n - (kTilesP - kHeldP));
        else if (n < kReads) at[1][n - (kTilesP - kHeldP + kTilesQ)] = a.read_p(p, at_p, 1, n - (kTilesP - kHeldP + kTilesQ));
      }
      if constexpr (kKind == kHalfQ) {
        // a part of them before each group of products, none left before their own
        constexpr int kEach = (kTilesQ + kTilesP / 2 - 1) / (kTilesP / 2);
#pragma unroll
        for (int n = (i - (kTilesP - kTilesP / 2)) * kEach; n < (i - (kTilesP - kTilesP / 2) + 1) * kEach; ++n)
          if (i < kTilesP && n >= 0 && n < kTilesQ) held.last_q[n] = half_to_bf16(held.last_q[n]);
      }
      if (i < kTilesP) products(i, at[0][i % kTilesP], held.q);
      else products(i - kTilesP, at[1][i % kTilesP], held.last_q);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < kTail; ++i) held.last_p[i] = at[1][kTilesP - kTail + i];
  }

  // Behind it this stage is everyone's, and the stage before has been read by everyone.
  // kLeft: this wave's loads that may still be on their way.
  template <int kLeft>
  __device__ __forceinline__ static void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // A sum over the steps [k0, k1), whole stages: begin() asks for the first ones, run()
  // forms it in acc. Between the two, `lds` is free from kFree on.
  static constexpr int kFree = (kSlotsP - 1) * SideP::kBytes;   // a slot that begin() leaves
  struct Work {
    Place a;
    int k0, k1;
    bool busy;               // the wave has items of Q; one that has none leaves its share of a SIMD to another
    Next<kSlotsP> next_p;
    Next<kSlotsQ> next_q;
  };
  __device__ __forceinline__ static void begin(Work& w, char* lds, const Operand& p, const Operand& q, int64_t plane_p,
                                               int64_t plane_q, int k0, int k1) {
    w.a.lane = threadIdx.x & 63;
    w.a.wave = uniform(static_cast<int>(threadIdx.x >> 6));
    w.a.p.init(p, w.a.wave, w.a.lane);
    w.a.q.init(q, w.a.wave, w.a.lane);
    w.a.at_p = SideP::lane_at(w.a.wave % kWavesP * kWaveP, w.a.lane & 15, w.a.lane >> 4);
    w.a.at_q = SideQ::lane_at(w.a.wave / kWavesP * kWaveQ, w.a.lane & 15, w.a.lane >> 4);
    w.a.plane_p = plane_p;
    w.a.plane_q = plane_q;
    w.k0 = k0;
    w.k1 = k1;
    w.busy = w.a.wave / kWavesP * kWaveQ < uniform(q.items);
    w.next_p = {k0, 0, 0};
    w.next_q = {k0, 0, 0};
    auto all_p = [&] {
      w.a.p.turn(w.next_p.k, w.a.wave, w.a.lane);
      const Buffer from = w.a.from(w.next_p);
#pragma unroll
      for (int n = 0; n < SideP::kLoads; ++n) bring_p(n, lds, w.a, from, w.next_p);
      w.next_p.advance(k0, k1);
    };
    auto all_q = [&] {
      w.a.q.turn(w.next_q.k, w.a.wave, w.a.lane);
      const Buffer from = w.a.from(w.next_q, 0);
#pragma unroll
      for (int n = 0; n < SideQ::kLoads; ++n) bring_q(n, lds, w.a, from, w.next_q);
      w.next_q.advance(k0, k1);
    };
    if constexpr (kLead > 0) {
#pragma unroll
      for (int s = 0; s < kLead; ++s) all_p(), all_q();
    } else {
      all_p();
      all_q();
      kDeepP ? all_p() : all_q();
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kTilesP; ++i)
#pragma unroll
      for (int j = 0; j < kTilesQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The workgroup may use `lds` again once all of its waves have come back. A wave that is
  // not busy has no sums.
  __device__ __forceinline__ void run(Work& w, char* lds) {
    const int stages = (w.k1 - w.k0) / kStep * kParts;
    int slot_p = 0, slot_q = 0;
    Held held;
    auto next = [&] {
      w.next_p.advance(w.k0, w.k1);
      w.next_q.advance(w.k0, w.k1);
      slot_p = slot_p == kSlotsP - 1 ? 0 : slot_p + 1;
      slot_q = slot_q == kSlotsQ - 1 ? 0 : slot_q + 1;
    };
    auto turn = [&] {
      w.a.p.turn(w.next_p.k, w.a.wave, w.a.lane);
      w.a.q.turn(w.next_q.k, w.a.wave, w.a.lane);
    };
    auto one = [&](auto first) {
      turn();
      arrive<kBehind>();
      step<decltype(first)::value>(lds + w.next_p.slot * SideP::kBytes, lds + kPlaceQ + w.next_q.slot * SideQ::kBytes,
                                   lds + slot_p * SideP::kBytes, lds + kPlaceQ + slot_q * SideQ::kBytes, held, w.a, w.next_p,
                                   w.next_q);
      next();
    };
    if (w.busy) {
      clear();
      one(std::true_type());
      for (int s = 1; s < stages; ++s) one(std::false_type());
    } else {
      for (int s = 0; s < stages; ++s) {   // the same loads in the same order, and the same barriers
        turn();
        arrive<kBehind>();
        const Buffer from_p = w.a.from(w.next_p), from_q = w.a.from(w.next_q, 0);
        auto all_p = [&] {
#pragma unroll
          for (int n = 0; n < SideP::kLoads; ++n) bring_p(n, lds, w.a, from_p, w.next_p);
        };
        auto all_q = [&] {
#pragma unroll
          for (int n = 0; n < SideQ::kLoads; ++n) bring_q(n, lds, w.a, from_q, w.next_q);
        };
        if constexpr (kDeepP) all_q(), all_p();
        else all_p(), all_q();
        next();
      }
    }
    // by idle waves too, of nothing: in one block with what follows, which runs under them
#pragma unroll
    for (int i = 0; i < kTail; ++i) products(kTilesP - kTail + i, held.last_p[i], held.last_q);
    // the loads that were brought for no product, and everyone's reads
    arrive<0>();
  }
};

// Eight fp32 numbers as three bf16 each that add up to them: cut off, not rounded, so that
// the largest do not overflow.
__device__ __forceinline__ void thirds(const float (&x)[8], s16x8 (&part)[3]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x[e]) & 0xffff0000u), rest = x[e] - hi;
    const float mid = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, rest) & 0xffff0000u), lo = rest - mid;
    part[0][e] = static_cast<short>(__builtin_bit_cast(uint32_t, hi) >> 16);
    part[1][e] = static_cast<short>(__builtin_bit_cast(uint32_t, mid) >> 16);
    part[2][e] = static_cast<short>(__builtin_bit_cast(uint32_t, lo) >> 16);
  }
}

// The same for few q, where P is large, fp32, and read once: it is made three bf16 arrays
// on its way from LDS to the products, not in memory before. Q is three bf16 arrays in
// memory, by rows, `plane` bytes apart. Each wave has all of the tile's q.
constexpr int kFewStep = 32;
template <Layout kLayoutP, int kP, int kQ, int kWaves, bool kSpread, int kSlots = 3>
struct FewTile {
  static constexpr int kSteps = kFewStep, kItemsQ = kQ, kAcross = kWaves;
  static constexpr int kWaveP = kP / kWaves, kWaveQ = kQ, kTilesP = kWaveP / 16, kTilesQ = kQ / 16;
  static_assert(!kSpread || kWaveP % 32 == 0);
  using SideP = Side<kLayoutP, kP, kWaves, kSpread, kSteps, 4>;
  using SideQ = Side<kRows, kQ, kWaves, false, kSteps, 2>;
  static constexpr int kSlotBytes = SideP::kBytes + 3 * SideQ::kBytes, kLdsBytes = kSlots * kSlotBytes;
  static constexpr int kLoads = SideP::kLoads + 3 * SideQ::kLoads;
  static constexpr int kFree = (kSlots - 1) * kSlotBytes;

  f32x4 acc[kTilesP][kTilesQ];

  struct Work {
    SideP p;
    SideQ q;
    int64_t plane_q;
    int k0, k1, wave, lane;
  };
  __device__ __forceinline__ static void load(Work& w, char* to, int stage) {
    const int k = min(w.k0 + stage * kSteps, w.k1 - kSteps);   // past the last stage that one again
    w.p.turn(k, w.wave, w.lane);
    const Buffer from = w.p.stage(0, k);
#pragma unroll
    for (int n = 0; n < SideP::kLoads; ++n) w.p.load(n, to, from, w.wave);
#pragma unroll
    for (int plane = 0; plane < 3; ++plane) {
      const Buffer of = w.q.stage(plane * w.plane_q, k);
#pragma unroll
      for (int n = 0; n < SideQ::kLoads; ++n) w.q.load(n, to + SideP::kBytes + plane * SideQ::kBytes, of, w.wave);
    }
  }
  __device__ __forceinline__ static void begin(Work& w, char* lds, const Operand& p, const Operand& q, int64_t, int64_t plane_q,
                                               int k0, int k1) {
    w.lane = threadIdx.x & 63;
    w.wave = uniform(static_cast<int>(threadIdx.x >> 6));
    w.p.init(p, w.wave, w.lane);
    w.q.init(q, w.wave, w.lane);
    w.plane_q = plane_q;
    w.k0 = k0;
    w.k1 = k1;
#pragma unroll
    for (int s = 0; s < kSlots - 1; ++s) load(w, lds + s * kSlotBytes, s);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kTilesP; ++i)
#pragma unroll
      for (int j = 0; j < kTilesQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void step(char* __restrict to, const char* __restrict from, Work& w, int stage) {
    const int m = w.lane & 15, g = w.lane >> 4;
    load(w, to, stage);
    s16x8 q[kTilesQ][3];
#pragma unroll
    for (int j = 0; j < kTilesQ; ++j)
#pragma unroll
      for (int plane = 0; plane < 3; ++plane) q[j][plane] = w.q.read(from + SideP::kBytes + plane * SideQ::kBytes, 0, 0, 0, j, m, g);
#pragma unroll
    for (int i = 0; i < kTilesP; ++i) {
      float v[8];
      w.p.read(from, w.wave * kWaveP, i, m, g, v);
      s16x8 p[3];
      thirds(v, p);
#pragma unroll
      for (int part = 0; part < kThirdsParts; ++part)
#pragma unroll
        for (int j = 0; j < kTilesQ; ++j) acc[i][j] = multiply<false>(p[third_p(part)], q[j][third_q(part)], acc[i][j]);
    }
  }
  __device__ __forceinline__ void run(Work& w, char* lds) {
    clear();
    const int stages = (w.k1 - w.k0) / kSteps;
    int now = 0, free = kSlots - 1;
    for (int s = 0; s < stages; ++s) {
      // this wave's loads of stage s are here, and behind the barrier everyone's; and
      // everyone has read the stage that is overwritten next
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kSlots - 2) * kLoads) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      step(lds + free * kSlotBytes, lds + now * kSlotBytes, w, s + kSlots - 1);
      now = now == kSlots - 1 ? 0 : now + 1;
      free = free == kSlots - 1 ? 0 : free + 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

}  // namespace rwkv_tile
