// Log probability of a given token, entropy and most likely alternatives of
// rows of logits, and their gradient (include/rwkv_token_scores.h).
//
// With M = max_j x_j and d_j = (x_j - M) log2(e): s = sum 2^d_j, u = sum 2^d_j d_j.
// Then log p_j = x_j - M - ln s and the entropy is ln s - ln 2 u / s.
//
// Forward: a workgroup loads a row (or a chunk of a long one) into registers
// once, eight logits a piece, all loads in flight together, and everything else
// works on those: the maximum, the sums, and the alternatives. These are found
// through a bound: each of 64 groups of pieces (128 for more than 32 alternatives)
// has a largest logit, and the k-th largest of those is no larger than the k-th
// largest logit, so what reaches it goes to a list in LDS, whose items are then
// ranked against each other. Where large logits do not crowd into few groups that
// is a few more than k (of 64 groups for k = 20 about 24, for 32 44; of 128 for 64
// 89; of 64 they would be some 300). A list that overflows is replaced by k rounds
// of taking the largest that is left.
//
// us and what bounds it: 4096 x 65536 bf16 without alternatives 92 (5.8 TB/s, HBM),
// with 20 117, with 64 142 (vector instructions, some 13 for a logit, and the
// waits between the steps of the selection); with one of eight rows masked 119
// and 142. 1024 x 65536 fp32 with 20 47 (5.7 TB/s). Backward of 4096 x 65536 bf16
// 214 (5.0 TB/s, HBM).
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "token_scores_launch.hpp"

namespace rwkv_scores {
namespace {

constexpr int kPiece = 8;    // logits of a load (bf16: 16 bytes) or of two (fp32)
constexpr int kTopStep = 32;  // alternatives: up to two steps of these, for each of which there are 64 groups
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// 2^kFloor is 0: what lies below adds nothing, and 0 times it is 0
constexpr float kFloor = -256.f;

// Rows of a vocabulary that is no multiple of a piece begin anywhere; the
// hardware takes such addresses in one access.
struct __attribute__((packed, aligned(2))) Raw16 {
  uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) Raw32 {
  float v[8];
};
// The largest of three; fmaxf would have each operand's NaN made quiet first, an
// instruction for each logit.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

template <bool BF>
struct Piece;   // as loaded
template <>
struct alignas(16) Piece<true> {
  Raw16 raw;
  __device__ __forceinline__ float operator[](int e) const {
    const uint32_t w = raw.w[e >> 1];
    return __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ float largest() const {
    const Piece& p = *this;
    return max3(max3(p[0], p[1], p[2]), max3(p[3], p[4], p[5]), max3(p[6], p[7], p[7]));
  }
  __device__ __forceinline__ void clear() { raw = Raw16{{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}}; }
  // The values are taken out of the words again from here on, so that a pass
  // over the row does not hold every value of the pass before in a register.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(raw.w[i]));
  }
};
template <>
struct alignas(16) Piece<false> {
  Raw32 raw;
  __device__ __forceinline__ float operator[](int e) const { return raw.v[e]; }
  __device__ __forceinline__ float largest() const {
    const Piece& p = *this;
    return max3(max3(p[0], p[1], p[2]), max3(p[3], p[4], p[5]), max3(p[6], p[7], p[7]));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < 8; ++e) raw.v[e] = -INFINITY;
  }
  __device__ __forceinline__ void forget() {}
};

template <bool BF>
__host__ __device__ __forceinline__ const char* at(const void* base, int64_t i) {
  return static_cast<const char*>(base) + i * (BF ? 2 : 4);
}
template <bool BF>
__device__ __forceinline__ float load_one(const void* base, int64_t i) {
  if constexpr (BF) return __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(base)[i]) << 16);
  else return static_cast<const float*>(base)[i];
}
template <bool BF>
__device__ __forceinline__ void store_one(void* base, int64_t i, float v) {
  if constexpr (BF) static_cast<__bf16*>(base)[i] = static_cast<__bf16>(v);
  else static_cast<float*>(base)[i] = v;
}
template <bool BF>
__device__ __forceinline__ Piece<BF> load_piece(const char* chunk, uint32_t q) {
  Piece<BF> p;
  __builtin_memcpy(&p.raw, chunk + q * static_cast<uint32_t>(sizeof(p.raw)), sizeof(p.raw));
  return p;
}

// A logit with its index (or a piece's largest with the piece's number) as one
// number: of two, the larger logit is larger, then the lower index. Zeros of
// both signs are equal. No key is 0.
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, int j) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  const uint32_t o = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  return static_cast<Key>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(j));
}
__device__ __forceinline__ float key_x(Key k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int key_j(Key k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ Key larger(Key a, Key b) { return a > b ? a : b; }

// The value of another lane: xor 1 and xor 2 of four, then mirrors of 8 and 16
// lanes, which join what four and eight lanes already share.
template <int kStep>
__device__ __forceinline__ int swapped(int v) {
  constexpr int ctrl = kStep == 1 ? 0xb1 : kStep == 2 ? 0x4e : kStep == 4 ? 0x141 : 0x140;
  return __builtin_amdgcn_update_dpp(v, v, ctrl, 0xf, 0xf, false);
}
template <int kLanes>
__device__ __forceinline__ int sum_of(int v) {
  if constexpr (kLanes > 1) v += swapped<1>(v);
  if constexpr (kLanes > 2) v += swapped<2>(v);
  if constexpr (kLanes > 4) v += swapped<4>(v);
  if constexpr (kLanes > 8) v += swapped<8>(v);
  return v;
}
template <int kStep>
__device__ __forceinline__ Key swapped(Key k) {
  const uint32_t hi = swapped<kStep>(static_cast<int>(k >> 32)), lo = swapped<kStep>(static_cast<int>(k));
  return static_cast<Key>(hi) << 32 | lo;
}
template <int kLanes>
__device__ __forceinline__ Key largest_of(Key k) {
  if constexpr (kLanes > 1) k = larger(k, swapped<1>(k));
  if constexpr (kLanes > 2) k = larger(k, swapped<2>(k));
  if constexpr (kLanes > 4) k = larger(k, swapped<4>(k));
  if constexpr (kLanes > 8) k = larger(k, swapped<8>(k));
  return k;
}
// Of all lanes, in every lane: the row's shifts, then its last lane to the rows
// behind; lane 63 has it all.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float shifted(float v, float none) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                                              kCtrl, kRowMask, 0xf, false));
}
template <typename F>
__device__ __forceinline__ float wave_join(float v, float none, F f) {
  v = f(v, shifted<0x111, 0xf>(v, none));
  v = f(v, shifted<0x112, 0xf>(v, none));
  v = f(v, shifted<0x114, 0xf>(v, none));
  v = f(v, shifted<0x118, 0xf>(v, none));
  v = f(v, shifted<0x142, 0xa>(v, none));
  v = f(v, shifted<0x143, 0xc>(v, none));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_join(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_join(v, 0.f, [](float a, float b) { return a + b; });
}

// Pieces and candidates that the lists hold; a chunk that has more goes the
// other way. A row that a mask leaves fewer than k tokens has up to k pieces of
// minus infinity in them.
template <bool BF, int kWaves, int kTop>
struct Shared {
  static constexpr int kGroups = 64 * kTop, kMost = kTopStep * kTop;
  static constexpr int kPieces = 128 * kTop, kListed = 512 * kTop;
  Piece<BF> piece[kPieces];
  int piece_at[kPieces];
  Key key[kWaves][65];
  Key group[kGroups];
  Key list[kListed];
  Key best[2][kMost];        // the alternatives so far, in order
  Key bound;
  float max;
  int pieces, listed;
};
constexpr int kRanked = 128;   // more than these are cut to the most before they are ranked

// The largest of every thread's keys (`mine`; a group is a lane of kWaves / kTop
// waves) and the k-th largest of the groups' largest, into sh.max and sh.bound.
// Every group's largest is another item, so the bound is one of them. Where it is
// minus infinity (a mask has left fewer than k groups anything), the whole pieces
// of it count as the eight logits that they are: few of them are needed.
template <bool BF, int kWaves, int kTop>
__device__ __forceinline__ void find_bound(Shared<BF, kWaves, kTop>& sh, Key mine, int k, int Q) {
  static_assert(kWaves % kTop == 0 && kTop <= 2, "a thread's key is in one group");
  constexpr int kShare = kWaves / kTop, kCompared = 64 * kTop / kShare;
  const int tid = threadIdx.x, group = tid / kShare, sub = tid % kShare;
  Key key = mine;
  if constexpr (kShare > 1) {
    sh.key[tid >> 6][tid & 63] = mine;
    __syncthreads();
    key = largest_of<kShare>(sh.key[group / 64 * kShare + sub][group & 63]);
  }
  if (sub == 0) sh.group[group] = key;
  __syncthreads();
  int rank = 0;
#pragma unroll 16
  for (int i = 0; i < kCompared; ++i) rank += sh.group[sub * kCompared + i] > key;
  rank = sum_of<kShare>(rank);
  if (sub == 0) {
    if (rank == 0) sh.max = key_x(key);
    if (rank == k - 1) sh.bound = key;
  }
  if (tid == 0) sh.pieces = sh.listed = 0;
  __syncthreads();
  constexpr Key kSome = Key{0x00800000u} << 32;   // the least key of more than minus infinity
  const Key bound = sh.bound;
  if (bound >= kSome) return;
  int some = 0;
#pragma unroll 16
  for (int i = 0; i < kCompared; ++i) some += sh.group[sub * kCompared + i] >= kSome;
  some = sum_of<kShare>(some);
  __syncthreads();   // every thread has the bound that is replaced
  if (sub == 0 && rank == some + (k - some + kPiece - 1) / kPiece - 1 && key_j(key) < Q) sh.bound = key;
  __syncthreads();
}

// The list's n keys, more than k of them, cut to their k largest by the first
// wave: a key that k keys reach (they are all different, so there is one) is
// looked for among those that still can be it. Ranking n keys against each other
// is n^2 comparisons, this n for each of the about 2 ln n keys tried. (By halving
// the distance between the numbers, 54 steps where minus infinities differ in
// their index alone, a masked row took 9 us.)
template <bool BF, int kWaves, int kTop>
__device__ __forceinline__ void cut_list(Shared<BF, kWaves, kTop>& sh, int n, int k) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    auto each = [&](auto f) {   // of four keys a lane at a time, 0 for none
#pragma nounroll
      for (int j = lane; j - lane < n; j += 256) {
        Key v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = j + 64 * i < n ? sh.list[j + 64 * i] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) f(v[i]);
      }
    };
    Key low = 0, high = ~Key{0}, tried = sh.list[n / 2];
    while (true) {
      int count = 0;
      Key above = 0, below = 0;   // one of the lane's that can be it, on either side
      each([&](Key v) {
        count += __popcll(__ballot(v >= tried));
        if (v > tried && v < high) above = v;
        if (v < tried && v > low) below = v;
      });
      if (count == k) break;
      (count > k ? low : high) = tried;
      const Key next = count > k ? above : below;
      const unsigned long long have = __ballot(next != 0);
      if (have == 0) break;
      const int from = __ffsll(have) - 1;
      tried = static_cast<Key>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(next >> 32), from))) << 32 |
              static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(next), from));
    }
    int to = 0;   // a key's place is never behind its own
    each([&](Key v) {
      const unsigned long long hit = __ballot(v >= tried);
      const int place = to + __popcll(hit & ((1ull << lane) - 1));
      if (v >= tried && place < k) sh.list[place] = v;
      to += __popcll(hit);
    });
  }
  __syncthreads();
}

// How many of n keys a sixteenth of the lanes' share counts above `mine`: four
// reads at a time, so that a long list is not a chain of waits.
__device__ __forceinline__ int count_above(const Key* keys, int n, Key mine) {
  int count = 0;
#pragma nounroll
  for (int j = threadIdx.x & 15; j < n; j += 64) {
    Key k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = keys[min(j + 16 * i, n - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) count += j + 16 * i < n && k[i] > mine;
  }
  return count;
}

// Ranks the list's n keys together with the `held` best so far, and gives those
// before the k-th to keep(rank, key). Sixteen lanes count for a key.
template <bool BF, int kWaves, int kTop, typename F>
__device__ __forceinline__ void rank_keys(const Shared<BF, kWaves, kTop>& sh, int n, const Key* best, int held, int k, F&& keep) {
  const int sub = threadIdx.x & 15;
#pragma nounroll
  for (int i = threadIdx.x >> 4; i < n + held; i += kWaves * 4) {
    const Key mine = i < n ? sh.list[i] : best[i - n];
    int rank = count_above(sh.list, n, mine) + count_above(best, held, mine);
    rank = sum_of<16>(rank);
    if (sub == 0 && rank < k) keep(rank, mine);
  }
}

// The list by another way: sh.list becomes the k largest of what next(last)
// gives, each thread's largest key below `last`. Ends with a barrier.
template <bool BF, int kWaves, int kTop, typename F>
__device__ __forceinline__ void take_largest(Shared<BF, kWaves, kTop>& sh, int k, F&& next) {
  Key last = ~Key{0};
  __syncthreads();
#pragma nounroll
  for (int i = 0; i < k; ++i) {
    Key v = next(last);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = larger(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) sh.group[threadIdx.x >> 6] = v;
    __syncthreads();
    last = sh.group[0];
#pragma nounroll
    for (int w = 1; w < kWaves; ++w) last = larger(last, sh.group[w]);
    if (threadIdx.x == 0) sh.list[i] = last;
    __syncthreads();
  }
}

// Where d is measured from. For maxima of ordinary size d = x log2(e) - rounded(m
// log2(e)), one operation, in which the largest logit has d = off instead of 0;
// beyond kFar that would leave fp32's range, and d is (x - m) log2(e).
constexpr float kFar = 1048576.f;
struct Origin {
  float m, shift, off;   // shift: rounded m log2(e), or 0 beyond kFar
  __device__ __forceinline__ bool far() const { return !(fabsf(m) < kFar); }
};
__device__ __forceinline__ Origin origin(float m) {
  Origin o{m, 0.f, 0.f};
  if (!o.far()) {
    o.shift = m * kLog2E;
    o.off = fmaf(m, kLog2E, -o.shift);
  }
  return o;
}

// What the row's outputs are formed from.
struct Sums {
  Origin o;
  float s, u;
  __device__ __forceinline__ bool valid() const { return fabsf(o.m) < INFINITY && s == s; }
  // Neither the log of a sum that holds 1 nor an entropy is negative; what the
  // exponential and the logarithm round (about 2^-24) may be.
  __device__ __forceinline__ float log_sum() const { return fmaxf(logf(s) - kLn2 * o.off, 0.f); }
  __device__ __forceinline__ float entropy() const { return valid() ? fmaxf(logf(s) - kLn2 * (u / s), 0.f) : NAN; }
  __device__ __forceinline__ float log_p(float x, float log_sum) const { return valid() ? (x - o.m) - log_sum : NAN; }
};
// terms measured from `from`, from then on from `to`, whose m is no smaller
__device__ __forceinline__ void rescale(float& s, float& u, const Origin& from, const Origin& to) {
  if (from.m == to.m || from.m == -INFINITY) return;   // nothing changes, or nothing was added yet
  const float d = fmaxf(fmaf(from.m - to.m, kLog2E, to.off - from.off), kFloor), f = __builtin_amdgcn_exp2f(d);
  u = f * fmaf(d, s, u);
  s *= f;
}

template <bool BF>
__device__ __forceinline__ void write_row(const ForwardCall& c, int64_t row, const Sums& t, float log_sum) {
  const int64_t token = c.tokens[row];
  c.log_prob[row] = token >= 0 && token < c.vocab ? t.log_p(load_one<BF>(c.logits, row * c.vocab + token), log_sum) : NAN;
  c.entropy[row] = t.entropy();
  if (c.row_max) c.row_max[row] = t.o.m;
  if (c.log_sum) c.log_sum[row] = t.valid() ? log_sum : NAN;
}
__device__ __forceinline__ void write_top(const ForwardCall& c, int64_t row, int rank, Key v, const Sums& t, float log_sum) {
  c.top_log_probs[row * c.top + rank] = t.log_p(key_x(v), log_sum);
  c.top_ids[row * c.top + rank] = t.valid() ? key_j(v) : -1;
}

// The largest key below `last` of a thread's pieces of a chunk, which are read again.
template <bool BF, int kThreads>
__device__ __forceinline__ Key next_of(const void* row, int q0, int pieces, Key last) {
  Key v = 0;
#pragma unroll 2
  for (int q = threadIdx.x; q < pieces; q += kThreads) {
    const Piece<BF> p = load_piece<BF>(at<BF>(row, static_cast<int64_t>(q0) * kPiece), q);
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
      const Key y = key_of(p[e], (q0 + q) * kPiece + e);
      if (y < last) v = larger(v, y);
    }
  }
  return v;
}

// The row is Q pieces and, after them, up to seven single logits, one to a
// thread, which are numbered like pieces (Q, Q + 1, ..). A chunk is kPieces of
// them a thread.
// kTop: steps of alternatives, 0 for none.
template <bool BF, int kWaves, int kPieces, int kTop>
__global__ __launch_bounds__(kWaves * 64, 4) void forward_kernel(const ForwardCall c) {
  constexpr int kThreads = kWaves * 64, kChunk = kThreads * kPieces;
  typedef Shared<BF, kWaves, kTop> Lists;
  __shared__ std::conditional_t<kTop != 0, Lists, int> sh;
  __shared__ float part_max[kWaves], part_s[kWaves], part_u[kWaves];
  const int64_t row = blockIdx.x, V = c.vocab;
  const void* const x = at<BF>(c.logits, row * V);
  const int tid = threadIdx.x, wave = tid >> 6, k = c.top;
  const int Q = static_cast<int>(V / kPiece), rest = static_cast<int>(V % kPiece);
  Origin o = origin(-INFINITY);
  float s = 0.f, u = 0.f;
  int held = 0, now = 0;   // the alternatives so far: sh.best[now][0 .. held)
  for (int q0 = 0;; q0 += kChunk) {
    const bool final = Q - q0 <= kChunk;
    const int left = final ? Q - q0 : kChunk;   // pieces of this chunk
    int lane = tid;   // known anew in each chunk: its addresses are not kept from one to the next
    asm volatile("" : "+v"(lane));
    const char* const chunk = at<BF>(x, static_cast<int64_t>(q0) * kPiece);
    Piece<BF> p[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (i * kThreads + lane < left) p[i] = load_piece<BF>(chunk, i * kThreads + lane);
      else p[i].clear();
    }
    const bool has_single = final && lane < rest;
    const float single = has_single ? load_one<BF>(x, static_cast<int64_t>(Q) * kPiece + lane) : -INFINITY;
    // the thread's largest logit, with the first piece that holds it
    float piece_max[kPieces], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      piece_max[i] = p[i].largest();
      most = fmaxf(most, piece_max[i]);
    }
    int most_at = 0;
#pragma unroll
    for (int i = kPieces - 1; i > 0; --i) most_at = piece_max[i] == most ? i * kThreads : most_at;
    if (piece_max[0] == most) most_at = 0;
    most_at += q0 + lane;
    if (lane >= left) most_at += kPiece;   // a thread without a piece comes behind all that there is
    if (has_single && (lane >= left || single > most)) {
      most = single;
      most_at = Q + lane;
    }
    float chunk_max, bound_x = 0.f;
    int bound_q = 0;
    if constexpr (kTop != 0) {
      find_bound(sh, key_of(most, most_at), k, Q);
      chunk_max = sh.max;
      bound_x = key_x(sh.bound);
      bound_q = key_j(sh.bound);
      // the pieces that may hold an alternative; few of a wave's do
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (piece_max[i] >= bound_x) {
          const int q = q0 + i * kThreads + lane;
          if ((piece_max[i] > bound_x || q <= bound_q) && i * kThreads + lane < left) {
            const int n = atomicAdd(&sh.pieces, 1);
            if (n < Lists::kPieces) {
              sh.piece[n] = p[i];
              sh.piece_at[n] = q;
            }
          }
        }
    } else {
      const float v = wave_max(most);
      if ((tid & 63) == 0) part_max[wave] = v;
      __syncthreads();
      chunk_max = part_max[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) chunk_max = fmaxf(chunk_max, part_max[w]);
    }
    const Origin before = o;
    o = origin(fmaxf(o.m, chunk_max));
    rescale(s, u, before, o);
    auto add = [&](float d) {
      const float t = __builtin_amdgcn_exp2f(d);
      s += t;
      u = fmaf(t, fmaxf(d, kFloor), u);
    };
    auto add_all = [&](auto distance) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        if (i * kThreads >= left) break;
        p[i].forget();
#pragma unroll
        for (int e = 0; e < kPiece; ++e) add(distance(p[i][e]));
      }
      add(distance(single));
    };
    if (!o.far()) {
      add_all([&](float v) { return fmaf(v, kLog2E, -o.shift); });
    } else {
      const float base = o.m == -INFINITY ? 0.f : o.m;   // nothing but minus infinity so far: the terms are 0
      add_all([&](float v) { return (v - base) * kLog2E; });
    }
    if constexpr (kTop != 0) {
      __syncthreads();
      const int pieces = min(sh.pieces, Lists::kPieces);
      auto list = [&](float v, int q, int j) {
        if (v > bound_x || (v == bound_x && q <= bound_q)) {
          const int n = atomicAdd(&sh.listed, 1);
          if (n < Lists::kListed) sh.list[n] = key_of(v, j);
        }
      };
#pragma nounroll
      for (int e = tid; e < pieces * kPiece; e += kThreads) {
        const int q = sh.piece_at[e / kPiece];
        list(load_one<BF>(sh.piece, e), q, q * kPiece + e % kPiece);
      }
      if (has_single) list(single, Q + lane, Q * kPiece + lane);
      __syncthreads();
      int n = sh.listed;
      if (n > Lists::kListed || sh.pieces > Lists::kPieces) {
        const int singles = final ? rest : 0;
        n = static_cast<int>(min(static_cast<int64_t>(k), static_cast<int64_t>(left) * kPiece + singles));
        take_largest(sh, n, [&](Key last) {
          const Key v = next_of<BF, kThreads>(x, q0, left, last);
          const Key y = has_single ? key_of(single, Q * kPiece + lane) : 0;
          return y < last ? larger(v, y) : v;
        });
      }
      if (n > kRanked) {
        cut_list(sh, n, k);
        n = k;
      }
      rank_keys(sh, n, sh.best[now], held, k, [&](int rank, Key v) { sh.best[now ^ 1][rank] = v; });
      held = min(k, held + n);
      now ^= 1;
    }
    if (final) break;
    __syncthreads();
  }
  s = wave_sum(s);
  u = wave_sum(u);
  if ((tid & 63) == 0) {
    part_s[wave] = s;
    part_u[wave] = u;
  }
  __syncthreads();
  Sums t{o, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    t.s += part_s[w];
    t.u += part_u[w];
  }
  const float log_sum = t.log_sum();
  if (tid == 0) write_row<BF>(c, row, t, log_sum);
  if constexpr (kTop != 0)
    if (tid < k) write_top(c, row, tid, sh.best[now][tid], t, log_sum);
}

// ------------------------------------------------------------------ backward
// The gradient of a logit, but for the terms of the token and the alternatives:
// -p (slope d + rest), d = log2 p, with a NaN rest in a row without a distribution.
struct RowGrad {
  float m, log2_sum, slope, rest;
  __device__ __forceinline__ float of(float x) const {
    const float d = fmaxf(fmaf(x - m, kLog2E, -log2_sum), kFloor);
    return -__builtin_amdgcn_exp2f(d) * fmaf(slope, d, rest);
  }
};

template <bool BF>
__device__ __forceinline__ void store_piece(void* row, int64_t q, const float (&v)[kPiece]) {
  char* const to = static_cast<char*>(row) + q * kPiece * (BF ? 2 : 4);
  if constexpr (BF) {
    Raw16 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w.w[e] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<__bf16>(v[2 * e]))) |
               static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<__bf16>(v[2 * e + 1]))) << 16;
    __builtin_memcpy(to, &w, sizeof(w));
  } else {
    __builtin_memcpy(to, v, sizeof(v));
  }
}

// The last rows first: the forward has read them last, and what of them is still
// in the cache need not come from memory (us, forward and backward, 8192 x 65536
// bf16 611 / 596, 1024 x 65536 fp32 173 / 168).
// Blocks (row, y) take `share` pieces of a row each, the last one its single
// logits too. The elements with a term of their own are written again, whole, by
// the block that holds them.
constexpr int kThreads = 256;

template <bool BF>
__global__ __launch_bounds__(kThreads) void backward_kernel(const BackwardCall c, const int64_t share) {
  const int64_t row = c.rows - 1 - blockIdx.x, V = c.vocab, Q = V / kPiece;
  const int64_t begin = blockIdx.y * share, end = min(begin + share, Q);
  const void* const x = at<BF>(c.logits, row * V);
  void* const dx = const_cast<char*>(at<BF>(c.logits_grad, row * V));
  const int tid = threadIdx.x, lane = tid & 63;
  const float g = c.log_prob_grad ? c.log_prob_grad[row] : 0.f, h = c.entropy_grad ? c.entropy_grad[row] : 0.f;
  const float own = lane < c.top ? c.top_grad[row * c.top + lane] : 0.f;   // alternative `lane`'s
  const float log_sum = c.log_sum[row];
  RowGrad r;
  r.m = c.row_max[row];
  r.log2_sum = log_sum * kLog2E;
  r.slope = h * kLn2;
  r.rest = log_sum == log_sum ? fmaf(h, c.entropy[row], g + wave_sum(own)) : NAN;
  for (int64_t q = begin + tid; q < end; q += kThreads) {
    const Piece<BF> p = load_piece<BF>(at<BF>(x, q * kPiece), 0);
    float v[kPiece];
#pragma unroll
    for (int e = 0; e < kPiece; ++e) v[e] = r.of(p[e]);
    store_piece<BF>(dx, q, v);
  }
  const int64_t from = begin * kPiece, to = blockIdx.y + 1 == gridDim.y ? V : end * kPiece;
  if (blockIdx.y + 1 == gridDim.y && Q * kPiece + tid < V)
    store_one<BF>(dx, Q * kPiece + tid, r.of(load_one<BF>(x, Q * kPiece + tid)));
  __syncthreads();
  if (tid >= 64) return;
  const int64_t t = c.tokens[row], j = lane < c.top ? c.top_ids[row * c.top + lane] : -1;
  if (j >= from && j < to) store_one<BF>(dx, j, r.of(load_one<BF>(x, j)) + own + (j == t ? g : 0.f));
  if (!__any(j == t) && lane == 0 && t >= from && t < to) store_one<BF>(dx, t, r.of(load_one<BF>(x, t)) + g);
}

template <bool BF, int kTop, int kWaves, int kPieces>
void forward(const ForwardCall& c, hipStream_t s) {
  hipLaunchKernelGGL((forward_kernel<BF, kWaves, kPieces, kTop>), dim3(static_cast<unsigned>(c.rows)), dim3(kWaves * 64),
                     0, s, c);
}

// The smallest workgroup whose registers hold a row, up to 128 of a thread's: what
// the selection costs does not grow with the pieces a thread holds. us, bf16, 20
// alternatives (waves, pieces a thread): 8192 x 4096 (2, 4) 25, (4, 2) 31, (1, 8)
// 28; 8192 x 8192 (4, 4) 37, (2, 8) 40, (4, 8) 45; 2048 x 32768 (4, 16) 30, (8, 8)
// 36, (8, 16) 42. Longer bf16 rows: 4096 x 65536 (4, 16), two chunks in smaller
// workgroups that wait for each other less, 117, (8, 16) 121, (8, 8) 147, (16, 8)
// 171; with 64 alternatives, whose second list is longer, (4, 16) 160, (8, 16) 142;
// without any there is little to wait for, (4, 16) 95.9, (8, 16) 91.8, and with few
// rows the row's own time counts, 8 x 65536 (8, 16) 9.3, (4, 16) 15. fp32 pieces
// are twice the registers: 1024 x 65536 (8, 8) 47, (16, 8) 58; 256 x 65529 (16, 8)
// 17.4, (8, 8) 20.6.
constexpr int64_t kManyRows = 512, kOwnTimeRows = 256;
template <bool BF, int kTop>
hipError_t forward(const ForwardCall& c, hipStream_t s) {
  auto holds = [&](int waves, int pieces) { return c.vocab <= waves * 64 * pieces * kPiece; };
  if constexpr (kTop <= 1) {   // a wave is 64 groups
    if (holds(1, 1)) forward<BF, kTop, 1, 1>(c, s);
    else if (holds(1, 2)) forward<BF, kTop, 1, 2>(c, s);
    else if (holds(1, 4)) forward<BF, kTop, 1, 4>(c, s);
  } else {
    if (holds(2, 1)) forward<BF, kTop, 2, 1>(c, s);
  }
  if (holds(kTop <= 1 ? 1 : 2, kTop <= 1 ? 4 : 1)) return hipGetLastError();
  if (holds(2, 4)) forward<BF, kTop, 2, 4>(c, s);
  else if (holds(4, 4)) forward<BF, kTop, 4, 4>(c, s);
  else if (holds(4, 8)) forward<BF, kTop, 4, 8>(c, s);
  else if constexpr (BF) {
    if (holds(4, 16) || (kTop == 1 && c.rows > kManyRows)) forward<BF, kTop, 4, 16>(c, s);
    else forward<BF, kTop, 8, 16>(c, s);
  } else {
    if (c.rows <= kOwnTimeRows) forward<BF, kTop, 16, 8>(c, s);
    else forward<BF, kTop, 8, 8>(c, s);
  }
  return hipGetLastError();
}

template <bool BF>
hipError_t forward(const ForwardCall& c, hipStream_t s) {
  if (c.top == 0) return forward<BF, 0>(c, s);
  return c.top <= kTopStep ? forward<BF, 1>(c, s) : forward<BF, 2>(c, s);
}

// Workgroups enough to fill the chip, each with a run of pieces for every thread.
// us without / with: 8 x 65536 bf16 47 / 3.6, 256 x 65536 77 / 12.4.
constexpr int64_t kFillBlocks = 2048;

template <bool BF>
hipError_t backward(const BackwardCall& c, hipStream_t s) {
  const int64_t Q = c.vocab / kPiece, runs = (Q + kThreads - 1) / kThreads;
  const int64_t split = std::max<int64_t>(1, std::min<int64_t>(kFillBlocks / c.rows, runs));
  const int64_t share = std::max<int64_t>(1, (runs + split - 1) / split) * kThreads;
  const int64_t parts = std::max<int64_t>(1, (Q + share - 1) / share);
  hipLaunchKernelGGL(backward_kernel<BF>, dim3(static_cast<unsigned>(c.rows), static_cast<unsigned>(parts)), dim3(kThreads),
                     0, s, c, share);
  return hipGetLastError();
}

// A launch holds less than 2^32 threads: more rows go in several.
constexpr int64_t kRowsOfLaunch = int64_t(1) << 21;
template <typename T>
T* rows_on(T* p, int64_t n) {
  return p ? p + n : p;
}

}  // namespace

hipError_t launch_forward(const ForwardCall& c, hipStream_t stream) {
  for (int64_t r = 0; r < c.rows; r += kRowsOfLaunch) {
    ForwardCall d = c;
    d.rows = std::min(kRowsOfLaunch, c.rows - r);
    d.logits = c.bf16 ? at<true>(c.logits, r * c.vocab) : at<false>(c.logits, r * c.vocab);
    d.tokens = c.tokens + r;
    d.log_prob = c.log_prob + r;
    d.entropy = c.entropy + r;
    d.row_max = rows_on(c.row_max, r);
    d.log_sum = rows_on(c.log_sum, r);
    d.top_log_probs = rows_on(c.top_log_probs, r * c.top);
    d.top_ids = rows_on(c.top_ids, r * c.top);
    if (const hipError_t e = c.bf16 ? forward<true>(d, stream) : forward<false>(d, stream)) return e;
  }
  return hipSuccess;
}

hipError_t launch_backward(const BackwardCall& c, hipStream_t stream) {
  for (int64_t r = 0; r < c.rows; r += kRowsOfLaunch) {
    BackwardCall d = c;
    d.rows = std::min(kRowsOfLaunch, c.rows - r);
    d.logits = c.bf16 ? at<true>(c.logits, r * c.vocab) : at<false>(c.logits, r * c.vocab);
    d.logits_grad = const_cast<char*>(c.bf16 ? at<true>(c.logits_grad, r * c.vocab) : at<false>(c.logits_grad, r * c.vocab));
    d.tokens = c.tokens + r;
    d.row_max = c.row_max + r;
    d.log_sum = c.log_sum + r;
    d.entropy = c.entropy + r;
    d.top_ids = rows_on(c.top_ids, r * c.top);
    d.log_prob_grad = rows_on(c.log_prob_grad, r);
    d.entropy_grad = rows_on(c.entropy_grad, r);
    d.top_grad = rows_on(c.top_grad, r * c.top);
    if (const hipError_t e = c.bf16 ? backward<true>(d, stream) : backward<false>(d, stream)) return e;
  }
  return hipSuccess;
}

}  // namespace rwkv_scores
