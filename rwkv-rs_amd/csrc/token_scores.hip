// Log probability of a given token, entropy and most likely alternatives of
// rows of logits, and their gradient (include/rwkv_token_scores.h).
//
// With M = max_j x_j and d_j = (x_j - M) log2(e): s = sum 2^d_j, u = sum 2^d_j d_j.
// Then log p_j = x_j - M - ln s and the entropy is ln s - ln 2 u / s.
//
// Forward: a workgroup loads a row (or a chunk of a long one) into registers
// once, eight logits a piece, all loads in flight together, and everything else
// works on those: the maximum, the sums, and the alternatives. These are found
// through a bound: each of 64 groups of pieces has a largest logit, and the k-th
// largest of those is no larger than the k-th largest logit, so what reaches it
// (a few more than k logits, where large ones do not crowd into few groups) goes
// to a list in LDS, whose items are then ranked against each other. A list that
// overflows is replaced by k rounds of taking the largest that is left.
#include <algorithm>
#include <climits>
#include <cmath>

#include "token_scores_launch.hpp"

namespace rwkv_scores {
namespace {

constexpr int kPiece = 8;    // logits of a load (bf16: 16 bytes) or of two (fp32)
constexpr int kGroups = 64;  // also the most alternatives
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
    return fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
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
    return fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < 8; ++e) raw.v[e] = -INFINITY;
  }
  __device__ __forceinline__ void forget() {}
};

template <bool BF>
__device__ __forceinline__ const char* at(const void* base, int64_t i) {
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
// both signs are equal. No key is below kGroups.
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
__device__ __forceinline__ Key wave_largest(Key k) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) k = larger(k, __shfl_xor(k, o));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int>(k >> 32));
  return static_cast<Key>(hi) << 32 | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(k)));
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
// other way.
constexpr int max_pieces(int waves) { return waves == 1 ? 64 : waves <= 4 ? 128 : 256; }
constexpr int max_listed(int waves) { return waves == 1 ? 512 : 4 * max_pieces(waves); }
constexpr int kRanked = 128;   // more than these are cut to the most before they are ranked
template <bool BF, int kWaves>
struct Shared {
  Piece<BF> piece[max_pieces(kWaves)];
  int piece_at[max_pieces(kWaves)];
  Key key[kWaves][kGroups + 1];
  Key group[kGroups];
  Key list[max_listed(kWaves)];
  Key best[2][kGroups];        // the alternatives so far, in order
  Key bound;
  float max, part_max[kWaves], part_s[kWaves], part_u[kWaves];
  int pieces, listed;
};

// The largest of every thread's keys (`mine`; lane l of every wave belongs to
// group l) and the k-th largest of the groups' largest, into sh.max and
// sh.bound. Every group's largest is another item, so the bound is one of the 64.
template <bool BF, int kWaves>
__device__ __forceinline__ void find_bound(Shared<BF, kWaves>& sh, Key mine, int k) {
  const int tid = threadIdx.x, group = tid / kWaves, sub = tid % kWaves;
  Key key = mine;
  if constexpr (kWaves > 1) {
    sh.key[tid >> 6][tid & 63] = mine;
    __syncthreads();
    key = largest_of<kWaves>(sh.key[sub][group]);
  }
  if (sub == 0) sh.group[group] = key;
  __syncthreads();
  int rank = 0;
#pragma unroll
  for (int i = 0; i < kGroups / kWaves; ++i) rank += sh.group[sub * (kGroups / kWaves) + i] > key;
  rank = sum_of<kWaves>(rank);
  if (sub == 0) {
    if (rank == 0) sh.max = key_x(key);
    if (rank == k - 1) sh.bound = key;
  }
  if (tid == 0) sh.pieces = sh.listed = 0;
  __syncthreads();
}

// The list's n keys, more than k of them, cut to their k largest by the first
// wave: a number that k keys reach, by bisection (they are all different, so there
// is one). Ranking n keys against each other is n^2 / 2 comparisons; this is n for
// a step, of which there are some twenty.
template <bool BF, int kWaves>
__device__ __forceinline__ void cut_list(Shared<BF, kWaves>& sh, int n, int k) {
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
    Key low = ~Key{0}, high = 0;
    each([&](Key v) {
      if (v != 0 && v < low) low = v;
      high = larger(high, v);
    });
    low = ~wave_largest(~low);
    high = wave_largest(high) + 1;
    Key mid;
    while (true) {   // n keys reach low and none reaches high: what is between halves every time
      mid = low + (high - low) / 2;
      int count = 0;
      each([&](Key v) { count += __popcll(__ballot(v >= mid)); });
      if (count == k || mid == low) break;
      (count > k ? low : high) = mid;
    }
    int to = 0;   // a key's place is never behind its own
    each([&](Key v) {
      const unsigned long long hit = __ballot(v >= mid);
      const int place = to + __popcll(hit & ((1ull << lane) - 1));
      if (v >= mid && place < k) sh.list[place] = v;
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
template <bool BF, int kWaves, typename F>
__device__ __forceinline__ void rank_keys(const Shared<BF, kWaves>& sh, int n, const Key* best, int held, int k, F&& keep) {
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
template <bool BF, int kWaves, typename F>
__device__ __forceinline__ void take_largest(Shared<BF, kWaves>& sh, int k, F&& next) {
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
  __device__ __forceinline__ float log_sum() const { return logf(s) - kLn2 * o.off; }
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
  c.entropy[row] = t.valid() ? logf(t.s) - kLn2 * (t.u / t.s) : NAN;
  if (c.row_max) c.row_max[row] = t.o.m;
  if (c.log_sum) c.log_sum[row] = t.valid() ? log_sum : NAN;
}
__device__ __forceinline__ void write_top(const ForwardCall& c, int64_t row, int rank, Key v, const Sums& t, float log_sum) {
  c.top_log_probs[row * c.top + rank] = t.log_p(key_x(v), log_sum);
  c.top_ids[row * c.top + rank] = t.valid() ? key_j(v) : -1;
}

// The largest key below `last` of a thread's share of the row, which is read again.
template <bool BF>
__device__ __forceinline__ Key next_of(const void* row, int64_t begin, int64_t end, int stride, Key last) {
  Key v = 0;
#pragma nounroll
  for (int64_t j = begin + threadIdx.x; j < end; j += stride) {
    const Key y = key_of(load_one<BF>(row, j), static_cast<int>(j));
    if (y < last) v = larger(v, y);
  }
  return v;
}

// The row is Q pieces and, after them, up to seven single logits, one to a
// thread, which are numbered like pieces (Q, Q + 1, ..). A chunk is kPieces of
// them a thread.
template <bool BF, int kWaves, int kPieces, bool kTop>
__global__ __launch_bounds__(kWaves * 64, 4) void forward_kernel(const ForwardCall c) {
  constexpr int kThreads = kWaves * 64, kChunk = kThreads * kPieces;
  __shared__ Shared<BF, kWaves> sh;
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
    if constexpr (kTop) {
      find_bound(sh, key_of(most, most_at), k);
      chunk_max = sh.max;
      bound_x = key_x(sh.bound);
      bound_q = key_j(sh.bound);
      uint32_t reached = 0;   // the pieces that may hold an alternative
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if ((piece_max[i] > bound_x || (piece_max[i] == bound_x && q0 + i * kThreads + lane <= bound_q)) &&
            i * kThreads + lane < left)
          reached |= 1u << i;
      if (reached) {
        int n = atomicAdd(&sh.pieces, __popc(reached));
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          if (reached >> i & 1) {
            if (n < max_pieces(kWaves)) {
              sh.piece[n] = p[i];
              sh.piece_at[n] = q0 + i * kThreads + lane;
            }
            ++n;
          }
      }
    } else {
      const float v = wave_max(most);
      if ((tid & 63) == 0) sh.part_max[wave] = v;
      __syncthreads();
      chunk_max = sh.part_max[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) chunk_max = fmaxf(chunk_max, sh.part_max[w]);
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
    if constexpr (kTop) {
      __syncthreads();
      const int pieces = min(sh.pieces, max_pieces(kWaves));
      auto list = [&](float v, int q, int j) {
        if (v > bound_x || (v == bound_x && q <= bound_q)) {
          const int n = atomicAdd(&sh.listed, 1);
          if (n < max_listed(kWaves)) sh.list[n] = key_of(v, j);
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
      if (n > max_listed(kWaves) || sh.pieces > max_pieces(kWaves)) {
        const int64_t begin = static_cast<int64_t>(q0) * kPiece, end = final ? V : begin + kChunk * kPiece;
        n = static_cast<int>(min(static_cast<int64_t>(k), end - begin));
        take_largest(sh, n, [&](Key last) { return next_of<BF>(x, begin, end, kThreads, last); });
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
    sh.part_s[wave] = s;
    sh.part_u[wave] = u;
  }
  __syncthreads();
  Sums t{o, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    t.s += sh.part_s[w];
    t.u += sh.part_u[w];
  }
  const float log_sum = t.log_sum();
  if (tid == 0) write_row<BF>(c, row, t, log_sum);
  if constexpr (kTop)
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

// Blocks (row, y) take `share` pieces of a row each, the last one its single
// logits too. The elements with a term of their own are written again, whole, by
// the block that holds them.
constexpr int kThreads = 256;

template <bool BF>
__global__ __launch_bounds__(kThreads) void backward_kernel(const BackwardCall c, const int64_t share) {
  const int64_t row = blockIdx.x, V = c.vocab, Q = V / kPiece;
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

template <bool BF, int kWaves, int kPieces>
void forward(const ForwardCall& c, hipStream_t s) {
  auto* const kernel = c.top > 0 ? forward_kernel<BF, kWaves, kPieces, true> : forward_kernel<BF, kWaves, kPieces, false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(c.rows)), dim3(kWaves * 64), 0, s, c);
}

// The smallest workgroup whose registers hold a row, up to 128 of a thread's: what
// the selection costs does not grow with the pieces a thread holds. us, bf16, 20
// alternatives (waves, pieces a thread): 8192 x 4096 (2, 4) 26.5, (4, 2) 30.8, (1,
// 8) 27.6; 8192 x 8192 (4, 4) 39.2, (2, 8) 40.3, (4, 8) 45.2; 2048 x 32768 (4, 16)
// 33.8, (8, 8) 36.4, (8, 16) 42; 4096 x 65536 (8, 16) 132, (8, 8) in two chunks 147,
// (4, 16) 137, (16, 8) 171. fp32 pieces are twice the registers: 1024 x 65536 (8, 8)
// 48, (16, 8) 58; with a workgroup a compute unit or fewer the row's own time
// counts, 256 x 65529 (16, 8) 17.5, (8, 8) 20.6.
template <bool BF>
hipError_t forward(const ForwardCall& c, hipStream_t s) {
  if (c.vocab <= 64 * 1 * kPiece) forward<BF, 1, 1>(c, s);
  else if (c.vocab <= 64 * 2 * kPiece) forward<BF, 1, 2>(c, s);
  else if (c.vocab <= 64 * 4 * kPiece) forward<BF, 1, 4>(c, s);
  else if (c.vocab <= 128 * 4 * kPiece) forward<BF, 2, 4>(c, s);
  else if (c.vocab <= 256 * 4 * kPiece) forward<BF, 4, 4>(c, s);
  else if (c.vocab <= 256 * 8 * kPiece) forward<BF, 4, 8>(c, s);
  else if constexpr (BF) {
    if (c.vocab <= 256 * 16 * kPiece) forward<BF, 4, 16>(c, s);
    else forward<BF, 8, 16>(c, s);
  } else {
    if (c.rows <= 256) forward<BF, 16, 8>(c, s);
    else forward<BF, 8, 8>(c, s);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_forward(const ForwardCall& c, hipStream_t stream) {
  return c.bf16 ? forward<true>(c, stream) : forward<false>(c, stream);
}

// Workgroups enough to fill the chip, each with a run of pieces for every thread.
constexpr int64_t kFillBlocks = 2048;

hipError_t launch_backward(const BackwardCall& c, hipStream_t stream) {
  const int64_t Q = c.vocab / kPiece, runs = (Q + kThreads - 1) / kThreads;
  const int64_t split = std::max<int64_t>(1, std::min<int64_t>(kFillBlocks / c.rows, runs));
  const int64_t share = (runs + split - 1) / split * kThreads;
  const dim3 grid(static_cast<unsigned>(c.rows), static_cast<unsigned>(std::max<int64_t>(1, (Q + share - 1) / std::max<int64_t>(share, 1))));
  if (c.bf16) hipLaunchKernelGGL(backward_kernel<true>, grid, dim3(kThreads), 0, stream, c, share);
  else hipLaunchKernelGGL(backward_kernel<false>, grid, dim3(kThreads), 0, stream, c, share);
  return hipGetLastError();
}

}  // namespace rwkv_scores
