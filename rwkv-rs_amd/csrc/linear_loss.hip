// The cross entropy of a language model from its last hidden states x [rows, c] and
// its unembedding w [vocab, c], without the logits z = x w^T (include/
// rwkv_linear_loss.h). Three products, each by way of matrix_tile.hpp:
//
//   logits  z's tiles of 256 words by 128 rows; the forward reduces a tile to each
//           row's maximum, sum of exponentials and first index of the maximum
//           (join_kernel joins the tiles), the backward makes it D;
//   dw      = D^T x, of a piece of the vocabulary;
//   dx      = D w, summed over the pieces in fp32, the words of a piece shared
//           among `splits` workgroups that each keep a sum of their own.
//
// The backward forms z a second time instead of keeping it: 8 rows vocab c products
// and sums in all, where 6 would do with the logits in memory.
#include <algorithm>
#include <climits>
#include <cmath>

#include "linear_loss_launch.hpp"
#include "matrix_tile.hpp"

namespace rwkv_linear_loss {
namespace {

using namespace rwkv_tile;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kWords = 256, kRowsTile = 256;   // a tile of logits
constexpr int kWavesP = 2, kWavesQ = 4, kThreads = 512;
constexpr int kUnits = 256;                    // compute units
constexpr int kXcds = 8;
constexpr int kMaxBlocks = 256;                // of a maximum over an operand
constexpr int kHalfExponent = 13;              // fp16 arrays hold up to 2^14

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
__host__ __device__ int64_t ceil_div(int64_t n, int64_t by) { return (n + by - 1) / by; }

// An operand as the tiles read it: rows of `pitch` bytes, a multiple of kStep
// elements each; two arrays `plane` bytes apart for fp32.
struct Matrix {
  const char* data;
  int64_t pitch, plane;
};

// Numbers that a call's kernels leave to one another.
struct Scalars {
  float reference;             // the backward's: D is held over this
  int exponent[2];             // fp32 operands' fp16 arrays are 2^exponent as large: x, w
};

// Consecutive workgroups go to the eight XCDs in turn: give each XCD a run of
// consecutive tiles, which read the same operands, for its L2.
__device__ __forceinline__ int tile_of_block() {
  const int blocks = gridDim.x, block = blockIdx.x, x = block % kXcds;
  return x * (blocks / kXcds) + min(x, blocks % kXcds) + block / kXcds;
}

// ------------------------------------------------------------- operands as planes
__device__ __forceinline__ bool finite_bits(uint32_t magnitude) { return magnitude < 0x7f800000u; }

__global__ __launch_bounds__(256) void largest_kernel(const float* x, int64_t nx, const float* w, int64_t nw, float* out) {
  const float* const from = blockIdx.y ? w : x;
  const int64_t n = blockIdx.y ? nw : nx;
  uint32_t most = 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += kMaxBlocks * 256) {
    const uint32_t b = __builtin_bit_cast(uint32_t, from[i]) & 0x7fffffffu;
    if (finite_bits(b)) most = max(most, b);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), off)));
  __shared__ uint32_t part[4];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0)
    out[blockIdx.y * kMaxBlocks + blockIdx.x] = __builtin_bit_cast(float, max(max(part[0], part[1]), max(part[2], part[3])));
}

struct PackCall {
  const void* from[2];
  char* to[2];
  int64_t rows[2];
  int64_t c, padded;        // elements of a row, there and here
  const float* largest;     // fp32: kMaxBlocks of each
  Scalars* scalars;
};
// Rows of bf16 with zeros up to a whole step, or of fp32 as two fp16 arrays: x s = hi +
// lo with s the power of two that brings the largest magnitude to 2^13 .. 2^14, lo
// rounded to 11 bits or to a multiple of 2^-24.
template <bool BF>
__global__ __launch_bounds__(256) void pack_kernel(const PackCall c) {
  const int which = blockIdx.y;
  const int64_t n = c.rows[which] * c.padded, plane = n;
  int exponent = 0;
  if constexpr (!BF) {
    float most = c.largest[which * kMaxBlocks + threadIdx.x];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off));
    __shared__ float part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    exponent = most > 0.f ? min(kHalfExponent - ilogbf(most), 120) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) c.scalars->exponent[which] = exponent;
  }
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / c.padded, k = i % c.padded;
    if constexpr (BF) {
      reinterpret_cast<uint16_t*>(c.to[which])[i] = k < c.c ? static_cast<const uint16_t*>(c.from[which])[row * c.c + k] : 0;
    } else {
      const float v = k < c.c ? ldexpf(static_cast<const float*>(c.from[which])[row * c.c + k], exponent) : 0.f;
      const _Float16 hi = static_cast<_Float16>(v);
      _Float16* const to = reinterpret_cast<_Float16*>(c.to[which]);
      to[i] = hi;
      to[plane + i] = static_cast<_Float16>(v - static_cast<float>(hi));
    }
  }
}

// ------------------------------------------------------------------------- logits
struct LogitsCall {
  Matrix x, w;
  int rows, vocab, steps;        // steps: c up to a whole step
  int first, words;              // the piece of the vocabulary, whole tiles
  const Scalars* scalars;
  const int64_t* targets;
  int64_t ignore_index;
  // forward: [tiles, rows] each, and the targets' logits
  float *part_max, *part_sum, *row_target;
  int* part_argmax;
  // backward
  const float *row_lse, *row_max, *row_grad;
  const int32_t* row_argmax;
  float l2wrap_scale;
  char* d;                       // [rows up to whole tiles, words] bf16, or two of fp16
  int64_t d_plane;
};

// A run of words whose rows of w stay in an XCD's L2 while the rows of x pass by.
constexpr int kWordTiles = 8;
template <bool BF>
using LogitsTile = Tile<kRows, kRows, kWords, kRowsTile, kWavesP, kWavesQ, true, true, BF ? 1 : 2>;

template <bool BF, bool kBackward>
__global__ __launch_bounds__(kThreads, 2) void logits_kernel(const LogitsCall c) {
  using T = LogitsTile<BF>;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const int row_tiles = (c.rows + kRowsTile - 1) / kRowsTile, word_tiles = c.words / kWords;
  const int at = tile_of_block();
  const int run = at / (kWordTiles * row_tiles), in_run = at % (kWordTiles * row_tiles);
  const int run_words = min(kWordTiles, word_tiles - run * kWordTiles);
  const int word_tile = run * kWordTiles + in_run % run_words, row_tile = in_run / run_words;
  const int v0 = c.first + word_tile * kWords, r0 = row_tile * kRowsTile;
  T t;
  t.sum(lds, Operand{c.w.data + int64_t{v0} * c.w.pitch, c.w.pitch, c.vocab - v0, c.steps},
        Operand{c.x.data + int64_t{r0} * c.x.pitch, c.x.pitch, c.rows - r0, c.steps}, c.w.plane, c.x.plane, 0, c.steps);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4, wp = wave % kWavesP, wq = wave / kWavesP;
  // lane's words: this + 64 (i / 4) + 4 (i % 4) + element
  const int word0 = v0 + wp * T::kWaveP + 16 * g;
  if constexpr (!BF) {
    const int exponent = -(c.scalars->exponent[0] + c.scalars->exponent[1]);
#pragma unroll
    for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
      for (int j = 0; j < T::kTilesQ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) t.acc[i][j][e] = ldexpf(t.acc[i][j][e], exponent);
  }
  if constexpr (!kBackward) {
    if (v0 + kWords > c.vocab) {
#pragma unroll
      for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (word0 + 64 * (i / 4) + 4 * (i % 4) + e >= c.vocab) {
#pragma unroll
            for (int j = 0; j < T::kTilesQ; ++j) t.acc[i][j][e] = -INFINITY;
          }
    }
    float* const maxima = reinterpret_cast<float*>(lds);      // [kWavesP][kRowsTile] each
    float* const sums = maxima + kWavesP * kRowsTile;
    int* const firsts = reinterpret_cast<int*>(sums + kWavesP * kRowsTile);
#pragma unroll
    for (int j = 0; j < T::kTilesQ; ++j) {
      const int in_tile = wq * T::kWaveQ + 16 * j + m;
      const int row = r0 + in_tile;
      float most = t.acc[0][j][0];
#pragma unroll
      for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, t.acc[i][j][e]);
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      float sum = 0.f;
      int first = INT_MAX;
#pragma unroll
      for (int i = T::kTilesP - 1; i >= 0; --i)
#pragma unroll
        for (int e = 3; e >= 0; --e) {
          const float z = t.acc[i][j][e];
          sum += __expf(z - most);
          first = z == most ? 64 * (i / 4) + 4 * (i % 4) + e : first;
        }
      if (first != INT_MAX) first += wp * T::kWaveP + 16 * g;
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      first = min(first, __shfl_xor(first, 16));
      first = min(first, __shfl_xor(first, 32));
      if (g == 0) {
        maxima[wp * kRowsTile + in_tile] = most;
        sums[wp * kRowsTile + in_tile] = sum;
        firsts[wp * kRowsTile + in_tile] = first;
      }
      if (row < c.rows) {
        const int64_t own = c.targets[row] - word0;
        if (own >= 0 && own < T::kWaveP && (own & 63) < 16) {
#pragma unroll
          for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (own == 64 * (i / 4) + 4 * (i % 4) + e) c.row_target[row] = t.acc[i][j][e];
        }
      }
    }
    __syncthreads();
    if (threadIdx.x < kRowsTile && r0 + threadIdx.x < c.rows) {
      const int q = threadIdx.x;
      const float a = maxima[q], b = maxima[kRowsTile + q];
      const float most = fmaxf(a, b), sa = sums[q], sb = sums[kRowsTile + q];
      const int64_t to = int64_t{v0 / kWords} * c.rows + r0 + q;
      const int fa = firsts[q], fb = firsts[kRowsTile + q];
      c.part_max[to] = most;
      // a half without a word (or all of minus infinity) has a NaN for a sum
      c.part_sum[to] = (a == -INFINITY ? 0.f : sa * __expf(a - most)) + (b == -INFINITY ? 0.f : sb * __expf(b - most));
      const int f = a >= b ? fa : fb;
      c.part_argmax[to] = f == INT_MAX ? INT_MAX : static_cast<int>(v0) + f;
    }
  } else {
    const float reference = c.scalars->reference;
#pragma unroll
    for (int j = 0; j < T::kTilesQ; ++j) {
      const int row = r0 + wq * T::kWaveQ + 16 * j + m, known = min(row, c.rows - 1);
      const int64_t target = c.targets[known];
      const bool dead = row >= c.rows || target == c.ignore_index;
      const float lse = c.row_lse[known], h = c.row_grad[known] / reference;
      const float wrap = c.l2wrap_scale * c.row_max[known] / reference;
      const int64_t own = target - word0;
      const int top = c.row_argmax[known] - word0;
#pragma unroll
      for (int half = 0; half < T::kTilesP / 4; ++half) {
        float v[16];
#pragma unroll
        for (int n = 0; n < 16; ++n) v[n] = h * __expf(t.acc[4 * half + n / 4][j][n % 4] - lse);
        if (own >= 64 * half && own < 64 * half + 16) {
#pragma unroll
          for (int n = 0; n < 16; ++n)
            if (own == 64 * half + n) v[n] -= h;
        }
        if (top >= 64 * half && top < 64 * half + 16) {
#pragma unroll
          for (int n = 0; n < 16; ++n)
            if (top == 64 * half + n) v[n] += wrap;
        }
        if (dead) {
#pragma unroll
          for (int n = 0; n < 16; ++n) v[n] = 0.f;
        }
        const int word = word0 + 64 * half;
        if (word + 16 > c.vocab) {
#pragma unroll
          for (int n = 0; n < 16; ++n)
            if (word + n >= c.vocab) v[n] = 0.f;
        }
        char* const to = c.d + (static_cast<int64_t>(row) * c.words + word - c.first) * 2;
        if constexpr (BF) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            bf16x8 o;
#pragma unroll
            for (int n = 0; n < 8; ++n) o[n] = static_cast<__bf16>(v[8 * q + n]);
            reinterpret_cast<bf16x8*>(to)[q] = o;
          }
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            f16x8 hi, lo;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const float s = ldexpf(v[8 * q + n], kHalfExponent);
              hi[n] = static_cast<_Float16>(s);
              lo[n] = static_cast<_Float16>(s - static_cast<float>(hi[n]));
            }
            reinterpret_cast<f16x8*>(to)[q] = hi;
            reinterpret_cast<f16x8*>(to + c.d_plane)[q] = lo;
          }
        }
      }
    }
  }
}

// Joins the tiles of each row: 16 rows a workgroup, their tiles among 16 threads.
struct JoinCall {
  const float *part_max, *part_sum, *row_target;
  const int* part_argmax;
  const int64_t* targets;
  int64_t rows, vocab, ignore_index;
  float *row_loss, *row_lse, *row_max;
  int32_t* row_argmax;
};
struct Run {
  float most, sum;
  int first;
};
__device__ __forceinline__ Run combine(const Run& a, const Run& b) {
  Run r;
  r.most = fmaxf(a.most, b.most);
  r.sum = (a.most == -INFINITY && a.sum == 0.f ? 0.f : a.sum * __expf(a.most - r.most)) +
          (b.most == -INFINITY && b.sum == 0.f ? 0.f : b.sum * __expf(b.most - r.most));
  r.first = a.most > b.most ? a.first : b.most > a.most ? b.first : min(a.first, b.first);
  return r;
}
__global__ __launch_bounds__(256) void join_kernel(const JoinCall c) {
  __shared__ Run part[16][17];
  const int own = threadIdx.x & 15, share = threadIdx.x >> 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + own, tiles = ceil_div(c.vocab, kWords);
  Run run{-INFINITY, 0.f, INT_MAX};
  if (row < c.rows) {
#pragma unroll 4
    for (int64_t t = share; t < tiles; t += 16) {
      const int64_t at = t * c.rows + row;
      run = combine(run, Run{c.part_max[at], c.part_sum[at], c.part_argmax[at]});
    }
  }
  part[share][own] = run;
  __syncthreads();
  if (share > 0 || row >= c.rows) return;
#pragma unroll
  for (int s = 1; s < 16; ++s) run = combine(run, part[s][own]);
  const float lse = run.most + logf(run.sum);
  const int64_t target = c.targets[row];
  c.row_lse[row] = lse;
  c.row_max[row] = run.most;
  c.row_argmax[row] = run.first;
  // a logit is at most the sum's logarithm: no rounding makes a loss negative
  c.row_loss[row] = target == c.ignore_index ? 0.f
                    : target < 0 || target >= c.vocab ? NAN
                    : lse != lse ? NAN
                                 : fmaxf(lse - c.row_target[row], 0.f);
}

// ---------------------------------------------------------------------- gradients
// What D is held over: the largest of the rows' factors. A gradient that is the same
// for all rows leaves exactly one, and so its own rounding out of D.
struct ReferenceCall {
  const float *row_grad, *row_max;
  const int64_t* targets;
  int64_t rows, ignore_index;
  float l2wrap_scale;
  Scalars* scalars;
};
__global__ __launch_bounds__(1024) void reference_kernel(const ReferenceCall c) {
  uint32_t most = 0;
  for (int64_t r = threadIdx.x; r < c.rows; r += 1024) {
    if (c.targets[r] == c.ignore_index) continue;
    const uint32_t g = __builtin_bit_cast(uint32_t, c.row_grad[r]) & 0x7fffffffu;
    const uint32_t w = __builtin_bit_cast(uint32_t, c.l2wrap_scale * c.row_max[r]) & 0x7fffffffu;
    if (finite_bits(g)) most = max(most, g);
    if (finite_bits(w)) most = max(most, w);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), off)));
  __shared__ uint32_t part[16];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 16; ++w) most = max(most, part[w]);
    c.scalars->reference = most == 0 ? 1.f : __builtin_bit_cast(float, most);
  }
}

template <bool BF>
__device__ __forceinline__ float unscaled(float sum, float reference, int exponent) {
  return BF ? sum * reference : ldexpf(sum, -(kHalfExponent + exponent)) * reference;
}

template <bool BF>
__device__ __forceinline__ void store4(void* base, int64_t at, f32x4 v, int64_t left, bool whole) {
  if (whole) {
    if constexpr (BF) {
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = static_cast<__bf16>(v[e]);
      *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(base) + at) = o;
    } else {
      *reinterpret_cast<f32x4*>(static_cast<float*>(base) + at) = v;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) {
      if constexpr (BF) static_cast<__bf16*>(base)[at + e] = static_cast<__bf16>(v[e]);
      else static_cast<float*>(base)[at + e] = v[e];
    }
}

struct WeightGradCall {
  Matrix x;
  const char* d;
  int64_t d_plane;
  int words, padded_rows, rows, vocab, c, first;
  const Scalars* scalars;
  void* grad;
};
// dw of the piece's words: steps are rows; those past the last have D = 0.
template <bool BF, int kChannels>
__global__ __launch_bounds__(kThreads, 2) void weight_grad_kernel(const WeightGradCall c) {
  using T = Tile<kSteps, kSteps, kChannels, 256, kWavesP, kWavesQ, false, false, BF ? 1 : 2>;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const int channel_tiles = (c.c + kChannels - 1) / kChannels;
  const int at = tile_of_block();
  const int c0 = at % channel_tiles * kChannels, w0 = at / channel_tiles * 256;
  const int steps = (c.rows + kStep - 1) / kStep * kStep;
  T t;
  t.sum(lds, Operand{c.x.data + c0 * 2, c.x.pitch, c.c - c0, c.rows},
        Operand{c.d + w0 * 2, int64_t{c.words} * 2, c.words - w0, c.padded_rows}, c.x.plane, c.d_plane, 0, steps);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4, wp = wave % kWavesP, wq = wave / kWavesP;
  const float reference = c.scalars->reference;
  const int exponent = BF ? 0 : c.scalars->exponent[0];
  const bool whole = c.c % 4 == 0;
#pragma unroll
  for (int j = 0; j < T::kTilesQ; ++j) {
    const int word = c.first + w0 + wq * T::kWaveQ + 16 * j + m;
    if (word >= c.vocab) continue;
#pragma unroll
    for (int i = 0; i < T::kTilesP; ++i) {
      const int channel = c0 + wp * T::kWaveP + 16 * i + 4 * g;
      if (channel >= c.c) continue;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = unscaled<BF>(t.acc[i][j][e], reference, exponent);
      store4<BF>(c.grad, int64_t{word} * c.c + channel, v, c.c - channel, whole);
    }
  }
}

struct HiddenGradCall {
  Matrix w;
  const char* d;
  int64_t d_plane;
  int words, rows, vocab, c, first;
  int share;                 // words of a workgroup
  bool begin;                // the first piece: nothing to add to
  float* sums;               // [splits, rows, pitch]
  int pitch;
};
template <bool BF, int kChannels>
__global__ __launch_bounds__(kThreads, 2) void hidden_grad_kernel(const HiddenGradCall c) {
  using T = Tile<kSteps, kRows, kChannels, 256, kWavesP, kWavesQ, false, true, BF ? 1 : 2>;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const int channel_tiles = (c.c + kChannels - 1) / kChannels, row_tiles = (c.rows + 255) / 256;
  const int at = tile_of_block();
  const int c0 = at % channel_tiles * kChannels, r0 = at / channel_tiles % row_tiles * 256;
  const int split = at / channel_tiles / row_tiles;
  const int k0 = split * c.share, k1 = min(k0 + c.share, c.words);
  T t;
  t.sum(lds, Operand{c.w.data + int64_t{c.first} * c.w.pitch + c0 * 2, c.w.pitch, c.c - c0, c.vocab - c.first},
        Operand{c.d + int64_t{r0} * c.words * 2, int64_t{c.words} * 2, 256, c.words}, c.w.plane, c.d_plane, k0, k1);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4, wp = wave % kWavesP, wq = wave / kWavesP;
#pragma unroll
  for (int j = 0; j < T::kTilesQ; ++j) {
    const int row = r0 + wq * T::kWaveQ + 16 * j + m;
    if (row >= c.rows) continue;
#pragma unroll
    for (int i = 0; i < T::kTilesP; ++i) {
      const int channel = c0 + wp * T::kWaveP + 16 * i + 4 * g;
      if (channel >= c.pitch) continue;
      f32x4* const to = reinterpret_cast<f32x4*>(c.sums + (int64_t{split} * c.rows + row) * c.pitch + channel);
      *to = c.begin ? t.acc[i][j] : *to + t.acc[i][j];
    }
  }
}

// The splits' sums of dx in order, in the operands' type.
struct HiddenSumCall {
  const float* sums;
  int64_t rows, c, pitch;
  int splits;
  const Scalars* scalars;
  void* grad;
};
template <bool BF>
__global__ __launch_bounds__(256) void hidden_sum_kernel(const HiddenSumCall c) {
  const float reference = c.scalars->reference;
  const int exponent = BF ? 0 : c.scalars->exponent[1];
  const int64_t fours = c.pitch / 4, n = c.rows * fours;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t row = i / fours, channel = i % fours * 4;
  if (channel >= c.c) return;
  f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < c.splits; ++s) v += reinterpret_cast<const f32x4*>(c.sums)[s * n + i];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = unscaled<BF>(v[e], reference, exponent);
  store4<BF>(c.grad, row * c.c + channel, v, c.c - channel, c.c % 4 == 0);
}

__global__ __launch_bounds__(256) void clear_kernel(uint32_t* to, int64_t words, int64_t bytes) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < words) to[i] = 0;
  else if (i == words && bytes % 4) *reinterpret_cast<uint16_t*>(to + words) = 0;
}

// ------------------------------------------------------------------ plan, workspace
// The bf16 operands whose rows are whole steps are read where they are.
bool packed(int64_t c, bool bf16) { return !bf16 || c % kStep != 0; }

struct Places {
  int64_t scalars, largest, x, w, x_plane, w_plane;   // byte offsets; planes' sizes
  int64_t end;
};
int64_t take(int64_t& end, int64_t bytes) {
  const int64_t at = end;
  end += up(bytes, 256);
  return at;
}
Places operands(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  Places p{};
  const int64_t pitch = up(c, kStep) * 2, planes = bf16 ? 1 : 2;
  p.scalars = take(p.end, sizeof(Scalars));
  if (packed(c, bf16)) {
    p.largest = take(p.end, 2 * kMaxBlocks * 4);
    p.x_plane = rows * pitch;
    p.w_plane = vocab * pitch;
    p.x = take(p.end, planes * p.x_plane);
    p.w = take(p.end, planes * p.w_plane);
  }
  return p;
}

// Two workgroups of a tile fill a compute unit.
constexpr int64_t kSlots = kUnits;
constexpr int64_t kMaxD = int64_t{512} << 20;   // bytes of D of a piece
struct Plan {
  int channels;                     // of a gradient's tile
  int64_t words, pieces;            // of a piece
  int64_t padded_rows, splits, share, pitch;
};
Plan plan(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  Plan p{};
  p.channels = (c - 1) % 256 < 128 ? 128 : 256;
  p.padded_rows = up(rows, kRowsTile);
  p.pitch = up(c, 4);
  const int64_t channel_tiles = ceil_div(c, p.channels), planes = bf16 ? 1 : 2;
  const int64_t all = up(vocab, kWords);
  const int64_t most = std::max<int64_t>(kWords, kMaxD / (p.padded_rows * 2 * planes) / kWords * kWords);
  // pieces of whole rounds of the weight gradient's tiles of 128 words
  const int64_t round = std::max<int64_t>(kSlots / channel_tiles, 1) * 256;
  p.words = std::min(all, most >= round ? most / round * round : most);
  p.pieces = ceil_div(all, p.words);
  p.words = std::min(p.words, up(ceil_div(all, p.pieces), kWords) );
  const int64_t tiles = channel_tiles * ceil_div(rows, 256);
  p.splits = std::max<int64_t>(1, std::min<int64_t>(kSlots * 4 / tiles, p.words / 512));
  p.share = up(ceil_div(p.words, p.splits), kStep);
  p.splits = ceil_div(p.words, p.share);
  return p;
}

struct BackwardPlaces {
  Places operands;
  int64_t d, d_plane, sums, end;
};
BackwardPlaces backward_places(const Plan& p, int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  BackwardPlaces b{};
  b.operands = operands(rows, vocab, c, bf16);
  b.end = b.operands.end;
  b.d_plane = p.padded_rows * p.words * 2;
  b.d = take(b.end, b.d_plane * (bf16 ? 1 : 2));
  b.sums = take(b.end, p.splits * rows * p.pitch * 4);
  return b;
}

struct ForwardPlaces {
  Places operands;
  int64_t part_max, part_sum, part_argmax, row_target, end;
};
ForwardPlaces forward_places(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  ForwardPlaces f{};
  f.operands = operands(rows, vocab, c, bf16);
  f.end = f.operands.end;
  const int64_t parts = ceil_div(vocab, kWords) * rows * 4;
  f.part_max = take(f.end, parts);
  f.part_sum = take(f.end, parts);
  f.part_argmax = take(f.end, parts);
  f.row_target = take(f.end, rows * 4);
  return f;
}

// x and w as the tiles read them, made first where they are not so in memory.
template <bool BF>
void prepare(const Call& c, const Places& p, Matrix* x, Matrix* w, hipStream_t s) {
  const int64_t padded = up(c.c, kStep);
  if (!packed(c.c, BF)) {
    *x = Matrix{static_cast<const char*>(c.hidden), c.c * 2, 0};
    *w = Matrix{static_cast<const char*>(c.weight), c.c * 2, 0};
    return;
  }
  float* const largest = reinterpret_cast<float*>(c.workspace + p.largest);
  if (!BF)
    hipLaunchKernelGGL(largest_kernel, dim3(kMaxBlocks, 2), dim3(256), 0, s, static_cast<const float*>(c.hidden),
                       c.rows * c.c, static_cast<const float*>(c.weight), c.vocab * c.c, largest);
  PackCall k{};
  k.from[0] = c.hidden;
  k.from[1] = c.weight;
  k.to[0] = c.workspace + p.x;
  k.to[1] = c.workspace + p.w;
  k.rows[0] = c.rows;
  k.rows[1] = c.vocab;
  k.c = c.c;
  k.padded = padded;
  k.largest = largest;
  k.scalars = reinterpret_cast<Scalars*>(c.workspace + p.scalars);
  const int64_t blocks = std::min<int64_t>(ceil_div(std::max(c.rows, c.vocab) * padded, 1024), 4096);
  hipLaunchKernelGGL(pack_kernel<BF>, dim3(static_cast<unsigned>(blocks), 2), dim3(256), 0, s, k);
  *x = Matrix{k.to[0], padded * 2, p.x_plane};
  *w = Matrix{k.to[1], padded * 2, p.w_plane};
}

template <bool BF>
void forward(const ForwardCall& c, hipStream_t s) {
  const ForwardPlaces f = forward_places(c.rows, c.vocab, c.c, BF);
  LogitsCall l{};
  prepare<BF>(c, f.operands, &l.x, &l.w, s);
  l.rows = static_cast<int>(c.rows);
  l.vocab = static_cast<int>(c.vocab);
  l.steps = static_cast<int>(up(c.c, kStep));
  l.words = static_cast<int>(up(c.vocab, kWords));
  l.scalars = reinterpret_cast<const Scalars*>(c.workspace + f.operands.scalars);
  l.targets = c.targets;
  l.part_max = reinterpret_cast<float*>(c.workspace + f.part_max);
  l.part_sum = reinterpret_cast<float*>(c.workspace + f.part_sum);
  l.part_argmax = reinterpret_cast<int*>(c.workspace + f.part_argmax);
  l.row_target = reinterpret_cast<float*>(c.workspace + f.row_target);
  const int64_t tiles = l.words / kWords * ceil_div(c.rows, kRowsTile);
  hipLaunchKernelGGL((logits_kernel<BF, false>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, s, l);
  const JoinCall j{l.part_max, l.part_sum, l.row_target, l.part_argmax, c.targets, c.rows, c.vocab, c.ignore_index,
                   c.row_loss, c.row_lse, c.row_max, c.row_argmax};
  hipLaunchKernelGGL(join_kernel, dim3(static_cast<unsigned>(ceil_div(c.rows, 16))), dim3(256), 0, s, j);
}

template <bool BF, int kChannels>
void gradients(const BackwardCall& c, const Plan& p, const BackwardPlaces& b, const LogitsCall& l, bool first, hipStream_t s) {
  const int64_t channel_tiles = ceil_div(c.c, kChannels);
  if (c.weight_grad) {
    const WeightGradCall w{l.x, l.d, l.d_plane, l.words, static_cast<int>(p.padded_rows), l.rows, l.vocab, static_cast<int>(c.c),
                           l.first, l.scalars, c.weight_grad};
    const int words = std::min(l.words, l.vocab - l.first);
    hipLaunchKernelGGL((weight_grad_kernel<BF, kChannels>), dim3(static_cast<unsigned>(channel_tiles * ceil_div(words, 256))),
                       dim3(kThreads), 0, s, w);
  }
  if (c.hidden_grad) {
    const int64_t splits = ceil_div(l.words, p.share);
    const HiddenGradCall h{l.w, l.d, l.d_plane, l.words, l.rows, l.vocab, static_cast<int>(c.c), l.first,
                           static_cast<int>(p.share), first, reinterpret_cast<float*>(c.workspace + b.sums),
                           static_cast<int>(p.pitch)};
    hipLaunchKernelGGL((hidden_grad_kernel<BF, kChannels>),
                       dim3(static_cast<unsigned>(channel_tiles * ceil_div(c.rows, 256) * splits)), dim3(kThreads), 0, s, h);
  }
}

template <bool BF>
void backward(const BackwardCall& c, hipStream_t s) {
  const Plan p = plan(c.rows, c.vocab, c.c, BF);
  const BackwardPlaces b = backward_places(p, c.rows, c.vocab, c.c, BF);
  LogitsCall l{};
  prepare<BF>(c, b.operands, &l.x, &l.w, s);
  Scalars* const scalars = reinterpret_cast<Scalars*>(c.workspace + b.operands.scalars);
  const ReferenceCall r{c.row_grad, c.row_max, c.targets, c.rows, c.ignore_index, c.l2wrap_scale, scalars};
  hipLaunchKernelGGL(reference_kernel, dim3(1), dim3(1024), 0, s, r);
  l.rows = static_cast<int>(c.rows);
  l.vocab = static_cast<int>(c.vocab);
  l.steps = static_cast<int>(up(c.c, kStep));
  l.scalars = scalars;
  l.targets = c.targets;
  l.ignore_index = c.ignore_index;
  l.row_lse = c.row_lse;
  l.row_max = c.row_max;
  l.row_grad = c.row_grad;
  l.row_argmax = c.row_argmax;
  l.l2wrap_scale = c.l2wrap_scale;
  l.d = c.workspace + b.d;
  l.d_plane = b.d_plane;
  for (int64_t first = 0; first < c.vocab; first += p.words) {
    l.first = static_cast<int>(first);
    l.words = static_cast<int>(std::min(p.words, up(c.vocab - first, kWords)));
    const int64_t tiles = l.words / kWords * ceil_div(c.rows, kRowsTile);
    hipLaunchKernelGGL((logits_kernel<BF, true>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, s, l);
    if (p.channels == 128) gradients<BF, 128>(c, p, b, l, first == 0, s);
    else gradients<BF, 256>(c, p, b, l, first == 0, s);
  }
  if (c.hidden_grad) {
    const HiddenSumCall h{reinterpret_cast<const float*>(c.workspace + b.sums), c.rows, c.c, p.pitch,
                          static_cast<int>(p.splits), scalars, c.hidden_grad};
    hipLaunchKernelGGL(hidden_sum_kernel<BF>, dim3(static_cast<unsigned>(ceil_div(c.rows * p.pitch / 4, 256))), dim3(256),
                       0, s, h);
  }
}

}  // namespace

int64_t forward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  return rows == 0 ? 0 : forward_places(rows, vocab, c, bf16).end;
}

int64_t backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  return rows == 0 ? 0 : backward_places(plan(rows, vocab, c, bf16), rows, vocab, c, bf16).end;
}

hipError_t launch_forward(const ForwardCall& c, hipStream_t s) {
  c.bf16 ? forward<true>(c, s) : forward<false>(c, s);
  return hipGetLastError();
}

hipError_t launch_backward(const BackwardCall& c, hipStream_t s) {
  if (c.rows == 0) {   // no row: no gradient of the weight
    const int64_t bytes = c.vocab * c.c * (c.bf16 ? 2 : 4);
    hipLaunchKernelGGL(clear_kernel, dim3(static_cast<unsigned>(ceil_div(bytes / 4 + 1, 256))), dim3(256), 0, s,
                       static_cast<uint32_t*>(c.weight_grad), bytes / 4, bytes);
  } else {
    c.bf16 ? backward<true>(c, s) : backward<false>(c, s);
  }
  return hipGetLastError();
}

}  // namespace rwkv_linear_loss
