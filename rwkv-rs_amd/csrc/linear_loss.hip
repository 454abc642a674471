// The cross entropy of a language model from its last hidden states x [rows, c] and
// its unembedding w [vocab, c], without the logits z = x w^T (include/
// rwkv_linear_loss.h). Three products, each by way of matrix_tile.hpp:
//
//   logits  tiles of z; the forward reduces a tile to each row's maximum, sum of
//           exponentials and first index of the maximum (join_kernel joins the tiles),
//           the backward makes it D;
//   dw      = D^T x, of a piece of the vocabulary;
//   dx      = D w, summed over the pieces in fp32, the words of a piece shared
//           among `splits` workgroups that each keep a sum of their own.
//
// The backward forms z a second time instead of keeping it: 8 rows vocab c products
// and sums in all, where 6 would do with the logits in memory. The matrix cores, and the
// power that they take, bound all three for many rows. For 7168 learned rows of 8192, c =
// 768, 65536 words in bf16 (us, PFLOP/s; torch's own products of 8192 rows in brackets):
// logits 623 to 690, 1.05 to 1.16 (812, 1.02); D 746 to 802, 0.9 (as the logits, and 1
// GiB written); dw and dx together 1280 to 1380, 1.05 to 1.13 (858 and 848, 0.97).
// A product of 8192 cubed reaches 1.49 here, one of 16384 cubed 1.65.
// For few rows it is memory: 64 rows of the same, 26 us for the loss, of which 20 are
// w's bytes at a copy's rate.
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

// A tile of logits: words by rows, on waves by waves. 256 by 256 reads each operand's
// element once for 256 products, which the matrix cores need to be fed from L2: on tiles of
// 128 by 128 the forward of 8192 x 768 x 65536 takes 823 us for 687, of 2048 x 4096 x 65536
// 1005 for 721. Two smaller ones, of which a compute unit has two and four at a time, for
// few rows or words, where large ones leave units idle: 30 x 2048 x 8000 19 us on the small
// one and 31 on the large one, 1000 x 512 x 1000 13 and 26.
struct Big {
  static constexpr int kWords = 256, kRows = 256, kWavesP = 2, kWavesQ = 4, kEach = 1, kLead = 0;
};
struct Middle {
  static constexpr int kWords = 128, kRows = 128, kWavesP = 2, kWavesQ = 2, kEach = 2, kLead = 0;
};
struct Small {
  static constexpr int kWords = 64, kRows = 64, kWavesP = 2, kWavesQ = 2, kEach = 4, kLead = 0;
};
// The same with eight stages on their way, one to a compute unit, for few tiles of many
// channels: 64 x 4096 x 16000 28 us and 34, fp32 7 x 2944 x 70 50 and 59.
struct Deep {
  static constexpr int kWords = 64, kRows = 64, kWavesP = 2, kWavesQ = 2, kEach = 1, kLead = 8;
};
// Of fp32 operands where there are few rows: w is split on its way to the products. 256
// words a workgroup keep 64 KiB of w on their way to each compute unit; the small one is
// for up to 64 rows of 12288 (below, this form does not run) to 16384 words, of which the
// large one makes a workgroup on a quarter of the units at most: both calls, us, on the large
// one and on the small, 64 x 344 x 12288 85 and 71, 8 x 768 x 12288 126 and 98, 64 x 2048 x
// 12288 249 and 178, 64 x 4096 x 16384 518 and 373.
struct Few {
  static constexpr int kWords = 256, kRows = 64, kWavesP = 4, kWavesQ = 1, kEach = 1, kSlots = 3;
};
struct FewSmall {
  static constexpr int kWords = 64, kRows = 64, kWavesP = 2, kWavesQ = 1, kEach = 1, kSlots = 5;
};
template <typename Shape>
constexpr bool kIsFew = std::is_same<Shape, Few>::value || std::is_same<Shape, FewSmall>::value;
template <typename Shape, Kind kKind, bool kFew = kIsFew<Shape>>
struct LogitsTile {
  using T = Tile<kRows, kRows, Shape::kWords, Shape::kRows, Shape::kWavesP, Shape::kWavesQ, true, true, kKind, Shape::kLead>;
};
template <typename Shape, Kind kKind>
struct LogitsTile<Shape, kKind, true> {
  using T = FewTile<kRows, Shape::kWords, Shape::kRows, Shape::kWavesP, true, Shape::kSlots>;
};
constexpr int kWholeWords = 256;               // a piece of the vocabulary is whole tiles of any size
constexpr int kWavesP = 2, kWavesQ = 4, kThreads = 512;   // of a gradient's tile
constexpr int kUnits = 256;                    // compute units; a tile's LDS leaves room for one workgroup on each
constexpr int kXcds = 8;
constexpr int kMaxBlocks = 256;                // of a maximum over an operand
constexpr int kHalfExponent = 13;              // fp16 arrays hold up to 2^14

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t ceil_div(int64_t n, int64_t by) { return (n + by - 1) / by; }

// An operand as the tiles read it: rows of `pitch` bytes, whole steps; two arrays `plane`
// bytes apart for fp32.
struct Matrix {
  const char* data;
  int64_t pitch, plane;
};

// What a call's kernels leave to one another.
struct Scalars {
  float mantissa;      // of the rows' largest factor, 1 to 2: D is held over this,
  int scale;           // and over 2^this, or what is less for a row of smaller factors
  int exponent[2];     // the fp16 arrays of x and w are 2^exponent as large
};

// Workgroups go to the eight XCDs in turn. Each XCD gets a run of consecutive tiles,
// which read the same operands, for its L2: the tile of workgroup `block` of `blocks`.
__device__ __forceinline__ int tile_of_block(int block, int blocks) {
  const int x = block % kXcds;
  return x * (blocks / kXcds) + min(x, blocks % kXcds) + block / kXcds;
}

// ------------------------------------------------------------- operands as fp16 arrays
__device__ __forceinline__ uint32_t finite_magnitude(float v) {   // as an integer of the same order; 0 for the others
  const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off)));
  return v;
}
template <int kWaves>
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  __shared__ uint32_t part[kWaves];
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = max(v, part[w]);
  return v;
}

// The rows that are not ignored, in order, and where each row is among them (-1: not).
// The products are formed of these alone: fine-tuning leaves out prompts and padding. One
// workgroup of kWide threads: each wave takes a run of rows, counts them, then numbers them.
constexpr int kWide = 1024;
struct RowsCall {
  const int64_t* targets;
  int64_t ignore_index;
  int rows;
  int *index, *place, *count;   // null: the rows as they are
};
__device__ __forceinline__ void number_rows(const RowsCall& c) {
  __shared__ int counts[kWide / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int each = (c.rows + kWide - 1) / kWide * 64, first = wave * each, last = min(first + each, c.rows);
  int n = 0;
#pragma unroll 8
  for (int r = first + lane; r - lane < last; r += 64)
    n += __popcll(__ballot(r < last && c.targets[min(r, c.rows - 1)] != c.ignore_index));
  if (lane == 0) counts[wave] = n;
  __syncthreads();
  int at = 0;
#pragma unroll
  for (int w = 0; w < kWide / 64; ++w) {
    if (w == wave) n = at;
    at += counts[w];
  }
  if (threadIdx.x == 0) *c.count = at;
#pragma unroll 4
  for (int r = first + lane; r - lane < last; r += 64) {
    const bool kept = r < last && c.targets[min(r, c.rows - 1)] != c.ignore_index;
    const uint64_t all = __ballot(kept);
    const int own = n + __popcll(all & ((uint64_t{1} << lane) - 1));
    if (kept) c.index[own] = r;
    if (r < last) c.place[r] = kept ? own : -1;
    n += __popcll(all);
  }
}
__global__ __launch_bounds__(kWide) void rows_kernel(const RowsCall c) { number_rows(c); }

// The largest magnitudes: of x but for the rows that are ignored (whatever stands there
// is nobody's measure), of w, and of the rows' factors of D. Row y of the grid takes
// array y; each workgroup leaves one number. A fourth row numbers the rows.
//
// A row's own power of two: D of each row is held over its own, so that a row of small
// weight has as many bits of its hidden gradient as any other. The weight gradient, in which
// the rows meet, takes the powers back on x (pack_kernel).
constexpr int kLargestScale = INT_MAX;         // a row without a finite factor, or any of fp32 with few rows: as the largest
struct SurveyCall {
  const void* from[2];       // null: not wanted
  int64_t n[2];              // rows
  int64_t c;
  const float *row_grad, *row_max;   // null: no backward
  const int64_t* targets;
  int64_t rows, ignore_index;
  float l2wrap_scale;
  float* residuals;          // [2, rows], cleared; may be null
  int* row_scale;            // [rows]
  bool own_scales;           // or all rows' as the largest
  uint32_t* largest;         // [3, kMaxBlocks]
  RowsCall numbered;
};
template <bool BF>
__global__ __launch_bounds__(kWide) void survey_kernel(const SurveyCall c) {
  const int which = blockIdx.y;
  uint32_t most = 0;
  if (which == 3) {
    if (blockIdx.x == 0) number_rows(c.numbered);
    return;
  }
  if (which < 2) {
    if (!c.from[which]) return;
    constexpr int kPer = BF ? 8 : 4;       // elements of 16 bytes
    const int lane = threadIdx.x & 63;
    const int pieces = (reinterpret_cast<uintptr_t>(c.from[which]) & 15) == 0 && c.c % kPer == 0 ? static_cast<int>(c.c / kPer) : 0;
    for (int64_t row = blockIdx.x * (kWide / 64) + (threadIdx.x >> 6); row < c.n[which]; row += kMaxBlocks * (kWide / 64)) {
      if (which == 0 && c.targets[row] == c.ignore_index) continue;
      const u32x4* const v = reinterpret_cast<const u32x4*>(static_cast<const char*>(c.from[which]) + row * c.c * (BF ? 2 : 4));
#pragma unroll 4
      for (int i = lane; i < pieces; i += 64) {
        const u32x4 p = v[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BF) {
            most = max(most, finite_magnitude(__builtin_bit_cast(float, p[e] << 16)));
            most = max(most, finite_magnitude(__builtin_bit_cast(float, p[e] & 0xffff0000u)));
          } else {
            most = max(most, finite_magnitude(__builtin_bit_cast(float, static_cast<uint32_t>(p[e]))));
          }
        }
      }
      if (pieces == 0) {
        for (int64_t i = row * c.c + lane; i < (row + 1) * c.c; i += 64) {
          if constexpr (BF) most = max(most, finite_magnitude(static_cast<float>(static_cast<const __bf16*>(c.from[which])[i])));
          else most = max(most, finite_magnitude(static_cast<const float*>(c.from[which])[i]));
        }
      }
    }
  } else {
    if (!c.row_grad) return;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWide + threadIdx.x; r < c.rows; r += kMaxBlocks * kWide) {
      if (c.residuals) c.residuals[r] = c.residuals[c.rows + r] = 0.f;
      const uint32_t own = c.targets[r] == c.ignore_index ? 0 : max(finite_magnitude(c.row_grad[r]), finite_magnitude(c.l2wrap_scale * c.row_max[r]));
      c.row_scale[r] = c.own_scales && own ? ilogbf(__builtin_bit_cast(float, own)) : kLargestScale;
      most = max(most, own);
    }
  }
  most = block_max<kWide / 64>(most);
  if (threadIdx.x == 0) c.largest[which * kMaxBlocks + blockIdx.x] = most;
}

// One array made of another: rows of `padded` elements, zeros behind the c there are.
// bf16 as it is; bf16 to fp16; fp32 to two of fp16, or to three of bf16; fp32 as it is, in
// rows of whole eights
enum PackKind { kCopy, kToHalf, kToHalves, kToThirds, kEights };
struct PackJob {
  const void* from;
  char* to;
  int64_t rows;
  int kind, which;           // which: of the largest magnitudes
  bool weighted;             // rows with the powers of two that D's rows are without
};
struct PackCall {
  PackJob job[3];
  int jobs, c, padded;
  bool factors;              // the backward's mantissa and scale are wanted
  const int* row_scale;
  const int64_t* targets;
  int64_t ignore_index;
  const int *index, *count;  // of x's rows that are taken; null: all
  const uint32_t* largest;
  Scalars* scalars;
};
// fp16 arrays are of x s, s the power of two that brings the largest magnitude to 2^13
// .. 2^14: bf16 numbers of 2^-27 of it and more are held whole, smaller ones to 2^-38 of
// it; of fp32 ones the second array holds what is left, rounded to 11 bits or likewise. For
// the weight gradient a row is smaller by the power of two that its weight is below the
// largest one's: its D is not, and what is lost is below 2^-38 of the largest of both.
// Ignored rows of x are left out or become zeros: a NaN there does not reach the weight's
// gradient.
__device__ __forceinline__ int exponent_of(uint32_t largest) {
  return largest ? min(kHalfExponent - ilogbf(__builtin_bit_cast(float, largest)), 120) : 0;
}
__global__ __launch_bounds__(256) void pack_kernel(const PackCall c) {
  const PackJob job = c.job[blockIdx.y];
  const bool writes = blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0;
  int exponent = 0, scale = 0;
  if (c.factors && ((blockIdx.x == 0 && blockIdx.y == 0) || job.weighted)) {
    const uint32_t most = block_max<4>(c.largest[2 * kMaxBlocks + threadIdx.x]);
    const float largest = most ? __builtin_bit_cast(float, most) : 1.f;
    scale = ilogbf(largest);
    // a gradient that is the same for all rows leaves a power of two, and so its own rounding out of D
    if (writes) {
      c.scalars->mantissa = ldexpf(largest, -scale);
      c.scalars->scale = scale;
    }
  }
  if (static_cast<int>(blockIdx.y) >= c.jobs) return;
  if (job.kind == kToThirds) {
    if (blockIdx.x == 0 && threadIdx.x == 0) c.scalars->exponent[0] = c.scalars->exponent[1] = 0;
  } else if (job.kind != kCopy && job.kind != kEights) {
    exponent = exponent_of(block_max<4>(c.largest[job.which * kMaxBlocks + threadIdx.x]));
    if (blockIdx.x == 0 && threadIdx.x == 0) c.scalars->exponent[job.which] = exponent;
  }
  const int lane = threadIdx.x & 63;
  if (job.kind == kEights) {
    const int64_t eights = (c.c + 7) / 8 * 8;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); row < job.rows; row += gridDim.x * int64_t{4}) {
      const float* const from = static_cast<const float*>(job.from) + row * c.c;
      float* const to = reinterpret_cast<float*>(job.to) + row * eights;
#pragma unroll 4
      for (int i = lane; i < eights; i += 64) to[i] = i < c.c ? from[i] : 0.f;
    }
    return;
  }
  const int pieces = c.padded / 8;
  const int64_t plane = job.rows * c.padded;
  const bool whole = c.c % 8 == 0;
  const bool some = c.index && job.which == 0;
  const int64_t rows = some ? *c.count : job.rows;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); row < rows; row += gridDim.x * int64_t{4}) {
    const int64_t source = some ? c.index[row] : row;
    const bool ignored = !some && job.kind != kCopy && job.which == 0 && c.targets[row] == c.ignore_index;
    const int shift = exponent + (job.weighted ? min(c.row_scale[source], scale) - scale : 0);
    for (int i = lane; i < pieces; i += 64) {
      const int64_t at = source * c.c + 8 * i;
      if (ignored) {
        char* const to = job.to + (row * c.padded + 8 * i) * 2;
        *reinterpret_cast<u32x4*>(to) = u32x4{0, 0, 0, 0};
        if (job.kind == kToHalves || job.kind == kToThirds) *reinterpret_cast<u32x4*>(to + plane * 2) = u32x4{0, 0, 0, 0};
        if (job.kind == kToThirds) *reinterpret_cast<u32x4*>(to + plane * 4) = u32x4{0, 0, 0, 0};
      } else if (job.kind == kToHalves || job.kind == kToThirds) {
        float v[8];
        const float* const from = static_cast<const float*>(job.from) + at;
        if (whole && 8 * i < c.c) {
          const f32x4 a = reinterpret_cast<const f32x4*>(from)[0], b = reinterpret_cast<const f32x4*>(from)[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 8 * i + e < c.c ? from[e] : 0.f;
        }
        if (job.kind == kToThirds) {
          s16x8 part[3];
          thirds(v, part);
#pragma unroll
          for (int k = 0; k < 3; ++k) *reinterpret_cast<s16x8*>(job.to + (row * c.padded + 8 * i + k * plane) * 2) = part[k];
          continue;
        }
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float s = ldexpf(v[e], shift);
          hi[e] = static_cast<_Float16>(s);
          lo[e] = static_cast<_Float16>(s - static_cast<float>(hi[e]));
        }
        _Float16* const to = reinterpret_cast<_Float16*>(job.to) + row * c.padded + 8 * i;
        *reinterpret_cast<f16x8*>(to) = hi;
        *reinterpret_cast<f16x8*>(to + plane) = lo;
      } else {
        const __bf16* const from = static_cast<const __bf16*>(job.from) + at;
        bf16x8 raw;
        if (whole && 8 * i < c.c) {
          raw = *reinterpret_cast<const bf16x8*>(from);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) raw[e] = 8 * i + e < c.c ? from[e] : static_cast<__bf16>(0.f);
        }
        char* const to = job.to + (row * c.padded + 8 * i) * 2;
        if (job.kind == kCopy) {
          *reinterpret_cast<bf16x8*>(to) = raw;
        } else {
          f16x8 h;
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = static_cast<_Float16>(ldexpf(static_cast<float>(raw[e]), shift));
          *reinterpret_cast<f16x8*>(to) = h;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------- logits
struct LogitsCall {
  Matrix x, w;
  int rows, vocab, c, steps;     // c up to whole eights, and up to whole stages
  int first, words;              // the piece of the vocabulary, whole tiles
  const int *index, *count;      // the rows that x's are, and how many; null: all as they are
  const Scalars* scalars;
  const int64_t* targets;
  int64_t ignore_index;
  // forward: [tiles of words, rows] each, and the targets' logits
  float *part_max, *part_sum, *row_target;
  int* part_argmax;
  // backward
  const float *row_log_sum, *row_max, *row_grad;
  const int32_t* row_argmax;
  const int* row_scale;
  float l2wrap_scale;
  // [rows up to whole tiles, words] fp16, each row over its own power of two, so 2^15 at most;
  // for fp32 two of them, or three of bf16
  char* d;
  int64_t d_plane;
  float* residuals;              // [2, rows], bf16 operands: what rounding took from D at the target and at the argmax
};

// D as hidden_grad's products see it: rounded to fp16 and then to bf16.
__device__ __forceinline__ float as_read(float v) {
  return static_cast<float>(static_cast<__bf16>(static_cast<float>(static_cast<_Float16>(v))));
}

// What a sum of exponentials over the maximum `own` counts among ones over `most`.
__device__ __forceinline__ float share_of(float own, float most) { return own == most ? 1.f : __expf(own - most); }

// A run of words whose rows of w stay in an XCD's L2 while the rows of x pass by: eight
// tiles of 256 words of c = 768 are 3 MiB of its 4.
//
// Persistent: as many workgroups as fit take the tiles in turn, and ask for a tile's first
// operands before they are done with the one before, so that only the first tile's loads
// are waited for. What follows the products bounds a tile of few channels beside them: a
// tile of 256 by 256 takes 1.5 us for 64 channels and 5 for the maximum, the exponentials and
// the first index, ten instructions' time an element.
constexpr int kWordTiles = 8;
template <bool BF, bool kBackward, typename Shape>
__global__ __launch_bounds__(64 * Shape::kWavesP * Shape::kWavesQ,
                             std::max(Shape::kWavesP* Shape::kWavesQ* Shape::kEach / 4, 1)) void logits_kernel(const LogitsCall c) {
  constexpr int kWords = Shape::kWords, kRowsTile = Shape::kRows, kWavesP = Shape::kWavesP;
  constexpr bool kFew = kIsFew<Shape>;
  using T = typename LogitsTile<Shape, BF ? kBf16 : kHalves>::T;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const int rows = c.count ? *c.count : c.rows;
  // the backward's D is made up to whole pieces, of zeros past the vocabulary
  const int words = kBackward ? c.words : min(c.words, c.vocab - c.first);
  const int row_tiles = (rows + kRowsTile - 1) / kRowsTile, word_tiles = (words + kWords - 1) / kWords, tiles = row_tiles * word_tiles;
  // each XCD has a run of tiles, and its workgroups take them in turn
  const int xcd = blockIdx.x % kXcds, local = blockIdx.x / kXcds, locals = (static_cast<int>(gridDim.x) - xcd + kXcds - 1) / kXcds;
  const int each = tiles / kXcds, rest = tiles % kXcds;
  const int last = (xcd + 1) * each + min(xcd + 1, rest);
  int at = xcd * each + min(xcd, rest) + local;
  T t;
  typename T::Work work;
  int v0, r0;
  auto begin = [&](int tile) {
    const int run = tile / (kWordTiles * row_tiles), in_run = tile % (kWordTiles * row_tiles);
    const int run_words = min(kWordTiles, word_tiles - run * kWordTiles);
    v0 = c.first + (run * kWordTiles + in_run % run_words) * kWords;
    r0 = in_run / run_words * kRowsTile;
    T::begin(work, lds,
             Operand{c.w.data + int64_t{min(v0, c.vocab - 1)} * c.w.pitch, c.w.pitch, max(c.vocab - v0, 1), kFew ? c.c : c.steps},
             Operand{c.x.data + int64_t{r0} * c.x.pitch, c.x.pitch, rows - r0, c.steps}, c.w.plane, c.x.plane, 0, c.steps);
  };
  if (at < last) begin(at);
  for (; at < last; at += locals) {
    t.run(work, lds);
    const int v = v0, r = r0;
    // a wave whose rows are all behind the last one, and behind the steps of D's other product
    const bool idle = T::kWaveQ % kStep == 0 && r + uniform(static_cast<int>(threadIdx.x >> 6)) / kWavesP * T::kWaveQ >= rows;
    if (at + locals < last) begin(at + locals);   // its loads run under what follows
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4, wp = wave % kWavesP, wq = wave / kWavesP;
    // lane's words: this + 32 (i / 2) + 4 (i % 2) + element
    const int word0 = v + wp * T::kWaveP + 8 * g;
    if constexpr (!BF && !kFew) {
      const int exponent = -(c.scalars->exponent[0] + c.scalars->exponent[1]);
#pragma unroll
      for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
        for (int j = 0; j < T::kTilesQ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) t.acc[i][j][e] = ldexpf(t.acc[i][j][e], exponent);
    }
    if constexpr (!kBackward) {
      if (v + kWords > c.vocab) {
#pragma unroll
        for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (word0 + 32 * (i / 2) + 4 * (i % 2) + e >= c.vocab) {
#pragma unroll
              for (int j = 0; j < T::kTilesQ; ++j) t.acc[i][j][e] = -INFINITY;
            }
      }
      float* const maxima = reinterpret_cast<float*>(lds + T::kFree);      // [kWavesP][kRowsTile] each
      float* const sums = maxima + kWavesP * kRowsTile;
      int* const firsts = reinterpret_cast<int*>(sums + kWavesP * kRowsTile);
      if (!idle) {
#pragma unroll
        for (int j = 0; j < T::kTilesQ; ++j) {
          const int in_tile = wq * T::kWaveQ + 16 * j + m;
          const int row = r + in_tile;
          float most = t.acc[0][j][0];
#pragma unroll
          for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, t.acc[i][j][e]);
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          const float base = most == -INFINITY ? 0.f : most;   // words of minus infinity alone: nothing, but a NaN among them
          float sum = 0.f;
          int first = INT_MAX;
#pragma unroll
          for (int i = T::kTilesP - 1; i >= 0; --i)
#pragma unroll
            for (int e = 3; e >= 0; --e) {
              const float z = t.acc[i][j][e];
              sum += __expf(z - base);
              first = z == most ? 32 * (i / 2) + 4 * (i % 2) + e : first;
            }
          if (first != INT_MAX) first += wp * T::kWaveP + 8 * g;
          sum += __shfl_xor(sum, 16);
          sum += __shfl_xor(sum, 32);
          first = min(first, __shfl_xor(first, 16));
          first = min(first, __shfl_xor(first, 32));
          if (g == 0) {
            maxima[wp * kRowsTile + in_tile] = most;
            sums[wp * kRowsTile + in_tile] = sum;
            firsts[wp * kRowsTile + in_tile] = first;
          }
          if (row < rows) {
            const int64_t target = c.targets[c.index ? c.index[row] : row];
            const int own = target >= 0 && target < c.vocab ? static_cast<int>(target) - word0 : -1;
            if (own >= 0 && own < T::kWaveP && (own & 31) < 8) {
#pragma unroll
              for (int i = 0; i < T::kTilesP; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (own == 32 * (i / 2) + 4 * (i % 2) + e) c.row_target[row] = t.acc[i][j][e];
            }
          }
        }
      }
      __syncthreads();
      if (threadIdx.x < kRowsTile && r + static_cast<int>(threadIdx.x) < rows) {
        const int q = threadIdx.x;
        float most = maxima[q];
#pragma unroll
        for (int w = 1; w < kWavesP; ++w) most = fmaxf(most, maxima[w * kRowsTile + q]);
        float sum = 0.f;
        int f = INT_MAX;
#pragma unroll
        for (int w = kWavesP - 1; w >= 0; --w) {
          const float own = maxima[w * kRowsTile + q];
          sum += sums[w * kRowsTile + q] * share_of(own, most);
          if (own == most) f = firsts[w * kRowsTile + q];
        }
        const int64_t to = int64_t{v / kWords} * c.rows + r + q;
        c.part_max[to] = most;
        c.part_sum[to] = sum;
        c.part_argmax[to] = f == INT_MAX ? INT_MAX : v + f;
      }
    } else if (!idle) {
      const float mantissa = c.scalars->mantissa;
      const int scale = c.scalars->scale;
      struct Row {
        float log_sum, h, most;
        int own, top, exponent;
        bool dead;
      } of[T::kTilesQ];
#pragma unroll
      for (int j = 0; j < T::kTilesQ; ++j) {      // all rows' numbers are asked for at once
        const int row = r + wq * T::kWaveQ + 16 * j + m, some = min(row, rows - 1), known = c.index ? c.index[some] : some;
        const int64_t target = c.targets[known];
        of[j].dead = row >= rows || target == c.ignore_index;
        of[j].own = target >= 0 && target < c.vocab ? static_cast<int>(target) - word0 : -1;
        of[j].top = c.row_argmax[known] - word0;
        of[j].log_sum = c.row_log_sum[known];
        of[j].h = c.row_grad[known];
        of[j].most = c.row_max[known];
        of[j].exponent = kHalfExponent - min(c.row_scale[known], scale);
      }
#pragma unroll
      for (int j = 0; j < T::kTilesQ; ++j) {
        const int row = r + wq * T::kWaveQ + 16 * j + m;
        const float most = of[j].most, h = ldexpf(of[j].h, of[j].exponent) / mantissa;
        const float wrap = ldexpf(c.l2wrap_scale * most, of[j].exponent) / mantissa;
        // exp(z - max) is as exact as z, however large that is, which max + log_sum in one number would not leave it
        const float share = h * expf(-of[j].log_sum);
        const int own = of[j].own, top = of[j].top;
        const bool dead = of[j].dead;
#pragma unroll
        for (int pair = 0; pair < T::kTilesP / 2; ++pair) {
          float d[8];
#pragma unroll
          for (int n = 0; n < 8; ++n) d[n] = share * __expf(t.acc[2 * pair + n / 4][j][n % 4] - most);
          const bool has_own = own >= 32 * pair && own < 32 * pair + 8, has_top = top >= 32 * pair && top < 32 * pair + 8;
          if (has_own || has_top) {
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const bool is_own = own == 32 * pair + n, is_top = top == 32 * pair + n;
              if (is_own) d[n] -= h;
              if (is_top) d[n] += wrap;
              if constexpr (BF) {
                if (!dead && is_own) c.residuals[row] = d[n] - as_read(d[n]);
                else if (!dead && is_top) c.residuals[c.rows + row] = d[n] - as_read(d[n]);
              }
            }
          }
          const int word = word0 + 32 * pair;
          if (dead || word + 8 > c.vocab) {
#pragma unroll
            for (int n = 0; n < 8; ++n)
              if (dead || word + n >= c.vocab) d[n] = 0.f;
          }
          char* const to = c.d + (static_cast<int64_t>(row) * c.words + word - c.first) * 2;
          if constexpr (kFew) {
            s16x8 part[3];
            thirds(d, part);
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<s16x8*>(to + k * c.d_plane) = part[k];
            continue;
          }
          f16x8 hi;
#pragma unroll
          for (int n = 0; n < 8; ++n) hi[n] = static_cast<_Float16>(d[n]);
          *reinterpret_cast<f16x8*>(to) = hi;
          if constexpr (!BF) {
            f16x8 lo;
#pragma unroll
            for (int n = 0; n < 8; ++n) lo[n] = static_cast<_Float16>(d[n] - static_cast<float>(hi[n]));
            *reinterpret_cast<f16x8*>(to + c.d_plane) = lo;
          }
        }
      }
    }
  }
}

// Joins the tiles of each row: 16 rows a workgroup, their tiles among 64 threads. Loads
// that wait for one another bound it: 16 threads took 13 us for 64 rows of 1024 tiles.
constexpr int kJoinRows = 16, kJoinShares = 64;
struct JoinCall {
  const float *part_max, *part_sum, *row_target;
  const int* part_argmax;
  const int64_t* targets;
  const int* place;          // of each row among the parts' rows; null: as it is
  int64_t rows, vocab, ignore_index;
  int words;                 // of a tile
  float *row_loss, *row_log_sum, *row_max;
  int32_t* row_argmax;
};
struct Run {
  float most, sum;
  int first;
};
__device__ __forceinline__ Run combine(const Run& a, const Run& b) {
  Run r;
  r.most = fmaxf(a.most, b.most);
  r.sum = a.sum * share_of(a.most, r.most) + b.sum * share_of(b.most, r.most);
  r.first = a.most > b.most ? a.first : b.most > a.most ? b.first : min(a.first, b.first);
  return r;
}
__global__ __launch_bounds__(kJoinRows * kJoinShares) void join_kernel(const JoinCall c) {
  __shared__ Run part[kJoinShares][kJoinRows + 1];
  const int own = threadIdx.x % kJoinRows, share = threadIdx.x / kJoinRows;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kJoinRows + own, tiles = (c.vocab + c.words - 1) / c.words;
  Run run{-INFINITY, 0.f, INT_MAX};
  const int64_t part_row = row >= c.rows ? -1 : c.place ? c.place[row] : row;
  if (part_row >= 0) {
#pragma unroll 4
    for (int64_t t = share; t < tiles; t += kJoinShares) {
      const int64_t at = t * c.rows + part_row;
      run = combine(run, Run{c.part_max[at], c.part_sum[at], c.part_argmax[at]});
    }
  }
#pragma unroll
  for (int s = kJoinShares / 2; s > 0; s /= 2) {   // the upper half of the shares gives its runs to the lower
    if (share >= s && share < 2 * s) part[share][own] = run;
    __syncthreads();
    if (share < s) run = combine(run, part[share + s][own]);
  }
  if (share > 0 || row >= c.rows) return;
  const float log_sum = logf(run.sum);
  const int64_t target = c.targets[row];
  c.row_log_sum[row] = log_sum;
  c.row_max[row] = run.most;
  c.row_argmax[row] = run.first;
  float loss = target == c.ignore_index ? 0.f : NAN;
  if (target != c.ignore_index && target >= 0 && target < c.vocab && log_sum == log_sum) {
    loss = run.most - c.row_target[part_row] + log_sum;   // of two large logits the difference first
    loss = loss < 0.f ? 0.f : loss;   // a logit is at most the sum's logarithm: no rounding makes a loss negative
  }
  c.row_loss[row] = loss;
}

// ---------------------------------------------------------------------- gradients
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

// dx of four channels from its sum, in the operands' type. For bf16 operands, what D's
// rounding took at the target and at the argmax is put back: mostly that is nearly all
// of a row's D, and its error would be as large as the result's own rounding.
struct HiddenCall {
  void* grad;
  int64_t c, rows;
  const float* residuals;
  const int64_t* targets;
  const int32_t* row_argmax;
  const int* row_scale;
  const __bf16* weight;
};
// What the sums are multiplied with: one number from 1 to 2, then one power of two, so that
// nothing on the way is larger or smaller than the result.
struct Factor {
  float mantissa;
  int exponent, scale;       // of a row of dx of smaller factors: its own scale's
  __device__ __forceinline__ Factor of_row(int row_scale) const { return Factor{mantissa, exponent + min(row_scale, scale) - scale, scale}; }
};
__device__ __forceinline__ f32x4 times(f32x4 v, Factor f) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e] * f.mantissa, f.exponent);
  return v;
}
__device__ __forceinline__ Factor factor_of(const Scalars* s, int exponent) {
  return Factor{s->mantissa, s->scale - kHalfExponent - exponent, s->scale};
}
__device__ __forceinline__ Factor weight_factor(const Scalars* s) { return factor_of(s, s->exponent[0]); }
template <bool BF>
__device__ __forceinline__ Factor hidden_factor(const Scalars* s) { return factor_of(s, BF ? 0 : s->exponent[1]); }
template <bool BF>
__device__ __forceinline__ void finish_hidden(const HiddenCall& c, Factor f, int64_t row, int64_t part_row, int64_t channel, f32x4 v) {
  const bool whole = c.c % 8 == 0;
  if constexpr (BF) {
    const int64_t words[2] = {c.targets[row], c.row_argmax[row]};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float r = c.residuals[k * c.rows + part_row];
      // read whether it is wanted or not, so that nothing waits for the residual first; where
      // there is none, there may be no such word
      const __bf16* const from = c.weight + (r != 0.f ? words[k] : 0) * c.c + channel;
      bf16x4 w;
      if (whole) {
        w = *reinterpret_cast<const bf16x4*>(from);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = from[min(static_cast<int64_t>(e), c.c - 1 - channel)];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += r != 0.f ? r * static_cast<float>(w[e]) : 0.f;
    }
  }
  store4<BF>(c.grad, row * c.c + channel, times(v, f.of_row(c.row_scale[row])), c.c - channel, whole);
}

constexpr int kGradTile = 256;   // words or rows of a gradient's tile
struct GradientsCall {
  Matrix x, w;               // x: fp16, weighted; w: bf16, or fp16 for fp32
  const char* d;
  int64_t d_plane;
  int first, words, padded_rows, rows, vocab, c;
  const int* count;          // of x's and D's rows; null: all
  const Scalars* scalars;
  int weight_tiles, weight_blocks;   // dw's workgroups: its tiles, up to whole rounds of the XCDs
  int hidden_blocks;                 // dx's, likewise
  bool hidden_first;
  void* weight_grad;
  int row_share;             // rows of a workgroup of dw
  float* weight_sums;        // [row shares, vocab, pitch]; null: one share, dw itself is stored
  int share;                 // words of a workgroup of dx
  bool begin;                // the first piece: no sums to add to
  float* sums;               // [splits, rows, pitch]; null (of fp32): dx itself is stored
  int pitch;
  HiddenCall hidden;
};

// Tiles of 256 by 256 (or 128 channels) as the logits' are. Workgroups of both gradients in
// one launch: either alone would leave units idle in its last round. The backward with one
// after the other: 8192 x 768 x 65536 2377 us for 2090, 512 rows of that 250 for 205,
// 2048 x 4096 x 65536 2494 for 2479, fp32 1024 x 1024 x 32000 690 for 583.
//
// The tiles of a gradient in an order in which those that an XCD has at a time share
// both operands: runs of up to five tiles of channels, in each the other tiles.
constexpr int kMaxRun = 5;
__device__ __forceinline__ void place(int at, int channel_tiles, int others, int& channel_tile, int& other) {
  const int runs = (channel_tiles + kMaxRun - 1) / kMaxRun, run = (channel_tiles + runs - 1) / runs;
  const int first = at / (run * others) * run, in_run = at % (run * others), width = min(run, channel_tiles - first);
  channel_tile = first + in_run % width;
  other = in_run / width;
}

// dw of four channels from its sum, in the operands' type.
template <bool BF>
__device__ __forceinline__ void finish_weight(void* grad, Factor f, int64_t word, int64_t channel, int64_t c, f32x4 v) {
  store4<BF>(grad, word * c + channel, times(v, f), c - channel, c % 8 == 0);
}

// A tile of dw, of the piece's words over a share of the rows: steps are rows; those past
// the last have D = 0.
template <bool BF, int kChannels, bool kFew>
__device__ __forceinline__ void weight_tile(const GradientsCall& c, char* lds, int tile) {
  using T = Tile<kSteps, kSteps, kChannels, kGradTile, kWavesP, kWavesQ, false, false, BF ? kHalf : kFew ? kThirds : kHalves>;
  const int channel_tiles = (c.c + kChannels - 1) / kChannels, word_tiles = c.words / kGradTile;
  const int split = tile / (channel_tiles * word_tiles);
  int channel_tile, word_tile;
  place(tile % (channel_tiles * word_tiles), channel_tiles, word_tiles, channel_tile, word_tile);
  const int c0 = channel_tile * kChannels, w0 = word_tile * kGradTile;
  const int rows = c.count ? *c.count : c.rows;
  const Factor factor = weight_factor(c.scalars);
  const int k0 = split * c.row_share, k1 = min(k0 + c.row_share, (rows + kStep - 1) / kStep * kStep);
  T t;
  if (k0 >= k1) {
    t.clear();
  } else {
    typename T::Work work;
    T::begin(work, lds, Operand{c.x.data + c0 * 2, c.x.pitch, c.c - c0, rows},
             Operand{c.d + w0 * 2, int64_t{c.words} * 2, c.words - w0, c.padded_rows}, c.x.plane, c.d_plane, k0, k1);
    t.run(work, lds);
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4, wp = wave % kWavesP, wq = wave / kWavesP;
  auto all_of = [&](auto store) {
#pragma unroll
    for (int j = 0; j < T::kTilesQ; ++j) {
      const int word = c.first + w0 + wq * T::kWaveQ + 16 * j + m;
      if (word >= c.vocab) continue;
#pragma unroll
      for (int i = 0; i < T::kTilesP; ++i) {
        const int channel = c0 + wp * T::kWaveP + 16 * i + 4 * g;
        if (channel < c.c) store(word, channel, t.acc[i][j]);
      }
    }
  };
  if (c.weight_sums) {
    float* const sums = c.weight_sums + int64_t{split} * c.vocab * c.pitch;
    all_of([&](int word, int channel, f32x4 v) { *reinterpret_cast<f32x4*>(sums + int64_t{word} * c.pitch + channel) = v; });
  } else {
    all_of([&](int word, int channel, f32x4 v) { finish_weight<BF>(c.weight_grad, factor, word, channel, c.c, v); });
  }
}

template <bool BF, int kChannels, bool kFew>
struct HiddenTile {
  using T = Tile<kSteps, kRows, kChannels, kGradTile, kWavesP, kWavesQ, false, true, BF ? kHalfQ : kHalves>;
};
template <int kChannels>
struct HiddenTile<false, kChannels, true> {
  using T = FewTile<kSteps, kChannels, Few::kRows, Few::kWavesP, false>;
};

// A tile of dx, over a share of the piece's words; the words past the vocabulary have D =
// 0. There are as many workgroups as all rows would need.
template <bool BF, int kChannels, bool kFew>
__device__ __forceinline__ void hidden_tile(const GradientsCall& c, char* lds, int block) {
  using T = typename HiddenTile<BF, kChannels, kFew>::T;
  constexpr int kTileRows = T::kItemsQ, kWavesP = T::kAcross;
  const int rows = c.count ? *c.count : c.rows;
  const int channel_tiles = (c.c + kChannels - 1) / kChannels, row_tiles = (rows + kTileRows - 1) / kTileRows;
  const int each = channel_tiles * row_tiles, all = each * ((c.words + c.share - 1) / c.share);
  if (block >= all) return;
  const int at = tile_of_block(block, all), split = at / each;
  int channel_tile, row_tile;
  place(at % each, channel_tiles, row_tiles, channel_tile, row_tile);
  const int c0 = channel_tile * kChannels, r0 = row_tile * kTileRows;
  const int k0 = split * c.share, k1 = min(k0 + c.share, c.words);
  const Factor factor = hidden_factor<BF>(c.scalars);
  T t;
  typename T::Work work;
  T::begin(work, lds, Operand{c.w.data + int64_t{c.first} * c.w.pitch + c0 * (kFew ? 4 : 2), c.w.pitch, c.c - c0, c.vocab - c.first},
           Operand{c.d + int64_t{r0} * c.words * 2, int64_t{c.words} * 2, (rows + kStep - 1) / kStep * kStep - r0, c.words},
           c.w.plane, c.d_plane, k0, k1);
  t.run(work, lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4, wp = wave % kWavesP, wq = wave / kWavesP;
  auto all_of = [&](auto store) {
#pragma unroll
    for (int j = 0; j < T::kTilesQ; ++j) {
      const int row = r0 + wq * T::kWaveQ + 16 * j + m;
      if (row >= rows) continue;
#pragma unroll
      for (int i = 0; i < T::kTilesP; ++i) {
        const int channel = c0 + wp * T::kWaveP + 16 * i + 4 * g;
        if (channel < c.pitch) store(row, channel, t.acc[i][j]);
      }
    }
  };
  if (BF || c.sums) {
    float* const sums = c.sums + int64_t{split} * c.rows * c.pitch;
    all_of([&](int row, int channel, f32x4 v) {
      f32x4* const to = reinterpret_cast<f32x4*>(sums + int64_t{row} * c.pitch + channel);
      *to = c.begin ? v : *to + v;
    });
  } else {
    all_of([&](int row, int channel, f32x4 v) { finish_hidden<false>(c.hidden, factor, row, row, channel, v); });
  }
}

// Both gradients of a piece side by side: first the longer tiles, then the shorter ones,
// which fill the compute units that have none of the last of those.
template <int kChannels>
constexpr int kWeightLds = Tile<kSteps, kSteps, kChannels, kGradTile, kWavesP, kWavesQ, false, false, kHalves>::kLdsBytes;
template <bool BF, int kChannels>
__global__ __launch_bounds__(kThreads, 2) void gradients_kernel(const GradientsCall c) {
  __shared__ __attribute__((aligned(16))) char lds[std::max(HiddenTile<BF, kChannels, false>::T::kLdsBytes, kWeightLds<kChannels>)];
  const int weight = static_cast<int>(blockIdx.x) - (c.hidden_first ? c.hidden_blocks : 0);
  if (weight >= 0 && weight < c.weight_blocks) {
    const int at = tile_of_block(weight, c.weight_blocks);
    if (at < c.weight_tiles) weight_tile<BF, kChannels, false>(c, lds, at);
  } else {
    hidden_tile<BF, kChannels, false>(c, lds, c.hidden_first ? static_cast<int>(blockIdx.x) : weight - c.weight_blocks);
  }
}

// Of few rows of fp32, one after the other: memory bounds both. 64 x 768 x 65536: dw 67 us,
// of which 41 are what it writes, dx 61, of which 41 are w.
template <int kChannels>
__global__ __launch_bounds__(kThreads, 2) void few_weight_kernel(const GradientsCall c) {
  __shared__ __attribute__((aligned(16))) char lds[kWeightLds<kChannels>];
  const int at = tile_of_block(blockIdx.x, c.weight_blocks);
  if (at < c.weight_tiles) weight_tile<false, kChannels, true>(c, lds, at);
}
template <int kChannels>
__global__ __launch_bounds__(64 * Few::kWavesP, 1) void few_hidden_kernel(const GradientsCall c) {
  __shared__ __attribute__((aligned(16))) char lds[HiddenTile<false, kChannels, true>::T::kLdsBytes];
  hidden_tile<false, kChannels, true>(c, lds, blockIdx.x);
}

// The shares' sums of dx and of dw, in order.
struct SumCall {
  const float *hidden_sums, *weight_sums;   // null: nothing to add
  int64_t rows, vocab, pitch;
  int splits, row_splits;
  const int* place;          // of each row among the sums' rows; null: as it is
  const Scalars* scalars;
  HiddenCall hidden;
  void* weight_grad;
};
__device__ __forceinline__ f32x4 sum_of(const float* sums, int64_t n, int64_t at, int splits) {
  f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) v += reinterpret_cast<const f32x4*>(sums)[s * n + at];
  return v;
}
template <bool BF>
__global__ __launch_bounds__(256) void sum_kernel(const SumCall c) {
  const int64_t fours = c.pitch / 4, step = static_cast<int64_t>(gridDim.x) * 256;
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (blockIdx.y == 0 && c.hidden_sums) {
    const int64_t n = c.rows * fours;
    const Factor factor = hidden_factor<BF>(c.scalars);
    for (; i < n; i += step) {
      const int64_t row = i / fours, four = i % fours, part_row = c.place ? c.place[row] : row;
      if (part_row < 0)
        store4<BF>(c.hidden.grad, row * c.hidden.c + 4 * four, f32x4{0.f, 0.f, 0.f, 0.f}, c.hidden.c - 4 * four, c.hidden.c % 8 == 0);
      else
        finish_hidden<BF>(c.hidden, factor, row, part_row, 4 * four, sum_of(c.hidden_sums, n, part_row * fours + four, c.splits));
    }
  } else if (blockIdx.y == 1 && c.weight_sums) {
    const int64_t n = c.vocab * fours;
    const Factor factor = weight_factor(c.scalars);
    for (; i < n; i += step)
      finish_weight<BF>(c.weight_grad, factor, i / fours, i % fours * 4, c.hidden.c, sum_of(c.weight_sums, n, i, c.row_splits));
  }
}

// by elements: where c is no multiple of 8, a gradient may begin at any of them
template <typename Element>
__global__ __launch_bounds__(256) void clear_kernel(Element* to, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) to[i] = 0;
}

// ------------------------------------------------------------------ plan, workspace
// fp32 operands with few rows and many words, w being nearly all there is to read: w is read
// where it is, three times in the two calls, where packing it to fp16 reads or writes it
// eleven times in all. Against the packed form, us for both calls: 1 to 64 rows of 768 with
// 65536 words 230 and 480, 128 rows 352 and 514, 192 rows 490 and 531, 256 rows 634 and 571;
// 64 of 768 with 16000 words 107 and 131, with 8000 97 and 91; 64 of 4096 with 4000 242 and
// 229; 64 of 512 with 2000, whose launches are what counts, 78 and 64. Rows that do not begin
// at whole 16 bytes are copied to rows of whole eights first: 40 of 333 with 100000 words 396
// and 517, 64 of 1001 with 65536 777 and 921, with 20000 294 and 276.
constexpr int64_t kFewRows = 128, kManyWords = 12288, kLargeWeight = int64_t{1} << 22;
bool few(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  return !bf16 && rows <= kFewRows && vocab >= kManyWords && vocab * c >= (c % 8 ? 6 : 1) * kLargeWeight;
}
int64_t planes_of(int64_t rows, int64_t vocab, int64_t c, bool bf16) { return bf16 ? 1 : few(rows, vocab, c, bf16) ? 3 : 2; }

// The rows that are not ignored are numbered, and x's brought together, where that is a
// small part of the work: two launches more for bf16 operands, 10 us; fp32 ones are packed
// anyhow. With an eighth of the rows ignored, both calls, us, numbered and not: 8192 x 768
// x 65536 2780 and 3010, 700 x 2048 x 65536 721 and 754, 512 x 768 x 65536 262 and 264, 300
// rows of that 231 and 222, 2000 x 768 x 8000 146 and 139; fp32 600 x 1024 x 32000 684 and
// 699.
constexpr int64_t kLargeWork = int64_t{1} << 36;
bool numbered(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  return rows > kFewRows && rows * c * (bf16 ? 1 : 4) >= kLargeWork / vocab;   // rows c is below 2^34
}
// bf16 operands whose rows are whole steps are read where they are.
bool packed(int64_t c, bool bf16) { return !bf16 || c % kStep != 0; }

int64_t take(int64_t& end, int64_t bytes) {
  const int64_t at = end;
  end += up(bytes, 256);
  return at;
}
// Byte offsets of the operands in the workspace.
struct Places {
  int64_t scalars, largest, index, place, count, x, w, x_weighted, x_plane, w_plane;
  int64_t end;
};
Places operands(int64_t rows, int64_t vocab, int64_t c, bool bf16, bool backward) {
  Places p{};
  const int64_t pitch = up(c, kStep) * 2, planes = planes_of(rows, vocab, c, bf16);
  p.scalars = take(p.end, sizeof(Scalars));
  p.largest = take(p.end, 3 * kMaxBlocks * 4);
  p.x_plane = rows * pitch;
  p.w_plane = vocab * pitch;
  if (numbered(rows, vocab, c, bf16)) {
    p.index = take(p.end, rows * 4);
    p.place = take(p.end, rows * 4);
    p.count = take(p.end, 4);
  }
  if (packed(c, bf16) || numbered(rows, vocab, c, bf16)) p.x = take(p.end, planes * p.x_plane);
  if (few(rows, vocab, c, bf16)) {
    if (c % 8 != 0) p.w = take(p.end, vocab * up(c, 8) * 4);
  } else if (packed(c, bf16)) {
    p.w = take(p.end, planes * p.w_plane);
  }
  if (backward && !few(rows, vocab, c, bf16)) p.x_weighted = take(p.end, planes * p.x_plane);
  return p;
}

// D of a piece takes at most kMaxD bytes, of which the least is a tile of words. The
// gradients' shares, of dx over the words and, of a vocabulary in one piece, of dw over
// the rows: those with which the tiles, handed to the compute units in turn, the longer
// ones first, are done first, in stages. A tile's first loads and its stores count as
// kOverhead stages, the launch that adds shares up as kLaunch, and the sums' way to memory
// and back as kBytesPerStage has it.
constexpr int64_t kMaxD = int64_t{512} << 20, kOverhead = 4, kLaunch = 4, kMaxSplits = 64, kBytesPerStage = int64_t{8} << 20;
struct Plan {
  int channels;                     // of a gradient's tile
  int64_t words, pieces;            // of a piece
  int64_t padded_rows, pitch;
  int64_t splits, share, row_splits, row_share;
  bool hidden_first;
};
// When `all_more` tiles of `more_each` are done behind `all` longer ones of `each`. An XCD
// has an eighth of each, whatever the others do: 102 and 768 tiles of 512 x 768 x 65536 look
// better than 96 and 768 on 256 units (65 stages and 68), but not on 32 (214 us and 175).
int64_t finish(int64_t all, int64_t each, int64_t all_more, int64_t more_each) {
  constexpr int64_t kOwn = kUnits / kXcds;
  const int64_t tiles = ceil_div(all, kXcds), more = ceil_div(all_more, kXcds);
  const int64_t whole = tiles / kOwn * each, late = tiles % kOwn, at = whole + (late ? each : 0);
  for (int64_t k = std::max((at - whole) / more_each, more / kOwn);; ++k) {   // before, too few are done
    const int64_t t = std::max(at, whole + k * more_each);
    if ((kOwn - late) * ((t - whole) / more_each) + late * ((t - at) / more_each) >= more) return t;
  }
}
Plan plan(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  Plan p{};
  p.channels = (c - 1) % 256 < 128 ? 128 : 256;
  p.padded_rows = up(rows, kGradTile);
  p.pitch = up(c, 4);
  const int64_t channel_tiles = ceil_div(c, p.channels), planes = planes_of(rows, vocab, c, bf16);
  const int64_t all = up(vocab, kWholeWords);
  const int64_t most = std::max<int64_t>(kWholeWords, kMaxD / (p.padded_rows * 2 * planes) / kWholeWords * kWholeWords);
  p.pieces = ceil_div(all, most);
  p.words = up(ceil_div(all, p.pieces), kWholeWords);
  p.pieces = ceil_div(all, p.words);
  if (few(rows, vocab, c, bf16)) {
    const int64_t splits = std::max<int64_t>(kUnits / (channel_tiles * ceil_div(rows, Few::kRows)), 1);
    p.share = up(ceil_div(p.words, splits), kStep);
    p.splits = ceil_div(p.words, p.share);
    p.row_splits = 1;
    p.row_share = up(rows, kStep);
    return p;
  }
  const int64_t weight_tiles = channel_tiles * ceil_div(p.words, kGradTile), hidden_tiles = channel_tiles * p.padded_rows / kGradTile;
  const int64_t parts = bf16 ? 1 : 3;
  int64_t least = INT64_MAX;
  for (int64_t r = 1; r <= (p.pieces == 1 ? kMaxSplits : 1); r *= 2) {
    const int64_t row_share = up(ceil_div(rows, r), kStep), row_splits = ceil_div(rows, row_share);
    if (row_splits < r) break;
    const int64_t weight_time = row_share / kStep * parts + kOverhead;
    const int64_t weight_moved = row_splits > 1 ? kLaunch + row_splits * vocab * p.pitch * 8 / kBytesPerStage : 0;
    for (int64_t s = 1; s <= kMaxSplits; ++s) {
      const int64_t share = up(ceil_div(p.words, s), kStep), splits = ceil_div(p.words, share);
      if (splits < s) continue;
      const int64_t hidden_time = share / kStep * parts + kOverhead;
      const int64_t moved = (bf16 || splits > 1 ? kLaunch + splits * rows * p.pitch * 8 / kBytesPerStage : 0) + weight_moved;
      if (moved >= least) break;
      const int64_t time = moved + (hidden_time > weight_time ? finish(hidden_tiles * splits, hidden_time, weight_tiles * row_splits, weight_time)
                                                              : finish(weight_tiles * row_splits, weight_time, hidden_tiles * splits, hidden_time));
      if (time >= least) continue;
      least = time;
      p.splits = splits;
      p.share = share;
      p.row_splits = row_splits;
      p.row_share = row_share;
      p.hidden_first = hidden_time > weight_time;
    }
  }
  return p;
}

// dx goes by way of sums, unless one workgroup has the whole of a row's, no row is left out
// and nothing is put back, which a tile's end would wait for (96 x 256 x 256 in bf16 45 us
// then, 41 with the launch).
bool needs_sums(const Plan& p, int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  return bf16 || p.splits > 1 || p.pieces > 1 || numbered(rows, vocab, c, bf16);
}
struct BackwardPlaces {
  Places operands;
  int64_t d, d_plane, sums, weight_sums, residuals, row_scale, end;
};
BackwardPlaces backward_places(const Plan& p, int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  BackwardPlaces b{};
  b.operands = operands(rows, vocab, c, bf16, true);
  b.end = b.operands.end;
  b.d_plane = p.padded_rows * p.words * 2;
  b.d = take(b.end, b.d_plane * planes_of(rows, vocab, c, bf16));
  b.sums = !needs_sums(p, rows, vocab, c, bf16) ? 0 : take(b.end, p.splits * rows * p.pitch * 4);
  b.weight_sums = p.row_splits == 1 ? 0 : take(b.end, p.row_splits * vocab * p.pitch * 4);
  b.residuals = take(b.end, 2 * rows * 4);
  b.row_scale = take(b.end, rows * 4);
  return b;
}

// The tile with which the logits are done first: as many workgroups as there are places
// for them take the tiles in turn, each `first` and `stage` times the steps of a tile, in
// ns.
enum { kBig, kMiddle, kSmall, kDeep, kFew, kFewSmall };
struct Shape {
  int words, rows, places;
  int64_t first, stage;
};
constexpr Shape kShapes[] = {{Big::kWords, Big::kRows, kUnits * Big::kEach, 6000, 1200},
                             {Middle::kWords, Middle::kRows, kUnits * Middle::kEach, 4000, 900},
                             {Small::kWords, Small::kRows, kUnits * Small::kEach, 3000, 700},
                             {Deep::kWords, Deep::kRows, kUnits * Deep::kEach, 13000, 200},
                             {Few::kWords, Few::kRows, kUnits * Few::kEach, 2000, 1300},
                             {FewSmall::kWords, FewSmall::kRows, kUnits * FewSmall::kEach, 2000, 700}};
int shape_of(int64_t rows, int64_t words, int64_t c, bool bf16, bool split) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = split ? kFew : kBig; i <= (split ? kFewSmall : kDeep); ++i) {
    const Shape& t = kShapes[i];
    const int64_t tiles = ceil_div(words, t.words) * ceil_div(rows, t.rows);
    const int64_t stages = split ? ceil_div(c, kFewStep) : ceil_div(c, kStep) * (bf16 ? 1 : 3);
    const int64_t time = ceil_div(tiles, t.places) * (t.first + t.stage * stages);
    if (time >= least) continue;
    least = time;
    best = i;
  }
  return best;
}
int shape_words(int shape) { return kShapes[shape].words; }

struct ForwardPlaces {
  Places operands;
  int64_t part_max, part_sum, part_argmax, row_target, end;
};
ForwardPlaces forward_places(int64_t rows, int64_t vocab, int64_t c, bool bf16) {
  ForwardPlaces f{};
  f.operands = operands(rows, vocab, c, bf16, false);
  f.end = f.operands.end;
  const int64_t parts = ceil_div(vocab, shape_words(shape_of(rows, vocab, c, bf16, few(rows, vocab, c, bf16)))) * rows * 4;
  f.part_max = take(f.end, parts);
  f.part_sum = take(f.end, parts);
  f.part_argmax = take(f.end, parts);
  f.row_target = take(f.end, rows * 4);
  return f;
}

// x and w as the tiles read them, and x as the weight gradient does (in fp16, with the rows'
// powers of two), made first where they are not so in memory; the rows' numbers; the
// backward's factors.
struct Operands {
  Matrix x, w, x_weighted;
  const int *index, *place, *count;
};
template <bool BF>
Operands prepare(const Call& c, const Places& p, const BackwardCall* b, float* residuals, int* row_scale, hipStream_t s) {
  const int64_t padded = up(c.c, kStep);
  Operands o{};
  o.x = Matrix{static_cast<const char*>(c.hidden), c.c * 2, 0};
  o.w = Matrix{static_cast<const char*>(c.weight), c.c * (BF ? 2 : 4), 0};
  const bool split = few(c.rows, c.vocab, c.c, BF);
  RowsCall r{c.targets, c.ignore_index, static_cast<int>(c.rows), nullptr, nullptr, nullptr};
  if (numbered(c.rows, c.vocab, c.c, BF)) {
    o.index = r.index = reinterpret_cast<int*>(c.workspace + p.index);
    o.place = r.place = reinterpret_cast<int*>(c.workspace + p.place);
    o.count = r.count = reinterpret_cast<int*>(c.workspace + p.count);
  }
  PackCall k{};
  auto pack = [&](const void* from, int64_t to, int64_t rows, int kind, int which, int64_t plane, bool weighted = false) {
    k.job[k.jobs++] = PackJob{from, c.workspace + to, rows, kind, which, weighted};
    return Matrix{c.workspace + to, padded * 2, plane};
  };
  if (packed(c.c, BF) || r.index) o.x = pack(c.hidden, p.x, c.rows, BF ? kCopy : split ? kToThirds : kToHalves, 0, p.x_plane);
  if (split && c.c % 8 != 0) {
    k.job[k.jobs++] = PackJob{c.weight, c.workspace + p.w, c.vocab, kEights, 1, false};
    o.w = Matrix{c.workspace + p.w, up(c.c, 8) * 4, 0};
  }
  if (packed(c.c, BF) && !split) o.w = pack(c.weight, p.w, c.vocab, BF ? kCopy : kToHalves, 1, p.w_plane);
  o.x_weighted = o.x;
  if (b && b->weight_grad && !split) o.x_weighted = pack(c.hidden, p.x_weighted, c.rows, BF ? kToHalf : kToHalves, 0, BF ? 0 : p.x_plane, true);
  if (k.jobs == 0 && !b) return o;
  k.c = static_cast<int>(c.c);
  k.padded = static_cast<int>(padded);
  k.factors = b != nullptr;
  k.row_scale = row_scale;
  k.index = o.index;
  k.count = o.count;
  uint32_t* const largest = reinterpret_cast<uint32_t*>(c.workspace + p.largest);
  k.largest = largest;
  k.scalars = reinterpret_cast<Scalars*>(c.workspace + p.scalars);
  SurveyCall v{};
  if ((!BF && !split) || (b && BF && b->weight_grad)) v.from[0] = c.hidden;
  if (!BF && !split) v.from[1] = c.weight;
  v.n[0] = c.rows;
  v.n[1] = c.vocab;
  v.c = c.c;
  v.largest = largest;
  v.numbered = r;
  k.targets = v.targets = c.targets;
  k.ignore_index = v.ignore_index = c.ignore_index;
  if (b) {
    v.row_grad = b->row_grad;
    v.row_max = b->row_max;
    v.rows = c.rows;
    v.l2wrap_scale = b->l2wrap_scale;
    v.residuals = residuals;
    v.row_scale = row_scale;
    v.own_scales = !split;
  }
  if (v.from[0] || b) hipLaunchKernelGGL(survey_kernel<BF>, dim3(kMaxBlocks, r.index ? 4 : b ? 3 : 2), dim3(kWide), 0, s, v);
  else if (r.index) hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(kWide), 0, s, r);
  int64_t rows = 1;
  for (int i = 0; i < k.jobs; ++i) rows = std::max(rows, k.job[i].rows);
  hipLaunchKernelGGL(pack_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(rows, 4), 2048)), std::max(k.jobs, 1)),
                     dim3(256), 0, s, k);
  return o;
}

// workgroups of 256 for n threads; a launch has fewer than 2^32 of these
dim3 grid_of(int64_t n) { return dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(n, 256), 1 << 22))); }

template <bool BF, bool kBackward, typename Shape>
void logits(const LogitsCall& l, hipStream_t s) {
  const int64_t tiles = l.words / Shape::kWords * ceil_div(l.rows, Shape::kRows);
  hipLaunchKernelGGL((logits_kernel<BF, kBackward, Shape>), dim3(static_cast<unsigned>(std::min<int64_t>(tiles, kUnits * Shape::kEach))),
                     dim3(64 * Shape::kWavesP * Shape::kWavesQ), 0, s, l);
}
template <bool BF, bool kBackward>
void logits(const LogitsCall& l, int shape, hipStream_t s) {
  if constexpr (!BF) {
    if (shape == kFew) return logits<BF, kBackward, Few>(l, s);
    if (shape == kFewSmall) return logits<BF, kBackward, FewSmall>(l, s);
  }
  if (shape == kBig) logits<BF, kBackward, Big>(l, s);
  else if (shape == kMiddle) logits<BF, kBackward, Middle>(l, s);
  else if (shape == kSmall) logits<BF, kBackward, Small>(l, s);
  else logits<BF, kBackward, Deep>(l, s);
}

template <bool BF>
void forward(const ForwardCall& c, hipStream_t s) {
  const ForwardPlaces f = forward_places(c.rows, c.vocab, c.c, BF);
  const Operands o = prepare<BF>(c, f.operands, nullptr, nullptr, nullptr, s);
  LogitsCall l{};
  l.x = o.x;
  l.w = o.w;
  l.index = o.index;
  l.count = o.count;
  l.rows = static_cast<int>(c.rows);
  l.vocab = static_cast<int>(c.vocab);
  l.c = static_cast<int>(up(c.c, 8));
  l.steps = static_cast<int>(up(c.c, few(c.rows, c.vocab, c.c, BF) ? kFewStep : kStep));
  l.words = static_cast<int>(up(c.vocab, kWholeWords));
  l.scalars = reinterpret_cast<const Scalars*>(c.workspace + f.operands.scalars);
  l.targets = c.targets;
  l.part_max = reinterpret_cast<float*>(c.workspace + f.part_max);
  l.part_sum = reinterpret_cast<float*>(c.workspace + f.part_sum);
  l.part_argmax = reinterpret_cast<int*>(c.workspace + f.part_argmax);
  l.row_target = reinterpret_cast<float*>(c.workspace + f.row_target);
  const int shape = shape_of(c.rows, c.vocab, c.c, BF, few(c.rows, c.vocab, c.c, BF));
  logits<BF, false>(l, shape, s);
  const JoinCall j{l.part_max, l.part_sum, l.row_target, l.part_argmax, c.targets, o.place, c.rows, c.vocab, c.ignore_index, shape_words(shape),
                   c.row_loss, c.row_log_sum, c.row_max, c.row_argmax};
  hipLaunchKernelGGL(join_kernel, dim3(static_cast<unsigned>(ceil_div(c.rows, kJoinRows))), dim3(kJoinRows * kJoinShares), 0, s, j);
}

template <int kChannels>
void few_gradients(const GradientsCall& g, hipStream_t s) {
  const dim3 weight(static_cast<unsigned>(g.weight_blocks)), hidden(static_cast<unsigned>(g.hidden_blocks));
  if (g.weight_blocks) hipLaunchKernelGGL(few_weight_kernel<kChannels>, weight, dim3(kThreads), 0, s, g);
  if (g.hidden_blocks) hipLaunchKernelGGL(few_hidden_kernel<kChannels>, hidden, dim3(64 * Few::kWavesP), 0, s, g);
}

template <bool BF>
void backward(const BackwardCall& c, hipStream_t s) {
  const Plan p = plan(c.rows, c.vocab, c.c, BF);
  const BackwardPlaces b = backward_places(p, c.rows, c.vocab, c.c, BF);
  float* const residuals = BF ? reinterpret_cast<float*>(c.workspace + b.residuals) : nullptr;
  int* const row_scale = reinterpret_cast<int*>(c.workspace + b.row_scale);
  const Operands o = prepare<BF>(c, b.operands, &c, residuals, row_scale, s);
  const Scalars* const scalars = reinterpret_cast<const Scalars*>(c.workspace + b.operands.scalars);
  LogitsCall l{};
  l.x = o.x;
  l.w = o.w;
  l.index = o.index;
  l.count = o.count;
  l.rows = static_cast<int>(c.rows);
  l.vocab = static_cast<int>(c.vocab);
  l.c = static_cast<int>(up(c.c, 8));
  l.steps = static_cast<int>(up(c.c, few(c.rows, c.vocab, c.c, BF) ? kFewStep : kStep));
  l.scalars = scalars;
  l.targets = c.targets;
  l.ignore_index = c.ignore_index;
  l.row_log_sum = c.row_log_sum;
  l.row_max = c.row_max;
  l.row_grad = c.row_grad;
  l.row_argmax = c.row_argmax;
  l.row_scale = row_scale;
  l.l2wrap_scale = c.l2wrap_scale;
  l.d = c.workspace + b.d;
  l.d_plane = b.d_plane;
  l.residuals = residuals;
  GradientsCall g{};
  g.x = o.x_weighted;
  g.w = o.w;
  g.count = o.count;
  g.d = l.d;
  g.d_plane = l.d_plane;
  g.padded_rows = static_cast<int>(p.padded_rows);
  g.rows = l.rows;
  g.vocab = l.vocab;
  g.c = static_cast<int>(c.c);
  g.scalars = scalars;
  g.weight_grad = c.weight_grad;
  g.row_share = static_cast<int>(p.row_share);
  g.weight_sums = p.row_splits == 1 ? nullptr : reinterpret_cast<float*>(c.workspace + b.weight_sums);
  g.share = static_cast<int>(p.share);
  const bool direct = !needs_sums(p, c.rows, c.vocab, c.c, BF);
  g.sums = direct ? nullptr : reinterpret_cast<float*>(c.workspace + b.sums);
  g.hidden = HiddenCall{c.hidden_grad, c.c, c.rows, residuals, c.targets, c.row_argmax, row_scale,
                        BF ? static_cast<const __bf16*>(c.weight) : nullptr};
  g.pitch = static_cast<int>(p.pitch);
  const int64_t channel_tiles = ceil_div(c.c, p.channels);
  for (int64_t first = 0; first < c.vocab; first += p.words) {
    g.first = l.first = static_cast<int>(first);
    g.words = l.words = static_cast<int>(std::min(p.words, up(c.vocab - first, kWholeWords)));
    logits<BF, true>(l, shape_of(c.rows, l.words, c.c, BF, few(c.rows, c.vocab, c.c, BF)), s);
    g.begin = first == 0;
    g.weight_tiles = c.weight_grad ? static_cast<int>(channel_tiles * (l.words / kGradTile) * p.row_splits) : 0;
    g.weight_blocks = static_cast<int>(up(g.weight_tiles, kXcds));
    const int64_t row_tiles = ceil_div(c.rows, few(c.rows, c.vocab, c.c, BF) ? Few::kRows : kGradTile);
    g.hidden_blocks = c.hidden_grad ? static_cast<int>(up(channel_tiles * row_tiles * ceil_div(l.words, p.share), kXcds)) : 0;
    g.hidden_first = p.hidden_first;
    const dim3 grid(static_cast<unsigned>(g.weight_blocks + g.hidden_blocks));
    if constexpr (!BF) {
      if (few(c.rows, c.vocab, c.c, BF)) {
        if (p.channels == 128) few_gradients<128>(g, s);
        else few_gradients<256>(g, s);
        continue;
      }
    }
    if (p.channels == 128) hipLaunchKernelGGL((gradients_kernel<BF, 128>), grid, dim3(kThreads), 0, s, g);
    else hipLaunchKernelGGL((gradients_kernel<BF, 256>), grid, dim3(kThreads), 0, s, g);
  }
  SumCall u{};
  u.hidden_sums = c.hidden_grad ? g.sums : nullptr;
  u.weight_sums = c.weight_grad ? g.weight_sums : nullptr;
  if (u.hidden_sums || u.weight_sums) {
    u.rows = c.rows;
    u.vocab = c.vocab;
    u.pitch = p.pitch;
    u.splits = static_cast<int>(p.splits);
    u.row_splits = static_cast<int>(p.row_splits);
    u.place = o.place;
    u.scalars = scalars;
    u.hidden = g.hidden;
    u.weight_grad = c.weight_grad;
    dim3 grid = grid_of(std::max(u.hidden_sums ? c.rows : 0, u.weight_sums ? c.vocab : 0) * p.pitch / 4);
    grid.y = u.weight_sums ? 2 : 1;
    hipLaunchKernelGGL(sum_kernel<BF>, grid, dim3(256), 0, s, u);
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
    const int64_t n = c.vocab * c.c;
    if (c.bf16) hipLaunchKernelGGL(clear_kernel<uint16_t>, grid_of(n), dim3(256), 0, s, static_cast<uint16_t*>(c.weight_grad), n);
    else hipLaunchKernelGGL(clear_kernel<uint32_t>, grid_of(n), dim3(256), 0, s, static_cast<uint32_t*>(c.weight_grad), n);
  } else {
    c.bf16 ? backward<true>(c, s) : backward<false>(c, s);
  }
  return hipGetLastError();
}

}  // namespace rwkv_linear_loss
