// C ABI of the token scores (include/rwkv_token_scores.h): argument checks on
// the host, before any HIP call, and dispatch.
#include "../../include/rwkv_token_scores.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "token_scores_launch.hpp"
#include "wkv7_launch.hpp"

namespace {

struct Range {
  const void* p;
  int64_t bytes;
};
typedef std::initializer_list<Range> Ranges;

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool overlaps(const Range& x, const Range& y) {
  if (!x.p || !y.p || x.bytes <= 0 || y.bytes <= 0) return false;
  const auto a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
  return a < b + static_cast<uintptr_t>(y.bytes) && b < a + static_cast<uintptr_t>(x.bytes);
}
// every output against every other output and every input
bool any_overlap(Ranges outs, Ranges ins) {
  for (const Range* o = outs.begin(); o != outs.end(); ++o) {
    for (const Range* i = o + 1; i != outs.end(); ++i)
      if (overlaps(*o, *i)) return true;
    for (const Range& i : ins)
      if (overlaps(*o, i)) return true;
  }
  return false;
}

bool sizes_ok(int64_t rows, int64_t vocab, int64_t top) {
  if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > INT32_MAX) return false;
  if (rows > 0 && vocab > INT64_MAX / 4 / rows) return false;   // byte sizes fit int64
  return top >= 0 && top <= RWKV_TOKEN_SCORES_MAX_TOP && top <= vocab;
}
int64_t size_of(int dtype) { return dtype == WKV7_DTYPE_BF16 ? 2 : 4; }

}  // namespace

extern "C" {

int rwkv_token_scores_forward(const void* logits, const int64_t* tokens, int64_t rows, int64_t vocab,
                              int64_t top, int dtype, float* log_prob, float* entropy, float* row_max,
                              float* row_log_sum, float* top_log_probs, int64_t* top_ids, void* stream) {
  if (dtype != WKV7_DTYPE_F32 && dtype != WKV7_DTYPE_BF16) return WKV7_ERR_DTYPE;
  if (!sizes_ok(rows, vocab, top)) return WKV7_ERR_SHAPE;
  if (rows == 0) return WKV7_OK;
  if (!logits || !tokens || !log_prob || !entropy ||
      (top > 0 && (!top_log_probs || !top_ids)))
    return WKV7_ERR_NULL_POINTER;
  if (!aligned(logits, size_of(dtype)) || !aligned(tokens, 8) || !aligned(log_prob, 4) || !aligned(entropy, 4) ||
      !aligned(row_max, 4) || !aligned(row_log_sum, 4) || (top > 0 && (!aligned(top_log_probs, 4) || !aligned(top_ids, 8))))
    return WKV7_ERR_ALIGNMENT;
  const int64_t rb = rows * 4;
  if (any_overlap({{log_prob, rb}, {entropy, rb}, {row_max, rb}, {row_log_sum, rb}, {top_log_probs, rb * top},
                   {top_ids, 2 * rb * top}},
                  {{logits, rows * vocab * size_of(dtype)}, {tokens, rows * 8}}))
    return WKV7_ERR_OVERLAP;
  rwkv_scores::ForwardCall c{};
  c.logits = logits;
  c.tokens = tokens;
  c.rows = rows;
  c.vocab = vocab;
  c.top = static_cast<int>(top);
  c.bf16 = dtype == WKV7_DTYPE_BF16;
  c.log_prob = log_prob;
  c.entropy = entropy;
  c.row_max = row_max;
  c.log_sum = row_log_sum;
  c.top_log_probs = top_log_probs;
  c.top_ids = top_ids;
  return wkv7::hip_status(rwkv_scores::launch_forward(c, static_cast<hipStream_t>(stream)));
}

int rwkv_token_scores_backward(const void* logits, const int64_t* tokens, const float* row_max,
                               const float* row_log_sum, const float* entropy, const int64_t* top_ids, const float* log_prob_grad,
                               const float* entropy_grad, const float* top_grad, int64_t rows, int64_t vocab,
                               int64_t top, int dtype, void* logits_grad, void* stream) {
  if (dtype != WKV7_DTYPE_F32 && dtype != WKV7_DTYPE_BF16) return WKV7_ERR_DTYPE;
  if (!sizes_ok(rows, vocab, top)) return WKV7_ERR_SHAPE;
  if (rows == 0) return WKV7_OK;
  if (!logits || !tokens || !row_max || !row_log_sum || !entropy || !logits_grad || (top > 0 && top_grad && !top_ids))
    return WKV7_ERR_NULL_POINTER;
  if (!aligned(logits, size_of(dtype)) || !aligned(logits_grad, size_of(dtype)) || !aligned(tokens, 8) ||
      !aligned(row_max, 4) || !aligned(row_log_sum, 4) || !aligned(entropy, 4) || !aligned(top_ids, 8) || !aligned(log_prob_grad, 4) ||
      !aligned(entropy_grad, 4) || !aligned(top_grad, 4))
    return WKV7_ERR_ALIGNMENT;
  const int64_t rb = rows * 4, lb = rows * vocab * size_of(dtype);
  if (any_overlap({{logits_grad, lb}},
                  {{logits, lb}, {tokens, rows * 8}, {row_max, rb}, {row_log_sum, rb}, {entropy, rb}, {top_ids, 2 * rb * top},
                   {log_prob_grad, rb}, {entropy_grad, rb}, {top_grad, rb * top}}))
    return WKV7_ERR_OVERLAP;
  rwkv_scores::BackwardCall c{};
  c.logits = logits;
  c.tokens = tokens;
  c.row_max = row_max;
  c.log_sum = row_log_sum;
  c.entropy = entropy;
  c.top_ids = top_ids;
  c.log_prob_grad = log_prob_grad;
  c.entropy_grad = entropy_grad;
  c.top_grad = top_grad;
  c.rows = rows;
  c.vocab = vocab;
  c.top = top_grad ? static_cast<int>(top) : 0;
  c.bf16 = dtype == WKV7_DTYPE_BF16;
  c.logits_grad = logits_grad;
  return wkv7::hip_status(rwkv_scores::launch_backward(c, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
