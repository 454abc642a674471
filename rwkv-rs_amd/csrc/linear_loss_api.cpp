// C ABI of the loss from hidden states and unembedding
// (include/rwkv_linear_loss.h): argument checks on the host, before any HIP call,
// and dispatch.
#include "../../include/rwkv_linear_loss.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "linear_loss_launch.hpp"
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

bool sizes_ok(int64_t rows, int64_t vocab, int64_t c) {
  return rows >= 0 && rows <= RWKV_LINEAR_LOSS_MAX_ROWS && vocab > 0 && vocab <= RWKV_LINEAR_LOSS_MAX_VOCAB &&
         c > 0 && c <= RWKV_LINEAR_LOSS_MAX_C && rows * c <= RWKV_LINEAR_LOSS_MAX_ELEMENTS &&
         vocab * c <= RWKV_LINEAR_LOSS_MAX_ELEMENTS;
}
bool dtype_ok(int dtype) { return dtype == WKV7_DTYPE_F32 || dtype == WKV7_DTYPE_BF16; }
int64_t size_of(int dtype) { return dtype == WKV7_DTYPE_BF16 ? 2 : 4; }
uintptr_t row_alignment(int64_t c, int dtype) { return c % 8 == 0 ? 16 : static_cast<uintptr_t>(size_of(dtype)); }

}  // namespace

extern "C" {

int64_t rwkv_linear_loss_forward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, int dtype) {
  if (!dtype_ok(dtype) || !sizes_ok(rows, vocab, c)) return -1;
  return rwkv_linear_loss::forward_workspace_bytes(rows, vocab, c, dtype == WKV7_DTYPE_BF16);
}

int64_t rwkv_linear_loss_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, int dtype) {
  if (!dtype_ok(dtype) || !sizes_ok(rows, vocab, c)) return -1;
  return rwkv_linear_loss::backward_workspace_bytes(rows, vocab, c, dtype == WKV7_DTYPE_BF16);
}

int rwkv_linear_loss_forward(const void* hidden, const void* weight, const int64_t* targets, int64_t rows,
                             int64_t vocab, int64_t c, int dtype, int64_t ignore_index, float* row_loss,
                             float* row_log_sum, float* row_max, int32_t* row_argmax, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return WKV7_ERR_DTYPE;
  if (!sizes_ok(rows, vocab, c)) return WKV7_ERR_SHAPE;
  if (rows == 0) return WKV7_OK;
  const bool bf16 = dtype == WKV7_DTYPE_BF16;
  const int64_t need = rwkv_linear_loss::forward_workspace_bytes(rows, vocab, c, bf16);
  if (workspace_bytes < need) return WKV7_ERR_SHAPE;
  if (!hidden || !weight || !targets || !row_loss || !row_log_sum || !row_max || !row_argmax || !workspace)
    return WKV7_ERR_NULL_POINTER;
  const uintptr_t a = row_alignment(c, dtype);
  if (!aligned(hidden, a) || !aligned(weight, a) || !aligned(targets, 8) || !aligned(row_loss, 4) ||
      !aligned(row_log_sum, 4) || !aligned(row_max, 4) || !aligned(row_argmax, 4) || !aligned(workspace, 16))
    return WKV7_ERR_ALIGNMENT;
  const int64_t rb = rows * 4;
  if (any_overlap({{row_loss, rb}, {row_log_sum, rb}, {row_max, rb}, {row_argmax, rb}, {workspace, need}},
                  {{hidden, rows * c * size_of(dtype)}, {weight, vocab * c * size_of(dtype)}, {targets, rows * 8}}))
    return WKV7_ERR_OVERLAP;
  rwkv_linear_loss::ForwardCall f{};
  f.hidden = hidden;
  f.weight = weight;
  f.targets = targets;
  f.rows = rows;
  f.vocab = vocab;
  f.c = c;
  f.ignore_index = ignore_index;
  f.bf16 = bf16;
  f.workspace = static_cast<char*>(workspace);
  f.row_loss = row_loss;
  f.row_log_sum = row_log_sum;
  f.row_max = row_max;
  f.row_argmax = row_argmax;
  return wkv7::hip_status(rwkv_linear_loss::launch_forward(f, static_cast<hipStream_t>(stream)));
}

int rwkv_linear_loss_backward(const void* hidden, const void* weight, const int64_t* targets, const float* row_log_sum,
                              const float* row_max, const int32_t* row_argmax, const float* row_loss_grad,
                              float l2wrap_scale, int64_t rows, int64_t vocab, int64_t c, int dtype,
                              int64_t ignore_index, void* hidden_grad, void* weight_grad, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return WKV7_ERR_DTYPE;
  if (!sizes_ok(rows, vocab, c) || !std::isfinite(l2wrap_scale)) return WKV7_ERR_SHAPE;
  if (!hidden_grad && !weight_grad) return WKV7_OK;
  const bool bf16 = dtype == WKV7_DTYPE_BF16;
  const uintptr_t a = row_alignment(c, dtype);
  if (rows == 0 && !weight_grad) return WKV7_OK;
  const int64_t need = rwkv_linear_loss::backward_workspace_bytes(rows, vocab, c, bf16);
  if (workspace_bytes < need) return WKV7_ERR_SHAPE;
  if (rows > 0 && (!hidden || !weight || !targets || !row_log_sum || !row_max || !row_argmax || !row_loss_grad || !workspace))
    return WKV7_ERR_NULL_POINTER;
  if (!aligned(hidden, a) || !aligned(weight, a) || !aligned(hidden_grad, a) || !aligned(weight_grad, a) ||
      !aligned(targets, 8) || !aligned(row_log_sum, 4) || !aligned(row_max, 4) || !aligned(row_argmax, 4) ||
      !aligned(row_loss_grad, 4) || !aligned(workspace, 16))
    return WKV7_ERR_ALIGNMENT;
  const int64_t rb = rows * 4, hb = rows * c * size_of(dtype), wb = vocab * c * size_of(dtype);
  if (any_overlap({{hidden_grad, hb}, {weight_grad, wb}, {workspace, need}},
                  {{hidden, hb}, {weight, wb}, {targets, rows * 8}, {row_log_sum, rb}, {row_max, rb}, {row_argmax, rb},
                   {row_loss_grad, rb}}))
    return WKV7_ERR_OVERLAP;
  rwkv_linear_loss::BackwardCall b{};
  b.hidden = hidden;
  b.weight = weight;
  b.targets = targets;
  b.rows = rows;
  b.vocab = vocab;
  b.c = c;
  b.ignore_index = ignore_index;
  b.bf16 = bf16;
  b.workspace = static_cast<char*>(workspace);
  b.row_log_sum = row_log_sum;
  b.row_max = row_max;
  b.row_argmax = row_argmax;
  b.row_grad = row_loss_grad;
  b.l2wrap_scale = l2wrap_scale;
  b.hidden_grad = hidden_grad;
  b.weight_grad = weight_grad;
  return wkv7::hip_status(rwkv_linear_loss::launch_backward(b, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
