// Launchers of the loss from hidden states and unembedding (linear_loss.hip); the C
// ABI (linear_loss_api.cpp) checks every argument before it calls them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rwkv_linear_loss {

struct Call {
  const void *hidden, *weight;   // [rows, c], [vocab, c]
  const int64_t* targets;
  int64_t rows, vocab, c, ignore_index;
  bool bf16;
  char* workspace;
};
struct ForwardCall : Call {
  float *row_loss, *row_log_sum, *row_max;
  int32_t* row_argmax;
};
struct BackwardCall : Call {
  const float *row_log_sum, *row_max;
  const int32_t* row_argmax;
  const float* row_grad;
  float l2wrap_scale;
  void *hidden_grad, *weight_grad;   // each may be null
};

int64_t forward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, bool bf16);
int64_t backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, bool bf16);
// rows > 0
hipError_t launch_forward(const ForwardCall& c, hipStream_t s);
hipError_t launch_backward(const BackwardCall& c, hipStream_t s);

}  // namespace rwkv_linear_loss
