// Launchers of the token score kernels (token_scores.hip); the C ABI
// (token_scores_api.cpp) checks every argument before it calls them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rwkv_scores {

struct ForwardCall {
  const void* logits;        // [rows, vocab]
  const int64_t* tokens;     // [rows]
  int64_t rows, vocab;
  int top;
  bool bf16;
  float *log_prob, *entropy, *row_max, *log_sum, *top_log_probs;   // row_max, log_sum: may be null
  int64_t* top_ids;
};
struct BackwardCall {
  const void* logits;
  const int64_t* tokens;
  const float *row_max, *log_sum, *entropy;
  const int64_t* top_ids;
  const float *log_prob_grad, *entropy_grad, *top_grad;   // each may be null: zeros
  int64_t rows, vocab;
  int top;
  bool bf16;
  void* logits_grad;
};

hipError_t launch_forward(const ForwardCall& c, hipStream_t s);
hipError_t launch_backward(const BackwardCall& c, hipStream_t s);

}  // namespace rwkv_scores
