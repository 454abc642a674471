// Launcher of the dropout kernel (dropout.hip); the C ABI (dropout_api.cpp) checks
// every argument before it calls it.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rwkv_drop {

struct Call {
  const void *x, *residual;    // residual: may be null
  const int64_t* rng;
  uint32_t site, threshold;    // kept: numbers below it, of 65536
  int64_t n;
  bool bf16, out_bf16;
  void* out;
};

// n > 0
hipError_t launch(const Call& c, hipStream_t s);

}  // namespace rwkv_drop
