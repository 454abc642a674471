// Launchers of the 4-bit weight kernels (w4.hip); the C ABI (w4_api.cpp)
// checks every argument before it calls them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rwkv_w4 {

constexpr int kRows = 16, kInputs = 128;   // of a block of packed weights

constexpr int64_t blocks_out(int64_t out) { return (out + kRows - 1) / kRows; }
constexpr int64_t blocks_in(int64_t in) { return (in + kInputs - 1) / kInputs; }
constexpr int64_t packed_bytes(int64_t out, int64_t in) { return blocks_out(out) * blocks_in(in) * 1024; }
constexpr int64_t scales_bytes(int64_t out, int64_t in, int64_t group) {
  return blocks_out(out) * blocks_in(in) * kRows * (kInputs / group) * 2;
}

struct WeightCall {           // quantize: weight to packed and scales; dequantize: back
  void* weight;               // [out, in]
  void *packed, *scales;
  int64_t out, in;
  int group;
  bool bf16;
};
// What becomes of a product's results, rounded to y's type. The last two take bf16
// activations; kAddTo's y is the fp32 rows that the results are added to.
enum Finish { kStore, kSquaredRelu, kAddTo };
struct LinearCall {
  const void* x;              // [rows, in]
  const void *packed, *scales;
  void* y;                    // [rows, out]
  int64_t rows, out, in;
  int group;
  bool bf16;
  float* partial;             // workspace of workspace_bytes, or null: no inputs are shared among workgroups
  Finish finish;              // kStore with a workspace
};

hipError_t launch_quantize(const WeightCall& c, hipStream_t s);
hipError_t launch_dequantize(const WeightCall& c, hipStream_t s);
// What a product of these sizes asks for.
int64_t workspace_bytes(int64_t rows, int64_t out, int64_t in, bool bf16);
hipError_t launch_linear(const LinearCall& c, hipStream_t s);

}  // namespace rwkv_w4
