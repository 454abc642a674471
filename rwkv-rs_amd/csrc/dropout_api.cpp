// C ABI of the dropout (include/rwkv_dropout.h): argument checks on the host, before
// any HIP call, and dispatch.
#include "../../include/rwkv_dropout.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "dropout_launch.hpp"
#include "wkv7_launch.hpp"

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool overlaps(const void* x, int64_t nx, const void* y, int64_t ny) {
  if (!x || !y) return false;
  const auto a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
  return a < b + static_cast<uintptr_t>(ny) && b < a + static_cast<uintptr_t>(nx);
}

bool dtype_ok(int dtype) { return dtype == WKV7_DTYPE_F32 || dtype == WKV7_DTYPE_BF16; }
int64_t size_of(int dtype) { return dtype == WKV7_DTYPE_BF16 ? 2 : 4; }

}  // namespace

extern "C" {

int rwkv_dropout(const void* x, const void* residual, const int64_t* rng, int64_t site, double p, int64_t n,
                 int dtype, int out_dtype, void* out, void* stream) {
  if (!dtype_ok(dtype) || !dtype_ok(out_dtype)) return WKV7_ERR_DTYPE;
  if (n < 0 || n > RWKV_DROPOUT_MAX_N || site < 0 || site > UINT32_MAX || !(p >= 0.0 && p <= 1.0)) return WKV7_ERR_SHAPE;
  if (n == 0) return WKV7_OK;
  if (!x || !rng || !out) return WKV7_ERR_NULL_POINTER;
  if (!aligned(x, size_of(dtype)) || !aligned(residual, size_of(out_dtype)) || !aligned(out, size_of(out_dtype)) ||
      !aligned(rng, 8))
    return WKV7_ERR_ALIGNMENT;
  const int64_t bytes = n * size_of(out_dtype);
  if (overlaps(out, bytes, x, n * size_of(dtype)) || overlaps(out, bytes, residual, bytes) || overlaps(out, bytes, rng, 16))
    return WKV7_ERR_OVERLAP;
  rwkv_drop::Call c{};
  c.x = x;
  c.residual = residual;
  c.rng = rng;
  c.site = static_cast<uint32_t>(site);
  c.threshold = static_cast<uint32_t>(std::nearbyint((1.0 - p) * 65536.0));
  c.n = n;
  c.bf16 = dtype == WKV7_DTYPE_BF16;
  c.out_bf16 = out_dtype == WKV7_DTYPE_BF16;
  c.out = out;
  return wkv7::hip_status(rwkv_drop::launch(c, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
