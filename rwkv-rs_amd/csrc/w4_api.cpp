// C ABI of the 4-bit weight products (include/rwkv_w4.h): argument checks on
// the host, before any HIP call, and dispatch.
#include "../../include/rwkv_w4.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "w4_launch.hpp"
#include "wkv7_launch.hpp"

namespace {

struct Range {
  const void* p;
  int64_t bytes;
};
typedef std::initializer_list<Range> Ranges;

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool overlaps(const Range& x, const Range& y) {
  if (x.bytes <= 0 || y.bytes <= 0) return false;
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

bool dims_ok(int64_t out, int64_t in) {
  return out > 0 && out <= RWKV_W4_MAX_DIM && in > 0 && in <= RWKV_W4_MAX_DIM &&
         rwkv_w4::blocks_out(out) * rwkv_w4::blocks_in(in) <= INT32_MAX;
}
bool group_ok(int64_t group) { return group == 32 || group == 64 || group == 128; }
int64_t size_of(int dtype) { return dtype == WKV7_DTYPE_BF16 ? 2 : 4; }
int check_weight(const void* weight, const void* packed, const void* scales, int64_t out, int64_t in,
                 int64_t group, int dtype) {
  if (dtype != WKV7_DTYPE_F32 && dtype != WKV7_DTYPE_BF16) return WKV7_ERR_DTYPE;
  if (!dims_ok(out, in) || !group_ok(group)) return WKV7_ERR_SHAPE;
  if (!weight || !packed || !scales) return WKV7_ERR_NULL_POINTER;
  if (!aligned(packed, 16) || !aligned(scales, 16) || !aligned(weight, size_of(dtype)))
    return WKV7_ERR_ALIGNMENT;
  return WKV7_OK;
}

rwkv_w4::WeightCall weight_call(const void* weight, const void* packed, const void* scales, int64_t out,
                                int64_t in, int64_t group, int dtype) {
  rwkv_w4::WeightCall c{};
  c.weight = const_cast<void*>(weight);
  c.packed = const_cast<void*>(packed);
  c.scales = const_cast<void*>(scales);
  c.out = out;
  c.in = in;
  c.group = static_cast<int>(group);
  c.bf16 = dtype == WKV7_DTYPE_BF16;
  return c;
}

}  // namespace

extern "C" {

int64_t rwkv_w4_packed_bytes(int64_t out, int64_t in) {
  return dims_ok(out, in) ? rwkv_w4::packed_bytes(out, in) : -1;
}

int64_t rwkv_w4_scales_bytes(int64_t out, int64_t in, int64_t group) {
  return dims_ok(out, in) && group_ok(group) ? rwkv_w4::scales_bytes(out, in, group) : -1;
}

int64_t rwkv_w4_linear_workspace_bytes(int64_t rows, int64_t out, int64_t in, int dtype) {
  if (rows < 0 || rows > RWKV_W4_MAX_ROWS || !dims_ok(out, in)) return -1;
  if (dtype != WKV7_DTYPE_F32 && dtype != WKV7_DTYPE_BF16) return -1;
  return rwkv_w4::workspace_bytes(rows, out, in, dtype == WKV7_DTYPE_BF16);
}

int rwkv_w4_quantize(const void* weight, int64_t out, int64_t in, int64_t group, int dtype, void* packed,
                     void* scales, void* stream) {
  if (int rc = check_weight(weight, packed, scales, out, in, group, dtype)) return rc;
  if (any_overlap({{packed, rwkv_w4::packed_bytes(out, in)}, {scales, rwkv_w4::scales_bytes(out, in, group)}},
                  {{weight, out * in * size_of(dtype)}}))
    return WKV7_ERR_OVERLAP;
  return wkv7::hip_status(rwkv_w4::launch_quantize(weight_call(weight, packed, scales, out, in, group, dtype),
                                                   static_cast<hipStream_t>(stream)));
}

int rwkv_w4_dequantize(const void* packed, const void* scales, int64_t out, int64_t in, int64_t group,
                       int dtype, void* weight, void* stream) {
  if (int rc = check_weight(weight, packed, scales, out, in, group, dtype)) return rc;
  if (any_overlap({{weight, out * in * size_of(dtype)}},
                  {{packed, rwkv_w4::packed_bytes(out, in)}, {scales, rwkv_w4::scales_bytes(out, in, group)}}))
    return WKV7_ERR_OVERLAP;
  return wkv7::hip_status(rwkv_w4::launch_dequantize(weight_call(weight, packed, scales, out, in, group, dtype),
                                                     static_cast<hipStream_t>(stream)));
}

int rwkv_w4_linear(const void* x, const void* packed, const void* scales, int64_t rows, int64_t out,
                   int64_t in, int64_t group, int dtype, void* y, void* workspace, int64_t workspace_bytes,
                   void* stream) {
  if (dtype != WKV7_DTYPE_F32 && dtype != WKV7_DTYPE_BF16) return WKV7_ERR_DTYPE;
  if (!dims_ok(out, in) || !group_ok(group) || rows < 0 || rows > RWKV_W4_MAX_ROWS) return WKV7_ERR_SHAPE;
  if (!packed || !scales || (rows > 0 && (!x || !y))) return WKV7_ERR_NULL_POINTER;
  if (!aligned(packed, 16) || !aligned(scales, 16) || !aligned(x, size_of(dtype)) ||
      !aligned(y, size_of(dtype)))
    return WKV7_ERR_ALIGNMENT;
  if (rows == 0) return WKV7_OK;
  const int64_t needed = rwkv_w4::workspace_bytes(rows, out, in, dtype == WKV7_DTYPE_BF16);
  if (workspace_bytes < needed) return WKV7_ERR_SHAPE;
  if (needed > 0 && !workspace) return WKV7_ERR_NULL_POINTER;
  if (needed > 0 && !aligned(workspace, 16)) return WKV7_ERR_ALIGNMENT;
  if (any_overlap({{y, rows * out * size_of(dtype)}, {workspace, needed}},
                  {{x, rows * in * size_of(dtype)}, {packed, rwkv_w4::packed_bytes(out, in)},
                   {scales, rwkv_w4::scales_bytes(out, in, group)}}))
    return WKV7_ERR_OVERLAP;
  rwkv_w4::LinearCall c{};
  c.x = x;
  c.packed = packed;
  c.scales = scales;
  c.y = y;
  c.rows = rows;
  c.out = out;
  c.in = in;
  c.group = static_cast<int>(group);
  c.bf16 = dtype == WKV7_DTYPE_BF16;
  c.partial = static_cast<float*>(workspace);
  return wkv7::hip_status(rwkv_w4::launch_linear(c, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
