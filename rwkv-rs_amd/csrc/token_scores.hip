// Log probability of a given token, entropy and most likely alternatives of
// rows of logits, and their gradient (include/rwkv_token_scores.h).
//
// With M = max_j x_j and d_j = (x_j - M) log2(e): s = sum 2^d_j, u = sum 2^d_j d_j.
// Then log p_j = x_j - M - ln 2 log2 s and the entropy is ln 2 (log2 s - u / s).
// M is subtracted before the product, so that logits as low as the type goes
// (another form of a mask) stay in range and equal ones stay equal.
#include <climits>
#include <cmath>

#include "token_scores_launch.hpp"

namespace rwkv_scores {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// 2^kFloor is 0: what lies below adds nothing, and 0 times it is 0
constexpr float kFloor = -256.f;

template <bool BF>
__device__ __forceinline__ float load_one(const void* base, int64_t i) {
  if constexpr (BF) return __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(base)[i]) << 16);
  else return static_cast<const float*>(base)[i];
}

template <bool BF>
__device__ __forceinline__ void store_one(void* base, int64_t i, float v) {
  if constexpr (BF) static_cast<__bf16*>(base)[i] = static_cast<__bf16>(v);
  else static_cast<float*>(base)[i] = v;
}

// a logit with its index; the larger logit is before, then the lower index
struct Item {
  float x;
  int j;
};
__device__ __forceinline__ bool before(const Item& a, const Item& b) { return a.x > b.x || (a.x == b.x && a.j < b.j); }

__device__ __forceinline__ float exchange(float v, int o) { return __shfl_xor(v, o); }
__device__ __forceinline__ Item exchange(const Item& v, int o) { return {__shfl_xor(v.x, o), __shfl_xor(v.j, o)}; }

// v of all threads joined by f, in every thread
template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* part, F f) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v = f(v, exchange(v, o));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < kThreads / 64; ++w) v = f(v, part[w]);
  return v;
}

template <bool BF>
__global__ __launch_bounds__(kThreads) void forward_kernel(const ForwardCall c) {
  __shared__ float part[kThreads / 64];
  __shared__ Item item_part[kThreads / 64];
  const int64_t row = blockIdx.x, V = c.vocab, base = row * V;
  const int tid = threadIdx.x;
  float m = -INFINITY;
  for (int64_t j = tid; j < V; j += kThreads) m = fmaxf(m, load_one<BF>(c.logits, base + j));
  m = block_reduce(m, part, [](float a, float b) { return fmaxf(a, b); });
  float s = 0.f, u = 0.f;
  for (int64_t j = tid; j < V; j += kThreads) {
    const float d = (load_one<BF>(c.logits, base + j) - m) * kLog2E;
    const float e = __builtin_amdgcn_exp2f(d);
    s += e;
    u = fmaf(e, fmaxf(d, kFloor), u);
  }
  s = block_reduce(s, part, [](float a, float b) { return a + b; });
  u = block_reduce(u, part, [](float a, float b) { return a + b; });
  const bool valid = fabsf(m) < INFINITY && s == s;
  const float log_sum = logf(s);
  auto log_p = [&](float x) { return valid ? (x - m) - log_sum : NAN; };
  if (tid == 0) {
    const int64_t t = c.tokens[row];
    c.log_prob[row] = t >= 0 && t < V ? log_p(load_one<BF>(c.logits, base + t)) : NAN;
    c.entropy[row] = valid ? log_sum - kLn2 * (u / s) : NAN;
    c.row_max[row] = m;
    c.log_sum[row] = valid ? log_sum : NAN;
  }
  Item last{INFINITY, -1};
  for (int i = 0; i < c.top; ++i) {
    Item best{-INFINITY, INT_MAX};
    for (int64_t j = tid; j < V; j += kThreads) {
      const Item x{load_one<BF>(c.logits, base + j), static_cast<int>(j)};
      if (before(last, x) && before(x, best)) best = x;
    }
    last = block_reduce(best, item_part, [](Item a, Item b) { return before(a, b) ? a : b; });
    if (tid == 0) {
      c.top_log_probs[row * c.top + i] = log_p(last.x);
      c.top_ids[row * c.top + i] = valid ? last.j : -1;
    }
  }
}

// the gradient of logit j, but for the terms of the token and the alternatives
struct RowGrad {
  float m, log_sum, total, h, entropy;
  __device__ __forceinline__ float at(float x) const {
    const float d = (x - m) - log_sum, p = __builtin_amdgcn_exp2f(d * kLog2E);
    return p == 0.f ? 0.f : -p * fmaf(h, d + entropy, total);
  }
};

template <bool BF>
__global__ __launch_bounds__(kThreads) void backward_kernel(const BackwardCall c) {
  const int64_t row = blockIdx.x, V = c.vocab, base = row * V;
  const int tid = threadIdx.x;
  const float g = c.log_prob_grad ? c.log_prob_grad[row] : 0.f;
  RowGrad r;
  r.m = c.row_max[row];
  r.log_sum = c.log_sum[row];
  r.total = g;
  for (int i = 0; i < c.top; ++i) r.total += c.top_grad[row * c.top + i];
  r.h = c.entropy_grad ? c.entropy_grad[row] : 0.f;
  r.entropy = c.entropy[row];
  for (int64_t j = tid; j < V; j += kThreads) store_one<BF>(c.logits_grad, base + j, r.at(load_one<BF>(c.logits, base + j)));
  __syncthreads();   // the token's and the alternatives' own terms: their gradient is written again
  const int64_t t = c.tokens[row];
  if (tid < c.top) {
    const int64_t j = c.top_ids[row * c.top + tid];
    if (j >= 0 && j < V) {
      float v = r.at(load_one<BF>(c.logits, base + j)) + c.top_grad[row * c.top + tid];
      if (j == t) v += g;
      store_one<BF>(c.logits_grad, base + j, v);
    }
  }
  if (tid == kThreads - 1 && t >= 0 && t < V) {
    bool among = false;
    for (int i = 0; i < c.top; ++i) among |= c.top_ids[row * c.top + i] == t;
    if (!among) store_one<BF>(c.logits_grad, base + t, r.at(load_one<BF>(c.logits, base + t)) + g);
  }
}

}  // namespace

int64_t workspace_bytes(int64_t rows, int64_t vocab, int64_t top) { return 0; }

hipError_t launch_forward(const ForwardCall& c, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(c.rows)), block(kThreads);
  if (c.bf16) hipLaunchKernelGGL(forward_kernel<true>, grid, block, 0, stream, c);
  else hipLaunchKernelGGL(forward_kernel<false>, grid, block, 0, stream, c);
  return hipGetLastError();
}

hipError_t launch_backward(const BackwardCall& c, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(c.rows)), block(kThreads);
  if (c.bf16) hipLaunchKernelGGL(backward_kernel<true>, grid, block, 0, stream, c);
  else hipLaunchKernelGGL(backward_kernel<false>, grid, block, 0, stream, c);
  return hipGetLastError();
}

}  // namespace rwkv_scores
