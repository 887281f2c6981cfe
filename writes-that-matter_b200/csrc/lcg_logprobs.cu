// Log probabilities of given tokens, the entropy of each row, and its most likely tokens.
//
// With m = max x, S = sum e^(x - m) and T = sum e^(x - m) (x - m) over a row (a masked value, -inf,
// adds nothing to either):  log p(token) = (x[token] - m) - ln S,  H = ln S - T / S.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "lcg_common.h"

namespace lcg {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Order of the alternatives: larger value first, lower id first among equals (0 and -0 alike); a
// NaN counts as -inf there (a row that holds one has no log probabilities at all).
__device__ __forceinline__ uint32_t order_key(float v) {
  v = v + 0.0f;
  if (v != v) v = -CUDART_INF_F;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long full_key(float v, uint32_t id) {
  return (static_cast<unsigned long long>(order_key(v)) << 32) | (0xffffffffu - id);
}

__device__ float block_max(float v, float* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, s[w]);
  return v;
}
__device__ float block_sum(float v, float* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < kThreads / 32; ++w) v += s[w];
  return v;
}

// One CTA per row, one pass for the maximum, one for the sums, one for each alternative.
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_token_logprobs(const T* __restrict__ logits, int64_t V, int64_t ld, const void* __restrict__ tokens, int token_bytes,
                 int top, float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_logprobs,
                 int64_t* __restrict__ top_ids) {
  __shared__ float s_red[32];
  __shared__ unsigned long long s_key[32];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  float m = -CUDART_INF_F;
  for (int64_t i = threadIdx.x; i < V; i += kThreads) m = fmaxf(m, to_float(x[i]));
  m = block_max(m, s_red);
  float S = 0.f, Tm = 0.f;
  for (int64_t i = threadIdx.x; i < V; i += kThreads) {
    const float v = to_float(x[i]);
    const float y = v - m;          // NaN where the row is all -inf, or holds +inf or NaN
    const float e = expf(y);
    S += e;
    if (v != -CUDART_INF_F && e != 0.f) Tm = fmaf(e, y, Tm);
  }
  S = block_sum(S, s_red);
  Tm = block_sum(Tm, s_red);
  const float lse = logf(S);
  if (threadIdx.x == 0) {
    const int64_t t = token_bytes == 8 ? static_cast<const int64_t*>(tokens)[row] : static_cast<const int32_t*>(tokens)[row];
    logprob[row] = t >= 0 && t < V ? (to_float(x[t]) - m) - lse : __int_as_float(0x7fc00000);
    entropy[row] = lse - Tm / S;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int64_t i = threadIdx.x; i < V; i += kThreads) {
      const unsigned long long key = full_key(to_float(x[i]), static_cast<uint32_t>(i));
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_key[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) best = max(best, s_key[w]);
    last = best;
    if (threadIdx.x == 0) {
      const uint32_t id = 0xffffffffu - static_cast<uint32_t>(best);
      top_ids[row * top + k] = id;
      top_logprobs[row * top + k] = (to_float(x[id]) - m) - lse;
    }
  }
}

}  // namespace
}  // namespace lcg

using namespace lcg;

extern "C" int lcg_token_logprobs(const void* logits, int dtype, int64_t M, int64_t V, int64_t ld, const void* tokens,
                                  int token_bytes, int top, float* logprob, float* entropy, float* top_logprobs,
                                  int64_t* top_ids, void* stream) {
  if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (M < 1 || M > 0x7fffffffLL || V < 1 || V > 0x7fffff00LL)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "bad extents M=%lld V=%lld", (long long)M, (long long)V);
  if (ld < V && M > 1) return fail(LCG_ERR_BAD_ARG, "leading dimension below extent");
  if (token_bytes != 4 && token_bytes != 8) return fail(LCG_ERR_BAD_ARG, "token ids must have 4 or 8 bytes");
  if (top < 0 || top > kMaxTop || top > V)
    return fail(LCG_ERR_BAD_ARG, "top must be between 0 and min(%d, V), got %d", kMaxTop, top);
  auto st = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(M);
  switch (dtype) {
    case LCG_DTYPE_BF16:
      k_token_logprobs<<<grid, kThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(logits), V, ld, tokens, token_bytes,
                                                  top, logprob, entropy, top_logprobs, top_ids);
      break;
    case LCG_DTYPE_FP16:
      k_token_logprobs<<<grid, kThreads, 0, st>>>(static_cast<const __half*>(logits), V, ld, tokens, token_bytes, top,
                                                  logprob, entropy, top_logprobs, top_ids);
      break;
    case LCG_DTYPE_FP32:
      k_token_logprobs<<<grid, kThreads, 0, st>>>(static_cast<const float*>(logits), V, ld, tokens, token_bytes, top,
                                                  logprob, entropy, top_logprobs, top_ids);
      break;
    default:
      return fail(LCG_ERR_BAD_ARG, "unknown dtype %d", dtype);
  }
  LCG_CUDA_OK(cudaGetLastError());
  count_launch();
  return LCG_OK;
}
