// Log probabilities of given tokens with entropy and top alternatives, and
// their gradient.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include "profile.h"
#include "serving.cuh"

namespace grx {

namespace {

constexpr int kThreads = 512;
// lse in 32 bits moves every probability of its row by up to 2^-25 |lse|: 2^-16 of itself at this size.
constexpr float kFarLse = 512.f;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float block_sum(float v, float* red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 15];
  for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

__device__ __forceinline__ float block_maxf(float v, float* red) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 15];
  for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* red) {
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 15];
  for (int o = 8; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

// (value, token) as one integer: larger value first, then smaller token; NaN
// below -inf, -0 as 0.
__device__ __forceinline__ unsigned long long rank_of(float x, int c) {
  const uint32_t u = __float_as_uint(x + 0.f);
  uint32_t key = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (x != x) key = 0;
  return (unsigned long long)key << 32 | (uint32_t)~c;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_score_kernel(TokenScoreArgs a) {
  __shared__ float red[kThreads / 32];
  __shared__ unsigned long long red64[kThreads / 32];
  const int r = blockIdx.x;
  const T* x = (const T*)a.logits + (long long)r * a.ld;
  unsigned long long best = 0;
  bool nan = false;
  for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
    best = max(best, rank_of(to_f(x[c]) * a.scale, c));
    nan |= isnan(to_f(x[c]));
  }
  nan = __syncthreads_or(nan);
  best = block_max(best, red64);
  const float top = to_f(x[(int)~(uint32_t)best]);
  const bool empty = top == -INFINITY;
  float sum = 0.f, dot = 0.f;
  for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
    const float d = (to_f(x[c]) - top) * a.scale, e = expf(d);
    sum += e;
    dot += e > 0.f ? e * d : 0.f;
  }
  sum = block_sum(sum, red);
  dot = block_sum(dot, red);
  const float total = nan ? NAN : logf(sum);
  const float lse = empty && !nan ? -INFINITY : top * a.scale + total;
  const float entropy = empty && !nan ? 0.f : total - dot / sum;
  // From the largest logit, not from lse: near the type's lowest value lse has no digits left after the point.
  auto log_prob = [&](float v) { return empty && !nan ? -INFINITY : (v - top) * a.scale - total; };
  if (threadIdx.x == 0) {
    const int t = a.tokens ? a.tokens[r] : -1;
    if (a.logp)
      a.logp[r] = (unsigned)t < (unsigned)a.vocab ? log_prob(to_f(x[t])) : 0.f;
    if (a.lse) a.lse[r] = lse;
    if (a.entropy) a.entropy[r] = entropy;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long v = 0;
    for (int c = threadIdx.x; c < a.vocab; c += kThreads) {
      const unsigned long long q = rank_of(to_f(x[c]) * a.scale, c);
      if (q < last) v = max(v, q);
    }
    last = block_max(v, red64);
    if (threadIdx.x == 0) {
      const int c = (int)~(uint32_t)last;
      if (a.top_tokens) a.top_tokens[(long long)r * a.top + k] = c;
      if (a.top_logp) a.top_logp[(long long)r * a.top + k] = log_prob(to_f(x[c]));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_score_bwd_kernel(TokenScoreBwdArgs a) {
  const int r = blockIdx.x / 8;
  const T* x = (const T*)a.logits + (long long)r * a.ld;
  T* dx = (T*)a.dlogits + (long long)r * a.ldd;
  const float lse = a.lse[r];
  __shared__ float red[kThreads / 32];
  // x - lse = (x - top) - total. A large lse has too few digits after the point for that: the row is summed again.
  // One CTA does that, and the row, since the others might be overwriting it.
  float top = 0.f, total = lse;
  long long first = blockIdx.x % 8 * kThreads, step = 8 * kThreads;
  if (fabsf(lse) > kFarLse && lse != -INFINITY) {
    if (first) return;
    step = kThreads;
    float m = -INFINITY;
    for (int c = threadIdx.x; c < a.vocab; c += kThreads) m = fmaxf(m, to_f(x[c]));
    top = block_maxf(m, red);
    float sum = 0.f;
    for (int c = threadIdx.x; c < a.vocab; c += kThreads) sum += expf((to_f(x[c]) - top) * a.scale);
    total = logf(block_sum(sum, red));
  }
  const int t = a.dlogp && lse != -INFINITY ? a.tokens[r] : -1;
  const float gl = (unsigned)t < (unsigned)a.vocab ? a.dlogp[r] : 0.f;
  const float ge = a.dentropy ? a.dentropy[r] : 0.f, ent = a.dentropy ? a.entropy[r] : 0.f;
  for (long long c = first + threadIdx.x; c < a.vocab; c += step) {
    const float d = (to_f(x[c]) - top) * a.scale - total;
    const float p = lse == -INFINITY ? 0.f : expf(d);
    float g = -p * gl;
    if (p != 0.f) g -= ge * p * (d + ent);
    if (c == t) g += gl;
    dx[c] = from_f<T>(g * a.scale);
  }
}

}  // namespace

cudaError_t launch_token_score(const TokenScoreArgs& a, int, cudaStream_t s) {
  ProfLaunch prof("token_score_kernel", dim3(a.rows), dim3(kThreads), 0, s);
  if (a.dtype == 0) token_score_kernel<float><<<a.rows, kThreads, 0, s>>>(a);
  else if (a.dtype == 1) token_score_kernel<__nv_bfloat16><<<a.rows, kThreads, 0, s>>>(a);
  else token_score_kernel<__half><<<a.rows, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_token_score_bwd(const TokenScoreBwdArgs& a, int, cudaStream_t s) {
  if (a.rows > INT_MAX / 8) return cudaErrorInvalidValue;
  const dim3 grid(8 * a.rows);
  ProfLaunch prof("token_score_bwd_kernel", grid, dim3(kThreads), 0, s);
  if (a.dtype == 0) token_score_bwd_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else if (a.dtype == 1) token_score_bwd_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  else token_score_bwd_kernel<__half><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace grx
