// Attention of one new token over a paged key-value cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "profile.h"
#include "serving.cuh"

namespace grx {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ float2 to_f2(uint32_t u, int dtype) {
  if (dtype == 1) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// One CTA per (sequence, kv head) walks its query heads; each warp takes every
// kWarps-th key, its lanes share the row.
__global__ void __launch_bounds__(kWarps * 32) paged_attn_kernel(PagedAttnArgs a) {
  constexpr int kPairs = 4;  // pairs of elements a lane holds, headDim 256 at most
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][256];
  const int b = blockIdx.x / a.cache.kv_heads, h = blockIdx.x % a.cache.kv_heads;
  const int group = a.heads / a.cache.kv_heads, dim = a.cache.head_dim;
  const int n = a.cache.clamp_len(a.lens[b]);
  const int first = a.window ? max(0, n - a.window) : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint16_t* kp = (const uint16_t*)a.k_pages + h * a.cache.s_head;
  const uint16_t* vp = (const uint16_t*)a.v_pages + h * a.cache.s_head;
  for (int g = 0; g < group; ++g) {
    const int qh = h * group + g;
    const uint16_t* q = (const uint16_t*)a.q + b * a.q_sb + qh * a.q_sh;
    float2 qv[kPairs], o[kPairs];
    for (int p = 0; p < kPairs; ++p) {
      const int d = 2 * (lane + 32 * p);
      qv[p] = d < dim ? to_f2(*(const uint32_t*)(q + d), a.dtype) : make_float2(0.f, 0.f);
      o[p] = make_float2(0.f, 0.f);
    }
    auto score = [&](long long at) {
      float s = 0.f;
      for (int p = 0; p < kPairs; ++p) {
        const int d = 2 * (lane + 32 * p);
        if (d >= dim) break;
        const float2 kv = to_f2(*(const uint32_t*)(kp + at + d), a.dtype);
        s = fmaf(qv[p].x, kv.x, fmaf(qv[p].y, kv.y, s));
      }
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
      return s * a.scale;
    };
    float m = -INFINITY, l = 0.f;
    for (int j = first + warp; j < n; j += kWarps) {
      const long long at = a.cache.offset(b, j);
      if (at < 0) {
        if (lane == 0) a.cache.report_bad_page();
        continue;
      }
      const float s = score(at);
      const float nm = fmaxf(m, s);
      const float c = m == -INFINITY ? 0.f : expf(m - nm), e = nm == -INFINITY ? 0.f : expf(s - nm);
      m = nm;
      l = l * c + e;
      for (int p = 0; p < kPairs; ++p) {
        const int d = 2 * (lane + 32 * p);
        if (d >= dim) break;
        const float2 v = to_f2(*(const uint32_t*)(vp + at + d), a.dtype);
        o[p].x = fmaf(e, v.x, o[p].x * c);
        o[p].y = fmaf(e, v.y, o[p].y * c);
      }
    }
    __syncthreads();
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    for (int p = 0; p < kPairs; ++p)
      if (2 * (lane + 32 * p) < dim) *(float2*)&so[warp][2 * (lane + 32 * p)] = o[p];
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < kWarps; ++w) total += sm[w] == -INFINITY ? 0.f : sl[w] * expf(sm[w] - top);
    for (int d = threadIdx.x; d < dim; d += kWarps * 32) {
      float x = 0.f;
      for (int w = 0; w < kWarps; ++w) x += sm[w] == -INFINITY ? 0.f : so[w][d] * expf(sm[w] - top);
      x = total > 0.f ? x / total : 0.f;
      uint16_t* op = (uint16_t*)a.o + b * a.o_sb + qh * a.o_sh + d;
      if (a.dtype == 1) *(__nv_bfloat16*)op = __float2bfloat16_rn(x);
      else *(__half*)op = __float2half_rn(x);
    }
    const float lse = total > 0.f ? top + logf(total) : -INFINITY;
    if (a.lse && threadIdx.x == 0) a.lse[(long long)b * a.heads + qh] = lse;
    if (a.weights) {
      float* w = a.weights + (long long)blockIdx.x * a.weights_stride;
      for (int j = first + warp; j < n; j += kWarps) {
        const long long at = a.cache.offset(b, j);
        if (at < 0) continue;
        const float s = score(at);
        if (lane == 0) w[j] += expf(s - lse);
      }
    }
  }
}

}  // namespace

size_t paged_attention_workspace_bytes(const PagedAttnArgs&, int) { return 0; }

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int, void*, cudaStream_t s) {
  const int grid = a.cache.batch * a.cache.kv_heads;
  ProfLaunch prof("paged_attn_kernel", dim3(grid), dim3(kWarps * 32), 0, s);
  paged_attn_kernel<<<grid, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace grx
