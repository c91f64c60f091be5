// Host/device interface of the token-serving kernels: the paged key-value
// cache (kv_cache.cu), the attention of one new token over it
// (paged_attention.cu) and the scoring of given tokens (token_score.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#include "per_device.h"
#include "ptx.cuh"
#endif

namespace grx {

// n / d and n % d for 0 <= n < 2^31 by one high multiplication: with
// 2^(s-1) < d <= 2^s and mul = floor(2^32 (2^s - d) / d) + 1, the quotient is
// (hi32(n mul) + n) >> s (Granlund & Montgomery 1994, division by invariant
// integers). The sum stays below 2^32 because n < 2^31.
struct FastDiv {
  uint32_t d = 1, mul = 1, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << shift) < div) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - div)) / div + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
#endif
};

// One sequence-major view of a paged cache; K and V pools share it.
struct PagedView {
  int batch, kv_heads, head_dim;
  int num_pages, capacity;  // capacity: max_pages * page_size tokens
  FastDiv page;             // by page_size
  const int* table;
  long long table_stride;
  long long s_page, s_token, s_head;  // elements
  int* err_word;

#ifdef __CUDACC__
  // Tokens that the sequence holds.
  __device__ __forceinline__ int clamp_len(int n) const { return min(max(n, 0), capacity); }
  // Element offset of (token, head 0) of sequence b, or -1 for a token whose
  // table entry names no page. 0 <= token < capacity.
  __device__ __forceinline__ long long offset(int b, int token) const {
    const uint32_t p = page.div((uint32_t)token);
    const int id = table[(long long)b * table_stride + p];
    if ((unsigned)id >= (unsigned)num_pages) return -1;
    return (long long)id * s_page + (long long)(token - (int)(p * page.d)) * s_token;
  }
  __device__ __forceinline__ void report_bad_page() const {
    if (err_word) atomicCAS(err_word, 0, (int)kErrBadPage);
  }
#endif
};

#ifdef __CUDACC__
// The serving kernels are short and follow one another: each is launched so
// that it may take its place on the SMs while the kernel before it ends, and
// waits, before anything else, for that one's end and its writes. A kernel may
// let the next one in before its own end, where its own CTAs have all started.
// Lengths, tables and weights may be what that kernel writes: they are read by
// plain loads, never through the read-only path (__ldg), which takes them for
// unchanged since before this kernel began.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_in() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches `kernel` so, in clusters of `cluster` CTAs along x. The answer is
// this launch's own: the runtime's last error may be an earlier call's, and one
// that is left behind would be taken for a later call's.
template <typename... Params, typename... Args>
cudaError_t launch_next(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, int cluster,
                        Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}
#endif

struct KvAppendArgs {
  PagedView cache;
  void* k_pages;
  void* v_pages;
  const int* lens;
  int tokens;  // seq of the new K and V
  const void* k; long long k_sb, k_sh, k_ss;
  const void* v; long long v_sb, v_sh, v_ss;
  const int* counts;  // or null
  int* lens_out;      // or null; may be lens
};
cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s);

struct PagedAttnArgs {
  PagedView cache;
  int dtype;  // 1 bf16, 2 f16
  const void* k_pages;
  const void* v_pages;
  const int* lens;
  int heads;
  const void* q; long long q_sb, q_sh;
  void* o; long long o_sb, o_sh;
  float scale;
  int window;
  float* lse;
  float* weights; long long weights_stride;
};
size_t paged_attention_workspace_bytes(const PagedAttnArgs& a, int num_sms);
// Zero before the first call, and after each.
size_t paged_attention_counter_bytes(const PagedAttnArgs& a);
cudaError_t launch_paged_attention(const PagedAttnArgs& a, int num_sms, void* ws, int* counters, cudaStream_t s);

struct KvEvictArgs {
  PagedView in, out;
  const void* k_in;
  const void* v_in;
  void* k_out;
  void* v_out;
  const int* lens;
  int* lens_out;
  const float* weights; long long weights_stride;
  float* weights_out; long long weights_out_stride;
  int keep, recent;
  int* indices;  // [batch, kv_heads, keep] or null
};
size_t kv_evict_workspace_bytes(const KvEvictArgs& a);
cudaError_t launch_kv_evict(const KvEvictArgs& a, int num_sms, void* ws, cudaStream_t s);

constexpr int kMaxTop = 32;

struct TokenScoreArgs {
  int rows, vocab, dtype;  // dtype 0 f32, 1 bf16, 2 f16
  const void* logits; long long ld;
  float scale;
  const int* tokens;
  float* logp;
  float* entropy;
  float* lse;
  int top;
  int* top_tokens;
  float* top_logp;
};
cudaError_t launch_token_score(const TokenScoreArgs& a, int num_sms, cudaStream_t s);

struct TokenScoreBwdArgs {
  int rows, vocab, dtype;
  const void* logits; long long ld;
  float scale;
  const int* tokens;
  const float* lse;
  const float* entropy;
  const float* dlogp;
  const float* dentropy;
  void* dlogits; long long ldd;
};
cudaError_t launch_token_score_bwd(const TokenScoreBwdArgs& a, int num_sms, cudaStream_t s);

}  // namespace grx
