// The paged key-value cache: append and eviction. Both move rows of headDim
// 2-byte elements as 16-byte vectors and compute nothing on them.
#include <limits.h>

#include "profile.h"
#include "serving.cuh"

namespace grx {

namespace {

constexpr int kAppendThreads = 256;

__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(KvAppendArgs a, int tokens_per_cta, int chunks) {
  const int b = blockIdx.x / chunks;
  const int held = a.cache.clamp_len(a.lens[b]);
  int count = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
  if (count > a.cache.capacity - held) {
    count = a.cache.capacity - held;
    if (threadIdx.x == 0) a.cache.report_bad_page();
  }
  const int vecs = a.cache.head_dim / 8;
  const int row = 2 * a.cache.kv_heads * vecs;  // vectors of one token, K then V
  const int t0 = (int)(blockIdx.x % chunks) * tokens_per_cta;
  const int t1 = min(t0 + tokens_per_cta, count);
  for (long long i = threadIdx.x; i < (long long)(t1 - t0) * row; i += kAppendThreads) {
    const int t = t0 + (int)(i / row);
    int r = (int)(i % row);
    const bool is_v = r >= row / 2;
    r -= is_v ? row / 2 : 0;
    const int h = r / vecs, d = r % vecs * 8;
    const long long to = a.cache.offset(b, held + t);
    if (to < 0) {
      a.cache.report_bad_page();
      continue;
    }
    const uint16_t* src = is_v ? (const uint16_t*)a.v + b * a.v_sb + h * a.v_sh + t * a.v_ss
                               : (const uint16_t*)a.k + b * a.k_sb + h * a.k_sh + t * a.k_ss;
    uint16_t* dst = (uint16_t*)(is_v ? a.v_pages : a.k_pages) + to + h * a.cache.s_head;
    *(uint4*)(dst + d) = *(const uint4*)(src + d);
  }
}

__global__ void kv_lens_kernel(KvAppendArgs a) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= a.cache.batch) return;
  const int held = a.cache.clamp_len(a.lens[b]);
  const int count = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
  a.lens_out[b] = held + min(count, a.cache.capacity - held);
}

// ------------------------------------------------------------------ eviction

constexpr int kSelectThreads = 512;

// Weights as integers of the same order: larger weight, larger key; -0 as 0
// and NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per (sequence, kv head): the slots it keeps, in rising order, into
// kept[0..count). The threshold is the largest key that at least `need` of the
// older slots reach, found bit by bit.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(KvEvictArgs a, int* kept_all) {
  __shared__ int red[kSelectThreads / 32 + 1];
  const int b = blockIdx.x / a.in.kv_heads;
  const int n = a.in.clamp_len(a.lens[b]);
  const int count = min(n, a.keep);
  const int old = n - min(n, a.recent);  // slots before the recent ones
  const int need = count - (n - old);    // of them stay
  const float* w = a.weights + (long long)blockIdx.x * a.weights_stride;
  int* kept = kept_all + (long long)blockIdx.x * a.keep;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t bound = 0;
  int above = 0;
  auto count_from = [&](uint32_t key) {  // older slots whose key is at least `key`
    int c = 0;
    for (int j = threadIdx.x; j < old; j += kSelectThreads) c += order_key(w[j]) >= key;
    c = __reduce_add_sync(~0u, c);
    __syncthreads();
    if (lane == 0) red[warp] = c;
    __syncthreads();
    return __reduce_add_sync(~0u, lane < kSelectThreads / 32 ? red[lane] : 0);
  };
  if (need > 0 && need < old) {
    for (int bit = 31; bit >= 0; --bit)
      if (count_from(bound | 1u << bit) >= need) bound |= 1u << bit;
    above = bound == ~0u ? 0 : count_from(bound + 1);
  }
  const bool all = need >= old;
  const int ties = need - above;  // of the slots at the bound, the oldest
  int base = 0, ties_seen = 0;
  for (int j0 = 0; j0 < old; j0 += kSelectThreads) {
    const int j = j0 + threadIdx.x;
    const uint32_t key = j < old ? order_key(w[j]) : 0;
    const bool tie = !all && need > 0 && j < old && key == bound;
    const uint32_t tie_mask = __ballot_sync(~0u, tie);
    __syncthreads();
    if (lane == 0) red[warp] = __popc(tie_mask);
    __syncthreads();
    int t = lane < kSelectThreads / 32 ? red[lane] : 0;
    const int tie_before = __reduce_add_sync(~0u, lane < warp ? t : 0) + __popc(tie_mask & ((1u << lane) - 1));
    const int tie_total = __reduce_add_sync(~0u, t);
    const bool keep = j < old && need > 0 && (all || key > bound || (tie && ties_seen + tie_before < ties));
    const uint32_t mask = __ballot_sync(~0u, keep);
    __syncthreads();
    if (lane == 0) red[warp] = __popc(mask);
    __syncthreads();
    t = lane < kSelectThreads / 32 ? red[lane] : 0;
    const int before = __reduce_add_sync(~0u, lane < warp ? t : 0) + __popc(mask & ((1u << lane) - 1));
    if (keep) kept[base + before] = j;
    base += __reduce_add_sync(~0u, t);
    ties_seen += tie_total;
  }
  for (int j = old + threadIdx.x; j < n; j += kSelectThreads) kept[base + j - old] = j;
  for (int i = count + threadIdx.x; i < a.keep; i += kSelectThreads) kept[i] = -1;
}

constexpr int kMoveThreads = 256;

// One CTA per (sequence, kv head, K or V): moves the kept rows in rising
// order, a chunk at a time. Kept slot i came from slot j >= i, so a chunk's
// destinations lie before every source of the chunks after it: reading a chunk
// whole before writing it makes the move safe in place.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(KvEvictArgs a, const int* kept_all) {
  const int item = blockIdx.x, b = item / a.in.kv_heads, h = item % a.in.kv_heads;
  const int* kept = kept_all + (long long)item * a.keep;
  const uint16_t* src = (const uint16_t*)(blockIdx.y ? a.v_in : a.k_in) + h * a.in.s_head;
  uint16_t* dst = (uint16_t*)(blockIdx.y ? a.v_out : a.k_out) + h * a.out.s_head;
  const int vecs = a.in.head_dim / 8;
  const int rows = kMoveThreads / vecs;
  const int r = threadIdx.x / vecs, d = threadIdx.x % vecs * 8;
  int count = 0;
  for (int i0 = 0; i0 < a.keep; i0 += rows) {
    const int i = i0 + r;
    const int j = i < a.keep ? kept[i] : -1;
    uint4 x = make_uint4(0, 0, 0, 0);
    long long to = -1;
    if (j >= 0) {
      const long long from = a.in.offset(b, j);
      to = a.out.offset(b, i);
      if (from < 0 || to < 0) a.in.report_bad_page();
      if (from < 0) to = -1;
      if (to >= 0) x = *(const uint4*)(src + from + d);
    }
    __syncthreads();
    if (to >= 0) *(uint4*)(dst + to + d) = x;
  }
  if (blockIdx.y == 0) {  // the weights follow their rows
    const float* w = a.weights + (long long)item * a.weights_stride;
    float* wo = a.weights_out + (long long)item * a.weights_out_stride;
    for (int i0 = 0; i0 < a.out.capacity; i0 += kMoveThreads) {
      const int i = i0 + threadIdx.x;
      const int j = i < a.keep ? kept[i] : -1;
      const float x = j >= 0 ? w[j] : 0.f;
      __syncthreads();
      if (i < a.out.capacity) wo[i] = x;
      if (a.indices && i < a.keep) a.indices[(long long)item * a.keep + i] = j;
      count += __syncthreads_count(j >= 0);
    }
    if (h == 0 && threadIdx.x == 0) a.lens_out[b] = count;
  }
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s) {
  // A sequence of a few tokens stays in one CTA, whose last act may then be
  // to overwrite its own length.
  const int per_cta = 16;
  const int chunks = a.tokens > 0 ? (a.tokens + per_cta - 1) / per_cta : 0;
  if ((long long)chunks * a.cache.batch > INT_MAX) return cudaErrorInvalidValue;
  if (chunks > 0) {
    const int grid = chunks * a.cache.batch;
    ProfLaunch prof("kv_append_kernel", dim3(grid), dim3(kAppendThreads), 0, s);
    kv_append_kernel<<<grid, kAppendThreads, 0, s>>>(a, per_cta, chunks);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  if (a.lens_out) {
    const int grid = (a.cache.batch + 255) / 256;
    ProfLaunch prof("kv_lens_kernel", dim3(grid), dim3(256), 0, s);
    kv_lens_kernel<<<grid, 256, 0, s>>>(a);
  }
  return cudaGetLastError();
}

size_t kv_evict_workspace_bytes(const KvEvictArgs& a) {
  return (size_t)a.in.batch * a.in.kv_heads * a.keep * sizeof(int);
}

cudaError_t launch_kv_evict(const KvEvictArgs& a, int num_sms, void* ws, cudaStream_t s) {
  (void)num_sms;
  const int items = a.in.batch * a.in.kv_heads;
  int* kept = static_cast<int*>(ws);
  {
    ProfLaunch prof("evict_select_kernel", dim3(items), dim3(kSelectThreads), 0, s);
    evict_select_kernel<<<items, kSelectThreads, 0, s>>>(a, kept);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  ProfLaunch prof("evict_move_kernel", dim3(items, 2), dim3(kMoveThreads), 0, s);
  evict_move_kernel<<<dim3(items, 2), kMoveThreads, 0, s>>>(a, kept);
  return cudaGetLastError();
}

}  // namespace grx
