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
//
// Two kernels: the slots that every (sequence, kv head) keeps, then the move.
// Bound by HBM: the kept rows are read once and written once, which the move
// reaches by keeping a chunk's loads under way while the one before is stored.

constexpr int kSelectThreads = 1024;
constexpr int kEach = 16;                             // weights of a thread
constexpr int kSpan = kSelectThreads * kEach;         // weights that the CTA holds at a time
constexpr int kBins = 2048;  // of a digit: 11, 11 and 10 bits

// Weights as integers of the same order: larger weight, larger key; -0 as 0
// and NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of the earlier threads' values, and of all threads'. All threads.
__device__ __forceinline__ int2 scan_block(int v, int* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int w = red[lane];  // one for each of the 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, w, o);
    if (lane >= o) w += y;
  }
  const int base = __shfl_sync(~0u, w, max(warp - 1, 0));
  return make_int2((warp ? base : 0) + x - v, __shfl_sync(~0u, w, 31));
}

// One CTA per (sequence, kv head): the slots it keeps, in rising order, into
// kept[0..count). The older slots compete for `need` places: their smallest
// kept key is found digit by digit, from histograms; of the slots at that key
// the oldest stay. A thread holds kEach neighbouring weights, in registers
// throughout where the CTA holds them all.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ KvEvictArgs a, int* kept_all, int* counts) {
  __shared__ int bins[kBins];
  __shared__ int red[32];
  __shared__ int found[2];
  asm volatile("griddepcontrol.launch_dependents;");
  const int b = blockIdx.x / a.in.kv_heads;
  const int n = a.in.clamp_len(a.lens[b]);
  const int count = min(n, a.keep);
  const int old = n - min(n, a.recent);  // slots before the recent ones
  const int need = count - (n - old);    // of them stay
  const float* w = a.weights + (long long)blockIdx.x * a.weights_stride;
  int* kept = kept_all + (long long)blockIdx.x * a.keep;
  if (threadIdx.x == 0) counts[blockIdx.x] = count;
  for (int i = need + threadIdx.x; i < a.keep; i += kSelectThreads) kept[i] = i < count ? old + i - need : -1;
  if (need == old) {
    for (int i = threadIdx.x; i < need; i += kSelectThreads) kept[i] = i;
    return;
  }
  if (need == 0) return;

  uint32_t key[kEach];
  int held = -1;  // first slot of the span in the registers
  auto hold = [&](int from) {
    if (held == from) return;
    held = from;
    const int j = from + threadIdx.x * kEach;
    const bool vectors = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
      if (vectors && j + i + 4 <= old) {
        const float4 x = *reinterpret_cast<const float4*>(w + j + i);
        key[i] = order_key(x.x);
        key[i + 1] = order_key(x.y);
        key[i + 2] = order_key(x.z);
        key[i + 3] = order_key(x.w);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) key[i + k] = j + i + k < old ? order_key(w[j + i + k]) : 0;  // 0 is no weight's key
      }
    }
  };

  uint32_t bound = 0, known = 0;  // the digits found so far, and which bits those are
  int places = need;              // for keys that share them
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, width = digit < 2 ? 11 : 10;
    for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (int from = 0; from < old; from += kSpan) {
      hold(from);
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (key[i] && (key[i] & known) == bound) {
          // equal weights are common (zeros, a handful of values): one addition for a warp's equal digits
          const int bin = key[i] >> shift & ((1 << width) - 1);
          const uint32_t same = __match_any_sync(__activemask(), bin);
          if ((threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&bins[bin], __popc(same));
        }
    }
    __syncthreads();
    // Bins from the highest down: the one in which the places run out.
    const int hi = kBins - 1 - 2 * (int)threadIdx.x, c0 = bins[hi], c1 = bins[hi - 1];
    const int2 sum = scan_block(c0 + c1, red);
    if (sum.x < places && places <= sum.x + c0 + c1) {
      const bool first = places <= sum.x + c0;
      found[0] = first ? hi : hi - 1;
      found[1] = places - sum.x - (first ? 0 : c0);
    }
    __syncthreads();
    bound |= (uint32_t)found[0] << shift;
    known |= (uint32_t)((1 << width) - 1) << shift;
    places = found[1];
  }

  // `places` of the keys at the bound stay, the oldest.
  int kept_before = 0, ties_before = 0;
  for (int from = 0; from < old; from += kSpan) {
    hold(from);
    int ties = 0, above = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      ties += key[i] == bound;
      above += key[i] > bound;
    }
    const int2 t = scan_block(ties, red);
    int tie = ties_before + t.x;
    const int mine = above + max(0, min(places - tie, ties));
    const int2 s = scan_block(mine, red);
    int at = kept_before + s.x;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      bool stays = key[i] > bound;
      if (key[i] == bound) stays = tie++ < places;
      if (stays) kept[at++] = from + threadIdx.x * kEach + i;
    }
    ties_before += t.y;
    kept_before += s.y;
  }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 8;  // vectors of a thread under way

// A CTA moves one run of columns of the K or V rows of one (sequence, kv head),
// chunk by chunk in rising order. Kept slot i came from slot j >= i, so a
// chunk's destinations lie before every source of the chunks after it: once all
// of a chunk is read (the barrier) it may be written while the next one is
// read, in place too. CTAs along y: K and V, each in `slices` runs of columns,
// and one for the weights, the slots and the length.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ KvEvictArgs a, const int* kept_all,
                                                                  const int* counts, int slices) {
  __shared__ long long from_at[2][kMoveThreads * kMoveRows / 2], to_at[2][kMoveThreads * kMoveRows / 2];
  const int item = blockIdx.x, b = item / a.in.kv_heads, h = item % a.in.kv_heads;
  const int* kept = kept_all + (long long)item * a.keep;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int count = counts[item];
  if (blockIdx.y == 2 * slices) {
    const float* w = a.weights + (long long)item * a.weights_stride;
    float* wo = a.weights_out + (long long)item * a.weights_out_stride;
    for (int i0 = 0; i0 < count; i0 += kMoveThreads * kMoveRows) {
      float x[kMoveRows];
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        const int i = i0 + u * kMoveThreads + threadIdx.x;
        x[u] = i < count ? w[kept[i]] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kMoveRows; ++u) {
        const int i = i0 + u * kMoveThreads + threadIdx.x;
        if (i < count) wo[i] = x[u];
      }
    }
    __syncthreads();
    for (int i = count + threadIdx.x; i < a.out.capacity; i += kMoveThreads) wo[i] = 0.f;
    if (a.indices)
      for (int i = threadIdx.x; i < a.keep; i += kMoveThreads) a.indices[(long long)item * a.keep + i] = kept[i];
    if (h == 0 && threadIdx.x == 0) a.lens_out[b] = count;
    return;
  }
  const bool is_v = (int)blockIdx.y >= slices;
  const int vecs = a.in.head_dim / 8 / slices;  // of a row in this CTA's columns: a power of two
  const int column = ((int)blockIdx.y - (is_v ? slices : 0)) * vecs * 8;
  const uint16_t* src = (const uint16_t*)(is_v ? a.v_in : a.k_in) + h * a.in.s_head + column;
  uint16_t* dst = (uint16_t*)(is_v ? a.v_out : a.k_out) + h * a.out.s_head + column;
  const int step = kMoveThreads / vecs, chunk = step * kMoveRows;  // rows at a time, rows of a chunk
  const int row = threadIdx.x / vecs, d = threadIdx.x % vecs * 8;

  // Offsets of a chunk's rows, -1 for one that stays where it is or has no page.
  auto look_up = [&](int i0) {
    for (int k = threadIdx.x; k < chunk; k += kMoveThreads) {
      const int i = i0 + k;
      long long from = -1, to = -1;
      if (i < count) {
        from = a.in.offset(b, kept[i]);
        to = a.out.offset(b, i);
        if (from < 0 || to < 0) {
          a.in.report_bad_page();
          from = -1;
        } else if (src + from == dst + to) {
          from = -1;
        }
      }
      const int slot = (i0 / chunk) & 1;
      from_at[slot][k] = from;
      to_at[slot][k] = to;
    }
  };
  uint4 x[kMoveRows], y[kMoveRows];
  auto load = [&](uint4 (&v)[kMoveRows], int i0) {
    const int slot = (i0 / chunk) & 1;
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const long long from = from_at[slot][u * step + row];
      if (from >= 0) v[u] = *reinterpret_cast<const uint4*>(src + from + d);
    }
  };
  auto store = [&](const uint4 (&v)[kMoveRows], int i0) {
    const int slot = (i0 / chunk) & 1;
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (from_at[slot][u * step + row] >= 0) *reinterpret_cast<uint4*>(dst + to_at[slot][u * step + row] + d) = v[u];
  };
  if (count == 0) return;
  look_up(0);
  __syncthreads();
  load(x, 0);
  for (int i0 = 0;; i0 += 2 * chunk) {
    if (i0 + chunk < count) look_up(i0 + chunk);
    __syncthreads();  // chunk i0 is read, the next one's offsets are known
    if (i0 + chunk < count) load(y, i0 + chunk);
    store(x, i0);
    if (i0 + chunk >= count) break;
    __syncthreads();  // the first chunk's offsets are no longer needed
    if (i0 + 2 * chunk < count) look_up(i0 + 2 * chunk);
    __syncthreads();
    if (i0 + 2 * chunk < count) load(x, i0 + 2 * chunk);
    store(y, i0 + chunk);
    if (i0 + 2 * chunk >= count) break;
    __syncthreads();
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
  return (size_t)a.in.batch * a.in.kv_heads * (a.keep + 1) * sizeof(int);
}

cudaError_t launch_kv_evict(const KvEvictArgs& a, int num_sms, void* ws, cudaStream_t s) {
  if ((long long)a.in.batch * a.in.kv_heads > INT_MAX) return cudaErrorInvalidValue;
  const int items = a.in.batch * a.in.kv_heads;
  int* counts = static_cast<int*>(ws);
  int* kept = counts + items;
  {
    ProfLaunch prof("evict_select_kernel", dim3(items), dim3(kSelectThreads), 0, s);
    evict_select_kernel<<<items, kSelectThreads, 0, s>>>(a, kept, counts);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // Runs of columns while CTAs are few, of 32 bytes (a sector) at least.
  int slices = 1;
  while (items * 2ll * slices < 4 * num_sms && a.in.head_dim / 8 / slices > 2) slices *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(items, 2 * slices + 1);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ProfLaunch prof("evict_move_kernel", cfg.gridDim, cfg.blockDim, 0, s);
  e = cudaLaunchKernelEx(&cfg, evict_move_kernel, a, (const int*)kept, (const int*)counts, slices);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace grx
