// Log probabilities of given tokens with entropy and top alternatives, and
// their gradient.
//
// Forward, x the scaled logits of a row, t its largest:
//   S = sum_c exp(x - t),  E = sum_c exp(x - t) (x - t)
//   lse = t + log S,  logp = x_token - t - log S,  entropy = log S - E / S
// in one pass over the row with a running largest (S and E are scaled when it
// grows). The top tokens come from the same pass: k elements of its first part
// give a bound that no element of the row's best k lies below, the few elements
// that pass it are collected, sorted by (value, token) and raise the bound; so do
// the largest elements of the threads.
//
// Without top tokens bound by HBM (4096 x 50257 bf16 with entropy 77 us = 5.35 TB/s,
// 82 % of a plain copy; device time, replays of a graph, like all here), with them by
// what a row does besides: its first bound, its queue and the chains of barriers and
// shuffles there (top 5: 94 us = 4.4 TB/s; with a scale and masked tokens 99, and 104
// in calls among others). 8 x 131072 with top 20 takes 9.9 us, such a chain. Fewer
// instructions an element (packed maxima, floors in 16 bits) changed nothing.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include "profile.h"
#include "serving.cuh"

namespace cg = cooperative_groups;

namespace grx {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// lse in 32 bits moves every probability of its row by up to 2^-25 |lse|: 2^-16 of itself at this size.
constexpr float kFarLse = 512.f;

// ------------------------------------------------------ pairs of fp32 values

struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pair(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ------------------------------------------------ 16 bytes of a row's elements

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ uint32_t none() { return 0xff800000u; }
  static __device__ __forceinline__ float largest(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  // Pair i of the vector, no element below `floor`.
  static __device__ __forceinline__ F2 at_least(const uint4& v, int i, float floor) {
    const float x = __uint_as_float(i ? v.z : v.x), y = __uint_as_float(i ? v.w : v.y);
    return pair(max_nan(x, floor), max_nan(y, floor));
  }
  static __device__ __forceinline__ F2 get(const uint4& v, int i) {
    return pair(__uint_as_float(i ? v.z : v.x), __uint_as_float(i ? v.w : v.y));
  }
  static __device__ __forceinline__ void put(uint4& v, int i, float2 f) {
    (i ? v.z : v.x) = __float_as_uint(f.x);
    (i ? v.w : v.y) = __float_as_uint(f.y);
  }
};
__device__ __forceinline__ uint32_t& word(uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ uint32_t none() { return 0xff80ff80u; }
  static __device__ __forceinline__ __nv_bfloat162 b2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const __nv_bfloat162 m = __hmax2(__hmax2(b2(v.x), b2(v.y)), __hmax2(b2(v.z), b2(v.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ F2 unpack(uint32_t u) {
    return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ F2 at_least(const uint4& v, int i, float floor) {
    const __nv_bfloat162 m = __hmax2_nan(b2(word(v, i)), __bfloat162bfloat162(__float2bfloat16_rd(floor)));
    return unpack(*reinterpret_cast<const uint32_t*>(&m));
  }
  static __device__ __forceinline__ F2 get(const uint4& v, int i) { return unpack(word(v, i)); }
  static __device__ __forceinline__ void put(uint4& v, int i, float2 f) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    word(v, i) = *reinterpret_cast<const uint32_t*>(&b);
  }
};
template <>
struct Elem<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ uint32_t none() { return 0xfc00fc00u; }
  static __device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const __half2 m = __hmax2(__hmax2(h2(v.x), h2(v.y)), __hmax2(h2(v.z), h2(v.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ F2 at_least(const uint4& v, int i, float floor) {
    const float2 f = __half22float2(h2(word(v, i)));  // the floor may lie past the type's range
    return pair(max_nan(f.x, floor), max_nan(f.y, floor));
  }
  static __device__ __forceinline__ F2 get(const uint4& v, int i) {
    const float2 f = __half22float2(h2(word(v, i)));
    return pair(f.x, f.y);
  }
  static __device__ __forceinline__ void put(uint4& v, int i, float2 f) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    word(v, i) = *reinterpret_cast<const uint32_t*>(&h);
  }
};

// A row as aligned vectors: vector v holds elements v N - shift ... of it. The
// first and the last may reach past its ends; what does is never read.
template <typename T>
struct Row {
  static constexpr int N = Elem<T>::N;
  const T* x;
  int vocab, shift;
  __device__ __forceinline__ Row(const T* p, int vocab_)
      : x(p), vocab(vocab_), shift((int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T))) {}
  __device__ __forceinline__ int vectors() const { return (int)(((long long)vocab + shift + N - 1) / N); }
  __device__ __forceinline__ bool inside(int v) const { return v * N >= shift && v * N - shift + N <= vocab; }
  __device__ __forceinline__ const uint4* base() const { return reinterpret_cast<const uint4*>(x - shift); }
  __device__ __forceinline__ uint4 load(int v) const {
    if (inside(v)) return __ldcs(reinterpret_cast<const uint4*>(x - shift) + v);
    uint4 r = make_uint4(Elem<T>::none(), Elem<T>::none(), Elem<T>::none(), Elem<T>::none());
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = v * N - shift + i;
      if (c >= 0 && c < vocab) e[i] = x[c];
    }
    return r;
  }
};

// ------------------------------------------------------------------- ranking

using Key = unsigned long long;

// (scaled logit, token) as one integer, larger first, of equal ones the smaller
// token first; NaN below -inf, -0 as 0. Never 0, which stands for nothing.
__device__ __forceinline__ Key rank_of(float x, int c) {
  const uint32_t u = __float_as_uint(x + 0.f);
  uint32_t key = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (x != x) key = 0;
  return (Key)key << 32 | (uint32_t)~c;
}
__device__ __forceinline__ int token_of(Key k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float value_of(Key k) {
  const uint32_t key = (uint32_t)(k >> 32);
  if (key == 0) return NAN;
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ Key shfl_xor(Key k, int o) { return __shfl_xor_sync(~0u, k, o); }
// The warp's 32 keys in falling order (bitonic).
__device__ __forceinline__ Key sort32(Key k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o; o /= 2) {
      const Key other = shfl_xor(k, o);
      const bool first = ((lane & o) == 0) == ((lane & size) == 0);  // keeps the larger
      k = first == (k > other) ? k : other;
    }
  return k;
}
__device__ __forceinline__ float sort32(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o; o /= 2) {
      const float other = __shfl_xor_sync(~0u, v, o);
      v = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(v, other) : fminf(v, other);
    }
  return v;
}
__device__ __forceinline__ float merge32(float a, float b) {
  const int lane = threadIdx.x & 31;
  float v = fmaxf(a, __shfl_sync(~0u, b, 31 - lane));
#pragma unroll
  for (int o = 16; o; o /= 2) {
    const float other = __shfl_xor_sync(~0u, v, o);
    v = (lane & o) == 0 ? fmaxf(v, other) : fminf(v, other);
  }
  return v;
}
// The best 32 of two falling lists, falling.
__device__ __forceinline__ Key merge32(Key a, Key b) {
  const int lane = threadIdx.x & 31;
  const Key r = __shfl_sync(~0u, b, 31 - lane);
  Key k = a > r ? a : r;
#pragma unroll
  for (int o = 16; o; o /= 2) {
    const Key other = shfl_xor(k, o);
    k = ((lane & o) == 0) == (k > other) ? k : other;
  }
  return k;
}

// ------------------------------------------------------------------- forward

// Warps of a CTA: one where rows are many, so that an SM has 28 at once, reads
// the others while one is finished and waits at no barrier; eight where they are
// few, and up to kMostSplit CTAs to a row; two and four between (rows of 50257
// bf16, entropy and top 5: 600 rows 25 us with four warps, 31 with eight, 38 with
// two; 1200 rows 41 with two, 43 with four; 2368 rows, a wave of two warps each,
// 60 with two, 62 with one; 3500 rows 90 and 84, of f32 132 and 128, 2400 of f32
// 113 and 89; 4096 rows 103 and 93).
constexpr int kOne = 1, kTwo = 2, kFour = 4, kEight = 8;
constexpr int kVecs = 4;       // vectors of a thread in a part of the row
constexpr int kMostSplit = 8;  // CTAs of a cluster that share a row
template <int WARPS>
struct Block {
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kPerSm = WARPS == kOne ? 28 : WARPS == kTwo ? 16 : WARPS == kFour ? 8 : 3;
  static constexpr int kStages = WARPS == kEight ? 3 : 2;  // parts in shared memory
  static constexpr int kPart = kVecs * kThreads;
  static constexpr int kSettle = WARPS == kEight ? 96 : 16;     // vectors of the queue that are settled together
  static constexpr int kSplit = WARPS == kEight ? kMostSplit : 1;
  static constexpr int kSmem = kStages * kPart * 16;
};

struct Sums {
  float top, sum, dot;  // the largest logit; sum and dot in units of log2
};

// Two parts of a row as one; c2 = scale log2 e.
__device__ __forceinline__ Sums join(Sums a, Sums b, float c2) {
  if (a.top < b.top) {
    const Sums t = a;
    a = b;
    b = t;
  }
  if (b.top == -INFINITY) {  // nothing in it but -inf, or a NaN
    a.sum += b.sum;
    a.dot += b.dot;
    return a;
  }
  const float d = (b.top - a.top) * c2, f = ex2_approx(d);
  if (f != 0.f || b.sum != b.sum) {
    a.sum = fmaf(b.sum, f, a.sum);
    a.dot = fmaf(f, fmaf(d, b.sum, b.dot), a.dot);
  }
  return a;
}
// The same over the warp, in every lane: the sums are moved to the largest of all, then added.
__device__ __forceinline__ Sums warp_join(Sums s, float c2) {
  float top = s.top;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  s = join(Sums{top, 0.f, 0.f}, s, c2);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s.sum += __shfl_xor_sync(~0u, s.sum, o);
    s.dot += __shfl_xor_sync(~0u, s.dot, o);
  }
  return s;
}

template <int WARPS>
struct Shared {
  Sums warp[WARPS];
  float first[WARPS][WARPS > 1 ? 32 : 1];
  int queued, passed, kept;
  // Vectors with an element above the bound: fewer than kSettle, then another part's and the row's ends.
  int queue[Block<WARPS>::kSettle + Block<WARPS>::kPart + 2];
  float most[Block<WARPS>::kSettle + Block<WARPS>::kPart + 2];  // their largest elements, scaled
  Key passing[Block<WARPS>::kSettle * 8];
  Key list[WARPS + 1][32];  // the first: the best so far
  uint4 end[2];             // the vectors at the row's ends
  float given;              // the given token's logit
  Sums part[Block<WARPS>::kSplit];  // of the CTAs that share the row
  Key best[Block<WARPS>::kSplit][Block<WARPS>::kSplit > 1 ? 32 : 1];
};

// lists[0] becomes the best 32 of `n` lists. All threads, between barriers.
template <int WARPS>
__device__ __forceinline__ void merge_lists(Key (*lists)[32], int n) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  while (n > 1) {
    const int half = (n + 1) / 2;
    for (int i = warp; i + half < n; i += WARPS) lists[i][lane] = merge32(lists[i][lane], lists[i + half][lane]);
    n = half;
    if (n > 1) __syncthreads();
  }
}

template <typename T, int VECS>
__device__ __forceinline__ float largest_of(const uint4 (&v)[VECS]) {
  float top = Elem<T>::largest(v[0]);
#pragma unroll
  for (int u = 1; u < VECS; ++u) top = fmaxf(top, Elem<T>::largest(v[u]));
  return top;
}

// sum and dot of one vector where the plain path does not do: everything masked
// so far, or a largest logit so far from 0 that no floor fits below it.
template <typename T>
__device__ __noinline__ float2 add_carefully(uint4 v, float top, float c2) {
  float sum = 0.f, dot = 0.f;
  for (int i = 0; i < Elem<T>::N / 2; ++i) {
    F2 p = Elem<T>::get(v, 0);
#pragma unroll
    for (int k = 1; k < Elem<T>::N / 2; ++k) p = k == i ? Elem<T>::get(v, k) : p;
    const float2 x = split(p);
    for (int k = 0; k < 2; ++k) {
      const float y = k ? x.y : x.x;
      if (y == -INFINITY) continue;
      const float d = (y - top) * c2, e = ex2_approx(d);
      sum += e;
      if (e != 0.f) dot += e * d;
    }
  }
  return make_float2(sum, dot);
}

// A thread's running sums over vectors of the row. They are relative to `top`,
// which follows the largest element only once that is 2^8 times as likely: a
// larger one before adds at most 8 bits to a sum.
template <bool ENTROPY>
struct Running {
  float top = -INFINITY, limit = -INFINITY;
  bool plain = false;  // a floor fits between -inf and the logits that count
  F2 sum = pair(0.f, 0.f), dot = pair(0.f, 0.f);

  __device__ __forceinline__ void rebase(float to, float c2) {
    if (top != -INFINITY) {
      float d = (top - to) * c2;
      const float f = ex2_approx(d);
      if (f == 0.f) d = 0.f;
      dot = mul2(fma2(sum, pair(d, d), dot), pair(f, f));
      sum = mul2(sum, pair(f, f));
    }
    top = to;
    limit = to + 8.f * __fdividef(1.f, c2);
    plain = (floor() - to) * c2 < -160.f && floor() > -1e37f;
  }

  // 400 units below `top` where 32 bits hold that; nearer, and `top` itself in the end, where 8 units are less than top's
  // last place. What `plain` is decided by is the value that add() uses.
  __device__ __forceinline__ float floor() const { return fmaf(-50.f, limit - top, top); }

  // Adds vectors, `largest` their largest element. A logit below the floor is
  // raised to it, where its exponential is 0 all the same and a product with
  // it is 0 too, which it is not with -inf.
  template <typename T, int VECS>
  __device__ __forceinline__ void add(const uint4 (&v)[VECS], float largest, float c2) {
    constexpr int PAIRS = Elem<T>::N / 2;
    if (largest > limit) rebase(largest, c2);
    if (plain) {
      const float low = floor();
      const F2 minus = pair(-top, -top), c = pair(c2, c2);
      F2 odd_sum = pair(0.f, 0.f), odd_dot = odd_sum;  // two chains of additions side by side
#pragma unroll
      for (int u = 0; u < VECS; ++u)
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const F2 x = ENTROPY ? Elem<T>::at_least(v[u], i, low) : Elem<T>::get(v[u], i);
          const F2 d = mul2(add2(x, minus), c);
          const float2 f = split(d);
          const F2 e = pair(ex2_approx(f.x), ex2_approx(f.y));
          F2& to = i & 1 ? odd_sum : sum;
          to = add2(to, e);
          if (ENTROPY) {
            F2& to_dot = i & 1 ? odd_dot : dot;
            to_dot = fma2(e, d, to_dot);
          }
        }
      sum = add2(sum, odd_sum);
      if (ENTROPY) dot = add2(dot, odd_dot);
      return;
    }
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      float any = -INFINITY;  // NaN goes on
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 x = split(Elem<T>::get(v[u], i));
        any = max_nan(any, max_nan(x.x, x.y));
      }
      if (any == -INFINITY) continue;
      const float2 more = add_carefully<T>(v[u], top, c2);
      sum = add2(sum, pair(more.x, 0.f));
      dot = add2(dot, pair(more.y, 0.f));
    }
  }

  __device__ __forceinline__ Sums total() const {
    const float2 a = split(sum), b = split(dot);
    return Sums{top, a.x + a.y, b.x + b.y};
  }
};

// Queues a vector if it has an element above the bound (or at it, where `with` is set); `largest` is its largest. Scaled
// values are compared: two that differ may be equal once scaled, and then the smaller token comes first. Says whether the
// queue should be settled.
template <int WARPS>
__device__ __forceinline__ bool enqueue(float largest, int vector, float bound, bool with, float scale, Shared<WARPS>& sh) {
  const float y = __fmul_rn(largest, scale);
  if (!(y > bound || (with && y == bound))) return false;
  const int at = atomicAdd(&sh.queued, 1);
  sh.queue[at] = vector;
  sh.most[at] = y;
  return at >= Block<WARPS>::kSettle - 1;
}

// The top-th largest of the threads' `best` and, where those are few for it, `second`: `top` elements lie at it or
// above. All threads, between barriers.
template <int WARPS>
__device__ __forceinline__ float bound_of(float best, float second, int top, Shared<WARPS>& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  best = sort32(best);
  if (WARPS < kFour && top * 4 > WARPS * 32) best = merge32(best, sort32(second));
  if (WARPS == 1) {
    __syncthreads();
    return __shfl_sync(~0u, best, top - 1);
  }
  sh.first[warp][lane] = best;
  __syncthreads();
#pragma unroll
  for (int n = WARPS / 2; n; n /= 2) {
    if (warp < n) sh.first[warp][lane] = merge32(sh.first[warp][lane], sh.first[warp + n][lane]);
    __syncthreads();
  }
  return sh.first[0][top - 1];
}

// Leaves in the queue the entries with an element at the bound or above. Returns their number. All threads, after a
// barrier.
template <int WARPS>
__device__ __forceinline__ int prune(Shared<WARPS>& sh, float bound) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    const int n = sh.queued;
    int kept = 0;
    for (int i = 0; i < n; i += 32) {
      const float y = i + lane < n ? sh.most[i + lane] : 0.f;
      const int entry = i + lane < n ? sh.queue[i + lane] : 0;
      const bool keep = i + lane < n && y >= bound;
      const uint32_t all = __ballot_sync(~0u, keep);
      const int to = kept + __popc(all & ((1u << lane) - 1));
      if (keep) {
        sh.queue[to] = entry;
        sh.most[to] = y;
      }
      kept += __popc(all);
      __syncwarp();
    }
    if (lane == 0) sh.queued = sh.kept = kept;
  }
  __syncthreads();
  return sh.kept;  // queued may grow before all have read it
}

// Sorts the queued elements into the best so far, which is what sets the new
// bound; the queue is empty then. All threads, after a barrier and before none.
template <int WARPS, typename T>
__device__ __noinline__ float settle(Shared<WARPS>& sh, const T* x, int vocab, int shift, float scale, int top, float bound) {
  constexpr int N = Elem<T>::N, kThreads = WARPS * 32, kSettle = Block<WARPS>::kSettle;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int queued = sh.queued;
  for (int q0 = 0; q0 < queued; q0 += kSettle) {
    const int n = min(queued - q0, kSettle);
#pragma unroll 4
    for (int i = threadIdx.x; i < n * N; i += kThreads) {
      const int c = sh.queue[q0 + i / N] * N - shift + i % N;
      const float y = (unsigned)c < (unsigned)vocab ? __fmul_rn(Elem<T>::to(x[c]), scale) : -INFINITY;
      // Those at the bound too, whatever their part: more than are needed do no harm.
      if (y >= bound && y > -INFINITY) sh.passing[atomicAdd(&sh.passed, 1)] = rank_of(y, c);
    }
    __syncthreads();
    const int passed = sh.passed, lists = min(WARPS, (passed + 31) / 32);
    if (warp < lists) {
      Key k = 0;
      for (int i = warp * 32; i < passed; i += kThreads) {
        const Key one = sort32(i + lane < passed ? sh.passing[i + lane] : 0);
        k = i == warp * 32 ? one : merge32(k, one);
      }
      sh.list[warp + 1][lane] = k;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      sh.passed = 0;
      if (q0 + kSettle >= queued) sh.queued = 0;
    }
    merge_lists<WARPS>(sh.list, lists + 1);
    __syncthreads();
    const Key worst = sh.list[0][top - 1];
    if (worst) bound = value_of(worst);
  }
  return bound;
}

// One CTA's run of a row's vectors: [in0, in1) whole ones, and where it has an
// end of the row that reaches past the row, the vector there.
template <typename T>
struct Run {
  Row<T> row;
  int in0, in1, head, tail;  // head, tail: such a vector, or -1
  __device__ __forceinline__ Run(const TokenScoreArgs& a, long long r, int rank, int split)
      : row((const T*)a.logits + r * a.ld, a.vocab) {
    const int vectors = row.vectors(), each = (vectors + split - 1) / split;
    in0 = min(rank * each, vectors);
    in1 = min(in0 + each, vectors);
    head = in0 < in1 && in0 == 0 && !row.inside(0) ? in0++ : -1;
    tail = in0 < in1 && in1 == vectors && !row.inside(vectors - 1) ? --in1 : -1;
  }
};

// Clusters of `split` CTAs share a row, each CTA a run of its vectors; single
// CTAs walk on through the rows. Every thread copies its own vectors to shared
// memory kStages parts ahead, of the next row too, so that the loads go on
// while a row is finished, and waits for nobody else's.
//
// A run is read in whole parts and what is left of it in one more. The bound
// comes from the first part. Whenever kSettle vectors are queued, the threads'
// largest elements so far raise it and vectors below it leave the queue; if many
// stay, they are settled (rows of 2048 x 50257 in rising order 161 us, with
// settling every time 680).
template <int WARPS, typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(Block<WARPS>::kThreads, Block<WARPS>::kPerSm) token_score_kernel(const __grid_constant__ TokenScoreArgs a, int split) {
  constexpr int kThreads = Block<WARPS>::kThreads, kPart = Block<WARPS>::kPart, kStages = Block<WARPS>::kStages;
  extern __shared__ __align__(16) uint4 ring[];  // [kStages][kVecs][kThreads]
  __shared__ Shared<WARPS> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % split, step = gridDim.x / split;
  const float c2 = a.scale * kLog2e;
  const uint4 none = make_uint4(Elem<T>::none(), Elem<T>::none(), Elem<T>::none(), Elem<T>::none());
  if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  wait_for_previous_kernel();
  if (TOP) {
    if (threadIdx.x == 0) sh.queued = sh.passed = 0;
    if (warp == 0) sh.list[0][lane] = 0;
  }

  unsigned r = blockIdx.x / split, ahead = r;  // the row worked on, the row being loaded
  Run<T> run(a, r, rank, split);
  const uint4* load_from = run.row.base() + run.in0 + threadIdx.x;
  int load_left = run.in1 - run.in0, load_slot = 0, slot = 0;
  auto feed = [&] {
    if (ahead < (unsigned)a.rows) {
      const uint32_t to = smem_u32(ring + load_slot * kPart + threadIdx.x);
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
        if (u * kThreads + (int)threadIdx.x < load_left)
          asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to + u * kThreads * 16),
                       "l"(load_from + u * kThreads)
                       : "memory");
      load_from += kPart;
      load_left -= kPart;
      if (load_left < 0) {  // that was the row's last part, whole or not
        ahead += step;
        if (ahead < (unsigned)a.rows) {
          const Run<T> next(a, ahead, rank, split);
          load_from = next.row.base() + next.in0 + threadIdx.x;
          load_left = next.in1 - next.in0;
        }
      }
    }
    load_slot = load_slot + 1 == kStages ? 0 : load_slot + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i + 1 < kStages; ++i) feed();

  while (true) {
    const T* x = run.row.x;
    Running<ENTROPY> sums;
    const int end_at = warp || lane > 1 ? -1 : lane ? run.tail : run.head;
    if (end_at >= 0) sh.end[lane] = run.row.load(end_at);
    if (threadIdx.x == kThreads - 1 && a.logp) {
      const int t = a.tokens[r];
      if ((unsigned)t < (unsigned)a.vocab) sh.given = Elem<T>::to(x[t]);
    }

    const uint4* part;
    auto next_part = [&] {
      feed();
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      part = ring + slot * kPart + threadIdx.x;
      slot = slot + 1 == kStages ? 0 : slot + 1;
    };
    next_part();
    int left = run.in1 - run.in0;  // vectors from this part on
    float bound = -INFINITY, best = -INFINITY, second = -INFINITY;  // best, second: of this thread's vectors
    if (TOP) {
#pragma unroll 1
      for (int u = 0; u < kVecs; ++u)
        if (u * kThreads + (int)threadIdx.x < left) {
          const float y = fmaxf(Elem<T>::largest(part[u * kThreads]), -INFINITY);  // NaN is none
          second = fmaxf(second, fminf(best, y));
          best = fmaxf(best, y);
        }
      bound = bound_of<WARPS>(__fmul_rn(best, a.scale), __fmul_rn(second, a.scale), a.top, sh);
      best = second = -INFINITY;
    }
    // Of elements equal to the bound, those of the first part come first, and are enough.
    bool with = bound > -INFINITY;
    int at = run.in0 + threadIdx.x;
    const bool tighten = a.top * 2 <= kThreads;  // more leave too few of the queue's vectors out
    for (; left >= kPart; left -= kPart) {
      uint4 v[kVecs];
#pragma unroll
      for (int u = 0; u < kVecs; ++u) v[u] = part[u * kThreads];
      const float largest = largest_of<T>(v);
      sums.template add<T>(v, largest, c2);
      if (TOP) {
        const float y = __fmul_rn(largest, a.scale);
        bool full = false;
        if (y > bound || (with && y == bound)) {
#pragma unroll
          for (int u = 0; u < kVecs; ++u)
            full |= enqueue<WARPS>(Elem<T>::largest(v[u]), at + u * kThreads, bound, with, a.scale, sh);
        }
        second = fmaxf(second, fminf(best, fmaxf(y, -INFINITY)));
        best = fmaxf(best, y);
        if (__syncthreads_or(full)) {
          if (tighten) bound = fmaxf(bound, bound_of<WARPS>(best, second, a.top, sh));
          if (!tighten || prune<WARPS>(sh, bound) > Block<WARPS>::kSettle / 2)
            bound = settle<WARPS, T>(sh, x, a.vocab, run.row.shift, a.scale, a.top, bound);
        }
      }
      with = false;
      at += kPart;
      next_part();
    }
#pragma unroll 1
    for (int u = 0; u <= kVecs; ++u) {
      uint4 v[1] = {none};
      if (u < kVecs) {
        if (u * kThreads + warp * 32 >= left) continue;  // no lane of the warp has one
        v[0] = u * kThreads + (int)threadIdx.x < left ? part[u * kThreads] : none;
      } else if (warp) {
        break;
      } else if (end_at >= 0) {
        v[0] = sh.end[lane];
      }
      const float largest = largest_of<T>(v);
      sums.template add<T>(v, largest, c2);
      if (TOP)
        enqueue<WARPS>(largest, u < kVecs ? at + u * kThreads : end_at, bound, u < kVecs ? with : bound > -INFINITY, a.scale, sh);
    }
    if (TOP) {
      __syncthreads();
      settle<WARPS, T>(sh, x, a.vocab, run.row.shift, a.scale, a.top, bound);
    }
    const unsigned r_next = r + step;

    Sums s = warp_join(sums.total(), c2);
    if (lane == 0) sh.warp[warp] = s;
    __syncthreads();
    if (warp == 0) s = warp_join(lane < WARPS ? sh.warp[lane] : Sums{-INFINITY, 0.f, 0.f}, c2);
    if constexpr (Block<WARPS>::kSplit > 1) if (split > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first CTA has started
      if (warp == 0) {
        Shared<WARPS>* to = cluster.map_shared_rank(&sh, 0);
        if (lane == 0) to->part[rank] = s;
        if (TOP) to->best[rank][lane] = sh.list[0][lane];
      }
      cluster.sync();
      if (rank != 0) return;
      if (TOP) {
        merge_lists<WARPS>(sh.best, split);
        __syncthreads();
      }
      if (warp == 0) s = warp_join(lane < split ? sh.part[lane] : Sums{-INFINITY, 0.f, 0.f}, c2);
    }
    if (warp == 0) {
      const bool empty = s.top == -INFINITY && s.sum == 0.f;
      const float total = log2f(s.sum) * kLn2, top = s.top == -INFINITY ? 0.f : __fmul_rn(s.top, a.scale);
      // Scaled, the largest logit may pass 32 bits (the type's lowest value by a scale above 1): then differences are
      // scaled, and lse, whose infinities stand for rows without and with infinite logits, is the last finite value.
      const bool past = isinf(top) && !isinf(s.top);
      // From the largest logit, not from lse: near the type's lowest value lse has no digits left after the point.
      auto log_prob = [&](float scaled, float raw) {
        return empty ? -INFINITY : past ? fmaf(raw - s.top, a.scale, -total) : scaled - top - total;
      };
      if (lane == 0) {
        if (a.logp)
          a.logp[r] = (unsigned)a.tokens[r] < (unsigned)a.vocab ? log_prob(__fmul_rn(sh.given, a.scale), sh.given) : 0.f;
        if (a.lse) a.lse[r] = empty ? -INFINITY : past && total == total ? copysignf(0x1.fffffep127f, top) : top + total;
        if (ENTROPY) a.entropy[r] = empty ? 0.f : (log2f(s.sum) - s.dot / s.sum) * kLn2;
      }
      if (TOP) {
        Key k = sh.list[0][lane];
        if (Block<WARPS>::kSplit > 1 && split > 1) k = sh.best[0][lane];
        // Fewer than `top` above -inf: -inf and then NaN follow, in the order of the tokens.
        int have = __popc(__ballot_sync(~0u, k != 0));
        for (int kind = 0; kind < 2; ++kind)
          for (int c0 = 0; have < a.top && c0 < a.vocab; c0 += 32) {
            const int c = c0 + lane;
            const float y = c < a.vocab ? __fmul_rn(Elem<T>::to(x[c]), a.scale) : 0.f;
            const bool hit = kind ? y != y : y == -INFINITY;
            const uint32_t hits = __ballot_sync(~0u, hit);
            for (int i = have; i < min(32, have + __popc(hits)); ++i) {
              const int from = __fns(hits, 0, i - have + 1);
              if (lane == i) k = rank_of(kind ? NAN : -INFINITY, c0 + from);
            }
            have = min(32, have + __popc(hits));
          }
        if (lane < a.top) {
          if (a.top_tokens) a.top_tokens[(long long)r * a.top + lane] = token_of(k);
          if (a.top_logp)
            a.top_logp[(long long)r * a.top + lane] = log_prob(value_of(k), past ? Elem<T>::to(x[token_of(k)]) : 0.f);
        }
      }
    }
    if (r_next >= (unsigned)a.rows) return;
    r = r_next;
    run = Run<T>(a, r, rank, split);
    __syncthreads();  // the shared arrays are free again
    if (TOP && warp == 0) sh.list[0][lane] = 0;
  }
}

// ------------------------------------------------------------------ backward

constexpr int kBwdThreads = 256;
constexpr int kBwdVecs = 4;  // vectors of a thread

__device__ __forceinline__ float block_reduce(float v, bool largest, float* red) {
  auto both = [&](float x, float y) { return largest ? fmaxf(x, y) : x + y; };
#pragma unroll
  for (int o = 16; o; o >>= 1) v = both(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kBwdThreads / 32; ++w) v = both(v, red[w]);
  return v;
}

// Element-wise, bound by HBM (2048 x 131072 bf16 with entropy 176 us = 6.1 TB/s,
// 94 % of a plain copy): a CTA takes one part of a row, a thread kBwdVecs vectors.
//   dlogits = scale (p (-dlogp - dentropy (x - lse + entropy)) + dlogp [c = token])
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kBwdThreads) token_score_bwd_kernel(const __grid_constant__ TokenScoreBwdArgs a, int parts) {
  constexpr int N = Elem<T>::N;
  __shared__ float red[kBwdThreads / 32];
  wait_for_previous_kernel();
  const int r = blockIdx.x / parts, part = blockIdx.x % parts;
  const T* x = (const T*)a.logits + (long long)r * a.ld;
  T* dx = (T*)a.dlogits + (long long)r * a.ldd;
  const Row<T> row(x, a.vocab);
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  const float lse = a.lse[r];
  const int token = a.dlogp && lse != -INFINITY ? a.tokens[r] : -1;
  const float gl = (unsigned)token < (unsigned)a.vocab ? a.dlogp[r] * a.scale : 0.f;
  const float ge = ENTROPY ? a.dentropy[r] * a.scale : 0.f;
  const float g0 = ENTROPY ? -fmaf(ge, a.entropy[r], gl) : -gl;
  const int vectors = row.vectors();
  int first = part * kBwdVecs * kBwdThreads, last = min(first + kBwdVecs * kBwdThreads, vectors);

  // x - lse = (x - top) - total. A large lse has too few digits after the
  // point for that: the row is summed again, by one CTA, which also writes all
  // of it (the others might overwrite what is being summed). That is the given
  // lse to more digits if it is this row's own, to the last place of 32 bits;
  // one of more than this row (of a vocabulary in shards) is taken as it is.
  float top = 0.f, total = lse;
  const bool far = fabsf(lse) > kFarLse && lse != -INFINITY;
  if (far) {
    if (part) return;
    last = vectors;
    float m = -INFINITY;
    for (int c = threadIdx.x; c < a.vocab; c += kBwdThreads) m = fmaxf(m, Elem<T>::to(x[c]));
    top = block_reduce(m, true, red);
    float sum = 0.f;
    for (int c = threadIdx.x; c < a.vocab; c += kBwdThreads) sum += expf((Elem<T>::to(x[c]) - top) * a.scale);
    total = logf(block_reduce(sum, false, red));
    const float own = __fadd_rn(__fmul_rn(top, a.scale), total);
    if (fabsf(lse - own) > 0x1p-23f * fabsf(own)) total = fmaf(-top, a.scale, lse);
    __syncthreads();
  }
  // Where p is 0 the distance from lse must not be infinite.
  const float floor = (lse - 200.f) / a.scale;
  const bool fast = !far && fabsf(floor) < 1e30f;
  const F2 scale = pair(a.scale, a.scale), minus = pair(-lse, -lse), log2e = pair(kLog2e, kLog2e);
  const F2 minus_ge = pair(-ge, -ge), base = pair(g0, g0);

  for (; first < last; first += kBwdVecs * kBwdThreads) {
    uint4 v[kBwdVecs];
#pragma unroll
    for (int u = 0; u < kBwdVecs; ++u) {
      const int i = first + u * kBwdThreads + threadIdx.x;
      if (i < last) v[u] = row.load(i);
    }
#pragma unroll
    for (int u = 0; u < kBwdVecs; ++u) {
      const int i = first + u * kBwdThreads + threadIdx.x;
      if (i >= last) break;
      const int c = i * N - row.shift;
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        float2 g;
        if (fast) {
          const F2 d = fma2(ENTROPY ? Elem<T>::at_least(v[u], k, floor) : Elem<T>::get(v[u], k), scale, minus);
          const float2 f = split(mul2(d, log2e));
          const F2 p = pair(ex2_approx(f.x), ex2_approx(f.y));
          g = split(mul2(p, ENTROPY ? fma2(d, minus_ge, base) : base));
        } else {
          const float2 y = split(Elem<T>::get(v[u], k));
          auto grad = [&](float z) {
            if (lse == -INFINITY || z == -INFINITY) return 0.f;
            const float d = (z - top) * a.scale - total, p = ex2_approx(d * kLog2e);
            return p == 0.f ? 0.f : p * fmaf(-ge, d, g0);
          };
          g = make_float2(grad(y.x), grad(y.y));
        }
        if (token - c == 2 * k) g.x += gl;
        if (token - c == 2 * k + 1) g.y += gl;
        Elem<T>::put(v[u], k, g);
      }
      if (same && row.inside(i)) {
        __stcs(reinterpret_cast<uint4*>(dx - row.shift) + i, v[u]);
      } else {
        const T* e = reinterpret_cast<const T*>(&v[u]);
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (c + k >= 0 && c + k < a.vocab) dx[c + k] = e[k];
      }
    }
  }
}

template <int WARPS, typename T, bool ENTROPY, bool TOP>
cudaError_t launch_score(const TokenScoreArgs& a, int split, int num_sms, cudaStream_t s) {
  using B = Block<WARPS>;
  static PerDevice allowed, resident;
  const cudaError_t set = allow_shared_memory(allowed, token_score_kernel<WARPS, T, ENTROPY, TOP>, B::kSmem);
  if (set != cudaSuccess) return set;
  const int per_sm = resident_ctas(resident, token_score_kernel<WARPS, T, ENTROPY, TOP>, B::kThreads, B::kSmem);
  const dim3 grid((unsigned)(split > 1 ? a.rows * split : a.rows < num_sms * per_sm ? a.rows : num_sms * per_sm));
  ProfLaunch prof("token_score_kernel", grid, dim3(B::kThreads), B::kSmem, s);
  return launch_next(token_score_kernel<WARPS, T, ENTROPY, TOP>, grid, B::kThreads, B::kSmem, s, split, a, split);
}

template <int WARPS, typename T>
cudaError_t score_by(const TokenScoreArgs& a, int split, int num_sms, cudaStream_t s) {
  if (a.top)
    return a.entropy ? launch_score<WARPS, T, true, true>(a, split, num_sms, s)
                     : launch_score<WARPS, T, false, true>(a, split, num_sms, s);
  return a.entropy ? launch_score<WARPS, T, true, false>(a, split, num_sms, s)
                   : launch_score<WARPS, T, false, false>(a, split, num_sms, s);
}

template <typename T>
cudaError_t score_of(const TokenScoreArgs& a, int num_sms, cudaStream_t s) {
  if (a.rows > 16ll * num_sms) return score_by<kOne, T>(a, 1, num_sms, s);
  if (a.rows >= 8ll * num_sms) return score_by<kTwo, T>(a, 1, num_sms, s);
  if (a.rows > (long long)Block<kEight>::kPerSm * num_sms) return score_by<kFour, T>(a, 1, num_sms, s);
  // Rows are split while that leaves SMs without work and a CTA at least 4096 elements.
  int split = 1;
  while (split < kMostSplit && (long long)a.rows * split * 2 <= 2ll * num_sms && a.vocab / (split * 2) >= 4096) split *= 2;
  return score_by<kEight, T>(a, split, num_sms, s);
}

template <typename T>
cudaError_t grad_of(const TokenScoreBwdArgs& a, cudaStream_t s) {
  constexpr int each = kBwdVecs * kBwdThreads * Elem<T>::N;
  const int parts = (int)(((long long)a.vocab + Elem<T>::N + each - 1) / each);
  if ((long long)a.rows * parts > INT_MAX) return cudaErrorInvalidValue;
  const int grid = a.rows * parts;
  ProfLaunch prof("token_score_bwd_kernel", dim3(grid), dim3(kBwdThreads), 0, s);
  return launch_next(a.dentropy ? token_score_bwd_kernel<T, true> : token_score_bwd_kernel<T, false>, dim3(grid), kBwdThreads, 0, s, 1,
                     a, parts);
}

}  // namespace

cudaError_t launch_token_score(const TokenScoreArgs& a, int num_sms, cudaStream_t s) {
  if (a.vocab > 1 << 30) return cudaErrorNotSupported;  // elements of a row are counted in 32 bits
  if (a.dtype == 0) return score_of<float>(a, num_sms, s);
  return a.dtype == 1 ? score_of<__nv_bfloat16>(a, num_sms, s) : score_of<__half>(a, num_sms, s);
}

cudaError_t launch_token_score_bwd(const TokenScoreBwdArgs& a, int, cudaStream_t s) {
  if (a.vocab > 1 << 30) return cudaErrorNotSupported;
  if (a.dtype == 0) return grad_of<float>(a, s);
  return a.dtype == 1 ? grad_of<__nv_bfloat16>(a, s) : grad_of<__half>(a, s);
}

}  // namespace grx
