// The paged key-value cache: append and eviction. Both move rows of headDim
// 2-byte elements as 16-byte vectors and compute nothing on them.
#include <limits.h>

#include "profile.h"
#include "serving.cuh"

namespace grx {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendVecs = 4;       // vectors of K, and as many of V, that a thread has under way
constexpr int kAppendTokens = 64;    // of a CTA at most

__device__ __forceinline__ int appended(const KvAppendArgs& a, int b, int held, bool& dropped) {
  const int count = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens, room = a.cache.capacity - held;
  dropped = count > room;
  return min(count, room);
}

// A CTA copies a run of one sequence's new tokens; their pages are looked up
// once, then neighbouring threads copy neighbouring 16 bytes of a head's row.
// Bound by HBM (each byte read once and written once); a single token by the
// chain lens -> page table -> copy. `write_lens`: this kernel also writes the
// new length, which it may where lens_out is not lens or the sequence is this
// CTA's alone.
template <int DIM>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ KvAppendArgs a, int tokens_per_cta,
                                                                   int chunks, FastDiv per_token, bool write_lens) {
  constexpr int VECS = DIM / 8;
  __shared__ long long at[kAppendTokens];
  wait_for_previous_kernel();
  const int b = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int held = a.cache.clamp_len(a.lens[b]);
  bool dropped;
  const int count = appended(a, b, held, dropped);
  if (dropped && threadIdx.x == 0) a.cache.report_bad_page();
  const int t0 = chunk * tokens_per_cta, n = min(tokens_per_cta, count - t0);
  if ((int)threadIdx.x < n) {
    const long long to = a.cache.offset(b, held + t0 + threadIdx.x);
    if (to < 0) a.cache.report_bad_page();
    at[threadIdx.x] = to;
  }
  __syncthreads();
  if (write_lens && chunk == 0 && threadIdx.x == 0) a.lens_out[b] = held + count;
  const int total = n * (int)per_token.d;  // vectors of K
  const uint16_t* k = (const uint16_t*)a.k + b * a.k_sb + t0 * a.k_ss;
  const uint16_t* v = (const uint16_t*)a.v + b * a.v_sb + t0 * a.v_ss;
  for (int i0 = threadIdx.x; i0 < total; i0 += kAppendThreads * kAppendVecs) {
    uint4 x[kAppendVecs], y[kAppendVecs];
    long long to[kAppendVecs];
#pragma unroll
    for (int u = 0; u < kAppendVecs; ++u) {
      const int i = i0 + u * kAppendThreads;
      to[u] = -1;
      if (i >= total) continue;
      const int t = per_token.div(i), r = i - t * (int)per_token.d, h = r / VECS, d = r % VECS * 8;
      x[u] = __ldcs(reinterpret_cast<const uint4*>(k + t * a.k_ss + h * a.k_sh + d));
      y[u] = __ldcs(reinterpret_cast<const uint4*>(v + t * a.v_ss + h * a.v_sh + d));
      if (at[t] >= 0) to[u] = at[t] + h * a.cache.s_head + d;
    }
#pragma unroll
    for (int u = 0; u < kAppendVecs; ++u)
      if (to[u] >= 0) {
        *reinterpret_cast<uint4*>((uint16_t*)a.k_pages + to[u]) = x[u];
        *reinterpret_cast<uint4*>((uint16_t*)a.v_pages + to[u]) = y[u];
      }
  }
}

__global__ void kv_lens_kernel(const __grid_constant__ KvAppendArgs a) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  wait_for_previous_kernel();
  if (b >= a.cache.batch) return;
  const int held = a.cache.clamp_len(a.lens[b]);
  bool dropped;
  a.lens_out[b] = held + appended(a, b, held, dropped);
}

template <int DIM>
cudaError_t launch_append(const KvAppendArgs& a, cudaStream_t s) {
  const FastDiv per_token((uint32_t)(a.cache.kv_heads * (DIM / 8)));
  // A CTA's tokens: one round of its threads (15288 tokens of 8 heads of 128: 22.6 us; four rounds: 26.9).
  const long long each = kAppendThreads * kAppendVecs / per_token.d;
  const int per_cta = each < 1 ? 1 : each > kAppendTokens ? kAppendTokens : (int)each;
  const int chunks = a.tokens > 0 ? (a.tokens - 1) / per_cta + 1 : 1;
  if ((long long)chunks * a.cache.batch > INT_MAX) return cudaErrorInvalidValue;
  const bool write_lens = a.lens_out && (a.lens_out != a.lens || chunks == 1);
  const int grid = chunks * a.cache.batch;
  {
    ProfLaunch prof("kv_append_kernel", dim3(grid), dim3(kAppendThreads), 0, s);
    const cudaError_t e = launch_next(kv_append_kernel<DIM>, dim3(grid), kAppendThreads, 0, s, 1, a, per_cta, chunks, per_token, write_lens);
    if (e != cudaSuccess || !a.lens_out || write_lens) return e;
  }
  // The lengths may change once no CTA needs the old ones any more.
  const dim3 lens_grid((a.cache.batch + 255) / 256);
  ProfLaunch prof("kv_lens_kernel", lens_grid, dim3(256), 0, s);
  return launch_next(kv_lens_kernel, lens_grid, 256, 0, s, 1, a);
}

// ------------------------------------------------------------------ eviction
//
// Two kernels: the slots that every (sequence, kv head) keeps, then the move.
// Bound by HBM: the kept rows are read once and written once, which the move
// reaches by keeping a chunk's loads under way while the one before is stored.

constexpr int kEach = 16;     // weights of a thread
constexpr int kBins = 2048;  // of a digit: 11, 11 and 10 bits

// Weights as integers of the same order: larger weight, larger key; -0 as 0
// and NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of the earlier threads' values, and of all threads'. All threads.
template <int THREADS>
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
  int w = lane < THREADS / 32 ? red[lane] : 0;
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
template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const __grid_constant__ KvEvictArgs a, int* kept_all, int* counts) {
  constexpr int SPAN = THREADS * kEach;        // weights that the CTA holds at a time
  constexpr int BINS = kBins / THREADS;        // of a thread
  __shared__ int bins[kBins];
  __shared__ int red[32];
  __shared__ int found[2];
  wait_for_previous_kernel();
  let_next_kernel_in();  // the move, whose CTAs are many
  const int b = blockIdx.x / a.in.kv_heads;
  const int n = a.in.clamp_len(a.lens[b]);
  const int count = min(n, a.keep);
  const int old = n - min(n, a.recent);  // slots before the recent ones
  const int need = count - (n - old);    // of them stay
  const float* w = a.weights + (long long)blockIdx.x * a.weights_stride;
  int* kept = kept_all + (long long)blockIdx.x * a.keep;
  if (threadIdx.x == 0) counts[blockIdx.x] = count;
  for (int i = need + threadIdx.x; i < a.keep; i += THREADS) kept[i] = i < count ? old + i - need : -1;
  if (need == old) {
    for (int i = threadIdx.x; i < need; i += THREADS) kept[i] = i;
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
    for (int i = threadIdx.x; i < kBins; i += THREADS) bins[i] = 0;
    __syncthreads();
    for (int from = 0; from < old; from += SPAN) {
      hold(from);
      // Neighbours with one digit (zeros, a handful of values) are added together.
      int run = -1, length = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const bool counts = key[i] && (key[i] & known) == bound;
        const int bin = key[i] >> shift & ((1 << width) - 1);
        if (counts && bin != run) {
          if (length) atomicAdd(&bins[run], length);
          run = bin;
          length = 0;
        }
        length += counts;
      }
      if (length) atomicAdd(&bins[run], length);
    }
    __syncthreads();
    // Bins from the highest down: the one in which the places run out.
    const int hi = kBins - 1 - BINS * (int)threadIdx.x;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < BINS; ++i) mine += bins[hi - i];
    int sum = scan_block<THREADS>(mine, red).x;
    if (sum < places && places <= sum + mine) {
      int i = 0;
      for (; places > sum + bins[hi - i]; ++i) sum += bins[hi - i];
      found[0] = hi - i;
      found[1] = places - sum;
    }
    __syncthreads();
    bound |= (uint32_t)found[0] << shift;
    known |= (uint32_t)((1 << width) - 1) << shift;
    places = found[1];
  }

  // `places` of the keys at the bound stay, the oldest.
  int kept_before = 0, ties_before = 0;
  for (int from = 0; from < old; from += SPAN) {
    hold(from);
    int ties = 0, above = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      ties += key[i] == bound;
      above += key[i] > bound;
    }
    const int2 t = scan_block<THREADS>(ties, red);
    int tie = ties_before + t.x;
    const int mine = above + max(0, min(places - tie, ties));
    const int2 s = scan_block<THREADS>(mine, red);
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
constexpr int kMoveVecs = 8;  // vectors of a thread under way
constexpr int kMostTeam = 8;

// A cluster ("team") of CTAs moves the K or the V rows of one (sequence, kv
// head), chunk by chunk in rising order, each CTA a run of the chunk's rows.
// Kept slot i came from slot j >= i, so a chunk's destinations lie before every
// source of the chunks after it: once all of a chunk is read (the barrier) it
// may be written while the next one is read, in place too. Along y: K, V, and
// one CTA of the team for the weights, the slots and the length.
template <int DIM>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ KvEvictArgs a, const int* kept_all,
                                                                  const int* counts, int team) {
  constexpr int VECS = DIM / 8, STEP = kMoveThreads / VECS, ROWS = STEP * kMoveVecs;  // rows of a CTA's chunk
  __shared__ long long from_at[3][ROWS], to_at[3][ROWS];
  const int item = blockIdx.x / team, rank = blockIdx.x % team, b = item / a.in.kv_heads, h = item % a.in.kv_heads;
  const int* kept = kept_all + (long long)item * a.keep;
  wait_for_previous_kernel();
  const int count = counts[item];
  if (blockIdx.y == 2) {
    if (rank) return;
    const float* w = a.weights + (long long)item * a.weights_stride;
    float* wo = a.weights_out + (long long)item * a.weights_out_stride;
    for (int i0 = 0; i0 < count; i0 += kMoveThreads * kMoveVecs) {
      float x[kMoveVecs];
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u) {
        const int i = i0 + u * kMoveThreads + threadIdx.x;
        x[u] = i < count ? w[kept[i]] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u) {
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
  const uint16_t* src = (const uint16_t*)(blockIdx.y ? a.v_in : a.k_in) + h * a.in.s_head;
  uint16_t* dst = (uint16_t*)(blockIdx.y ? a.v_out : a.k_out) + h * a.out.s_head;
  const int chunks = (count + team * ROWS - 1) / (team * ROWS);
  const int row = threadIdx.x / VECS, d = threadIdx.x % VECS * 8;
  auto first_row = [&](int c) { return (c * team + rank) * ROWS; };
  // The old slot of the chunk's row threadIdx.x, or -1.
  auto slot_of = [&](int c) {
    const int i = first_row(c) + threadIdx.x;
    return threadIdx.x < ROWS && i < count ? kept[i] : -1;
  };
  // Offsets of the chunk's rows, -1 for one that stays where it is or has no page.
  auto look_up = [&](int c, int j) {
    if (threadIdx.x >= ROWS) return;
    long long from = -1, to = -1;
    if (j >= 0) {
      from = a.in.offset(b, j);
      to = a.out.offset(b, first_row(c) + threadIdx.x);
      if (from < 0 || to < 0) {
        a.in.report_bad_page();
        from = -1;
      } else if (src + from == dst + to) {
        from = -1;
      }
    }
    from_at[c % 3][threadIdx.x] = from;
    to_at[c % 3][threadIdx.x] = to;
  };
  auto load = [&](uint4 (&v)[kMoveVecs], int c) {
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u) {
      const long long from = from_at[c % 3][u * STEP + row];
      if (from >= 0) v[u] = *reinterpret_cast<const uint4*>(src + from + d);
    }
  };
  auto store = [&](const uint4 (&v)[kMoveVecs], int c) {
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u)
      if (from_at[c % 3][u * STEP + row] >= 0) *reinterpret_cast<uint4*>(dst + to_at[c % 3][u * STEP + row] + d) = v[u];
  };
  auto team_barrier = [&] {
    if (team > 1) cluster_sync();
    else __syncthreads();
  };
  if (chunks == 0) return;
  uint4 x[kMoveVecs], y[kMoveVecs];
  look_up(0, slot_of(0));
  look_up(1, slot_of(1));
  int j = slot_of(2);
  __syncthreads();
  load(x, 0);
  auto step = [&](uint4 (&now)[kMoveVecs], uint4 (&next)[kMoveVecs], int c) {
    team_barrier();  // chunk c is read, the next one's offsets are known
    if (c + 1 < chunks) load(next, c + 1);
    if (c + 2 < chunks) {
      look_up(c + 2, j);
      j = slot_of(c + 3);
    }
    store(now, c);
  };
  for (int c = 0; c < chunks; c += 2) {
    step(x, y, c);
    if (c + 1 < chunks) step(y, x, c + 1);
  }
}

template <int DIM>
cudaError_t launch_move(const KvEvictArgs& a, int num_sms, const int* kept, const int* counts, cudaStream_t s) {
  const int items = a.in.batch * a.in.kv_heads;
  // A team while SMs are without work and its CTAs have rows of their own. At
  // 16 x 8 heads, 256 CTAs without teams, the move takes 92 us; teams of two
  // make it 110 and of four 118: more streams of reads and writes at a time.
  int team = 1;
  while (team < kMostTeam && items * 2ll * team < num_sms && a.keep > team * 32) team *= 2;
  if ((long long)items * team > INT_MAX) return cudaErrorInvalidValue;
  ProfLaunch prof("evict_move_kernel", dim3(items * team, 3), dim3(kMoveThreads), 0, s);
  return launch_next(evict_move_kernel<DIM>, dim3(items * team, 3), kMoveThreads, 0, s, team, a, kept, counts, team);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s) {
  switch (a.cache.head_dim) {
    case 64: return launch_append<64>(a, s);
    case 128: return launch_append<128>(a, s);
    case 256: return launch_append<256>(a, s);
    default: return cudaErrorNotSupported;
  }
}

size_t kv_evict_workspace_bytes(const KvEvictArgs& a) {
  return (size_t)a.in.batch * a.in.kv_heads * (a.keep + 1) * sizeof(int);
}

cudaError_t launch_kv_evict(const KvEvictArgs& a, int num_sms, void* ws, cudaStream_t s) {
  if ((long long)a.in.batch * a.in.kv_heads > INT_MAX) return cudaErrorInvalidValue;
  const int items = a.in.batch * a.in.kv_heads;
  int* counts = static_cast<int*>(ws);
  int* kept = counts + items;
  // Where a CTA of 256 threads holds all weights, its barriers are the cheaper ones.
  const int threads = a.in.capacity <= 256 * kEach ? 256 : 1024;
  {
    ProfLaunch prof("evict_select_kernel", dim3(items), dim3(threads), 0, s);
    const cudaError_t e = launch_next(threads == 256 ? evict_select_kernel<256> : evict_select_kernel<1024>, dim3(items), threads, 0, s,
                                      1, a, kept, counts);
    if (e != cudaSuccess) return e;
  }
  switch (a.in.head_dim) {
    case 64: return launch_move<64>(a, num_sms, kept, counts, s);
    case 128: return launch_move<128>(a, num_sms, kept, counts, s);
    case 256: return launch_move<256>(a, num_sms, kept, counts, s);
    default: return cudaErrorNotSupported;
  }
}

}  // namespace grx
