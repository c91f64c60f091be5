// The paged key-value cache: append and eviction. Both move rows of headDim
// 2-byte elements as 16-byte vectors and compute nothing on them.
#include <cooperative_groups.h>
#include <limits.h>

#include "profile.h"
#include "serving.cuh"

namespace cg = cooperative_groups;

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
// Bound by HBM (each byte read once and written once: 15288 tokens of 8 heads of
// 128 in 22.1 us, 5.7 TB/s); a single token by the chain lens -> page table ->
// copy (64 sequences 2.4 us). `write_lens`: this kernel also writes the
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
// reaches by keeping loads of two chunks under way while one is stored. 16
// sequences of 3000 to 16000 tokens cut to 4096 (8 heads of 128) take 104 us, of
// which the selection has 17 and the move runs at 6.1 TB/s; one sequence of
// 1051 cut to 1024 takes 12.7 us, a chain of accesses in both kernels (device
// times, replays of a graph).

constexpr int kBins = 2048;  // of a digit: 11, 11 and 10 bits
constexpr int kMostTeam = 8;

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

// A cluster of `team` CTAs per (sequence, kv head): the slots it keeps, in rising
// order, into kept[0..count). The older slots compete for `need` places: their
// smallest kept key is found digit by digit, from histograms; of the slots at
// that key the oldest stay. A CTA has a run of the older slots; a thread holds
// EACH neighbouring weights, in registers throughout where the CTA holds its
// whole run. The CTAs add up their histograms from each other's shared memory.
template <int THREADS, int EACH>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const __grid_constant__ KvEvictArgs a, int* kept_all, int* counts,
                                                               int team) {
  constexpr int SPAN = THREADS * EACH;  // weights that the CTA holds at a time
  constexpr int BINS = kBins / THREADS;  // of a thread
  __shared__ int bins[2][kBins];         // of a digit and of the next
  __shared__ int red[32];
  __shared__ int found[2];
  __shared__ int2 sums[kMostTeam];       // ties and kept slots of the team's CTAs
  wait_for_previous_kernel();
  let_next_kernel_in();  // the move, whose CTAs are many
  cg::cluster_group cluster = cg::this_cluster();
  auto team_barrier = [&] {
    if (team > 1) cluster.sync();
    else __syncthreads();
  };
  const int item = blockIdx.x / team, rank = blockIdx.x % team, b = item / a.in.kv_heads;
  const int n = a.in.clamp_len(a.lens[b]);
  const int count = min(n, a.keep);
  const int old = n - min(n, a.recent);  // slots before the recent ones
  const int need = count - (n - old);    // of them stay
  const float* w = a.weights + (long long)item * a.weights_stride;
  int* kept = kept_all + (long long)item * a.keep;
  const int thread = rank * THREADS + threadIdx.x, threads = team * THREADS;
  if (thread == 0) counts[item] = count;
  for (int i = need + thread; i < a.keep; i += threads) kept[i] = i < count ? old + i - need : -1;
  if (need == old) {
    for (int i = thread; i < need; i += threads) kept[i] = i;
    return;  // the whole team
  }
  if (need == 0) return;
  const int run = ((old + team - 1) / team + 3) & ~3;  // of whole vectors
  const int begin = min(rank * run, old), end = min(begin + run, old);

  uint32_t key[EACH];
  int held = -1;  // first slot of the span in the registers
  auto hold = [&](int from) {
    if (held == from) return;
    held = from;
    const int j = from + threadIdx.x * EACH;
    const bool vectors = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
#pragma unroll
    for (int i = 0; i < EACH; i += 4) {
      if (vectors && j + i + 4 <= end) {
        const float4 x = *reinterpret_cast<const float4*>(w + j + i);
        key[i] = order_key(x.x);
        key[i + 1] = order_key(x.y);
        key[i + 2] = order_key(x.z);
        key[i + 3] = order_key(x.w);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) key[i + k] = j + i + k < end ? order_key(w[j + i + k]) : 0;  // 0 is no weight's key
      }
    }
  };

  uint32_t bound = 0, known = 0;  // the digits found so far, and which bits those are
  int places = need;              // for keys that share them
  for (int i = threadIdx.x; i < kBins; i += THREADS) bins[0][i] = 0;
  __syncthreads();
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, width = digit < 2 ? 11 : 10;
    int* mine = bins[digit & 1];
    for (int from = begin; from < end; from += SPAN) {
      hold(from);
      // Neighbours with one digit (zeros, a handful of values) are added together.
      int same = -1, length = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const bool counts = key[i] && (key[i] & known) == bound;
        const int bin = key[i] >> shift & ((1 << width) - 1);
        if (counts && bin != same) {
          if (length) atomicAdd(&mine[same], length);
          same = bin;
          length = 0;
        }
        length += counts;
      }
      if (length) atomicAdd(&mine[same], length);
    }
    // The other histogram was read to its end before the last barrier.
    for (int i = threadIdx.x; i < kBins; i += THREADS) bins[1 - (digit & 1)][i] = 0;
    team_barrier();
    // Bins from the highest down: the one in which the places run out.
    const int hi = kBins - 1 - BINS * (int)threadIdx.x;
    int in_bin[BINS] = {}, all = 0;
    for (int c = 0; c < team; ++c) {
      const int* theirs = team > 1 ? cluster.map_shared_rank(mine, c) : mine;
#pragma unroll
      for (int i = 0; i < BINS; ++i) in_bin[i] += theirs[hi - i];
    }
#pragma unroll
    for (int i = 0; i < BINS; ++i) all += in_bin[i];
    int sum = scan_block<THREADS>(all, red).x;
    if (sum < places && places <= sum + all) {
#pragma unroll
      for (int i = 0; i < BINS; ++i) {
        if (sum < places && places <= sum + in_bin[i]) {
          found[0] = hi - i;
          found[1] = places - sum;
        }
        sum += in_bin[i];
      }
    }
    team_barrier();
    bound |= (uint32_t)found[0] << shift;
    known |= (uint32_t)((1 << width) - 1) << shift;
    places = found[1];
  }

  // `places` of the keys at the bound stay, the oldest: the CTAs before this one come first.
  int kept_before = 0, ties_before = 0;
  if (team > 1) {
    int ties = 0, above = 0;
    for (int from = begin; from < end; from += SPAN) {
      hold(from);
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        ties += key[i] == bound;
        above += key[i] > bound;
      }
    }
    const int t = scan_block<THREADS>(ties, red).y, s = scan_block<THREADS>(above, red).y;
    if ((int)threadIdx.x < team) *cluster.map_shared_rank(&sums[rank], threadIdx.x) = make_int2(t, s);
    team_barrier();
    for (int c = 0; c < rank; ++c) {
      kept_before += sums[c].y;
      ties_before += sums[c].x;
    }
    kept_before += min(ties_before, places);
  }
  for (int from = begin; from < end; from += SPAN) {
    hold(from);
    int ties = 0, above = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      ties += key[i] == bound;
      above += key[i] > bound;
    }
    const int2 t = scan_block<THREADS>(ties, red);
    int tie = ties_before + t.x;
    const int mine = above + max(0, min(places - tie, ties));
    const int2 s = scan_block<THREADS>(mine, red);
    int at = kept_before + s.x;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      bool stays = key[i] > bound;
      if (key[i] == bound) stays = tie++ < places;
      if (stays) kept[at++] = from + threadIdx.x * EACH + i;
    }
    ties_before += t.y;
    kept_before += s.y;
  }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 8;    // vectors of a thread in a chunk
constexpr int kMoveStages = 3;  // chunks in shared memory

template <int DIM>
struct Move {
  static constexpr int kVecs = DIM / 8, kStep = kMoveThreads / kVecs, kRows = kStep * kMoveVecs;  // rows of a CTA's chunk
  static constexpr int kRing = kMoveStages * kMoveVecs * kMoveThreads * 16;
  static constexpr int kSlots = kMoveStages + 1;  // chunks whose offsets are known
  static constexpr int kSmem = kRing + kSlots * kRows * 2 * 8;
};

// `team` CTAs move the K or the V rows of one (sequence, kv head), chunk by
// chunk in rising order, each CTA a run of the chunk's rows. Every thread copies
// its own vectors to shared memory, kMoveStages - 1 chunks ahead, and on to
// their places. In place (`together`, the team a cluster) a chunk may be written
// once all of it is read: kept slot i came from slot j >= i, so its destinations
// lie before every source of the chunks after it, whose reading goes on. Along
// y: K, V, and the weights with the length.
template <int DIM>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ KvEvictArgs a, const int* kept_all,
                                                                  const int* counts, int team, bool together) {
  using M = Move<DIM>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;                                      // [stage][vector][thread]
  long long(*from_at)[M::kRows] = reinterpret_cast<long long(*)[M::kRows]>(smem + M::kRing);     // [slot][row]
  long long(*to_at)[M::kRows] = from_at + M::kSlots;
  const int item = blockIdx.x / team, rank = blockIdx.x % team, b = item / a.in.kv_heads, h = item % a.in.kv_heads;
  const int* kept = kept_all + (long long)item * a.keep;
  wait_for_previous_kernel();
  const int count = counts[item];
  const bool barrier = together && team > 1;
  if (blockIdx.y == 2) {
    const float* w = a.weights + (long long)item * a.weights_stride;
    float* wo = a.weights_out + (long long)item * a.weights_out_stride;
    const int each = kMoveThreads * kMoveVecs;
    for (int i0 = 0; i0 < count; i0 += team * each) {
      float x[kMoveVecs];
      const int first = i0 + rank * each + threadIdx.x;
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u) {
        const int i = first + u * kMoveThreads;
        x[u] = i < count ? w[kept[i]] : 0.f;
      }
      if (barrier) cluster_sync();
      else __syncthreads();
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u) {
        const int i = first + u * kMoveThreads;
        if (i < count) wo[i] = x[u];
      }
    }
    // All weights are read. What lies behind the kept ones is 0.
    for (int i = count + rank * kMoveThreads + threadIdx.x; i < a.out.capacity; i += team * kMoveThreads) wo[i] = 0.f;
    if (h == 0 && rank == 0 && threadIdx.x == 0) a.lens_out[b] = count;
    return;
  }
  const uint16_t* src = (const uint16_t*)(blockIdx.y ? a.v_in : a.k_in) + h * a.in.s_head;
  uint16_t* dst = (uint16_t*)(blockIdx.y ? a.v_out : a.k_out) + h * a.out.s_head;
  const int chunks = (count + team * M::kRows - 1) / (team * M::kRows);
  const int row = threadIdx.x / M::kVecs, d = threadIdx.x % M::kVecs * 8;
  auto first_row = [&](int c) { return (c * team + rank) * M::kRows; };
  // The old slot of the chunk's row threadIdx.x, or -1.
  auto slot_of = [&](int c) {
    const int i = first_row(c) + threadIdx.x;
    return (int)threadIdx.x < M::kRows && c < chunks && i < count ? kept[i] : -1;
  };
  // Offsets of the chunk's row threadIdx.x, -1 for one that stays where it is or
  // has no page: asked for, and later put where the CTA sees them.
  long long from = -1, to = -1;
  auto ask = [&](int c, int j) {
    from = to = -1;
    if (j < 0) return;
    from = a.in.offset(b, j);
    to = a.out.offset(b, first_row(c) + threadIdx.x);
  };
  auto put = [&](int c, int j) {
    if ((int)threadIdx.x >= M::kRows) return;
    if (j >= 0 && (from < 0 || to < 0)) {
      a.in.report_bad_page();
      from = -1;
    } else if (src + from == dst + to) {
      from = -1;
    }
    from_at[c % M::kSlots][threadIdx.x] = from;
    to_at[c % M::kSlots][threadIdx.x] = to;
  };
  auto load = [&](int c) {
    if (c < chunks) {
#pragma unroll
      for (int u = 0; u < kMoveVecs; ++u) {
        const long long from = from_at[c % M::kSlots][u * M::kStep + row];
        if (from >= 0)
          asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(
                           smem_u32(ring + (c % kMoveStages * kMoveVecs + u) * kMoveThreads)),
                       "l"(src + from + d)
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (chunks == 0) return;
  // All slots, then all pages, then where they are put: the loads of a kind are under way together.
  int first[kMoveStages];
  long long from_of[kMoveStages], to_of[kMoveStages];
#pragma unroll
  for (int c = 0; c < kMoveStages; ++c) first[c] = slot_of(c);
  int j = slot_of(kMoveStages);
#pragma unroll
  for (int c = 0; c < kMoveStages; ++c) {
    ask(c, first[c]);
    from_of[c] = from;
    to_of[c] = to;
  }
#pragma unroll
  for (int c = 0; c < kMoveStages; ++c) {
    from = from_of[c];
    to = to_of[c];
    put(c, first[c]);
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c + 1 < kMoveStages; ++c) load(c);
  for (int c = 0; c < chunks; ++c) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kMoveStages - 2) : "memory");  // this thread's part of chunk c
    // All of chunk c is read; the offsets of chunk c + kMoveStages - 1 are known.
    if (barrier) cluster_sync();
    else __syncthreads();
    const int j_next = slot_of(c + kMoveStages + 1);
    ask(c + kMoveStages, j);
    load(c + kMoveStages - 1);
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u) {
      const int r = u * M::kStep + row;
      if (from_at[c % M::kSlots][r] >= 0)
        *reinterpret_cast<uint4*>(dst + to_at[c % M::kSlots][r] + d) = ring[(c % kMoveStages * kMoveVecs + u) * kMoveThreads];
    }
    put(c + kMoveStages, j);
    j = j_next;
  }
}

template <int DIM>
cudaError_t launch_move(const KvEvictArgs& a, int num_sms, const int* kept, const int* counts, cudaStream_t s) {
  using M = Move<DIM>;
  static PerDevice allowed;
  const cudaError_t set = allow_shared_memory(allowed, evict_move_kernel<DIM>, M::kSmem);
  if (set != cudaSuccess) return set;
  // Pools and weights of their own overlap nowhere: then the team needs no barrier.
  const bool together = a.k_in == a.k_out || a.v_in == a.v_out || a.k_in == a.v_out || a.v_in == a.k_out || a.weights == a.weights_out;
  const int items = a.in.batch * a.in.kv_heads;
  // Teams while CTAs are few and have rows of their own. Without a barrier they
  // even out the SMs' loads: 80 heads of 8115 kept tokens take 161 us without
  // teams, 142 in teams of four. In a cluster that barrier is dear (128 heads of
  // 4096: 124 us in teams of two, 107 without teams at that time): only where SMs
  // lie idle.
  const long long wanted = together ? num_sms : 3ll * num_sms, most = together ? kMostTeam : 256;
  int team = 1;
  while (team < most && items * 2ll * team < wanted && a.keep > team * M::kRows) team *= 2;
  if ((long long)items * team > INT_MAX) return cudaErrorInvalidValue;
  const dim3 grid(items * team, 3);
  ProfLaunch prof("evict_move_kernel", grid, dim3(kMoveThreads), M::kSmem, s);
  return launch_next(evict_move_kernel<DIM>, grid, kMoveThreads, M::kSmem, s, together ? team : 1, a, kept, counts, team, together);
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
  return (size_t)a.in.batch * a.in.kv_heads * (a.indices ? 1 : a.keep + 1) * sizeof(int);
}

cudaError_t launch_kv_evict(const KvEvictArgs& a, int num_sms, void* ws, cudaStream_t s) {
  if ((long long)a.in.batch * a.in.kv_heads > INT_MAX) return cudaErrorInvalidValue;
  const int items = a.in.batch * a.in.kv_heads;
  int* counts = static_cast<int*>(ws);
  int* kept = a.indices ? a.indices : counts + items;  // in the form that a caller is given
  // Where a CTA of 256 threads holds all weights, its barriers are the cheaper
  // ones. Where one of 1024 does not and SMs are without work, a team does; else
  // its threads hold twice as many (and read what is over again for each digit).
  const bool small = a.in.capacity <= 256 * 16;
  int team = 1;
  while (!small && team < kMostTeam && (long long)team * 1024 * 16 < a.in.capacity && items * 2ll * team <= num_sms) team *= 2;
  const bool large = !small && (long long)team * 1024 * 16 < a.in.capacity;
  if ((long long)items * team > INT_MAX) return cudaErrorInvalidValue;
  {
    const int threads = small ? 256 : 1024;
    ProfLaunch prof("evict_select_kernel", dim3(items * team), dim3(threads), 0, s);
    const auto kernel = small ? evict_select_kernel<256, 16> : large ? evict_select_kernel<1024, 32> : evict_select_kernel<1024, 16>;
    const cudaError_t e = launch_next(kernel, dim3(items * team), threads, 0, s, team, a, kept, counts, team);
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
