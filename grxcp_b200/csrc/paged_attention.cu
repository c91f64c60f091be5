// Attention of one new token over a paged key-value cache.
//
//   s_j = scale q . K_j,  o = sum_j p_j V_j / sum_j p_j,  p_j = exp(s_j - max s)
//
// Every key and value is read once for 4 operations a byte and query head, so
// the kernel is bound by HBM as long as its loads never pause.
//
// Split. The keys of one (sequence, kv head, chunk of up to 16 query heads) are
// an item; its keys are cut into tiles. All tiles of all items, in order, form
// one line that the CTAs cut into equal shares, whatever the lengths: a batch of
// ragged sequences and a single long one load every SM alike. Short lines are
// cut item by item instead, so that no CTA ends an item in mid-share. A CTA's
// warps take the tiles of its share in turn, each with its own ring of shared
// memory filled by cp.async, so that no warp waits for another until an item
// ends. Then the warps' partial results (running maximum, sum, output) are
// joined; an item that lies in one share is written out, one that crosses
// shares leaves its parts in memory, where the CTA that comes last, or
// paged_attn_join_kernel, joins them in the order of the keys.
//
// The query heads of an item are the rows of mma.sync (16 x 8 x 16, fp32
// accumulation): at 1 to 16 rows the 128-row tcgen05 tile would stay empty,
// and the tensor pipe is not what bounds this.
//
// Measured (calls among others, as a user makes them): caches of 100003 and
// 131072 tokens (64 query heads on 8, 128, f16) 154 us = 6.1 TB/s, 94 % of a plain
// copy; 64 sequences of 1 to 4096 tokens (32 on 8, 128, bf16) 89 us = 6.05 TB/s,
// 92 %; one of 417 tokens 8.5 us, and the same behind a page table of 131072
// tokens; 64 of up to 4096 of dim 256 5.6 TB/s, of dim 64 4.9; 4 of 16000 tokens (8
// kv heads, 128, bf16) 50 us with 4 query heads on each, 58 with 16: a join's time.
// Short of the copy's rate a warp's chain of look-up, copies, products and softmax
// (430 instructions a tile at 5.9 cycles each, by the counters) is what it waits for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include "profile.h"
#include "serving.cuh"

namespace grx {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;  // query heads of an item: the rows of one MMA
constexpr int kLongShare = 32;  // tiles from which ending an item in mid-share costs little
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int DIM>
struct Shape {
  static constexpr int kKeys = DIM == 64 ? 32 : 16;          // keys of a tile
  static constexpr int kStage = 2 * kKeys * DIM * 2;         // bytes of its K and V
  static constexpr int kStages = DIM == 64 ? 2 : 3;  // tiles of a warp in shared memory
  static constexpr int kSmem = kWarps * kStages * kStage;
  // What ending an item costs, in tiles (64 sequences of 1 to 4096 keys, dim 128: 89.8 us, 91.0 with 6, 92.2 with 20).
  static constexpr int kEnd = DIM == 128 ? 10 : DIM == 256 ? 12 : 6;
  // CTAs that share an SM. A tile's work is a long chain, so that warps count
  // for more than tiles under way: three CTAs with two tiles each against two
  // with three take 34.9 against 37.5 us at 24 x 16 heads of 64.
  static constexpr int kPerSm = DIM == 256 ? 1 : DIM == 128 ? 2 : 3;
  static_assert(kRows * DIM * 4 <= kStage, "a stage holds a warp's output");
};

// Where the parts of an item are: CTA first / 2 holds the first of `count`, in
// its slot first % 2; the next CTAs hold the others, each in its slot 0.
struct Span {
  int first, count;
  __device__ __forceinline__ int part(int k) const { return k ? (first / 2 + k) * 2 : first; }
};

struct Open {
  int b, head0, heads, item;
  Span span;
};

struct Workspace {
  float* part_o;   // [ctas][2][kRows][dim], not yet divided by the sum
  float2* part_ml; // [ctas][2][kRows]: maximum (times log2 e) and sum
  Span* span;      // [batch * kv_heads * chunks]
  float* lse2;     // [batch * heads], log2 of the sum, of the rows that the first kernel finishes; with weights
  float* scores;   // [batch * heads][pitch], times log2 e; with weights
  long long pitch; // the capacity in whole tiles
};

struct Params {
  PagedAttnArgs a;
  Workspace ws;
  int group, chunks;  // query heads of a kv head, and the items they make
  int min_tiles;      // of a share
  int* arrived;       // [items], 0: parts of an item that are written; null: the second kernel joins
};

// One tensor core product of 16-bit types: c += a b.
template <int DTYPE>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DTYPE == 1)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool TRANS>
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// 16 bytes to shared memory, zeros instead where !valid (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}

template <int DTYPE>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (DTYPE == 1) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// The keys that a sequence's query sees, in tiles.
template <int KEYS>
struct Range {
  int first, end, base, tiles;  // keys [first, end); tile t starts at base + t KEYS
  __device__ __forceinline__ Range(const PagedAttnArgs& a, int b) {
    end = a.cache.clamp_len(a.lens[b]);
    first = a.window ? max(0, end - a.window) : 0;
    base = first / KEYS * KEYS;
    tiles = (end - base + KEYS - 1) / KEYS;
  }
};

// A place on the line of all tiles. Each item's tiles follow kEnd places that
// stand for the cost of ending it, so that shares cost alike.
template <int KEYS, int END>
struct Cursor {
  int b, item, tile;  // item of the sequence, tile of the item
  int start;          // place of the item
  Range<KEYS> r;
  __device__ __forceinline__ Cursor(const PagedAttnArgs& a, int b_, int item_, int tile_, int start_)
      : b(b_), item(item_), tile(tile_), start(start_), r(a, b_) {}
  // Moves past the tiles that the item lacks; the caller stays on the line.
  __device__ __forceinline__ void settle(const PagedAttnArgs& a, int items) {
    while (tile >= r.tiles) {
      tile -= r.tiles;
      if (r.tiles) start += r.tiles + END;
      if (++item == items || r.tiles == 0) {
        item = 0;
        if (++b == a.cache.batch) return;
        r = Range<KEYS>(a, b);
      }
    }
  }
};

// Adds 1. What the CTA wrote before a barrier before this is seen by the CTA
// that counts to the end, past a barrier after this.
__device__ __forceinline__ int arrive(int* counter) {
  int v;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(v) : "l"(counter) : "memory");
  return v;
}

__device__ __forceinline__ int peek(const int* counter) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
  return v;
}

__device__ __forceinline__ int block_sum(int v, int* red) {
  v = __reduce_add_sync(~0u, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += red[w];
  return t;
}

// Four dims of a row: not yet divided by the sum, which like them is relative to 2^top.
struct Partial {
  float4 x;
  float top, sum;
};

// All parts of an item in the order of the keys, whoever joins them; part `mine`, if any, is in hand. kAhead parts are
// loaded at a time: in a loop that is only unrolled each cost a trip to L2 (4 x 16000 tokens, 16 query heads on each kv
// head: 66 us, 58 so; 16 at a time spill: 24 x 300 to 2050 tokens with weights 39 us, 32 so).
constexpr int kAhead = 8;
template <int DIM>
__device__ __noinline__ Partial join_parts(const Workspace& ws, Span span, int row, int d, int mine, Partial own) {
  Partial all{make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
  for (int k0 = 0; k0 < span.count; k0 += kAhead) {
    float2 ml[kAhead];
    float4 y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int k = k0 + i, at = span.part(k) * kRows + row;
      ml[i] = k == mine ? make_float2(own.top, own.sum) : make_float2(0.f, 0.f);
      y[i] = own.x;
      if (k < span.count && k != mine) {
        ml[i] = __ldcg(ws.part_ml + at);
        y[i] = __ldcg(reinterpret_cast<const float4*>(ws.part_o + (long long)at * DIM + d));
      }
    }
    float to = all.top;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (ml[i].y != 0.f) to = fmaxf(to, ml[i].x);
    const float was = all.sum == 0.f ? 0.f : ex2_approx(all.top - to);
    all = Partial{make_float4(all.x.x * was, all.x.y * was, all.x.z * was, all.x.w * was), to, all.sum * was};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (ml[i].y == 0.f) continue;  // no key of it weighs anything; a NaN goes on
      const float f = ex2_approx(ml[i].x - to);
      all.sum = fmaf(ml[i].y, f, all.sum);
      all.x.x = fmaf(y[i].x, f, all.x.x);
      all.x.y = fmaf(y[i].y, f, all.x.y);
      all.x.z = fmaf(y[i].z, f, all.x.z);
      all.x.w = fmaf(y[i].w, f, all.x.w);
    }
  }
  return all;
}

// HALF: items of up to 8 query heads; the MMAs' other 8 rows are left alone.
template <int DTYPE, int DIM, bool WEIGHTS, bool HALF>
__global__ void __launch_bounds__(kThreads, Shape<DIM>::kPerSm) paged_attn_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = HALF ? 1 : 2;  // of a thread: g and g + 8
  constexpr uint32_t ALL = Shape<DIM>::kKeys == 32 ? ~0u : (1u << Shape<DIM>::kKeys) - 1;
  constexpr int END = Shape<DIM>::kEnd;
  constexpr int KEYS = Shape<DIM>::kKeys, kStages = Shape<DIM>::kStages, CH = DIM / 8, STAGE = Shape<DIM>::kStage;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int red[kWarps], red_items[kWarps];
  __shared__ int found[4], flag[2];
  __shared__ float2 ml[kWarps][kRows];
  __shared__ Open opened[2];
  const PagedAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int items = a.cache.kv_heads * p.chunks;
  wait_for_previous_kernel();

  // The CTA's share.
  int mine = 0, mine_items = 0;
  for (int b = threadIdx.x; b < a.cache.batch; b += kThreads) {
    const int n = Range<KEYS>(a, b).tiles;
    mine += n;
    mine_items += n > 0;
  }
  const int total = block_sum(mine, red) * items, full = block_sum(mine_items, red) * items;
  if (p.arrived)  // sequences without keys are on nobody's share
    for (int b = blockIdx.x; b < a.cache.batch; b += gridDim.x)
      if (Range<KEYS>(a, b).tiles == 0) {
        for (int u = threadIdx.x; u < a.heads * CH; u += kThreads)
          *(uint4*)((uint16_t*)a.o + b * a.o_sb + (long long)(u / CH) * a.o_sh + u % CH * 8) = make_uint4(0, 0, 0, 0);
        if (a.lse)
          for (int i = threadIdx.x; i < a.heads; i += kThreads) a.lse[(long long)b * a.heads + i] = -INFINITY;
      }
  // Where shares are short each item is cut for itself, into parts of whole
  // rounds of the warps: an item has less than one part more than its tiles
  // fill, so this fits the grid.
  const int grid = gridDim.x, line = total + full * END;
  int share = max(p.min_tiles, (line + grid - 1) / grid);
  const bool by_item = share < kLongShare && (long long)full * 4 <= (long long)grid * 3;
  if (by_item) {
    share = max(p.min_tiles, (total + grid - full - 1) / (grid - full));
    share = (share + kWarps - 1) / kWarps * kWarps;
  }
  const int place = by_item ? blockIdx.x : blockIdx.x * share;  // in parts, or on the line
  if (threadIdx.x == 0) {
    found[0] = -1;
    found[3] = total;
  }
  int before = 0, before_items = 0;  // places and items (of one head) of the sequences before the chunk below
  for (int c = 0; c < a.cache.batch; c += kThreads) {
    const int b = c + threadIdx.x;
    const int tiles = b < a.cache.batch ? Range<KEYS>(a, b).tiles : 0;
    const int n = by_item ? (tiles + share - 1) / share : tiles ? tiles + END : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    const uint32_t some = __ballot_sync(~0u, n > 0);
    __syncthreads();
    if (lane == 31) {
      red[warp] = x;
      red_items[warp] = __popc(some);
    }
    __syncthreads();
    int at = before + x - n, at_items = before_items + __popc(some & ((1u << lane) - 1));
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        at += red[w];
        at_items += red_items[w];
      }
      before += red[w];
      before_items += red_items[w];
    }
    if (n > 0) {
      const int first = at * items, tiles_before = (at - at_items * END) * items;
      if (first <= place && place < first + n * items) {
        found[0] = b;
        found[1] = place - first;
        found[2] = tiles_before;
      }
      if (!by_item && first <= place + share && place + share < first + n * items) {  // where the share ends
        const int off = place + share - first;
        found[3] = tiles_before + off / n * tiles + max(off % n - END, 0);
      }
    }
    if (before * items > place + (by_item ? 0 : share)) break;
  }
  __syncthreads();
  const int b0 = found[0];
  if (b0 < 0) return;
  // Tiles [t0, t1): of all items, or of the one.
  const Range<KEYS> r0(a, b0);
  const int in_seq = found[1], per_item = by_item ? (r0.tiles + share - 1) / share : r0.tiles + END;
  const int item0 = in_seq / per_item, tile0 = by_item ? in_seq % per_item * share : max(in_seq % per_item - END, 0);
  const int start0 = place - in_seq % per_item;  // of the item on the line
  const int t0 = by_item ? tile0 : found[2] + item0 * r0.tiles + tile0, t1 = by_item ? min(t0 + share, r0.tiles) : found[3];
  if (t0 >= t1) return;

  const uint32_t ring = smem_u32(smem) + warp * (kStages * STAGE);
  // Loads: row_at is the offset of key `lane` of the tile after those already
  // under way, -1 where it has none; asked for one tile ahead, so that the page
  // table's latency passes during a tile's work.
  Cursor<KEYS, END> next(a, b0, item0, tile0 + warp, 0);
  int left = (t1 - t0 - warp + kWarps - 1) / kWarps;  // tiles of this warp not yet loaded
  if (left > 0) next.settle(a, items);
  long long row_at = -1;
  auto look_up = [&] {
    row_at = -1;
    if (left > 0) {
      const int j = next.r.base + next.tile * KEYS + lane % KEYS;
      if (j >= next.r.first && j < next.r.end) {
        row_at = a.cache.offset(next.b, j);
        if (row_at < 0) a.cache.report_bad_page();
        else row_at += (long long)(next.item / p.chunks) * a.cache.s_head;
      }
    }
  };
  uint32_t valid[kStages] = {};  // keys of the tiles in the ring, the oldest first
  int slot = 0;                  // where the next tile goes
  auto load = [&] {
#pragma unroll
    for (int s = 0; s + 1 < kStages; ++s) valid[s] = valid[s + 1];
    valid[kStages - 1] = __ballot_sync(~0u, row_at >= 0);
    if (left > 0) {
      const uint32_t dst = ring + slot * STAGE;
      constexpr int STEP = 32 / CH > 0 ? 32 / CH : 1;  // rows that the warp copies at a time
#pragma unroll
      for (int i = 0; i < KEYS / STEP; ++i) {
        const int row = i * STEP + lane / CH, c = lane % CH;
        const long long at = __shfl_sync(~0u, row_at, row);
        const uint32_t to = dst + row * (DIM * 2) + ((c ^ (row & 7)) * 16);
        const long long from = at < 0 ? 0 : at + c * 8;
        copy16(to, (const uint16_t*)a.k_pages + from, at >= 0);
        copy16(to + KEYS * DIM * 2, (const uint16_t*)a.v_pages + from, at >= 0);
      }
      --left;
      if (left > 0) {
        next.tile += kWarps;
        next.settle(a, items);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    slot = slot + 1 == kStages ? 0 : slot + 1;
    look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s + 1 < kStages; ++s) load();

  const float c2 = a.scale * kLog2e;
  const int g = lane >> 2, q4 = lane & 3;
  Cursor<KEYS, END> seg(a, b0, item0, tile0, start0);
  int t = t0 + warp;        // this warp's next tile
  int seg_start = t0;       // first tile of the segment within this share
  uint32_t q[DIM / 16][4];
  auto first_head = [&] { return seg.item / p.chunks * p.group + seg.item % p.chunks * kRows; };
  auto heads_of = [&](int head0) { return min(kRows, (seg.item / p.chunks + 1) * p.group - head0); };
  auto load_q = [&] {
    const int head0 = first_head(), heads = heads_of(head0);
    const uint16_t* qp = (const uint16_t*)a.q + seg.b * a.q_sb + (long long)head0 * a.q_sh + q4 * 2;
#pragma unroll
    for (int k = 0; k < DIM / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = g + (i & 1) * 8;
        q[k][i] = (!HALF || !(i & 1)) && row < heads ? *(const uint32_t*)(qp + row * a.q_sh + k * 16 + (i >> 1) * 8) : 0u;
      }
  };
  auto write_out = [&](int b, int head, int d, float4 x, float top, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key weighs anything
    uint16_t* op = (uint16_t*)a.o + b * a.o_sb + (long long)head * a.o_sh + d;
    *(uint2*)op = make_uint2(pack2<DTYPE>(x.x * inv, x.y * inv), pack2<DTYPE>(x.z * inv, x.w * inv));
    if (d == 0) {
      const float lse2 = sum == 0.f ? -INFINITY : top + log2f(sum);
      const long long at = (long long)b * a.heads + head;
      if (a.lse) a.lse[at] = lse2 * kLn2;
      if (WEIGHTS) p.ws.lse2[at] = lse2;
    }
  };
  int open = 0;           // items of which this CTA leaves a part: its first and its last at most
  int before_first = -1;  // parts of the first that were there before this CTA's
  load_q();
  while (seg_start < t1) {
    const int item_start = seg_start - seg.tile, item_tiles = seg.r.tiles, b = seg.b, item = seg.b * items + seg.item;
    const int seg_end = min(item_start + item_tiles, t1), base = seg.r.base;
    const int head0 = first_head(), heads = heads_of(head0);
    float o[DIM / 8][4];
    float m[ROWS], l[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DIM / 8; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] = 0.f;

    const int start = seg.start;
    const int first_cta = by_item ? (int)blockIdx.x - tile0 / share : (start + END) / share;
    const int parts = by_item ? (item_tiles + share - 1) / share : (start + END + item_tiles - 1) / share - first_cta + 1;
    const Span span{first_cta * 2 + (by_item || first_cta * share >= start ? 0 : 1), parts};
    const bool last = seg_end == t1;
    int seen = -1;  // parts of the CTA's last item that others have written
    for (; t < seg_end; t += kWarps) {
      if (last && threadIdx.x == 0 && p.arrived && t + kWarps >= seg_end) seen = peek(p.arrived + item);
      const int use = slot + 1 == kStages ? 0 : slot + 1;  // the oldest tile's slot once the next is under way
      load();
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint32_t kt = ring + use * STAGE, vt = kt + KEYS * DIM * 2;
      const uint32_t ok = valid[0];
      float s[KEYS / 8][4];
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < DIM / 16; ++k)
#pragma unroll
        for (int n = 0; n < KEYS / 16; ++n) {
          // matrices: keys 0-7 and 8-15 of the 16, each with both halves of the 16 dims
          const int row = n * 16 + (lane & 7) + (lane >> 4) * 8, c = k * 2 + ((lane >> 3) & 1);
          uint32_t kb[4];
          ldmatrix<false>(kb, kt + row * (DIM * 2) + ((c ^ (row & 7)) * 16));
          mma<DTYPE>(s[2 * n], q[k], kb[0], kb[1]);
          mma<DTYPE>(s[2 * n + 1], q[k], kb[2], kb[3]);
        }
      float top[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) top[i] = -INFINITY;
      if (ok != ALL) {
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
          for (int i = 0; i < 2 * ROWS; ++i)
            if (!(ok >> (n * 8 + q4 * 2 + (i & 1)) & 1)) s[n][i] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2 * ROWS; ++i) {
          s[n][i] *= c2;
          top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
        }
      if constexpr (WEIGHTS) {
        const int j = base + (t - item_start) * KEYS;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int row = g + i * 8;
          if (row >= heads) continue;
          float* to = p.ws.scores + ((long long)b * a.heads + head0 + row) * p.ws.pitch + j + q4 * 2;
#pragma unroll
          for (int n = 0; n < KEYS / 8; ++n) *(float2*)(to + n * 8) = make_float2(s[n][2 * i], s[n][2 * i + 1]);
        }
      }
      bool more = false;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 2));
        more |= top[i] > m[i];
      }
      if (__any_sync(~0u, more)) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const float n = fmaxf(m[i], top[i]);
          const float f = n == -INFINITY ? 1.f : ex2_approx(m[i] - n);
          m[i] = n;
          l[i] *= f;
#pragma unroll
          for (int d = 0; d < DIM / 8; ++d) {
            o[d][2 * i] *= f;
            o[d][2 * i + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float ref = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            s[n][2 * i + k] = ex2_approx(s[n][2 * i + k] - ref);
            l[i] += s[n][2 * i + k];
          }
      }
#pragma unroll
      for (int k = 0; k < KEYS / 16; ++k) {
        // p is at most 1 and its sum is kept in 32 bits: rounding it to the cache's type costs at most that
        // type's unit of each term, as rounding the output does.
        const uint32_t pa[4] = {pack2<DTYPE>(s[2 * k][0], s[2 * k][1]), HALF ? 0u : pack2<DTYPE>(s[2 * k][2], s[2 * k][3]),
                                pack2<DTYPE>(s[2 * k + 1][0], s[2 * k + 1][1]),
                                HALF ? 0u : pack2<DTYPE>(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d) {
          // matrices: keys 0-7 and 8-15 of the 16, for each of two runs of 8 dims
          const int row = k * 16 + (lane & 15), c = d * 2 + (lane >> 4);
          uint32_t vb[4];
          ldmatrix<true>(vb, vt + row * (DIM * 2) + ((c ^ (row & 7)) * 16));
          mma<DTYPE>(o[2 * d], pa, vb[0], vb[1]);
          mma<DTYPE>(o[2 * d + 1], pa, vb[2], vb[3]);
        }
      }
      __syncwarp();  // the slot is free again
    }

    const bool whole = seg_start == item_start && seg_end == item_start + item_tiles;
    const bool first_part = seg_start == t0;
    seg.tile += seg_end - seg_start;
    seg_start = seg_end;
    if (seg_start < t1) {
      seg.settle(a, items);
      load_q();  // while the warps are joined
    }

    // Join the warps. `slot` is the one place of a warp's ring that no load is
    // under way to: it holds the warp's output meanwhile.
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      l[i] += __shfl_xor_sync(~0u, l[i], 1);
      l[i] += __shfl_xor_sync(~0u, l[i], 2);
      if (q4 == 0) ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
    }
    float* mine_o = reinterpret_cast<float*>(smem + warp * (kStages * STAGE) + slot * STAGE);
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (g + 8 * i < heads && l[i] != 0.f)
#pragma unroll
        for (int d = 0; d < DIM / 8; ++d)
          *(float2*)(mine_o + (g + 8 * i) * DIM + d * 8 + q4 * 2) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
    if (lane == 0) red[warp] = slot;
    if (threadIdx.x == 0) {
      flag[0] = !whole && seen == parts - 1;  // they are all there: joined here and now
      if (flag[0]) __threadfence();
    }
    __syncthreads();
    const bool complete = flag[0];
    const int part = (blockIdx.x * 2 + (first_part ? 0 : 1)) * kRows;
    for (int u = threadIdx.x; u < heads * (DIM / 4); u += kThreads) {
      const int row = u / (DIM / 4), d = u % (DIM / 4) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w][row].x);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (ml[w][row].y == 0.f) continue;  // it has left no output; a NaN goes on
        const float f = ex2_approx(ml[w][row].x - top);
        const float4 y = *(const float4*)(smem + (w * kStages + red[w]) * STAGE + (row * DIM + d) * 4);
        sum = fmaf(ml[w][row].y, f, sum);
        x.x = fmaf(y.x, f, x.x);
        x.y = fmaf(y.y, f, x.y);
        x.z = fmaf(y.z, f, x.z);
        x.w = fmaf(y.w, f, x.w);
      }
      if (whole || complete) {
        Partial all{x, top, sum};
        if (!whole) all = join_parts<DIM>(p.ws, span, row, d, (int)blockIdx.x - first_cta, all);
        write_out(b, head0 + row, d, all.x, all.top, all.sum);
      } else {
        *(float4*)(p.ws.part_o + (long long)(part + row) * DIM + d) = x;
        if (d == 0) p.ws.part_ml[part + row] = make_float2(top, sum);
      }
    }
    if (!p.arrived) {
      if (threadIdx.x == 0 && first_cta == (int)blockIdx.x) p.ws.span[item] = span;
    } else if (complete) {
      if (threadIdx.x == 0) p.arrived[item] = 0;  // for the next call
    } else if (!whole) {
      if (threadIdx.x == 0) opened[open] = Open{b, head0, heads, item, span};
      ++open;
    }
    __syncthreads();
    // A first part is counted in at once, so that the CTA before this one finds it; the answer is read at the end.
    if (threadIdx.x == 0 && first_part && !last && open) before_first = arrive(p.arrived + item);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  let_next_kernel_in();

  // Who counts an item's parts to their end joins it.
  if (open == 0) return;
  if (threadIdx.x == 0)
    for (int i = 0; i < open; ++i) {
      const int n = i == 0 && before_first >= 0 ? before_first : arrive(p.arrived + opened[i].item);
      flag[i] = n == opened[i].span.count - 1;
    }
  __syncthreads();
  for (int i = 0; i < open; ++i) {
    if (!flag[i]) continue;
    const Open item = opened[i];
    for (int u = threadIdx.x; u < item.heads * (DIM / 4); u += kThreads) {
      const int row = u / (DIM / 4), d = u % (DIM / 4) * 4;
      const Partial all = join_parts<DIM>(p.ws, item.span, row, d, -1, Partial{});
      write_out(item.b, item.head0 + row, d, all.x, all.top, all.sum);
    }
    if (threadIdx.x == 0) p.arrived[item.item] = 0;  // for the next call
  }
}

// The parts of an item's row, joined in the order of the keys: maximum and sum.
__device__ __forceinline__ float2 join_row(const Workspace& ws, Span sp, int row) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.f;
  for (int k = lane; k < sp.count; k += 32) {
    const float2 x = ws.part_ml[sp.part(k) * kRows + row];
    if (x.y == 0.f) continue;  // no key weighs anything; a NaN goes on
    const float n = fmaxf(top, x.x);
    sum = (sum == 0.f ? 0.f : sum * ex2_approx(top - n)) + x.y * ex2_approx(x.x - n);
    top = n;
  }
  float all = top;
#pragma unroll
  for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(~0u, all, o));
  if (sum != 0.f) sum *= ex2_approx(top - all);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  return make_float2(all, sum);
}

constexpr int kWeightVecs = 2;  // keys of a thread of the second part
constexpr int kWeightKeys = kWeightVecs * kThreads;

// The first batch * heads CTAs, where the first kernel has not joined them: the
// outputs whose parts lie in several shares, and those of sequences without
// keys. The others: weights += sum over the group of 2^(score - lse2).
template <int DTYPE, int DIM, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads) paged_attn_join_kernel(const __grid_constant__ Params p, int splits) {
  constexpr int VEC = DIM / 32;
  __shared__ float sum_o[kWarps][DIM];
  __shared__ float lse2[kThreads];
  const PagedAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.arrived ? 0 : a.cache.batch * a.heads;
  wait_for_previous_kernel();
  if ((int)blockIdx.x < rows) {
    const int b = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const int in_group = head % p.group;
    const Range<Shape<DIM>::kKeys> r(a, b);
    uint16_t* op = (uint16_t*)a.o + b * a.o_sb + (long long)head * a.o_sh;
    if (r.tiles == 0) {
      for (int d = threadIdx.x * 8; d < DIM; d += kThreads * 8) *(uint4*)(op + d) = make_uint4(0, 0, 0, 0);
      if (a.lse && threadIdx.x == 0) a.lse[blockIdx.x] = -INFINITY;
      return;
    }
    const Span sp = p.ws.span[(b * a.cache.kv_heads + head / p.group) * p.chunks + in_group / kRows];
    if (sp.count == 1) return;
    const int row = in_group % kRows;
    const float2 all = join_row(p.ws, sp, row);
    float x[VEC] = {};
    for (int k = warp; k < sp.count; k += kWarps) {
      const int part = sp.part(k) * kRows + row;
      const float2 part_ml = p.ws.part_ml[part];
      if (part_ml.y == 0.f) continue;
      const float f = ex2_approx(part_ml.x - all.x);
      const float* y = p.ws.part_o + (long long)part * DIM + lane;
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = fmaf(y[v * 32], f, x[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) sum_o[warp][lane + v * 32] = x[v];
    __syncthreads();
    const float inv = all.y == 0.f ? 0.f : 1.f / all.y;
    for (int d = threadIdx.x * 2; d < DIM; d += kThreads * 2) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        s.x += sum_o[w][d];
        s.y += sum_o[w][d + 1];
      }
      *(uint32_t*)(op + d) = pack2<DTYPE>(s.x * inv, s.y * inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[blockIdx.x] = all.y == 0.f ? -INFINITY : (all.x + log2f(all.y)) * kLn2;
    return;
  }
  if constexpr (WEIGHTS) {
    const int pair = (blockIdx.x - rows) / splits, b = pair / a.cache.kv_heads, kvh = pair % a.cache.kv_heads;
    const Range<Shape<DIM>::kKeys> r(a, b);
    const int start = r.first + (int)((blockIdx.x - rows) % splits) * kWeightKeys;
    if (start >= r.end) return;
    float* w = a.weights + (long long)pair * a.weights_stride;
    for (int g0 = 0; g0 < p.group; g0 += kThreads) {
      const int n = min(kThreads, p.group - g0);
      __syncthreads();
      // log2 of the sums; +inf where no key weighs anything, so that no key does.
      const long long first = (long long)b * a.heads + kvh * p.group + g0;
      if (p.arrived) {
        if ((int)threadIdx.x < n) lse2[threadIdx.x] = p.ws.lse2[first + threadIdx.x];
      } else {
        for (int g = warp; g < n; g += kWarps) {
          const Span sp = p.ws.span[pair * p.chunks + (g0 + g) / kRows];
          float x;
          if (sp.count == 1) {
            x = p.ws.lse2[first + g];
          } else {
            const float2 all = join_row(p.ws, sp, (g0 + g) % kRows);
            x = all.y == 0.f ? -INFINITY : all.x + log2f(all.y);
          }
          if (lane == 0) lse2[g] = x;
        }
      }
      __syncthreads();
      if ((int)threadIdx.x < n && lse2[threadIdx.x] == -INFINITY) lse2[threadIdx.x] = INFINITY;
      __syncthreads();
      const float* s = p.ws.scores + first * p.ws.pitch;
      for (int j0 = start; j0 < r.end; j0 += splits * kWeightKeys) {
        float x[kWeightVecs] = {}, old[kWeightVecs];
        int at[kWeightVecs];
#pragma unroll
        for (int u = 0; u < kWeightVecs; ++u) {
          at[u] = min(j0 + u * kThreads + (int)threadIdx.x, r.end - 1);  // past the end: read, not written
          old[u] = w[at[u]];
        }
#pragma unroll 8
        for (int g = 0; g < n; ++g)
#pragma unroll
          for (int u = 0; u < kWeightVecs; ++u) x[u] += ex2_approx(s[g * p.ws.pitch + at[u]] - lse2[g]);
#pragma unroll
        for (int u = 0; u < kWeightVecs; ++u)
          if (j0 + u * kThreads + (int)threadIdx.x < r.end) w[at[u]] = old[u] + x[u];
      }
    }
  }
}

constexpr size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

int per_sm(int dim) { return dim == 256 ? Shape<256>::kPerSm : dim == 128 ? Shape<128>::kPerSm : Shape<64>::kPerSm; }

size_t lay_out(const PagedAttnArgs& a, int num_sms, uint8_t* base, Workspace* ws) {
  const size_t parts = (size_t)num_sms * per_sm(a.cache.head_dim) * 2 * kRows;
  const int group = a.heads / a.cache.kv_heads;
  const size_t items = (size_t)a.cache.batch * a.cache.kv_heads * ((group + kRows - 1) / kRows);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += up256(bytes);
    return base + was;
  };
  Workspace w{};
  w.part_o = (float*)take(parts * a.cache.head_dim * sizeof(float));
  w.part_ml = (float2*)take(parts * sizeof(float2));
  w.span = (Span*)take(items * sizeof(Span));
  if (a.weights) {
    w.lse2 = (float*)take((size_t)a.cache.batch * a.heads * sizeof(float));
    w.pitch = ((long long)a.cache.capacity + 31) / 32 * 32;
    w.scores = (float*)take((size_t)a.cache.batch * a.heads * w.pitch * sizeof(float));
  }
  if (ws) *ws = w;
  return at;
}

template <int DTYPE, int DIM, bool WEIGHTS, bool HALF>
cudaError_t launch(Params p, int num_sms, cudaStream_t s) {
  constexpr int smem = Shape<DIM>::kSmem;
  const PagedAttnArgs& a = p.a;
  static PerDevice allowed;
  const cudaError_t set = allow_shared_memory(allowed, paged_attn_kernel<DTYPE, DIM, WEIGHTS, HALF>, smem);
  if (set != cudaSuccess) return set;
  const long long tiles = (long long)a.cache.batch * a.cache.kv_heads * p.chunks *
                          ((a.cache.capacity + Shape<DIM>::kKeys - 1) / Shape<DIM>::kKeys + 1);
  const long long items = (long long)a.cache.batch * a.cache.kv_heads * p.chunks, cut = (tiles + p.min_tiles - 1) / p.min_tiles;
  const long long most = cut > 2 * items ? cut : 2 * items;
  const int grid = (int)(most < (long long)num_sms * Shape<DIM>::kPerSm ? most : num_sms * Shape<DIM>::kPerSm);
  // The last CTA of an item joins it while that is a few parts of each (on
  // average: how the lengths lie is not known here), which saves the second
  // launch; more parts take the second kernel, with a CTA for each query head.
  if (grid > 16 * items) p.arrived = nullptr;
  {
    ProfLaunch prof("paged_attn_kernel", dim3(grid), dim3(kThreads), smem, s);
    const cudaError_t e = launch_next(paged_attn_kernel<DTYPE, DIM, WEIGHTS, HALF>, dim3(grid), kThreads, smem, s, 1, p);
    if (e != cudaSuccess || (p.arrived && !WEIGHTS)) return e;
  }
  // Weights: enough CTAs to fill the GPU twice over, each striding on to its sequence's end.
  int splits = 1;
  const int pairs = a.cache.batch * a.cache.kv_heads;
  if (WEIGHTS) {
    const int want = (16 * num_sms + pairs - 1) / pairs, most_splits = (a.cache.capacity + kWeightKeys - 1) / kWeightKeys;
    splits = want < most_splits ? want : most_splits;
  }
  const long long ctas = (p.arrived ? 0 : (long long)a.cache.batch * a.heads) + (WEIGHTS ? (long long)pairs * splits : 0);
  if (ctas > INT_MAX) return cudaErrorInvalidValue;
  ProfLaunch prof("paged_attn_join_kernel", dim3((unsigned)ctas), dim3(kThreads), 0, s);
  return launch_next(paged_attn_join_kernel<DTYPE, DIM, WEIGHTS>, dim3((unsigned)ctas), kThreads, 0, s, 1, p, splits);
}

template <int DTYPE, int DIM>
cudaError_t by_weights(const Params& p, int num_sms, cudaStream_t s) {
  if (p.group <= 8) return p.a.weights ? launch<DTYPE, DIM, true, true>(p, num_sms, s) : launch<DTYPE, DIM, false, true>(p, num_sms, s);
  return p.a.weights ? launch<DTYPE, DIM, true, false>(p, num_sms, s) : launch<DTYPE, DIM, false, false>(p, num_sms, s);
}

template <int DTYPE>
cudaError_t by_dim(const Params& p, int num_sms, cudaStream_t s) {
  switch (p.a.cache.head_dim) {
    case 64: return by_weights<DTYPE, 64>(p, num_sms, s);
    case 128: return by_weights<DTYPE, 128>(p, num_sms, s);
    case 256: return by_weights<DTYPE, 256>(p, num_sms, s);
    default: return cudaErrorNotSupported;
  }
}

}  // namespace

size_t paged_attention_counter_bytes(const PagedAttnArgs& a) {
  const int group = a.heads / a.cache.kv_heads;
  return (size_t)a.cache.batch * a.cache.kv_heads * ((group + kRows - 1) / kRows) * sizeof(int);
}

size_t paged_attention_workspace_bytes(const PagedAttnArgs& a, int num_sms) { return lay_out(a, num_sms, nullptr, nullptr); }

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int num_sms, void* ws, int* counters, cudaStream_t s) {
  Params p{};
  p.a = a;
  p.arrived = counters;
  lay_out(a, num_sms, static_cast<uint8_t*>(ws), &p.ws);
  p.group = a.heads / a.cache.kv_heads;
  p.chunks = (p.group + kRows - 1) / kRows;
  p.min_tiles = kWarps;
  // The line of tiles is counted in 32 bits.
  const long long tiles = (long long)a.cache.batch * a.cache.kv_heads * p.chunks * (a.cache.capacity / 16 + 8);
  if (tiles > INT_MAX / 2) return cudaErrorNotSupported;
  return a.dtype == 1 ? by_dim<1>(p, num_sms, s) : by_dim<2>(p, num_sms, s);
}

}  // namespace grx
