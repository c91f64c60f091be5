// grxDNN host entry points of token serving: paged key-value cache, attention
// of one new token, eviction, token scoring. Validation as in dnn_host.cpp:
// null handle -> NOT_INITIALIZED, malformed arguments -> INVALID_VALUE, empty
// problem -> SUCCESS without a launch, a type or layout the kernels do not
// implement -> NOT_SUPPORTED.
#include <cuda_runtime.h>

#include <limits.h>
#include <math.h>

#include <atomic>
#include <new>

#include "dnn_context.h"
#include "serving.cuh"

// Held by the blocks of a capture and by its graph, whichever goes last.
struct GraphLease {
  std::atomic<int> holders{2};
  std::atomic<bool> graph_gone{false};
  void drop() {
    if (holders.fetch_sub(1) == 1) delete this;
  }
};

namespace {

// Called once the graph, all its executable copies and their last runs are over.
void CUDART_CB graph_is_gone(void* lease) {
  auto* l = static_cast<GraphLease*>(lease);
  l->graph_gone = true;
  l->drop();
}

// One for all blocks of a capture. It costs a launch of the graph 2 us (six attention calls on one sequence each, replayed
// back to back: 51.2 and 53.2 us); without it, a program that captures anew now and then would pile up scratch. Null where
// the graph cannot be made to tell its end: the block then stays until the handle goes.
GraphLease* lease_to(const grxdnnContext& ctx, const ScratchOwner& owner) {
  for (StreamScratch* b = ctx.scratch; b; b = b->next)
    if (b->owner.capture == owner.capture && b->lease) {
      ++b->lease->holders;
      return b->lease;
    }
  auto* l = new (std::nothrow) GraphLease();
  if (!l) return nullptr;
  cudaUserObject_t object;
  if (cudaUserObjectCreate(&object, l, graph_is_gone, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
    cudaGetLastError();
    delete l;
    return nullptr;
  }
  if (cudaGraphRetainUserObject(owner.graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
    cudaGetLastError();
    cudaUserObjectRelease(object, 1);  // calls graph_is_gone
    l->drop();
    return nullptr;
  }
  return l;
}

bool graph_gone(const StreamScratch& b) { return b.lease && b.lease->graph_gone; }

void free_block(StreamScratch* b) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // another thread's stream may be capturing
  cudaThreadExchangeStreamCaptureMode(&mode);
  cudaFree(b->ptr);  // waits for the kernels that use it
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (b->lease) b->lease->drop();
  delete b;
}

}  // namespace

ScratchOwner scratch_owner(const grxdnnContext& ctx) {
  ScratchOwner o;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(ctx.stream, &status, &id, &o.graph) != cudaSuccess) {
    cudaGetLastError();  // the default stream beside a capture, whose launch will say so
    status = cudaStreamCaptureStatusNone;
  }
  if (status == cudaStreamCaptureStatusActive) {
    o.capture = id + 1;
    o.stream = reinterpret_cast<uintptr_t>(ctx.stream);  // a capturing stream must not be asked for its id
    return o;
  }
  o.graph = nullptr;
  if (ctx.stream == nullptr || ctx.stream == cudaStreamLegacy) {
    o.stream = ~0ull;
  } else if (cudaStreamGetId(ctx.stream, &o.stream) != cudaSuccess) {
    cudaGetLastError();  // a capture that has failed, as the launch will
    o.stream = reinterpret_cast<uintptr_t>(ctx.stream);
    o.known = false;
  }
  return o;
}

void* stream_scratch(grxdnnContext& ctx, const ScratchOwner& owner, size_t bytes, ScratchKind kind) {
  std::lock_guard<std::mutex> lock(ctx.mutex);
  size_t had = 0;  // the newest block of an owner is its largest
  for (StreamScratch* b = ctx.scratch; b; b = b->next) {
    if (!(b->owner == owner) || b->kind != kind) continue;
    if (b->bytes >= bytes) return b->ptr;
    had = had > b->bytes ? had : b->bytes;
  }
  if (grx::fault_injected("alloc")) return nullptr;
  StreamScratch* found = nullptr;
  if (owner.capture) {
    // What a graph that is gone has left serves another one.
    for (StreamScratch* b = ctx.scratch; b && !found; b = b->next)
      if (graph_gone(*b) && b->kind == kind && b->bytes >= bytes) found = b;
    if (found) {
      found->lease->drop();
      found->lease = nullptr;
      found->lease = lease_to(ctx, owner);
      found->owner = owner;
      found->stream = ctx.stream;
    }
  } else {
    // Blocks that nobody asks for again: of graphs that are gone, and of a stream
    // whose handle this one has now, so that it is gone too (a thread's default
    // stream has the same handle in every thread).
    for (StreamScratch** at = &ctx.scratch; *at;) {
      StreamScratch* b = *at;
      const bool stream_gone = owner.known && !b->owner.capture && b->stream == ctx.stream &&
                               b->owner.stream != owner.stream && ctx.stream != cudaStreamPerThread;
      if (graph_gone(*b) || stream_gone) {
        *at = b->next;
        free_block(b);
      } else {
        at = &b->next;
      }
    }
  }
  auto* b = found ? nullptr : new (std::nothrow) StreamScratch();
  if (b) {
    b->owner = owner;
    b->stream = ctx.stream;
    b->kind = kind;
    // Doubling bounds what a growing problem leaves behind to one more block.
    b->bytes = bytes > 2 * had ? bytes : 2 * had;
    cudaError_t e = grx::allocate_now(&b->ptr, b->bytes, kind == kScratchZeroed);
    if (e != cudaSuccess && b->bytes > bytes) {
      b->bytes = bytes;
      e = grx::allocate_now(&b->ptr, b->bytes, kind == kScratchZeroed);
    }
    if (e == cudaSuccess) {
      b->lease = owner.capture ? lease_to(ctx, owner) : nullptr;
      b->next = ctx.scratch;
      ctx.scratch = found = b;
    } else {
      delete b;
    }
  }
  return found ? found->ptr : nullptr;
}

void release_stream_scratch(grxdnnContext& ctx) {
  while (StreamScratch* b = ctx.scratch) {
    ctx.scratch = b->next;
    free_block(b);
  }
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether the addresses are those of whole 4-byte values, or null.
template <typename... P>
bool aligned4(const P*... p) {
  return ((... | reinterpret_cast<uintptr_t>(p)) & 3) == 0;
}

// Whether `p` is the address of a whole element of a norm_dtype.
bool whole_element(const void* p, grxDataType_t type) {
  return (reinterpret_cast<uintptr_t>(p) & (type == GRX_R_32F ? 3 : 1)) == 0;
}

// What the kernels count in 32 bits, they count past its end by what a grid takes in one step: less than 2^20.
constexpr long long kMostCounted = INT_MAX - (1 << 20);

// Layout of a cache whose elements have 2 bytes: every row on 16 bytes.
grxdnnStatus_t check_cache(const grxdnnPagedCache_t* c, const void* k, const void* v, const int* table,
                           const int* lens) {
  if (c->kvHeads < 1 || c->headDim < 1 || c->numPages < 1 || c->pageSize < 1 || c->maxPages < 1)
    return GRXDNN_STATUS_INVALID_VALUE;
  if ((long long)c->pageSize * c->maxPages > INT_MAX) return GRXDNN_STATUS_INVALID_VALUE;
  if (c->strideTable < c->maxPages) return GRXDNN_STATUS_INVALID_VALUE;
  if ((c->numPages > 1 && c->stridePage < c->headDim) || (c->pageSize > 1 && c->strideToken < c->headDim) ||
      (c->kvHeads > 1 && c->strideHead < c->headDim))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (!k || !v || !table || !lens || !aligned4(table, lens)) return GRXDNN_STATUS_INVALID_VALUE;
  if (c->dtype != GRX_R_16BF && c->dtype != GRX_R_16F) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (c->headDim != 64 && c->headDim != 128 && c->headDim != 256) return GRXDNN_STATUS_NOT_SUPPORTED;
  if ((long long)c->pageSize * c->maxPages > kMostCounted || c->batch > kMostCounted ||
      (long long)c->kvHeads * c->headDim > kMostCounted)
    return GRXDNN_STATUS_NOT_SUPPORTED;
  if (((c->stridePage | c->strideToken | c->strideHead) & 7) || !aligned16(k) || !aligned16(v))
    return GRXDNN_STATUS_NOT_SUPPORTED;
  return GRXDNN_STATUS_SUCCESS;
}

grx::PagedView view_of(const grxdnnPagedCache_t* c, const int* table, int* err_word) {
  grx::PagedView v{};
  v.batch = c->batch;
  v.kv_heads = c->kvHeads;
  v.head_dim = c->headDim;
  v.num_pages = c->numPages;
  v.capacity = c->pageSize * c->maxPages;
  v.page = grx::FastDiv((uint32_t)c->pageSize);
  v.table = table;
  v.table_stride = c->strideTable;
  v.s_page = c->stridePage;
  v.s_token = c->strideToken;
  v.s_head = c->strideHead;
  v.err_word = err_word;
  return v;
}

bool rows_aligned(const grxdnnAttnTensor_t* d, const void* p) {
  return aligned16(p) && (d->batch < 2 || (d->strideBatch & 7) == 0) && (d->heads < 2 || (d->strideHead & 7) == 0) &&
         (d->seq < 2 || (d->strideSeq & 7) == 0);
}

}  // namespace

extern "C" {

grxdnnStatus_t grxdnnKvCacheAppend(grxdnnHandle_t handle, const grxdnnPagedCache_t* cache, void* kPages,
                                   void* vPages, const int* pageTable, const int* lens,
                                   const grxdnnAttnTensor_t* kd, const void* k, const grxdnnAttnTensor_t* vd,
                                   const void* v, const int* counts, int* lensOut) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!cache || !kd || !vd || cache->batch < 0) return GRXDNN_STATUS_INVALID_VALUE;
  for (auto* d : {kd, vd})
    if (d->batch != cache->batch || d->heads != cache->kvHeads || d->headDim != cache->headDim || d->seq < 0 ||
        d->seq != kd->seq || (d->seq > 1 && d->strideSeq < d->headDim))
      return GRXDNN_STATUS_INVALID_VALUE;
  if (cache->batch == 0) return GRXDNN_STATUS_SUCCESS;
  grxdnnStatus_t s = check_cache(cache, kPages, vPages, pageTable, lens);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if ((kd->seq > 0 && (!k || !v)) || !aligned4(counts, lensOut)) return GRXDNN_STATUS_INVALID_VALUE;
  if (kd->dtype != cache->dtype || vd->dtype != cache->dtype) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (kd->seq > 0 && (!rows_aligned(kd, k) || !rows_aligned(vd, v))) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (kd->seq == 0 && !lensOut) return GRXDNN_STATUS_SUCCESS;
  auto& ctx = *reinterpret_cast<grxdnnContext*>(handle);
  s = ensure(ctx, false);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  grx::KvAppendArgs a{};
  a.cache = view_of(cache, pageTable, ctx.dev.err_word);
  a.k_pages = kPages;
  a.v_pages = vPages;
  a.lens = lens;
  a.tokens = kd->seq;
  a.k = k; a.k_sb = kd->strideBatch; a.k_sh = kd->strideHead; a.k_ss = kd->strideSeq;
  a.v = v; a.v_sb = vd->strideBatch; a.v_sh = vd->strideHead; a.v_ss = vd->strideSeq;
  a.counts = counts;
  a.lens_out = lensOut;
  return from_cuda(grx::launch_kv_append(a, ctx.stream));
}

grxdnnStatus_t grxdnnPagedAttentionForward(grxdnnHandle_t handle, const grxdnnPagedCache_t* cache,
                                           const void* kPages, const void* vPages, const int* pageTable,
                                           const int* lens, const grxdnnAttnTensor_t* qd, const void* q,
                                           const grxdnnAttnTensor_t* od, void* o, float scale, int window,
                                           float* lse, float* weights, long long strideWeights) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!cache || !qd || !od || cache->batch < 0) return GRXDNN_STATUS_INVALID_VALUE;
  for (auto* d : {qd, od})
    if (d->batch != cache->batch || d->heads < 0 || d->heads != qd->heads || d->seq < 0 || d->seq != qd->seq ||
        d->headDim != cache->headDim)
      return GRXDNN_STATUS_INVALID_VALUE;
  if (cache->batch == 0 || qd->heads == 0 || qd->seq == 0) return GRXDNN_STATUS_SUCCESS;
  grxdnnStatus_t s = check_cache(cache, kPages, vPages, pageTable, lens);
  if (s == GRXDNN_STATUS_INVALID_VALUE) return s;
  if (qd->heads % cache->kvHeads != 0 || !q || !o || window < 0 || !aligned4(lse, weights)) return GRXDNN_STATUS_INVALID_VALUE;
  if (!(scale > 0.0f) || isinf(scale)) return GRXDNN_STATUS_INVALID_VALUE;
  if (weights && strideWeights < (long long)cache->pageSize * cache->maxPages) return GRXDNN_STATUS_INVALID_VALUE;
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if ((long long)qd->heads * qd->headDim > kMostCounted) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (qd->seq != 1 || qd->dtype != cache->dtype || od->dtype != cache->dtype) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!rows_aligned(qd, q) || !rows_aligned(od, o)) return GRXDNN_STATUS_NOT_SUPPORTED;
  auto& ctx = *reinterpret_cast<grxdnnContext*>(handle);
  s = ensure(ctx, true);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  grx::PagedAttnArgs a{};
  a.cache = view_of(cache, pageTable, ctx.dev.err_word);
  a.dtype = norm_dtype(cache->dtype);
  a.k_pages = kPages;
  a.v_pages = vPages;
  a.lens = lens;
  a.heads = qd->heads;
  a.q = q; a.q_sb = qd->strideBatch; a.q_sh = qd->strideHead;
  a.o = o; a.o_sb = od->strideBatch; a.o_sh = od->strideHead;
  a.scale = scale;
  a.window = window;
  a.lse = lse;
  a.weights = weights; a.weights_stride = strideWeights;
  const ScratchOwner owner = scratch_owner(ctx);
  void* ws = stream_scratch(ctx, owner, grx::paged_attention_workspace_bytes(a, ctx.dev.num_sms));
  void* counters = stream_scratch(ctx, owner, grx::paged_attention_counter_bytes(a), kScratchZeroed);
  if (!ws || !counters) return GRXDNN_STATUS_ALLOC_FAILED;
  return from_cuda(grx::launch_paged_attention(a, ctx.dev.num_sms, ws, static_cast<int*>(counters), ctx.stream));
}

grxdnnStatus_t grxdnnKvCacheEvict(grxdnnHandle_t handle, const grxdnnPagedCache_t* cache, const void* kPages,
                                  const void* vPages, const int* pageTable, const int* lens, const float* weights,
                                  long long strideWeights, int keep, int recent, const grxdnnPagedCache_t* outCache,
                                  void* kOut, void* vOut, const int* tableOut, int* lensOut, float* weightsOut,
                                  long long strideWeightsOut, int* indices) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!cache || !outCache || cache->batch < 0) return GRXDNN_STATUS_INVALID_VALUE;
  if (outCache->batch != cache->batch || outCache->kvHeads != cache->kvHeads || outCache->headDim != cache->headDim)
    return GRXDNN_STATUS_INVALID_VALUE;
  if (cache->batch == 0) return GRXDNN_STATUS_SUCCESS;
  const grxdnnStatus_t si = check_cache(cache, kPages, vPages, pageTable, lens);
  const grxdnnStatus_t so = check_cache(outCache, kOut, vOut, tableOut, lensOut);
  if (si == GRXDNN_STATUS_INVALID_VALUE || so == GRXDNN_STATUS_INVALID_VALUE) return GRXDNN_STATUS_INVALID_VALUE;
  const long long room = (long long)outCache->pageSize * outCache->maxPages;
  if (!weights || !weightsOut || strideWeights < (long long)cache->pageSize * cache->maxPages ||
      strideWeightsOut < room || (weights == weightsOut && strideWeights != strideWeightsOut))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (!aligned4(weights, weightsOut, indices)) return GRXDNN_STATUS_INVALID_VALUE;
  if (keep < 1 || recent < 0 || recent > keep || keep > room) return GRXDNN_STATUS_INVALID_VALUE;
  if (si != GRXDNN_STATUS_SUCCESS) return si;
  if (so != GRXDNN_STATUS_SUCCESS) return so;
  if (outCache->dtype != cache->dtype) return GRXDNN_STATUS_NOT_SUPPORTED;
  auto& ctx = *reinterpret_cast<grxdnnContext*>(handle);
  const grxdnnStatus_t s = ensure(ctx, false);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  grx::KvEvictArgs a{};
  a.in = view_of(cache, pageTable, ctx.dev.err_word);
  a.out = view_of(outCache, tableOut, ctx.dev.err_word);
  a.k_in = kPages;
  a.v_in = vPages;
  a.k_out = kOut;
  a.v_out = vOut;
  a.lens = lens;
  a.lens_out = lensOut;
  a.weights = weights; a.weights_stride = strideWeights;
  a.weights_out = weightsOut; a.weights_out_stride = strideWeightsOut;
  a.keep = keep;
  a.recent = recent;
  a.indices = indices;
  void* ws = stream_scratch(ctx, scratch_owner(ctx), grx::kv_evict_workspace_bytes(a));
  if (!ws) return GRXDNN_STATUS_ALLOC_FAILED;
  return from_cuda(grx::launch_kv_evict(a, ctx.dev.num_sms, ws, ctx.stream));
}

grxdnnStatus_t grxdnnTokenLogProbsForward(grxdnnHandle_t handle, int rows, int vocab, const void* logits,
                                          grxDataType_t type, long long ld, float scale, const int* tokens,
                                          float* logp, float* entropy, float* lse, int topK, int* topTokens,
                                          float* topLogp) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (rows < 0 || vocab < 0) return GRXDNN_STATUS_INVALID_VALUE;
  if (!(scale > 0.0f) || isinf(scale)) return GRXDNN_STATUS_INVALID_VALUE;
  if (topK < 0 || topK > GRXDNN_MAX_TOP) return GRXDNN_STATUS_INVALID_VALUE;
  if (rows == 0) return GRXDNN_STATUS_SUCCESS;
  if (vocab == 0 || topK > vocab || !logits || ld < vocab || (logp && !tokens)) return GRXDNN_STATUS_INVALID_VALUE;
  if (!aligned4(tokens, logp, entropy, lse, topTokens, topLogp)) return GRXDNN_STATUS_INVALID_VALUE;
  if (norm_dtype(type) < 0) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!whole_element(logits, type)) return GRXDNN_STATUS_INVALID_VALUE;
  if (!topTokens && !topLogp) topK = 0;
  if (!logp && !entropy && !lse && topK == 0) return GRXDNN_STATUS_SUCCESS;
  auto& ctx = *reinterpret_cast<grxdnnContext*>(handle);
  const grxdnnStatus_t s = ensure(ctx, false);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  grx::TokenScoreArgs a{};
  a.rows = rows;
  a.vocab = vocab;
  a.dtype = norm_dtype(type);
  a.logits = logits; a.ld = ld;
  a.scale = scale;
  a.tokens = tokens;
  a.logp = logp;
  a.entropy = entropy;
  a.lse = lse;
  a.top = topK;
  a.top_tokens = topTokens;
  a.top_logp = topLogp;
  return from_cuda(grx::launch_token_score(a, ctx.dev.num_sms, ctx.stream));
}

grxdnnStatus_t grxdnnTokenLogProbsBackward(grxdnnHandle_t handle, int rows, int vocab, const void* logits,
                                           grxDataType_t type, long long ld, float scale, const int* tokens,
                                           const float* lse, const float* entropy, const float* dlogp,
                                           const float* dentropy, void* dlogits, grxDataType_t dlogitsType,
                                           long long lddlogits) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (rows < 0 || vocab < 0) return GRXDNN_STATUS_INVALID_VALUE;
  if (!(scale > 0.0f) || isinf(scale)) return GRXDNN_STATUS_INVALID_VALUE;
  if (rows == 0) return GRXDNN_STATUS_SUCCESS;
  if (vocab == 0 || !logits || !dlogits || !lse || ld < vocab || lddlogits < vocab) return GRXDNN_STATUS_INVALID_VALUE;
  if ((!dlogp && !dentropy) || (dlogp && !tokens) || (dentropy && !entropy)) return GRXDNN_STATUS_INVALID_VALUE;
  if (logits == dlogits && ld != lddlogits) return GRXDNN_STATUS_INVALID_VALUE;
  if (!aligned4(tokens, lse, entropy, dlogp, dentropy)) return GRXDNN_STATUS_INVALID_VALUE;
  if (norm_dtype(type) < 0 || dlogitsType != type) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!whole_element(logits, type) || !whole_element(dlogits, type)) return GRXDNN_STATUS_INVALID_VALUE;
  auto& ctx = *reinterpret_cast<grxdnnContext*>(handle);
  const grxdnnStatus_t s = ensure(ctx, false);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  grx::TokenScoreBwdArgs a{};
  a.rows = rows;
  a.vocab = vocab;
  a.dtype = norm_dtype(type);
  a.logits = logits; a.ld = ld;
  a.scale = scale;
  a.tokens = tokens;
  a.lse = lse;
  a.entropy = entropy;
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  a.dlogits = dlogits; a.ldd = lddlogits;
  return from_cuda(grx::launch_token_score_bwd(a, ctx.dev.num_sms, ctx.stream));
}

}  // extern "C"
