// The grxDNN handle and the host helpers its entry points share
// (dnn_host.cpp, dnn_serving.cpp).
#pragma once

#include <cuda_runtime.h>

#include <mutex>

#include "grx/grxdnn.h"
#include "host_common.h"

// Whose work scratch is for: one stream's, or one stream's part of a captured
// graph, which may be replayed on any stream beside that one's own work.
struct ScratchOwner {
  unsigned long long stream = 0;   // the stream's id, which no other stream of the program ever has; in a capture its handle
  unsigned long long capture = 0;  // the capture's id and 1; 0 for work that is not captured
  cudaGraph_t graph = nullptr;     // being captured
  bool known = true;               // whether `stream` is what it says: not where a capture has failed
  bool operator==(const ScratchOwner& o) const { return stream == o.stream && capture == o.capture; }
};

// Scratch of one owner. A handle that moves to another stream, or calls of
// another capture, get another block, so that kernels still running for the old
// owner keep theirs. A block that turns out too small is kept, since a graph or
// a running kernel may hold its address: until the handle goes, or until the
// graph does.
struct GraphLease;
enum ScratchKind { kScratchAny, kScratchZeroed };  // Zeroed: 0 at first, and left so by every kernel
struct StreamScratch {
  ScratchOwner owner;
  cudaStream_t stream;
  GraphLease* lease;  // of a captured graph
  ScratchKind kind;
  void* ptr;
  size_t bytes;
  StreamScratch* next;
};

struct grxdnnContext {
  cudaStream_t stream = nullptr;
  std::mutex mutex;
  grx::DeviceState dev;
  void* ws = nullptr;  // grow-only, stream-ordered scratch (norm backward)
  size_t ws_bytes = 0;
  StreamScratch* scratch = nullptr;
};

// Whose work the next launch on the handle's stream is.
ScratchOwner scratch_owner(const grxdnnContext& ctx);
// At least `bytes` of device scratch (256-byte aligned) for that work, or null.
// Also inside a stream capture.
void* stream_scratch(grxdnnContext& ctx, const ScratchOwner& owner, size_t bytes, ScratchKind kind = kScratchAny);
void release_stream_scratch(grxdnnContext& ctx);

namespace {

inline grxdnnStatus_t from_cuda(cudaError_t e) {
  switch (e) {
    case cudaSuccess: return GRXDNN_STATUS_SUCCESS;
    case cudaErrorMemoryAllocation: return GRXDNN_STATUS_ALLOC_FAILED;
    case cudaErrorInvalidValue: return GRXDNN_STATUS_INVALID_VALUE;
    case cudaErrorNotSupported: return GRXDNN_STATUS_NOT_SUPPORTED;
    case cudaErrorNoKernelImageForDevice:
    case cudaErrorInvalidDeviceFunction: return GRXDNN_STATUS_ARCH_MISMATCH;
    default: return GRXDNN_STATUS_EXECUTION_FAILED;
  }
}

inline grxdnnStatus_t ensure(grxdnnContext& ctx, bool need_tensor) {
  std::lock_guard<std::mutex> lock(ctx.mutex);
  const int rc = grx::ensure_device(ctx.dev);
  if (rc == 1) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (rc == 2) return GRXDNN_STATUS_ALLOC_FAILED;
  if (need_tensor && ctx.dev.cc_major != 10) return GRXDNN_STATUS_ARCH_MISMATCH;
  return GRXDNN_STATUS_SUCCESS;
}

inline int norm_dtype(grxDataType_t t) {
  switch (t) {
    case GRX_R_32F: return 0;
    case GRX_R_16BF: return 1;
    case GRX_R_16F: return 2;
    default: return -1;
  }
}

}  // namespace
