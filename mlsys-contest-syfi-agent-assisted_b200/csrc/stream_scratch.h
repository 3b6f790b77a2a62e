// Scratch memory of the operators that have no context of their own: one buffer per stream, so that calls on one stream follow
// each other in theirs and calls on two streams never meet, and buffers of their own for captured graphs; and the driver functions
// they need without a link to libcuda.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>
#include <new>

#include "moe_internal.h"

namespace syfi {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

typedef CUresult (*IsCapturingFn)(CUstream, CUstreamCaptureStatus*);
typedef CUresult (*StreamIdFn)(CUstream, unsigned long long*);

// (The runtime has the two on streams as well; it takes 40 ns for each instead of 11, and a short call is bound by the
// host's part of it.)
struct Driver {
  EncodeTiledFn encode_tiled = nullptr;
  IsCapturingFn is_capturing = nullptr;
  StreamIdFn stream_id = nullptr;
};

template <typename Fn>
void driver_fn(const char* name, Fn* fn) {
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
    *fn = reinterpret_cast<Fn>(p);
}

inline const Driver& driver() {
  static Driver d;
  static std::once_flag once;
  std::call_once(once, [] {
    driver_fn("cuTensorMapEncodeTiled", &d.encode_tiled);
    driver_fn("cuStreamIsCapturing", &d.is_capturing);
    driver_fn("cuStreamGetId", &d.stream_id);
  });
  return d;
}

// Allocation must not end a capture that is going on, on this stream or another.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

struct ScratchBuffer {
  void* memory = nullptr;
  size_t bytes = 0;
};

// A stream is known by its id, which is never given out twice (a handle may be, after the stream was destroyed).
struct Scratch : ScratchBuffer {
  unsigned long long id = 0;
  uint64_t last_use = 0;     // 0: free
};
constexpr int kMaxScratch = 8;   // streams of a device that hold one at a time; the next one takes over the least recently used

// A captured graph uses its buffer whenever it is replayed, so that buffer is no stream's, is never freed, and is another graph's only when
// the graph is gone, which a user object of the graph tells.  Branches of a graph that may run at the same time are captured on
// different streams and have one each.
struct GraphScratch : ScratchBuffer {
  unsigned long long capture = 0;
  cudaStream_t stream = nullptr;
  std::atomic<bool> taken{false};
  GraphScratch* next = nullptr;
  static void CUDART_CB release(void* self) { static_cast<GraphScratch*>(self)->taken.store(false, std::memory_order_release); }
};

// One operator's buffers of one device.  The caller holds a lock.
struct ScratchPool {
  Scratch scratch[kMaxScratch];
  uint64_t calls = 0;
  GraphScratch* graphs = nullptr;

  // The stream's buffer of at least `need` bytes, or that of the graph that it captures; null with the error code in *rc when there is
  // none.  The first `zeroed` bytes of a new buffer are zero.
  ScratchBuffer* get(cudaStream_t st, size_t need, size_t zeroed, int error, int* rc);
  ScratchBuffer* get_for_graph(cudaStream_t st, size_t need, size_t zeroed, int error, int* rc);
};

inline bool zero_now(void* p, size_t bytes) {     // on a stream of its own: the caller's may be capturing
  if (bytes == 0) return true;
  cudaStream_t side;
  if (cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking) != cudaSuccess) return false;
  const bool ok = cudaMemsetAsync(p, 0, bytes, side) == cudaSuccess && cudaStreamSynchronize(side) == cudaSuccess;
  cudaStreamDestroy(side);
  return ok;
}

// Null memory when there is none to be had.
inline ScratchBuffer new_buffer(size_t bytes, size_t zeroed) {
  ScratchBuffer b;
  RelaxedCapture relaxed;
  if (cudaMalloc(&b.memory, bytes) != cudaSuccess) return {};
  if (!zero_now(b.memory, zeroed)) {
    cudaFree(b.memory);
    return {};
  }
  b.bytes = bytes;
  return b;
}

inline ScratchBuffer* ScratchPool::get_for_graph(cudaStream_t st, size_t need, size_t zeroed, int error, int* rc) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  cudaGraph_t graph = nullptr;
  if (cudaStreamGetCaptureInfo_v2(st, &status, &capture, &graph, nullptr, nullptr) != cudaSuccess || status != cudaStreamCaptureStatusActive) {
    *rc = set_last_error(error, "the stream's capture is not in order");
    return nullptr;
  }
  GraphScratch* g = nullptr;
  for (GraphScratch* c = graphs; c; c = c->next) {
    if (c->bytes < need) continue;
    const bool taken = c->taken.load(std::memory_order_acquire);
    if (taken && c->capture == capture && c->stream == st) return c;      // of an earlier call in this capture
    if (!taken && (!g || c->bytes < g->bytes)) g = c;
  }
  const bool fresh = !g;
  if (fresh) {
    const ScratchBuffer b = new_buffer(need, zeroed);
    g = b.memory ? new (std::nothrow) GraphScratch : nullptr;
    if (!g) {
      if (b.memory) cudaFree(b.memory);
      *rc = set_last_error(error, "out of memory for a graph's scratch buffer");
      return nullptr;
    }
    static_cast<ScratchBuffer&>(*g) = b;
    g->next = graphs;
    graphs = g;
  }
  g->capture = capture;
  g->stream = st;
  cudaUserObject_t object;
  g->taken.store(true, std::memory_order_relaxed);
  if (cudaUserObjectCreate(&object, g, GraphScratch::release, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
    g->taken.store(false, std::memory_order_relaxed);
    *rc = set_last_error(error, "cannot tie a scratch buffer to the graph");
    return nullptr;
  }
  if (cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
    cudaUserObjectRelease(object, 1);
    *rc = set_last_error(error, "cannot tie a scratch buffer to the graph");
    return nullptr;
  }
  return g;
}

inline ScratchBuffer* ScratchPool::get(cudaStream_t st, size_t need, size_t zeroed, int error, int* rc) {
  const Driver& drv = driver();
  CUstreamCaptureStatus capture = CU_STREAM_CAPTURE_STATUS_NONE;
  unsigned long long id = 0;
  bool known = drv.is_capturing && drv.stream_id;
  if (known && drv.is_capturing(st, &capture) != CUDA_SUCCESS) capture = CU_STREAM_CAPTURE_STATUS_NONE;   // the default stream beside a capture: the launch will say so
  if (known && capture != CU_STREAM_CAPTURE_STATUS_NONE) return get_for_graph(st, need, zeroed, error, rc);
  if (!known || drv.stream_id(st, &id) != CUDA_SUCCESS) {
    *rc = set_last_error(error, "not a stream of the current device");
    return nullptr;
  }
  Scratch *s = nullptr, *oldest = &scratch[0];
  for (Scratch& c : scratch) {
    if (c.last_use != 0 && c.id == id) s = &c;
    if (c.last_use < oldest->last_use) oldest = &c;
  }
  const bool other = !s && oldest->last_use != 0;      // takes over another stream's
  if (!s) s = oldest;
  if (other || (s->memory && s->bytes < need)) {
    if (cudaDeviceSynchronize() != cudaSuccess) {
      *rc = set_last_error(error, "device synchronisation failed");
      return nullptr;
    }
  }
  s->id = id;
  s->last_use = ++calls;
  if (s->bytes < need) {
    if (s->memory) cudaFree(s->memory);
    static_cast<ScratchBuffer&>(*s) = new_buffer(need, zeroed);
    if (!s->memory) {
      s->last_use = 0;
      *rc = set_last_error(error, "out of device memory for the scratch buffer");
      return nullptr;
    }
  }
  return s;
}

}  // namespace syfi
