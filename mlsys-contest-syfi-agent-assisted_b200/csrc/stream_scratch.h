// Scratch memory of the operators that have no context of their own: one buffer per stream, so that calls on one stream follow
// each other in theirs and calls on two streams never meet; and the driver functions they need without a link to libcuda.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

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

// A stream is known by its id, which is never given out twice (a handle may be, after the stream was destroyed); a stream
// that is being captured cannot be asked for it and is known by its handle.
struct Scratch {
  cudaStream_t handle = nullptr;
  unsigned long long id = 0; // 0: not known yet
  uint64_t last_use = 0;     // 0: free
  void* memory = nullptr;
  size_t bytes = 0;
  bool captured = false;     // a graph may use it
};
constexpr int kMaxScratch = 8;   // streams of a device that hold one at a time; the next one takes over the least recently used

// One operator's buffers of one device.  The caller holds a lock.
struct ScratchPool {
  Scratch scratch[kMaxScratch];
  uint64_t calls = 0;

  // The stream's buffer of at least `need` bytes; null with the error code in *rc when there is none.  The first `zeroed` bytes
  // of a new buffer are zero.
  Scratch* get(cudaStream_t st, size_t need, size_t zeroed, int error, int* rc);
};

inline bool zero_now(void* p, size_t bytes) {     // on a stream of its own: the caller's may be capturing
  if (bytes == 0) return true;
  cudaStream_t side;
  if (cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking) != cudaSuccess) return false;
  const bool ok = cudaMemsetAsync(p, 0, bytes, side) == cudaSuccess && cudaStreamSynchronize(side) == cudaSuccess;
  cudaStreamDestroy(side);
  return ok;
}

inline Scratch* ScratchPool::get(cudaStream_t st, size_t need, size_t zeroed, int error, int* rc) {
  const Driver& drv = driver();
  CUstreamCaptureStatus capture = CU_STREAM_CAPTURE_STATUS_NONE;
  unsigned long long id = 0;
  bool known = drv.is_capturing && drv.stream_id;
  if (known && drv.is_capturing(st, &capture) != CUDA_SUCCESS) capture = CU_STREAM_CAPTURE_STATUS_NONE;   // the default stream beside a capture: the launch will say so
  const bool capturing = capture != CU_STREAM_CAPTURE_STATUS_NONE;
  if (known && !capturing) known = drv.stream_id(st, &id) == CUDA_SUCCESS;
  if (!known) {
    *rc = set_last_error(error, "not a stream of the current device");
    return nullptr;
  }
  // The stream's own; of two (below) the larger.
  Scratch *s = nullptr, *spare = nullptr;
  for (Scratch& c : scratch) {
    if (c.last_use == 0) spare = &c;
    else if ((capturing || c.id == 0 ? c.handle == st : c.id == id) && (!s || c.bytes > s->bytes)) s = &c;
  }
  if (s && s->bytes < need && (capturing || s->captured) && spare) s = nullptr;   // a graph keeps the small one
  if (capturing && !spare && (!s || s->bytes < need)) {
    // Nothing may wait now, so nothing can be freed: whichever is large enough, as if the two streams were one.
    s = nullptr;
    for (Scratch& c : scratch)
      if (c.bytes >= need && (!s || c.last_use < s->last_use)) s = &c;
    if (!s) *rc = set_last_error(error, "no scratch buffer is large enough, and none can be had during a capture");
    else s->captured = true;
    return s;
  }
  if (!s) {
    s = spare;
    if (!s) {   // the one that was not used for longest, of those that no graph needs, if there is one
      for (Scratch& c : scratch)
        if (!s || (c.captured != s->captured ? s->captured : c.last_use < s->last_use)) s = &c;
      if (cudaDeviceSynchronize() != cudaSuccess) {
        *rc = set_last_error(error, "device synchronisation failed");
        return nullptr;
      }
    }
    s->handle = st;
    s->id = 0;
    s->captured = false;
  }
  if (need > s->bytes) {
    if (s->memory) {
      if (cudaDeviceSynchronize() != cudaSuccess) {
        *rc = set_last_error(error, "device synchronisation failed");
        return nullptr;
      }
      cudaFree(s->memory);
    }
    s->memory = nullptr;
    s->bytes = 0;
    RelaxedCapture relaxed;
    if (cudaMalloc(&s->memory, need) != cudaSuccess || !zero_now(s->memory, zeroed)) {
      if (s->memory) cudaFree(s->memory);
      s->memory = nullptr;
      s->last_use = 0;
      *rc = set_last_error(error, "out of device memory for the scratch buffer");
      return nullptr;
    }
    s->bytes = need;
  }
  if (id != 0) s->id = id;
  if (capturing) s->captured = true;
  s->last_use = ++calls;
  return s;
}

}  // namespace syfi
