// Workspaces of captured calls.
//
// A call inside a stream capture runs again with every replay of the graph, so its
// workspace has to outlive the graph, belong to that graph alone (two graphs may be
// replayed at the same time), and hold zeros before the first replay, whichever graph is
// replayed first. So it is neither the capturing stream's eager workspace nor memory of
// the capture: it is allocated and zero-filled at once, outside the capture, and a CUDA
// user object that the graph retains (as does everything instantiated from it, until its
// last execution has ended) reports when it is free for another capture.
#include <cuda_runtime.h>

#include <mutex>
#include <vector>

#include "cb200.h"
#include "cb_internal.h"

namespace cb {
namespace {

struct Held {
  void* p;
  size_t bytes;
  int device;
  uint64_t capture;
};

struct Registry {
  std::mutex lock;
  std::vector<Held*> live, spare;
  cudaStream_t zero[64] = {};  // per device: zero-fills, never captured
};

// Never destroyed: the user objects' callbacks may come while the process ends.
Registry& registry() {
  static Registry* r = new Registry;
  return *r;
}

// The graph is gone and its last execution over.
void CUDART_CB released(void* arg) {
  Registry& r = registry();
  const std::lock_guard<std::mutex> guard(r.lock);
  for (size_t i = 0; i < r.live.size(); ++i)
    if (r.live[i] == arg) {
      r.spare.push_back(r.live[i]);
      r.live.erase(r.live.begin() + i);
      return;
    }
}

// Allocation and synchronisation are allowed to this thread while it captures.
struct Relaxed {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

bool capture_of(cudaStream_t s, uint64_t* id, cudaGraph_t* graph) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long n = 0;
  if (cudaStreamGetCaptureInfo(s, &status, &n, graph) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  *id = n + 1;  // 0 stands for none
  return status == cudaStreamCaptureStatusActive;
}

// A zeroed buffer of the device: where released ones fit, the last of the smallest.
int acquire(Registry& r, size_t bytes, int device, Held** out) {
  if (device < 0 || device >= 64) return CB_ERR_UNSUPPORTED;
  size_t best = r.spare.size();
  for (size_t i = 0; i < r.spare.size(); ++i)
    if (r.spare[i]->device == device && r.spare[i]->bytes >= bytes && (best == r.spare.size() || r.spare[i]->bytes <= r.spare[best]->bytes))
      best = i;
  Held* h;
  if (best < r.spare.size()) {
    h = r.spare[best];
    r.spare.erase(r.spare.begin() + best);
  } else {
    void* p = nullptr;
    if (cudaMalloc(&p, bytes) != cudaSuccess) {
      cudaGetLastError();
      return CB_ERR_CUDA;
    }
    h = new Held{p, bytes, device, 0};
  }
  if ((!r.zero[device] && cudaStreamCreateWithFlags(&r.zero[device], cudaStreamNonBlocking) != cudaSuccess) ||
      cudaMemsetAsync(h->p, 0, h->bytes, r.zero[device]) != cudaSuccess || cudaStreamSynchronize(r.zero[device]) != cudaSuccess) {
    cudaGetLastError();
    r.spare.push_back(h);
    return CB_ERR_CUDA;
  }
  *out = h;
  return CB_OK;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" CB_API uint64_t cb_stream_capture_id(cb_stream_t stream) {
  uint64_t id = 0;
  cudaGraph_t graph = nullptr;
  return capture_of(reinterpret_cast<cudaStream_t>(stream), &id, &graph) ? id : 0;
}

extern "C" CB_API int cb_capture_workspace(cb_stream_t stream, size_t bytes, void** workspace) {
  if (!workspace || bytes == 0) return CB_ERR_INVALID_ARG;
  uint64_t id = 0;
  cudaGraph_t graph = nullptr;
  if (!capture_of(reinterpret_cast<cudaStream_t>(stream), &id, &graph)) return CB_ERR_INVALID_ARG;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return CB_ERR_CUDA;
  const Relaxed relaxed;
  Registry& r = registry();
  Held* h = nullptr;
  {
    const std::lock_guard<std::mutex> guard(r.lock);
    const int rc = acquire(r, bytes, device, &h);
    if (rc != CB_OK) return rc;
    h->capture = id;
    r.live.push_back(h);
  }
  // (without the lock: releasing an object may call back at once)
  cudaUserObject_t object = nullptr;
  if (cudaUserObjectCreate(&object, h, released, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
    cudaGetLastError();
    released(h);
    return CB_ERR_CUDA;
  }
  if (cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
    cudaGetLastError();
    cudaUserObjectRelease(object, 1);
    return CB_ERR_CUDA;
  }
  *workspace = h->p;
  return CB_OK;
}

extern "C" CB_API int cb_capture_live(uint64_t capture_id) {
  Registry& r = registry();
  const std::lock_guard<std::mutex> guard(r.lock);
  for (const Held* h : r.live)
    if (h->capture == capture_id) return 1;
  return 0;
}
