// Device scratch of launches that need more than one kernel: a buffer a (device, stream, user), and buffers of their own for
// captured launches.
#include <cuda_runtime.h>

#include <mutex>
#include <vector>

#include "launch.h"

namespace tsr {
namespace {

constexpr size_t kStep = 2u << 20;
size_t in_steps(size_t bytes) { return (bytes + kStep - 1) / kStep * kStep; }

struct Buffer {
  int device, slot;
  cudaStream_t stream;
  unsigned long long capture;  // 0: of plain launches
  unsigned char* ptr;
  size_t bytes;
  bool serves(int dev, cudaStream_t st, int s, unsigned long long c, size_t need) const {
    return device == dev && stream == st && slot == s && capture == c && bytes >= need;
  }
};

// Buffers that graphs hold, and those whose graphs are gone.  Its lock is never held across a call of the runtime, which may
// run give_back() on a thread of its own; it is never destroyed, since graphs may outlive the library's other objects.
struct GraphBuffers {
  std::mutex mutex;
  std::vector<Buffer> held, spare;
};
GraphBuffers& graph_buffers() {
  static GraphBuffers* const all = new GraphBuffers;
  return *all;
}

// The last graph or executable graph that could launch over `user`'s buffer is gone.
void CUDART_CB give_back(void* user) {
  GraphBuffers& all = graph_buffers();
  std::lock_guard<std::mutex> lock(all.mutex);
  for (size_t i = 0; i < all.held.size(); ++i)
    if (all.held[i].ptr == user) {
      all.spare.push_back(all.held[i]);  // (has room: see below)
      all.held.erase(all.held.begin() + static_cast<std::ptrdiff_t>(i));
      return;
    }
}

// A captured launch may be replayed on any stream, beside other graphs that were captured on this one and beside plain launches
// on it, so every capture has buffers of its own, which its graph keeps.
unsigned char* capture_scratch(int dev, cudaStream_t st, size_t bytes, int slot) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  if (cudaStreamGetCaptureInfo(st, &status, &id, &graph) != cudaSuccess || status != cudaStreamCaptureStatusActive) {
    cudaGetLastError();
    return nullptr;
  }
  const size_t want = in_steps(bytes);
  Buffer b{dev, slot, st, id, nullptr, want};
  GraphBuffers& all = graph_buffers();
  {
    std::lock_guard<std::mutex> lock(all.mutex);
    for (const Buffer& h : all.held)
      if (h.serves(dev, st, slot, id, bytes)) return h.ptr;
    size_t best = all.spare.size();
    for (size_t i = 0; i < all.spare.size(); ++i)
      if (all.spare[i].device == dev && all.spare[i].bytes >= want && all.spare[i].bytes <= 2 * want &&
          (best == all.spare.size() || all.spare[i].bytes < all.spare[best].bytes))
        best = i;
    if (best != all.spare.size()) {
      b.ptr = all.spare[best].ptr, b.bytes = all.spare[best].bytes;
      all.spare.erase(all.spare.begin() + static_cast<std::ptrdiff_t>(best));
    }
  }
  if (b.ptr == nullptr) {  // (an allocation is no work of the stream: it is made beside the capture)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    void* ptr = nullptr;
    const cudaError_t e = cudaMalloc(&ptr, want);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    b.ptr = static_cast<unsigned char*>(ptr);
  }
  {
    std::lock_guard<std::mutex> lock(all.mutex);
    all.held.push_back(b);
    all.spare.reserve(all.held.size() + all.spare.size());
  }
  cudaUserObject_t owner = nullptr;
  if (cudaUserObjectCreate(&owner, b.ptr, give_back, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
    cudaGetLastError();
    give_back(b.ptr);
    return nullptr;
  }
  if (cudaGraphRetainUserObject(graph, owner, 1, cudaGraphUserObjectMove) != cudaSuccess) {
    cudaGetLastError();
    cudaUserObjectRelease(owner, 1);  // gives it back
    return nullptr;
  }
  return b.ptr;
}

thread_local bool own_capture = false;

}  // namespace

OwnCapture::OwnCapture() { own_capture = true; }
OwnCapture::~OwnCapture() { own_capture = false; }

unsigned char* stream_scratch(cudaStream_t st, size_t bytes, int slot) try {
  static std::mutex mutex;
  static std::vector<Buffer> table;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &status) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  const bool capturing = status != cudaStreamCaptureStatusNone;
  {
    std::lock_guard<std::mutex> lock(mutex);
    unsigned char* plain = nullptr;
    for (const Buffer& b : table)
      if (b.serves(dev, st, slot, 0, bytes)) plain = b.ptr;
    if (plain != nullptr && (!capturing || own_capture)) return plain;
    if (capturing && plain == nullptr) return nullptr;
    if (!capturing) {
      // twice as large every time, so that what a stream outgrew is no more than what it uses (the delta rule's come in few
      // sizes already)
      size_t want = slot == kScratchDelta ? in_steps(bytes) : 4u << 20;
      while (want < bytes) want <<= 1;
      void* ptr = nullptr;
      if (cudaMallocAsync(&ptr, want, st) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
      }
      table.push_back(Buffer{dev, slot, st, 0, static_cast<unsigned char*>(ptr), want});
      return static_cast<unsigned char*>(ptr);
    }
  }
  return capture_scratch(dev, st, bytes, slot);
} catch (...) {  // no memory for a table
  return nullptr;
}

}  // namespace tsr
