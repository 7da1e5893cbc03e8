// Workspaces of calls that are being captured into a CUDA graph.
//
// An eager call uses the workspace of its (device, stream): calls on one stream are ordered.  Graphs are not tied to the
// stream they were captured on, so two of them may run side by side: each capture gets workspaces of its own, one per
// capturing stream (branches of one graph are captured on different streams).  A workspace is cleared once, when the
// capture takes it (every call leaves it clean), so a replay pays nothing; it returns to a free list when the last graph
// that uses it has been destroyed.
#include <cuda_runtime.h>

#include <map>
#include <mutex>
#include <stdexcept>
#include <utility>
#include <vector>

#include "fg_torch.h"

namespace {

struct Block {
  void* ptr;
  size_t bytes;
  int device;
  bool free;
};

// Never destroyed: graphs may outlive the interpreter's teardown of this module.
std::mutex& mu() {
  static std::mutex* m = new std::mutex;
  return *m;
}
std::vector<Block>& blocks() {
  static std::vector<Block>* v = new std::vector<Block>;
  return *v;
}
using Key = std::pair<unsigned long long, int64_t>;  // capture id, stream
std::map<Key, size_t>& taken() {
  static std::map<Key, size_t>* m = new std::map<Key, size_t>;
  return *m;
}

struct Release {
  size_t index;
  Key key;
};

// Runs when the graph (and every executable graph made of it) is gone; may not call CUDA.
void CUDART_CB release(void* p) {
  Release* r = static_cast<Release*>(p);
  {
    std::lock_guard<std::mutex> lk(mu());
    blocks()[r->index].free = true;
    taken().erase(r->key);
  }
  delete r;
}

void must(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("fastgate_b200: ") + cudaGetErrorString(e));
}

// Calls that a capture in progress on another stream would otherwise forbid.
struct RelaxedMode {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedMode() { must(cudaThreadExchangeStreamCaptureMode(&mode)); }
  ~RelaxedMode() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// On a stream of its own, to the end.
void clear(void* p, size_t bytes) {
  cudaStream_t side = nullptr;
  must(cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking));
  cudaError_t e = cudaMemsetAsync(p, 0, bytes, side);
  if (e == cudaSuccess) e = cudaStreamSynchronize(side);
  cudaStreamDestroy(side);
  must(e);
}

// `bytes` of zeros on the current device, also while a stream is being captured.
void* cleared(size_t bytes) {
  RelaxedMode relaxed;
  void* p = nullptr;
  must(cudaMalloc(&p, bytes));
  clear(p, bytes);
  return p;
}

}  // namespace

int* linear_status(int device) {
  static std::map<int, void*>* words = new std::map<int, void*>;
  std::lock_guard<std::mutex> lk(mu());
  void*& p = (*words)[device];
  if (p == nullptr) p = cleared(256);
  return static_cast<int*>(p);
}

void* graph_workspace(int device, cudaStream_t stream, size_t bytes) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  must(cudaStreamGetCaptureInfo(stream, &status, &id, &graph));
  if (status != cudaStreamCaptureStatusActive) return nullptr;
  const Key key{id, reinterpret_cast<int64_t>(stream)};
  std::lock_guard<std::mutex> lk(mu());
  const auto known = taken().find(key);
  if (known != taken().end() && blocks()[known->second].bytes >= bytes) return blocks()[known->second].ptr;
  // (A larger workspace than the one this capture has: the old one stays with the graph too, its calls are in it.)
  RelaxedMode relaxed;
  size_t index = blocks().size();
  for (size_t i = 0; i < blocks().size(); ++i)
    if (blocks()[i].free && blocks()[i].device == device && blocks()[i].bytes >= bytes && (index == blocks().size() || blocks()[i].bytes < blocks()[index].bytes)) index = i;
  if (index == blocks().size()) {
    Block b = {nullptr, bytes, device, true};
    must(cudaMalloc(&b.ptr, bytes));
    blocks().push_back(b);
  }
  Block& b = blocks()[index];
  clear(b.ptr, b.bytes);
  Release* r = new Release{index, key};
  cudaUserObject_t object = nullptr;
  cudaError_t e = cudaUserObjectCreate(&object, r, release, 1, cudaUserObjectNoDestructorSync);
  if (e != cudaSuccess) {
    delete r;
    must(e);
  }
  b.free = false;
  taken()[key] = index;
  e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
  if (e != cudaSuccess) {
    b.free = true;
    taken().erase(key);
    must(e);
  }
  return b.ptr;
}
