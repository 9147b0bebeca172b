// Device memory of the layer operators' handles (linear.h), shared with the
// graphs that are captured from their calls.
#include <mutex>

#include "linear.h"

namespace apk {

namespace {

// Allocating, freeing and waiting disturb no capture that the calling thread
// or another one has under way: they concern no captured stream.
class RelaxedCapture {
 public:
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode_); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode_); }

 private:
  cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
};

// What its last user has let go of, a graph perhaps: the callback that tells
// of a graph's end may not call CUDA.
struct Shared {
  std::mutex mu;  // of `gone`: held over no CUDA call, which may wait for a callback that wants it
  std::vector<std::pair<int, uint8_t*>> gone;
  std::mutex side_mu;
  std::vector<std::pair<int, cudaStream_t>> side;  // per device, for clearing new memory
};
Shared& shared() {
  static Shared* s = new Shared;  // never destroyed: a graph may end at the process's exit
  return *s;
}

// A stream that nothing else uses: the caller's may be captured, and the
// legacy one is not ordered before non-blocking ones.
apk_status side_stream(int device, cudaStream_t* out, Err* err) {
  Shared& g = shared();
  std::lock_guard<std::mutex> lock(g.side_mu);
  for (const auto& s : g.side)
    if (s.first == device) {
      *out = s.second;
      return APK_OK;
    }
  const apk_status st = cu_status(cudaStreamCreateWithFlags(out, cudaStreamNonBlocking), "cudaStreamCreate", err);
  if (st == APK_OK) g.side.emplace_back(device, *out);
  return st;
}

}  // namespace

apk_status cu_status(cudaError_t e, const char* what, Err* err) {
  if (e == cudaSuccess) return APK_OK;
  return err->fail(e == cudaErrorMemoryAllocation ? APK_ENOMEM : APK_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

Memory::~Memory() {
  if (!data_) return;
  Shared& g = shared();
  std::lock_guard<std::mutex> lock(g.mu);
  try {
    g.gone.emplace_back(device_, data_);
  } catch (...) {  // it stays allocated
  }
}

void Memory::free_gone() {
  std::vector<std::pair<int, uint8_t*>> list;
  {
    Shared& g = shared();
    std::lock_guard<std::mutex> lock(g.mu);
    list.swap(g.gone);
  }
  if (list.empty()) return;
  RelaxedCapture relaxed;
  for (const auto& m : list) {
    DeviceGuard guard(m.first);
    cudaFree(m.second);  // waits for the device
  }
}

apk_status Memory::make(int device, size_t bytes, size_t zeroed, std::shared_ptr<Memory>* out, Err* err) {
  free_gone();
  auto m = std::make_shared<Memory>();
  RelaxedCapture relaxed;
  void* q = nullptr;
  apk_status st = cu_status(cudaMalloc(&q, bytes), "cudaMalloc", err);
  if (st != APK_OK) return st;
  m->device_ = device;
  m->data_ = static_cast<uint8_t*>(q);
  m->bytes_ = bytes;
  cudaStream_t side = nullptr;
  st = side_stream(device, &side, err);
  if (st == APK_OK) st = cu_status(cudaMemsetAsync(q, 0, zeroed, side), "cudaMemset", err);
  if (st == APK_OK) st = cu_status(cudaStreamSynchronize(side), "cudaStreamSynchronize", err);
  if (st == APK_OK) *out = std::move(m);
  return st;
}

apk_status Memory::keep_for(cudaGraph_t graph, const std::shared_ptr<Memory>& m, Err* err) {
  auto* own = new std::shared_ptr<Memory>(m);
  cudaUserObject_t obj = nullptr;
  apk_status st = cu_status(cudaUserObjectCreate(
                                &obj, own, [](void* p) { delete static_cast<std::shared_ptr<Memory>*>(p); }, 1,
                                cudaUserObjectNoDestructorSync),
                            "cudaUserObjectCreate", err);
  if (st != APK_OK) {
    delete own;
    return st;
  }
  st = cu_status(cudaGraphRetainUserObject(graph, obj, 1, cudaGraphUserObjectMove), "cudaGraphRetainUserObject", err);
  if (st != APK_OK) cudaUserObjectRelease(obj, 1);
  return st;
}

apk_status Scratch::open(int device, Err* err) {
  device_ = device;
  return Memory::make(device, 256, 256, &status_, err);
}

apk_status Scratch::enter(cudaStream_t stream, Err* err) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  apk_status st = cu_status(cudaStreamGetCaptureInfo(stream, &cap, &id, &graph_), "cudaStreamGetCaptureInfo", err);
  if (st != APK_OK) return st;
  capturing_ = cap == cudaStreamCaptureStatusActive;
  stream_ = stream;
  now_ = nullptr;
  if (!capturing_ || id == capture_) return APK_OK;
  if ((st = Memory::keep_for(graph_, status_, err)) == APK_OK) capture_ = id;
  return st;
}

apk_status Scratch::begin(size_t bytes, size_t zeroed, Err* err) {
  apk_status st = APK_OK;
  if (capturing_) {
    if (bytes > most_)
      return err->fail(APK_ESTATE, "the scratch has to grow to %zu bytes: make one call of this size before the capture",
                       bytes);
    for (size_t i = captured_.size(); i-- > 0;)
      if (captured_[i].memory.expired()) {
        cudaEventDestroy(captured_[i].ev);
        captured_.erase(captured_.begin() + i);
      }
    for (Captured& c : captured_) {
      const std::shared_ptr<Memory> m = c.memory.lock();
      if (c.capture != capture_ || !m || m->bytes() < bytes) continue;
      // an edge from the last call that used it, which another branch may have made
      if (c.last != stream_ &&
          (st = cu_status(cudaStreamWaitEvent(stream_, c.ev, 0), "cudaStreamWaitEvent", err)) != APK_OK)
        return st;
      now_ = &c;
      data_ = m->data();
      return APK_OK;
    }
    captured_.reserve(captured_.size() + 1);
    Captured c;
    c.capture = capture_;
    std::shared_ptr<Memory> m;
    if ((st = Memory::make(device_, bytes, zeroed, &m, err)) != APK_OK ||
        (st = Memory::keep_for(graph_, m, err)) != APK_OK ||
        (st = cu_status(cudaEventCreateWithFlags(&c.ev, cudaEventDisableTiming), "cudaEventCreate", err)) != APK_OK)
      return st;
    c.memory = m;
    captured_.push_back(c);
    now_ = &captured_.back();
    data_ = m->data();
    return APK_OK;
  }
  if (!own_ || bytes > own_->bytes()) {
    if (used_) {
      RelaxedCapture relaxed;
      if ((st = cu_status(cudaEventSynchronize(ev_), "waiting for the scratch", err)) != APK_OK) return st;
    }
    used_ = false;
    own_.reset();
    if ((st = Memory::make(device_, bytes, zeroed, &own_, err)) != APK_OK) return st;
    most_ = bytes;
  }
  if (!ev_ && (st = cu_status(cudaEventCreateWithFlags(&ev_, cudaEventDisableTiming), "cudaEventCreate", err)) != APK_OK)
    return st;
  data_ = own_->data();
  // (on the same stream too: a handle's value may name another stream by now)
  return used_ ? cu_status(cudaStreamWaitEvent(stream_, ev_, 0), "cudaStreamWaitEvent", err) : APK_OK;
}

apk_status Scratch::end(Err* err) {
  const apk_status st = cu_status(cudaEventRecord(now_ ? now_->ev : ev_, stream_), "cudaEventRecord", err);
  if (now_) now_->last = stream_;
  else used_ = used_ || st == APK_OK;
  return st;
}

apk_status Scratch::clear(size_t bytes, cudaStream_t stream, Err* err) {
  std::vector<std::shared_ptr<Memory>> all;
  if (own_) all.push_back(own_);
  for (const Captured& c : captured_)
    if (auto m = c.memory.lock()) all.push_back(m);
  for (const auto& m : all) {
    const apk_status st = cu_status(cudaMemsetAsync(m->data(), 0, bytes, stream), "clearing the scratch", err);
    if (st != APK_OK) return st;
  }
  return cu_status(cudaStreamSynchronize(stream), "cudaStreamSynchronize", err);
}

Scratch::~Scratch() {
  own_.reset();
  status_.reset();
  for (const Captured& c : captured_) cudaEventDestroy(c.ev);
  if (ev_) cudaEventDestroy(ev_);
  Memory::free_gone();
}

}  // namespace apk
