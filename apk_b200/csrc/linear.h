// Shared by the layer operators (linear_gemm.cu, linear.cu, moe.cu): the
// GEMM problem the epilogue kernel runs, and host helpers.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>
#include <memory>
#include <string>
#include <vector>

#include "../../include/apk.h"

namespace apk {
namespace lin {

// One product out[r][c] = act(sum_k Q(r,k) P(k,c) + bias[c]) + res[r][c].
// P is the operand of the output's columns, Q that of its rows; either is
// K-major (k contiguous) or MN-major (its columns / rows contiguous).
struct Epilogue {
  const void* bias;
  const void* res;
  void* out;
  void* pre;  // bf16 pre-activation, or null
  long long ld_res, ld_out, ld_pre;
  int bias_f32, res_f32, out_f32, act;
};
struct alignas(64) Problem {
  CUtensorMap tmP, tmQ;
  Epilogue epi;
  int rows, cols, nkb;
  int tiles_r, tiles_c;
  int p_mn, q_mn;
  uint32_t idesc;
};
struct GemmParams {
  Problem pr[2];
  int nprob;
  int tiles0, tiles;  // tiles of problem 0 / of all
  int extra;          // tiles of problem 1 that take the time of one of problem 0
  int split;          // CTAs of a cluster that share one tile's K range (1: none)
  int* status;
  long long limit;
};

// An operand as the caller holds it: [outer][inner] bf16, `inner` contiguous.
struct Operand {
  const void* p;
  long long ld;
  int outer, inner;
  bool mn;  // the contiguous axis is the output's (MN-major), not k
};
struct Product {
  Operand P, Q;
  int rows, cols, k;
  Epilogue epi;
};

// Whether a product is faster through run_stream than through run_products.
// Up to 8 rows [n][k] weights always are (8 x 4096 x 8192: 14.0 against 15.6
// us).  Two MMA tiles of rows, or the narrower row pieces of [k][n], cost it
// bandwidth, so that only its smaller latency counts (16 rows, [n][k]: 2048 x
// 2048 3.2 against 7.0, 2048 x 4096 6.1 against 7.4, 4096 x 8192 20.6 against
// 16.1; [k][n]: 1 x 2048 x 2048 5.2 against 6.8, 8 x 2048 x 4096 8.4 against
// 7.4, 8 x 4096 x 8192 21.2 against 15.1).  Weights that TMA cannot address
// save it their copy.
inline bool streams(int rows, long long weight_bytes, bool nk, bool tma) {
  if (rows > 16) return false;
  const long long mb = weight_bytes >> 20;
  if (!tma) return mb < 16;
  return nk ? rows <= 8 || mb < 24 : mb < (rows <= 8 ? 16 : 4);
}
// Launches one or two products, in one launch where that is faster.  sms: the
// SMs it may fill; dev: the current device.  `why` receives a message on failure.
apk_status run_products(const Product* pr, int n, int sms, int dev, int* status, long long limit, cudaStream_t stream,
                        std::string* why);
// A product of at most 16 rows with weights [n][k] (nk) or [k][n] of any
// stride and alignment.
cudaError_t run_stream(const void* x, long long ldx, const void* w, long long ldw, bool nk, int rows, int n, int k,
                       const Epilogue& epi, int sms, cudaStream_t stream);
// Sets the kernels' attributes on the current device, once; before its first run_products.
cudaError_t prepare();

}  // namespace lin

// ---- host helpers -----------------------------------------------------------
struct Err {
  std::string text;
  apk_status fail(apk_status st, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    text = buf;
    return st;
  }
};

// The calling thread's device is put back when a call returns.
class DeviceGuard {
 public:
  explicit DeviceGuard(int dev) {
    cudaGetDevice(&old_);
    if (old_ != dev) cudaSetDevice(dev);
    else old_ = -1;
  }
  ~DeviceGuard() {
    if (old_ >= 0) cudaSetDevice(old_);
  }

 private:
  int old_ = -1;
};

// Device memory that a handle's calls and the graphs captured from them share.
// It is freed some time after the last of them has let go of it.
class Memory {
 public:
  // The first `zeroed` bytes are zero.  May be called while a stream is captured.
  static apk_status make(int device, size_t bytes, size_t zeroed, std::shared_ptr<Memory>* out, Err* err);
  // `graph`, and what is instantiated from it, hold m until they are destroyed.
  static apk_status keep_for(cudaGraph_t graph, const std::shared_ptr<Memory>& m, Err* err);
  static void free_gone();
  Memory() = default;
  Memory(const Memory&) = delete;
  ~Memory();
  uint8_t* data() const { return data_; }
  size_t bytes() const { return bytes_; }

 private:
  int device_ = 0;
  uint8_t* data_ = nullptr;
  size_t bytes_ = 0;
};

// Status word and scratch of one handle.
//
// Calls on one handle may come from different streams: a call that uses the
// scratch waits for the last one that did.  Nothing could order a graph's
// launches with them, or with another graph's, so the calls of one capture get
// scratch of their own, which lives as long as the graph does; branches of one
// capture are ordered by an edge between their calls.  What a capture
// allocates is bounded by what calls outside captures have needed: a larger
// call is refused.
class Scratch {
 public:
  Scratch() = default;
  Scratch(const Scratch&) = delete;
  ~Scratch();
  apk_status open(int device, Err* err);  // allocates the status word
  int* status() const { return status_ ? reinterpret_cast<int*>(status_->data()) : nullptr; }
  // The first thing of every call that uses the status word or the scratch.
  apk_status enter(cudaStream_t stream, Err* err);
  // At least `bytes` of scratch, the first `zeroed` of them zero when it was
  // allocated and left so by every kernel that uses them.
  apk_status begin(size_t bytes, size_t zeroed, Err* err);
  apk_status end(Err* err);
  uint8_t* data() const { return data_; }
  // Zeroes the first `bytes` of every buffer, those of graphs too, and waits for it.
  apk_status clear(size_t bytes, cudaStream_t stream, Err* err);

 private:
  struct Captured {
    unsigned long long capture = 0;
    std::weak_ptr<Memory> memory;
    cudaEvent_t ev = nullptr;      // the last call of the capture that used it
    cudaStream_t last = nullptr;   // and its stream
  };
  int device_ = 0;
  std::shared_ptr<Memory> status_, own_;
  size_t most_ = 0;  // bytes that a call outside captures needed
  cudaEvent_t ev_ = nullptr;
  bool used_ = false;
  std::vector<Captured> captured_;
  unsigned long long capture_ = 0;  // whose graph holds the status word
  // of the call under way
  cudaStream_t stream_ = nullptr;
  cudaGraph_t graph_ = nullptr;
  bool capturing_ = false;
  Captured* now_ = nullptr;
  uint8_t* data_ = nullptr;
};

// Ends the use of the scratch on every way out of a call.
class ScratchUse {
 public:
  ScratchUse(Scratch* s, Err* err) : s_(s), err_(err) {}
  ~ScratchUse() {
    if (begun_) {
      Err ignored;
      s_->end(&ignored);
    }
  }
  apk_status begin(size_t bytes, size_t zeroed) {
    const apk_status st = s_->begin(bytes, zeroed, err_);
    begun_ = st == APK_OK;
    return st;
  }
  apk_status end() {
    if (!begun_) return APK_OK;
    begun_ = false;
    return s_->end(err_);
  }

 private:
  Scratch* s_;
  Err* err_;
  bool begun_ = false;
};

// Launch configuration with a cluster size and programmatic stream
// serialization (every kernel launched with it calls pdl_wait first thing).
struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[3];
  Launch(dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster = 1) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = at;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
      at[1].id = cudaLaunchAttributeClusterDimension;
      at[1].val.clusterDim.x = cluster;
      at[1].val.clusterDim.y = 1;
      at[1].val.clusterDim.z = 1;
      cfg.numAttrs = 2;
    }
  }
};

apk_status cu_status(cudaError_t e, const char* what, Err* err);

}  // namespace apk
