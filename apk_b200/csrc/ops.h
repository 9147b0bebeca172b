// Host helpers shared by norm.cu, clip.cu, logprobs.cu and linear4.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <new>

#include "../../include/apk.h"
#include "linear.h"

#define APK_TRY(x)                    \
  do {                                \
    const apk_status st_ = (x);       \
    if (st_ != APK_OK) return st_;    \
  } while (0)

namespace apk {
namespace ops {

constexpr int MAX_SIZE = 1 << 30;  // of a 32-bit count: leaves room to step past the end

inline bool valid_dtype(int d) { return d == APK_F32 || d == APK_BF16; }
inline size_t esize(int d) { return d == APK_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }
template <class T>
constexpr T ceil_div(T a, T b) {
  return (a + b - 1) / b;
}

// Whether rows of `dtype` can be read in whole 16-byte pieces.
inline bool on16(const void* p, long long ld, int rows, int dtype) {
  return aligned(p, 16) && (rows <= 1 || ld % (16 / (long long)esize(dtype)) == 0);
}

// The device has to exist and be the one that the kernels are built for.
inline apk_status open_device(int device, int* sms, Err* err) {
  int ndev = 0, major = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
    cudaGetLastError();
    return err->fail(APK_ECUDA, "no CUDA device %d", device);
  }
  APK_TRY(cu_status(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device), "device query", err));
  APK_TRY(cu_status(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device), "device query", err));
  if (major != 10) return err->fail(APK_EUNSUPPORTED, "the kernels are built for sm_100a");
  return APK_OK;
}

// The bodies of the C entry points: no exception leaves them, and calls on one
// handle from several host threads are taken one at a time.  H has err, mu and opened.
template <class H, class Cfg, class F>
apk_status make(const Cfg* cfg, H** out, F&& create) {
  if (!out) return APK_EINVAL;
  *out = new (std::nothrow) H;
  if (!*out) return APK_ENOMEM;
  try {
    if (!cfg) return (*out)->err.fail(APK_EINVAL, "cfg is NULL");  // *out is set on failure too
    APK_TRY(create(cfg, *out));
    (*out)->opened = true;
    return APK_OK;
  } catch (...) {
    return APK_ENOMEM;
  }
}
template <class H, class F>
apk_status call(H* h, const void* arg, F&& f) {
  if (!h || !h->opened || !arg) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    return f();
  } catch (...) {
    return APK_ENOMEM;
  }
}

}  // namespace ops
}  // namespace apk
