// The global norm of many tensors, and scaling them to a bound (apk_clip_* of
// include/apk.h).  No counterpart in the reference, which multiplies bare
// matrices (src/tcyield.cu:91-356).
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   c = min(1, max_norm / (norm + 1e-6)),  g' = c g
//
// Bound by memory: the norm reads everything once; the scaling, which cannot
// begin before the norm is known, reads it again and writes it.  The tensors'
// addresses travel as kernel arguments, so that a captured graph holds them
// and no copy precedes the kernels.
#include <algorithm>
#include <vector>

#include "ops.cuh"
#include "ops.h"

namespace apk {
namespace clip {

constexpr int THREADS = 256, VECS = 4;            // 16-byte vectors of a thread and unit
constexpr int UNIT = THREADS * VECS;              // vectors of a unit
constexpr int BLOCKS = 4;                         // of an SM

struct Tensor {
  const uint8_t* in;
  uint8_t* out;
  long long n;
  unsigned first;  // its first unit
  int f32;
};
// Units are taken from the aligned 16-byte vector that holds a tensor's first element.
template <int N>
struct List {
  Tensor t[N];
  int count;
  unsigned units;
};
// (a launch copies its arguments: few tensors should not pay for many; 32,764 bytes
// is the most.  Clipping 4 tensors of 100,000 values together 4.8 us, by the list
// of 350 5.0, of 1000 5.1; 300 tensors of 8.4 million 22.7, by that of 1000 22.8)
constexpr int FEW = 60, SOME = 350, MANY = 1000;
struct Sum {
  unsigned* arrived;  // zero between launches; null: the scaling adds the blocks' sums up
  double* part;       // one of each block of all launches
  float* norm;
  float max_norm;
  unsigned first, blocks;  // of this launch, of all
};

// The elements of an incomplete vector, the first or the last of a tensor: [lo, hi) of those it has room for.
struct Span {
  long long vec;  // bytes from the tensor's aligned start
  int lo, hi;
  bool any, whole;
};
__device__ __forceinline__ Span span_of(const Tensor& t, unsigned unit, int j) {
  const int per = t.f32 ? 4 : 8, head = (int)(reinterpret_cast<uintptr_t>(t.in) & 15) / (t.f32 ? 4 : 2);
  const long long v = (long long)(unit - t.first) * UNIT + j * THREADS + threadIdx.x;
  const long long e0 = v * per - head;  // the vector's first element
  Span s;
  s.vec = v * 16;
  s.lo = e0 < 0 ? (int)-e0 : 0;
  s.hi = t.n - e0 < per ? (int)(t.n - e0) : per;
  s.any = s.hi > s.lo;
  s.whole = s.lo == 0 && s.hi == per;
  return s;
}
__device__ __forceinline__ uint4 load(const uint8_t* base, const Span& s, int f32, bool last_use) {
  const uint4* q = reinterpret_cast<const uint4*>(base + s.vec);
  if (s.whole) return last_use ? __ldcs(q) : *q;
  union {
    uint16_t h[8];
    uint32_t w[4];
    uint4 v;
  } u;
  u.v = make_uint4(0, 0, 0, 0);
  if (f32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i >= s.lo && i < s.hi) u.w[i] = reinterpret_cast<const uint32_t*>(q)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= s.lo && i < s.hi) u.h[i] = reinterpret_cast<const uint16_t*>(q)[i];
  }
  return u.v;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ double block_sum(double v, double (&sh)[8]) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += sh[i];
  return v;
}

// The sum of the squares of a vector's values.  Between 2^-45 and 2^45 fp32
// has room for them, and what lies far below the largest value of the eight
// is lost beside it; else in 64 bits.
__device__ __forceinline__ void add_squares(const float* v, int n, float& sum, double& total) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < n; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(v[i])));
  if (most >= 0x1p-45f && most <= 0x1p45f) {
#pragma unroll
    for (int i = 0; i < n; ++i) sum = fmaf(v[i], v[i], sum);
  } else if (most != 0.f) {
#pragma unroll
    for (int i = 0; i < n; ++i) total = fma((double)v[i], (double)v[i], total);
  }
}

// A block takes runs of up to 8 neighbouring units, of one tensor mostly: unit
// by unit, it stepped over ten tensors' entries for each where there are
// hundreds (300 tensors, 268 MB: 67 us); in one piece, blocks read far apart.
template <int N>
__device__ __forceinline__ unsigned run_of(const List<N>& list) {
  return min(max(list.units / (gridDim.x * 4), 1u), 8u);
}
// The last tensor that begins at unit u or before.
template <int N>
__device__ __forceinline__ int find(const List<N>& list, unsigned u) {
  int lo = 0, hi = list.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (list.t[mid].first <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The norm, from all blocks' sums, in their order.
__device__ __forceinline__ double total_norm(const Sum& p, double (&sh)[8]) {
  double total = 0.0;
  for (unsigned i = threadIdx.x; i < p.blocks; i += THREADS) total += __ldcg(p.part + i);
  return sqrt(block_sum(total, sh));
}
// Squares are added in fp32 within a thread's part of a unit (16 or 32 values)
// and in 64 bits beyond; for the norm alone the last block to arrive adds the
// blocks' sums.
template <int N>
__global__ void __launch_bounds__(THREADS, BLOCKS) norm(const __grid_constant__ List<N> list, const __grid_constant__ Sum p) {
  __shared__ double sh[8], sh2[8];
  __shared__ bool last;
  pdl_launch();
  pdl_wait();
  double total = 0.0;
  const unsigned run = run_of(list);
  for (unsigned first = blockIdx.x * run; first < list.units; first += gridDim.x * run) {
    const unsigned end = min(first + run, list.units);
    int at = find(list, first);
    for (unsigned u = first; u < end; u += 2) {  // two units' loads at once
      uint4 raw[2][VECS];
      int f32[2] = {};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (u + k >= end) break;
        while (at + 1 < list.count && u + k >= list.t[at + 1].first) ++at;
        const Tensor& t = list.t[at];
        const uint8_t* base = t.in - (reinterpret_cast<uintptr_t>(t.in) & 15);
        f32[k] = t.f32;
#pragma unroll
        for (int j = 0; j < VECS; ++j) {
          const Span s = span_of(t, u + k, j);
          raw[k][j] = s.any ? load(base, s, t.f32, false) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (u + k >= end) break;
        float sum[VECS] = {};
#pragma unroll
        for (int j = 0; j < VECS; ++j) {
          const uint4 q = raw[k][j];
          if (f32[k]) {
            const float v[4] = {__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w)};
            add_squares(v, 4, sum[j], total);
          } else {
            float v[8];
            ops::unpack(ops::Raw<false>{q}, v);
            add_squares(v, 8, sum[j], total);
          }
        }
        total += (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
      }
    }
  }
  total = block_sum(total, sh);
  if (!p.arrived) {
    if (threadIdx.x == 0) p.part[p.first + blockIdx.x] = total;
    return;
  }
  if (threadIdx.x == 0) {
    p.part[p.first + blockIdx.x] = total;
    __threadfence();
    last = atomicAdd(p.arrived, 1u) == p.blocks - 1;
    if (last) *p.arrived = 0;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const double n = total_norm(p, sh2);
  if (threadIdx.x == 0) *p.norm = (float)n;
}

// (An output at another place within 16 bytes is written element by element: 134
// million fp32 values into a flat buffer 270 us, shifted by one value 335.)
__device__ __forceinline__ void scale_unit(const Tensor& t, unsigned u, float c) {
  const int shift = (int)(reinterpret_cast<uintptr_t>(t.in) & 15);
  const uint8_t* base = t.in - shift;
  uint8_t* out = t.out - shift;
  const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  uint4 raw[VECS];
  Span sp[VECS];
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    sp[j] = span_of(t, u, j);
    if (sp[j].any) raw[j] = load(base, sp[j], t.f32, true);
  }
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    if (!sp[j].any) continue;
    union {
      uint16_t h[8];
      uint32_t w[4];
      uint4 v;
    } o;
    if (t.f32) {
      o.v = make_uint4(__float_as_uint(__uint_as_float(raw[j].x) * c), __float_as_uint(__uint_as_float(raw[j].y) * c),
                       __float_as_uint(__uint_as_float(raw[j].z) * c), __float_as_uint(__uint_as_float(raw[j].w) * c));
    } else {
      float v[8];
      ops::Raw<false> r{raw[j]};
      ops::unpack(r, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= c;
      ops::pack(v, r);
      o.v = r.a;
    }
    uint8_t* q = out + sp[j].vec;
    if (sp[j].whole && same) {
      __stcs(reinterpret_cast<uint4*>(q), o.v);
    } else if (t.f32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= sp[j].lo && i < sp[j].hi) reinterpret_cast<uint32_t*>(q)[i] = o.w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= sp[j].lo && i < sp[j].hi) reinterpret_cast<uint16_t*>(q)[i] = o.h[i];
    }
  }
}

// From the last unit to the first: what the norm read last is still in L2.
template <int N>
__global__ void __launch_bounds__(THREADS, BLOCKS) scale(const __grid_constant__ List<N> list, const __grid_constant__ Sum p) {
  __shared__ double sh[8];
  pdl_launch();
  pdl_wait();
  // every block adds the sums up for itself: a last block that did it for all
  // would be 2 us behind the others
  const double n = total_norm(p, sh), q = (double)p.max_norm / (n + 1e-6);
  const float c = q >= 1.0 ? 1.f : (float)q;  // (a NaN stays one)
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.norm = (float)n;
  const unsigned run = run_of(list);
  for (unsigned first = blockIdx.x * run; first < list.units; first += gridDim.x * run) {
    int at = find(list, list.units - 1 - first);
    for (unsigned k = first; k < min(first + run, list.units); ++k) {
      const unsigned u = list.units - 1 - k;
      while (u < list.t[at].first) --at;
      const Tensor& t = list.t[at];
      if (c != 1.f || t.in != t.out) scale_unit(t, u, c);
    }
  }
}

}  // namespace clip
}  // namespace apk

using namespace apk;

struct apk_clip {
  apk_clip_config cfg{};
  Err err;
  bool opened = false;
  int sms = 0;
  Scratch scratch;
  std::mutex mu;
};

namespace {

apk_status create(const apk_clip_config* cfg, apk_clip* h) {
  h->cfg = *cfg;
  APK_TRY(ops::open_device(h->cfg.device, &h->sms, &h->err));
  DeviceGuard guard(h->cfg.device);
  return h->scratch.open(h->cfg.device, &h->err);
}

unsigned long long units_of(const apk_clip_io* io, int i) {
  const size_t es = ops::esize(io->dtype[i]);
  const unsigned long long bytes = (reinterpret_cast<uintptr_t>(io->in[i]) & 15) + (unsigned long long)io->n[i] * es;
  return ops::ceil_div<unsigned long long>(bytes, 16ull * clip::UNIT);
}

// Every output is its own memory: no other tensor's, and its input's only where it is that.
apk_status check_apart(const apk_clip_io* io, Err* err) {
  struct Range {
    uintptr_t lo, hi;
    int i;
  };
  std::vector<Range> out;
  auto range = [&](const void* p, int i) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return Range{lo, lo + (uintptr_t)io->n[i] * ops::esize(io->dtype[i]), i};
  };
  for (int i = 0; i < io->count; ++i)
    if (io->n[i] > 0) out.push_back(range(io->out[i], i));
  std::sort(out.begin(), out.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  for (size_t j = 1; j < out.size(); ++j)
    if (out[j].lo < out[j - 1].hi)
      return err->fail(APK_EINVAL, "tensors %d and %d are written to the same memory", out[j - 1].i, out[j].i);
  for (int i = 0; i < io->count; ++i) {
    if (io->n[i] == 0 || io->in[i] == io->out[i]) continue;
    const Range r = range(io->in[i], i);
    // (the outputs do not overlap: the first that ends above r.lo is the one to look at)
    const auto it = std::upper_bound(out.begin(), out.end(), r.lo, [](uintptr_t at, const Range& o) { return at < o.hi; });
    if (it != out.end() && it->lo < r.hi)
      return err->fail(APK_EINVAL, "tensor %d is written to the memory that tensor %d is read from", it->i, i);
  }
  return APK_OK;
}

template <int N>
apk_status run(apk_clip* h, const apk_clip_io* io, bool scales, cudaStream_t s) {
  // the lists: of non-empty tensors, N at a time
  std::vector<clip::List<N>> lists;
  unsigned blocks = 0;
  auto grid = [&](const clip::List<N>& l) { return std::min<unsigned>(std::max(1u, l.units), h->sms * clip::BLOCKS); };
  for (int i = 0; i < io->count; ++i) {
    if (io->n[i] == 0) continue;
    const unsigned long long units = units_of(io, i);
    if (lists.empty() || lists.back().count == N || lists.back().units + units > 0xF0000000ull) {
      lists.emplace_back();
      lists.back().count = 0;
      lists.back().units = 0;
    }
    clip::List<N>& l = lists.back();
    l.t[l.count++] = {static_cast<const uint8_t*>(io->in[i]), scales ? static_cast<uint8_t*>(io->out[i]) : nullptr, io->n[i],
                      l.units, io->dtype[i] == APK_F32};
    l.units += (unsigned)units;
  }
  if (lists.empty()) {  // the norm of nothing
    lists.emplace_back();
    lists.back().count = 0;
    lists.back().units = 0;
  }
  for (const auto& l : lists) blocks += grid(l);
  APK_TRY(h->scratch.enter(s, &h->err));
  ScratchUse use(&h->scratch, &h->err);
  APK_TRY(use.begin(256 + ops::up256(blocks * sizeof(double)), 256));
  clip::Sum sum{scales ? nullptr : reinterpret_cast<unsigned*>(h->scratch.data()),
                reinterpret_cast<double*>(h->scratch.data() + 256), io->norm, io->max_norm, 0, blocks};
  for (const auto& l : lists) {
    Launch launch(dim3(grid(l)), clip::THREADS, 0, s);
    APK_TRY(cu_status(cudaLaunchKernelEx(&launch.cfg, clip::norm<N>, l, sum), "launching the norm", &h->err));
    sum.first += grid(l);
  }
  if (scales)
    for (size_t i = lists.size(); i-- > 0;) {
      Launch launch(dim3(grid(lists[i])), clip::THREADS, 0, s);
      APK_TRY(cu_status(cudaLaunchKernelEx(&launch.cfg, clip::scale<N>, lists[i], sum),
                        "launching the scaling", &h->err));
    }
  return use.end();
}

apk_status run(apk_clip* h, const apk_clip_io* io, bool scales) {
  if (io->count < 0) return h->err.fail(APK_EINVAL, "count is %d", io->count);
  if (!io->norm || !ops::aligned(io->norm, 4)) return h->err.fail(APK_EINVAL, "norm is NULL, or not aligned to its element");
  if (io->count > 0 && (!io->in || !io->n || !io->dtype || (scales && !io->out)))
    return h->err.fail(APK_EINVAL, "in, out, n or dtype is NULL");
  if (scales && !(io->max_norm >= 0.f)) return h->err.fail(APK_EINVAL, "max_norm is %g", io->max_norm);
  for (int i = 0; i < io->count; ++i) {
    if (io->n[i] < 0 || io->n[i] > 1ll << 40) return h->err.fail(APK_EINVAL, "tensor %d has %lld elements: at most 2^40", i, io->n[i]);
    if (io->n[i] == 0) continue;
    if (!ops::valid_dtype(io->dtype[i])) return h->err.fail(APK_EINVAL, "tensor %d: dtype %d", i, io->dtype[i]);
    if (!io->in[i] || (scales && !io->out[i])) return h->err.fail(APK_EINVAL, "tensor %d is NULL", i);
    const size_t es = ops::esize(io->dtype[i]);
    if (!ops::aligned(io->in[i], es) || (scales && !ops::aligned(io->out[i], es)))
      return h->err.fail(APK_EINVAL, "tensor %d is not aligned to its element", i);
  }
  if (scales) APK_TRY(check_apart(io, &h->err));
  DeviceGuard guard(h->cfg.device);
  const cudaStream_t s = static_cast<cudaStream_t>(io->stream);
  return io->count <= clip::FEW    ? run<clip::FEW>(h, io, scales, s)
         : io->count <= clip::SOME ? run<clip::SOME>(h, io, scales, s)
                                   : run<clip::MANY>(h, io, scales, s);
}

}  // namespace

extern "C" {

apk_status apk_clip_create(const apk_clip_config* cfg, apk_clip** out) { return ops::make(cfg, out, create); }

apk_status apk_clip_destroy(apk_clip* h) {
  delete h;
  return APK_OK;
}

const char* apk_clip_last_error(const apk_clip* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_clip_norm(apk_clip* h, const apk_clip_io* io) {
  return ops::call(h, io, [&] { return run(h, io, false); });
}

apk_status apk_clip_scale(apk_clip* h, const apk_clip_io* io) {
  return ops::call(h, io, [&] { return run(h, io, true); });
}

}  // extern "C"
