// Device helpers shared by norm.cu, clip.cu, logprobs.cu and linear4.cu:
// pieces of 8 elements, fp32 or bf16, and sums over warps.
#pragma once
#include <stdint.h>

#include "common.cuh"

namespace apk {
namespace ops {

__device__ __forceinline__ float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint16_t to_bf16(float v) {
  uint16_t r;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float ld_any(const void* p, long long i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : bf_lo(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void st_any(void* p, long long i, float v, bool f32) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = to_bf16(v);
}

// Eight elements as they lie in memory.
template <bool F32>
struct Raw;
template <>
struct Raw<false> {
  uint4 a;
};
template <>
struct Raw<true> {
  uint4 a, b;
};

__device__ __forceinline__ void unpack(const Raw<false>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf_lo(w[i]);
    v[2 * i + 1] = bf_hi(w[i]);
  }
}
__device__ __forceinline__ void unpack(const Raw<true>& r, float (&v)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw<false>& r) {
  r.a = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw<true>& r) {
  r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  r.b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}
// (ordinary loads, which stay behind pdl_wait; read once, so evicted first)
__device__ __forceinline__ void ld8(const void* p, long long i, Raw<false>& r) {
  r.a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
}
__device__ __forceinline__ void ld8(const void* p, long long i, Raw<true>& r) {
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
  r.a = __ldcs(q);
  r.b = __ldcs(q + 1);
}
__device__ __forceinline__ void st8(void* p, long long i, const Raw<false>& r) {
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = r.a;
}
__device__ __forceinline__ void st8(void* p, long long i, const Raw<true>& r) {
  uint4* q = reinterpret_cast<uint4*>(static_cast<float*>(p) + i);
  q[0] = r.a;
  q[1] = r.b;
}
// One element of eight, for rows that 16-byte pieces cannot address.
__device__ __forceinline__ void set1(Raw<false>& r, int i, const void* p, long long at) {
  const uint32_t v = static_cast<const uint16_t*>(p)[at];
  uint32_t& w = (&r.a.x)[i >> 1];
  w = (i & 1) ? (w & 0xFFFFu) | v << 16 : (w & 0xFFFF0000u) | v;
}
__device__ __forceinline__ void set1(Raw<true>& r, int i, const void* p, long long at) {
  (&(i < 4 ? r.a : r.b).x)[i & 3] = static_cast<const uint32_t*>(p)[at];
}

// Pairs of fp32 values, for instructions that take two at once.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pair2(v, v); }
__device__ __forceinline__ void unpair2(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ float sum2(f32x2 v) {
  float lo, hi;
  unpair2(v, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void unpack2(const Raw<false>& r, f32x2 (&v)[4]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pair2(bf_lo(w[i]), bf_hi(w[i]));
}
__device__ __forceinline__ void unpack2(const Raw<true>& r, f32x2 (&v)[4]) {
  float f[8];
  unpack(r, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pair2(f[2 * i], f[2 * i + 1]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

}  // namespace ops
}  // namespace apk
