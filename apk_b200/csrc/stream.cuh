// Products of a few rows with weights that are read once: the weights go
// from global memory straight into the A fragments of mma.m16n8k16 (the
// weights' rows are the MMA's M axis, the tokens its N axis), with no shared
// memory, barrier or descriptor between.  Such a product is bound by reading
// the weights, and its latency by what stands before the first load; the
// tensor pipe's rate does not matter.
//
// A fragment's k order is free as long as A and B agree, so a thread loads 16
// (8) contiguous bytes and deals them over the fragments:
//   [feature][k] weights: lane (g, t) holds features g and g + 8 at k = 8t..8t+7
//     of 32, two MMAs; its B values are token g at the same k.
//   [k][feature] weights: lane (g, t) holds features 4g..4g+3 of 32 at the
//     rows k = 4t..4t+3 of 16; byte permutes pair two rows into the two MMAs'
//     A registers.
#pragma once
#include <stdint.h>

namespace apk {
namespace stream {

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are read once by one SM: not kept in L1.  Through the read-only path:
// for a kernel that starts after whatever wrote them has ended.
__device__ __forceinline__ uint4 ld_weights(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The same for a kernel that may start while its predecessor still writes them
// (pdl_wait stands between): ordinary loads, which stay behind the wait.
__device__ __forceinline__ uint4 ld_late(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_late8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
// The few rows of the other operand, kept in L1.
__device__ __forceinline__ uint4 ld_rows(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_rows8(const void* p) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}

// The first n of 8 elements from p, the others zero, at any alignment.
__device__ __forceinline__ uint4 ld8_any(const uint16_t* p, int n) {
  union {
    uint16_t h[8];
    uint4 v;
  } u;
#pragma unroll
  for (int i = 0; i < 8; ++i) u.h[i] = i < n ? p[i] : (uint16_t)0;
  return u.v;
}
__device__ __forceinline__ uint2 ld4_any(const uint16_t* p, int n) {
  union {
    uint16_t h[4];
    uint2 v;
  } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.h[i] = i < n ? p[i] : (uint16_t)0;
  return u.v;
}

}  // namespace stream
}  // namespace apk
