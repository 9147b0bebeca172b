// The linear layer for up to 16 rows (decoding): weights streamed once from
// global memory into MMA fragments (stream.cuh).
//
// A CTA owns 16 output columns ([N][K] weights, 16 warps) or 32 ([K][N]:
// 64-byte row pieces, 8 warps) and splits K over its warps in chunks of 128 (64); a
// cluster of 2, 4 or 8 CTAs splits it further where the columns alone give
// too few CTAs.  The warps' partial sums meet in shared memory and are added
// in the order of (CTA rank, warp): the result does not depend on timing.
// Rows past the last and columns past the last are computed from the last
// one's data and not stored.
#include <algorithm>

#include "act.cuh"
#include "common.cuh"
#include "linear.h"
#include "stream.cuh"

namespace apk {
namespace lin {

struct StreamParams {
  const uint16_t* x;
  const uint16_t* w;
  long long ldx, ldw;
  int rows, n, k, split;
  Epilogue epi;
};

namespace {

template <bool NK>
constexpr int WARPS_OF = NK ? 16 : 8;
template <bool NK>
constexpr int FEATURES = NK ? 16 : 32;
template <bool NK>
constexpr int CHUNK = NK ? 128 : 64;  // k of one warp's round: 128 bytes a lane

__device__ __forceinline__ float ld_epi(const void* p, long long i, int f32) {
  return f32 ? static_cast<const float*>(p)[i]
             : __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
__device__ __forceinline__ void st_epi(void* p, long long i, float v, int f32) {
  if (f32) {
    static_cast<float*>(p)[i] = v;
  } else {
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
    static_cast<uint16_t*>(p)[i] = r;
  }
}

// The tensor core truncates as it adds, a bias that grows with the length of
// the chain (1e-6 of the result at 1024 k): every FLUSH k a warp adds its sum
// to a total with rounding.
constexpr int FLUSH = 512;
template <int N>
__device__ __forceinline__ void flush(float (&acc)[N][4], float (&total)[N][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      total[i][j] += acc[i][j];
      acc[i][j] = 0.f;
    }
}

// LONG: a warp's share of K exceeds FLUSH.
template <bool NK, int NT8, bool VEC, bool LONG>
__global__ void __launch_bounds__(32 * WARPS_OF<NK>, NT8 == 1 && VEC ? (NK ? 2 : 3) : NK ? 1 : VEC ? 3 : 2)
lin_stream(const __grid_constant__ StreamParams p) {
  constexpr int WARPS = WARPS_OF<NK>;
  constexpr int FT = FEATURES<NK>, KC = CHUNK<NK>, TOK = 8 * NT8;
  __shared__ float part[WARPS][TOK][FT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = (int)blockIdx.x % p.split;
  const int f0 = (int)blockIdx.x / p.split * FT;
  pdl_launch();
  pdl_wait();
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.x + min(8 * i + g, p.rows - 1) * p.ldx;

  if constexpr (NK) {
    float acc[NT8][4] = {}, total[NT8][4] = {};
    int round = 0;
    const uint16_t* w0 = p.w + min(f0 + g, p.n - 1) * p.ldw;
    const uint16_t* w1 = p.w + min(f0 + g + 8, p.n - 1) * p.ldw;
#pragma unroll 1
    for (int k0 = (rank * WARPS + warp) * KC; k0 < p.k; k0 += p.split * WARPS * KC) {
      uint4 a[4], b[4], c[NT8][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = k0 + 32 * u + 8 * t;
        if (VEC) {
          const uint4 zero = make_uint4(0, 0, 0, 0);
          const bool in = k < p.k;
          a[u] = in ? stream::ld_late(w0 + k) : zero;
          b[u] = in ? stream::ld_late(w1 + k) : zero;
#pragma unroll
          for (int i = 0; i < NT8; ++i) c[i][u] = in ? stream::ld_rows(xr[i] + k) : zero;
        } else {
          a[u] = stream::ld8_any(w0 + k, p.k - k);
          b[u] = stream::ld8_any(w1 + k, p.k - k);
#pragma unroll
          for (int i = 0; i < NT8; ++i) c[i][u] = stream::ld8_any(xr[i] + k, p.k - k);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < NT8; ++i) {
          stream::mma_bf16(acc[i], a[u].x, b[u].x, a[u].y, b[u].y, c[i][u].x, c[i][u].y);
          stream::mma_bf16(acc[i], a[u].z, b[u].z, a[u].w, b[u].w, c[i][u].z, c[i][u].w);
        }
      if (LONG && (++round & (FLUSH / KC - 1)) == 0) flush(acc, total);
    }
    flush(acc, total);
#pragma unroll
    for (int i = 0; i < NT8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[warp][8 * i + 2 * t + (j & 1)][g + 8 * (j >> 1)] = total[i][j];
  } else {
    float acc[2][NT8][4] = {}, total[2][NT8][4] = {};
    int round = 0;
    const int f = f0 + 4 * g;
    const uint16_t* w = p.w + (VEC ? min(f, p.n - 4) : f);
#pragma unroll 1
    for (int k0 = (rank * WARPS + warp) * KC; k0 < p.k; k0 += p.split * WARPS * KC) {
      constexpr int U = KC / 16;
      uint2 a[U][4], c[U][NT8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + 16 * u + 4 * t;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = k + r < p.k;
          if (VEC) a[u][r] = in ? stream::ld_late8(w + (long long)(k + r) * p.ldw) : make_uint2(0, 0);
          else a[u][r] = stream::ld4_any(w + (long long)(k + r) * p.ldw, in ? p.n - f : 0);
        }
#pragma unroll
        for (int i = 0; i < NT8; ++i) {
          if (VEC) c[u][i] = k < p.k ? stream::ld_rows8(xr[i] + k) : make_uint2(0, 0);
          else c[u][i] = stream::ld4_any(xr[i] + k, p.k - k);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint32_t r0 = m ? a[u][0].y : a[u][0].x, r1 = m ? a[u][1].y : a[u][1].x;
          const uint32_t r2 = m ? a[u][2].y : a[u][2].x, r3 = m ? a[u][3].y : a[u][3].x;
          const uint32_t a0 = __byte_perm(r0, r1, 0x5410), a1 = __byte_perm(r0, r1, 0x7632);
          const uint32_t a2 = __byte_perm(r2, r3, 0x5410), a3 = __byte_perm(r2, r3, 0x7632);
#pragma unroll
          for (int i = 0; i < NT8; ++i) stream::mma_bf16(acc[m][i], a0, a1, a2, a3, c[u][i].x, c[u][i].y);
        }
      if (LONG && (++round & (FLUSH / KC - 1)) == 0)
#pragma unroll
        for (int m = 0; m < 2; ++m) flush(acc[m], total[m]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) flush(acc[m], total[m]);
    // MMA m's rows g and g + 8 are the features 4g + 2m and 4g + 2m + 1
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < NT8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          part[warp][8 * i + 2 * t + (j & 1)][4 * g + 2 * m + (j >> 1)] = total[m][i][j];
  }
  __syncthreads();
  if (p.split > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int o = rank * 32 * WARPS + tid; o < TOK * FT; o += p.split * 32 * WARPS) {
    const int tok = o / FT, f = o % FT;
    if (tok >= p.rows || f0 + f >= p.n) continue;
    float z = 0.f;
    if (p.split == 1) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) z += part[w][tok][f];
    } else {
      for (int r = 0; r < p.split; ++r) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&part[0][tok][f])), "r"(r));
        float v[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[w]) : "r"(at + w * (uint32_t)(TOK * FT * 4)) : "memory");
#pragma unroll
        for (int w = 0; w < WARPS; ++w) z += v[w];
      }
    }
    const Epilogue& e = p.epi;
    const long long c = f0 + f;
    if (e.bias) z += ld_epi(e.bias, c, e.bias_f32);
    const float res = e.res ? ld_epi(e.res, tok * e.ld_res + c, e.res_f32) : 0.f;
    if (e.pre) st_epi(e.pre, tok * e.ld_pre + c, z, 0);
    with_act(e.act, [&](auto a) { st_epi(e.out, tok * e.ld_out + c, act_f<decltype(a)::value>(z) + res, e.out_f32); });
  }
  if (p.split > 1) {  // no read reaches a CTA that has left
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

template <bool NK, int NT8, bool VEC>
const void* fn(bool longer) {
  return longer ? reinterpret_cast<const void*>(&lin_stream<NK, NT8, VEC, true>)
                : reinterpret_cast<const void*>(&lin_stream<NK, NT8, VEC, false>);
}

}  // namespace

cudaError_t run_stream(const void* x, long long ldx, const void* w, long long ldw, bool nk, int rows, int n, int k,
                       const Epilogue& epi, int sms, cudaStream_t stream) {
  StreamParams p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(w), ldx, ldw, rows, n, k, 1, epi};
  auto a16 = [](const void* q, long long ld) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && ld % 8 == 0; };
  const bool vec = k % 8 == 0 && (nk || n % 8 == 0) && a16(w, ldw) && (a16(x, ldx) || (rows == 1 && a16(x, 8)));
  const int nt = rows <= 8 ? 1 : 2;
  const int ft = nk ? FEATURES<true> : FEATURES<false>, kc = nk ? CHUNK<true> : CHUNK<false>;
  const int warps = nk ? WARPS_OF<true> : WARPS_OF<false>;
  const int tiles = (n + ft - 1) / ft;
  // split K while a round of every warp remains and the CTAs do not exceed two per SM
  while (p.split < 8 && 2 * p.split * tiles <= 2 * sms && 2 * p.split * warps * kc <= k) p.split *= 2;
  const int round = p.split * warps * kc;
  const bool longer = (k + round - 1) / round * kc > FLUSH;
  const void* f = nk ? (nt == 1 ? (vec ? fn<true, 1, true>(longer) : fn<true, 1, false>(longer))
                                : (vec ? fn<true, 2, true>(longer) : fn<true, 2, false>(longer)))
                     : (nt == 1 ? (vec ? fn<false, 1, true>(longer) : fn<false, 1, false>(longer))
                                : (vec ? fn<false, 2, true>(longer) : fn<false, 2, false>(longer)));
  Launch l(dim3(tiles * p.split), 32 * warps, 0, stream, p.split);
  void* args[] = {&p};
  return cudaLaunchKernelExC(&l.cfg, f, args);
}

}  // namespace lin
}  // namespace apk
