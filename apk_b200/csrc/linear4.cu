// A linear layer with 4-bit weights and group scales (apk_linear4_* of
// include/apk.h).  No counterpart in the reference, which multiplies bare
// matrices (src/tcyield.cu:91-356).
//
//   W[n][k] = s[n][k / G] (q[n][k] - z[n][k / G]),  y = act(x W^T + b) + r
//
// Few rows are bound by reading the weights: they go from global memory
// straight into the A fragments of mma.m16n8k16, as in stream.cuh, the
// weights' rows on its M axis.  A nibble becomes a bf16 by an or: 0x4300 | q
// is 128 + q, and (128 + q) - (128 + z) is exact.  The scales are applied to
// a group's sums in fp32, so that weights are not rounded.
//
// A fragment's k order is free as long as A and B agree.  Of a 32-bit word's
// eight weights, shifts by 4 i yield the pairs (i, i + 4); B's values, eight
// contiguous ones of x, are put in the same order by four byte permutes.
//
// Many rows take the tensor cores' products (linear_gemm.cu) of weights that
// are written out as bf16 first.
#include <algorithm>

#include "act.cuh"
#include "common.cuh"
#include "ops.cuh"
#include "ops.h"
#include "stream.cuh"

namespace apk {
namespace lin4 {

struct Params {
  const uint16_t* x;
  const uint8_t* w;
  const void* s;
  const uint8_t* z;
  long long ldx, ldw;
  int rows, n, k, group, groups, split, s_f32;
  lin::Epilogue epi;
};

constexpr int WARPS = 8, FT = 16, CHUNK = 128;

// Eight weights less their zero point: h[i] is the pair (i, i + 4).
__device__ __forceinline__ void dequant(uint32_t w, uint32_t zero, uint32_t (&h)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(h[i]) : "r"(v), "r"(zero));
  }
}
// Eight values of x in the same order.
__device__ __forceinline__ void pairs(const uint4& v, uint32_t (&h)[4]) {
  h[0] = __byte_perm(v.x, v.z, 0x5410);
  h[1] = __byte_perm(v.x, v.z, 0x7632);
  h[2] = __byte_perm(v.y, v.w, 0x5410);
  h[3] = __byte_perm(v.y, v.w, 0x7632);
}
// 128 + z twice
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) { return 0x43004300u | (z & 15u) * 0x00010001u; }

// P: groups that a chunk of 128 k has (1 for groups of 128 and more).  A
// warp's lane (g, t) holds weights of the features g and g + 8; a group's
// 32 / P k-values of a lane lie together.
template <int NT8, int P, bool ZEROS, bool VEC>
__global__ void __launch_bounds__(32 * WARPS, 2) stream4(const __grid_constant__ Params p) {
  constexpr int TOK = 8 * NT8, WORDS = 4 / P;  // 32-bit words of a lane and group
  __shared__ float part[WARPS][TOK][FT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = (int)blockIdx.x % p.split;
  const int f0 = (int)blockIdx.x / p.split * FT, r0 = blockIdx.y * TOK;
  const int rows = p.rows - r0;
  pdl_launch();
  pdl_wait();
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.x + (r0 + min(8 * i + g, rows - 1)) * p.ldx;
  const int f[2] = {min(f0 + g, p.n - 1), min(f0 + g + 8, p.n - 1)};
  float total[NT8][4] = {};
#pragma unroll 1
  for (int k0 = (rank * WARPS + warp) * CHUNK; k0 < p.k; k0 += p.split * WARPS * CHUNK) {
    uint32_t w[2][4];
    uint4 c[NT8][4];
    float s[2];
    uint32_t z[2] = {8, 8};
#pragma unroll
    for (int h = 0; h < P; ++h) {
      const int k = k0 + h * (CHUNK / P) + t * (32 / P);
      const bool in = k < p.k;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* q = p.w + f[m] * p.ldw + k / 2;
        if constexpr (P == 1) {
          const uint4 v = in ? stream::ld_late(q) : make_uint4(0, 0, 0, 0);
          w[m][0] = v.x, w[m][1] = v.y, w[m][2] = v.z, w[m][3] = v.w;
        } else if constexpr (P == 2) {
          const uint2 v = in ? stream::ld_late8(q) : make_uint2(0, 0);
          w[m][2 * h] = v.x, w[m][2 * h + 1] = v.y;
        } else {
          w[m][h] = in ? *reinterpret_cast<const uint32_t*>(q) : 0u;
        }
      }
#pragma unroll
      for (int j = 0; j < WORDS; ++j)
#pragma unroll
        for (int i = 0; i < NT8; ++i) {
          uint4& v = c[i][h * WORDS + j];
          if (VEC) v = in ? stream::ld_rows(xr[i] + k + 8 * j) : make_uint4(0, 0, 0, 0);
          else v = stream::ld8_any(xr[i] + k + 8 * j, p.k - k - 8 * j);
        }
    }
    {  // lane t has the chunk's t-th group's scale and zero point (with fewer groups: of one of them)
      const int k = k0 + (t & (P - 1)) * (CHUNK / P);
      const int at = k / p.group;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const long long i = (long long)f[m] * p.groups + at;
        s[m] = k < p.k ? ops::ld_any(p.s, i, p.s_f32) : 0.f;
        if (ZEROS) z[m] = k < p.k ? p.z[i] : 0;
      }
    }
#pragma unroll
    for (int h = 0; h < P; ++h) {
      float acc[NT8][4] = {};
      float sh[2];
      uint32_t zh[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        sh[m] = P == 1 ? s[m] : __shfl_sync(0xFFFFFFFFu, s[m], (lane & ~3) | h);
        zh[m] = zero_pair(P == 1 || !ZEROS ? z[m] : __shfl_sync(0xFFFFFFFFu, z[m], (lane & ~3) | h));
      }
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        uint32_t a[4], b[4];
        dequant(w[0][h * WORDS + j], zh[0], a);
        dequant(w[1][h * WORDS + j], zh[1], b);
#pragma unroll
        for (int i = 0; i < NT8; ++i) {
          uint32_t x[4];
          pairs(c[i][h * WORDS + j], x);
          stream::mma_bf16(acc[i], a[0], b[0], a[1], b[1], x[0], x[1]);
          stream::mma_bf16(acc[i], a[2], b[2], a[3], b[3], x[2], x[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT8; ++i) {
        total[i][0] = fmaf(sh[0], acc[i][0], total[i][0]);
        total[i][1] = fmaf(sh[0], acc[i][1], total[i][1]);
        total[i][2] = fmaf(sh[1], acc[i][2], total[i][2]);
        total[i][3] = fmaf(sh[1], acc[i][3], total[i][3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[warp][8 * i + 2 * t + (j & 1)][g + 8 * (j >> 1)] = total[i][j];
  __syncthreads();
  if (p.split > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int o = rank * 32 * WARPS + tid; o < TOK * FT; o += p.split * 32 * WARPS) {
    const int tok = o / FT, c = o % FT;
    if (tok >= rows || f0 + c >= p.n) continue;
    float y = 0.f;
    if (p.split == 1) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) y += part[w][tok][c];
    } else {
      for (int r = 0; r < p.split; ++r) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&part[0][tok][c])), "r"(r));
        float v[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[w]) : "r"(at + w * (uint32_t)(TOK * FT * 4)) : "memory");
#pragma unroll
        for (int w = 0; w < WARPS; ++w) y += v[w];
      }
    }
    const lin::Epilogue& e = p.epi;
    const long long row = r0 + tok, col = f0 + c;
    if (e.bias) y += ops::ld_any(e.bias, col, e.bias_f32);
    const float res = e.res ? ops::ld_any(e.res, row * e.ld_res + col, e.res_f32) : 0.f;
    if (e.pre) ops::st_any(e.pre, row * e.ld_pre + col, y, false);
    with_act(e.act, [&](auto a) { ops::st_any(e.out, row * e.ld_out + col, act_f<decltype(a)::value>(y) + res, e.out_f32); });
  }
  if (p.split > 1) {  // no read reaches a CTA that has left
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// The weights as bf16, [n][ld]; with `low` also what that rounds away, in the
// next k columns, and x twice beside each other to go with it.
struct Expand {
  const uint8_t* w;
  const void* s;
  const uint8_t* z;
  uint16_t* out;
  const uint16_t* x;
  uint16_t* xx;
  long long ldw, ldx;
  int n, k, group, groups, s_f32, low, rows;
};
__global__ void __launch_bounds__(256) expand(const __grid_constant__ Expand p) {
  pdl_launch();
  pdl_wait();
  const int per = p.k / 32;  // a thread's piece
  const long long ld = p.low ? 2ll * p.k : p.k;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)p.n * per; i += (long long)gridDim.x * 256) {
    const int f = (int)(i / per), k = (int)(i - (long long)f * per) * 32;
    const long long at = (long long)f * p.groups + k / p.group;
    const float s = ops::ld_any(p.s, at, p.s_f32), z = p.z ? (float)(p.z[at] & 15) : 8.f;
    const uint4 v = stream::ld_late(p.w + f * p.ldw + k / 2);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint4* o = reinterpret_cast<uint4*>(p.out + f * ld + k);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = s * ((float)(w[j] >> (4 * e) & 15u) - z);
      ops::Raw<false> r;
      ops::pack(q, r);
      o[j] = r.a;
      if (p.low) {
        float hi[8];
        ops::unpack(r, hi);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] -= hi[e];
        ops::pack(q, r);
        reinterpret_cast<uint4*>(p.out + f * ld + p.k + k)[j] = r.a;
      }
    }
  }
  if (!p.xx) return;
  const int eights = p.k / 8;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)p.rows * eights; i += (long long)gridDim.x * 256) {
    const long long r = i / eights;
    const int k = (int)(i - r * eights) * 8;
    const uint4 v = stream::ld8_any(p.x + r * p.ldx + k, 8);
    *reinterpret_cast<uint4*>(p.xx + r * ld + k) = v;
    if (p.low) *reinterpret_cast<uint4*>(p.xx + r * ld + p.k + k) = v;
  }
}

template <int NT8, int P>
const void* fn(bool zeros, bool vec) {
  return zeros ? (vec ? reinterpret_cast<const void*>(&stream4<NT8, P, true, true>)
                      : reinterpret_cast<const void*>(&stream4<NT8, P, true, false>))
               : (vec ? reinterpret_cast<const void*>(&stream4<NT8, P, false, true>)
                      : reinterpret_cast<const void*>(&stream4<NT8, P, false, false>));
}
template <int NT8>
const void* fn(int group, bool zeros, bool vec) {
  return group == 32 ? fn<NT8, 4>(zeros, vec) : group == 64 ? fn<NT8, 2>(zeros, vec) : fn<NT8, 1>(zeros, vec);
}

}  // namespace lin4
}  // namespace apk

using namespace apk;

struct apk_linear4 {
  apk_linear4_config cfg{};
  Err err;
  int sms = 0;
  Scratch scratch;
  std::mutex mu;
};

namespace {

apk_status create(const apk_linear4_config* cfg, apk_linear4* h) {
  h->cfg = *cfg;
  const apk_linear4_config& c = h->cfg;
  if (c.in_features < 32 || c.out_features < 1 || c.in_features > ops::MAX_SIZE || c.out_features > ops::MAX_SIZE)
    return h->err.fail(APK_EINVAL, "in_features %d, out_features %d: 32 or 1 to 2^30", c.in_features, c.out_features);
  if (c.in_features % 32) return h->err.fail(APK_EINVAL, "in_features %d is not a multiple of 32", c.in_features);
  if (c.group != 32 && c.group != 64 && (c.group < 128 || c.group % 128))
    return h->err.fail(APK_EINVAL, "group is %d: 32, 64 or a multiple of 128", c.group);
  if (c.act < APK_ACT_NONE || c.act > APK_ACT_SILU) return h->err.fail(APK_EINVAL, "act %d", (int)c.act);
  if (!c.W || !c.scales) return h->err.fail(APK_EINVAL, "W or scales is NULL");
  if (c.ldw < c.in_features / 2 || c.ldw % 16 || !ops::aligned(c.W, 16))
    return h->err.fail(APK_EINVAL, "W's rows have to start on 16 bytes and not overlap (ldw %lld)", c.ldw);
  if (!ops::valid_dtype(c.scale_dtype) || (c.bias && !ops::valid_dtype(c.bias_dtype)))
    return h->err.fail(APK_EINVAL, "scale_dtype %d, bias_dtype %d", (int)c.scale_dtype, (int)c.bias_dtype);
  if (!ops::aligned(c.scales, ops::esize(c.scale_dtype)) || (c.bias && !ops::aligned(c.bias, ops::esize(c.bias_dtype))))
    return h->err.fail(APK_EINVAL, "scales or bias is not aligned to its element");
  if (c.wait_limit_ns < 0) return h->err.fail(APK_EINVAL, "wait_limit_ns is negative");
  if (c.wait_limit_ns == 0) h->cfg.wait_limit_ns = 2000000000ll;
  int sms = 0;
  APK_TRY(ops::open_device(c.device, &sms, &h->err));
  if (c.sms < 0 || c.sms > sms) return h->err.fail(APK_EINVAL, "sms %d of %d", c.sms, sms);
  h->sms = c.sms ? c.sms : sms;
  DeviceGuard guard(c.device);
  APK_TRY(cu_status(lin::prepare(), "preparing the linear kernels", &h->err));
  return h->scratch.open(c.device, &h->err);
}

// Rows up to here stream the weights, 16 rows at a time.
constexpr int STREAM_ROWS = 64;

apk_status stream(apk_linear4* h, const apk_linear_io* io, const lin::Epilogue& epi) {
  const apk_linear4_config& c = h->cfg;
  lin4::Params p{};
  p.x = static_cast<const uint16_t*>(io->x);
  p.w = static_cast<const uint8_t*>(c.W);
  p.s = c.scales;
  p.z = c.zeros;
  p.ldx = io->ldx;
  p.ldw = c.ldw;
  p.rows = io->rows;
  p.n = c.out_features;
  p.k = c.in_features;
  p.group = c.group;
  p.groups = ops::ceil_div(c.in_features, c.group);
  p.s_f32 = c.scale_dtype == APK_F32;
  p.epi = epi;
  const bool vec = ops::on16(io->x, io->ldx, io->rows, APK_BF16);
  const int nt = io->rows <= 8 ? 1 : 2;
  const int tiles = ops::ceil_div(p.n, lin4::FT), blocks = ops::ceil_div(p.rows, 8 * nt);
  // split K while every warp keeps a chunk and the blocks do not exceed two an SM
  p.split = 1;
  while (p.split < 8 && 2 * p.split * tiles * blocks <= 2 * h->sms && 2 * p.split * lin4::WARPS * lin4::CHUNK <= p.k) p.split *= 2;
  const void* f = nt == 1 ? lin4::fn<1>(c.group, c.zeros, vec) : lin4::fn<2>(c.group, c.zeros, vec);
  Launch l(dim3(tiles * p.split, blocks), 32 * lin4::WARPS, 0, static_cast<cudaStream_t>(io->stream), p.split);
  void* args[] = {&p};
  return cu_status(cudaLaunchKernelExC(&l.cfg, f, args), "launching the 4-bit product", &h->err);
}

apk_status forward(apk_linear4* h, const apk_linear_io* io) {
  const apk_linear4_config& c = h->cfg;
  const int K = c.in_features, N = c.out_features, M = io->rows;
  const cudaStream_t s = static_cast<cudaStream_t>(io->stream);
  if (M < 0 || M > ops::MAX_SIZE) return h->err.fail(APK_EINVAL, "rows is %d: at most 2^30", M);
  if (M == 0) return APK_OK;
  if (!io->x || !io->y) return h->err.fail(APK_EINVAL, "x or y is NULL");
  if (!ops::valid_dtype(io->y_dtype) || (io->residual && !ops::valid_dtype(io->residual_dtype)))
    return h->err.fail(APK_EINVAL, "y_dtype %d, residual_dtype %d", (int)io->y_dtype, (int)io->residual_dtype);
  if (io->ldx < K || io->ldy < N || (io->residual && io->ld_residual < N) || (io->preact && io->ld_preact < N))
    return h->err.fail(APK_EINVAL, "a row stride is below its row: ldx %lld, ldy %lld, ld_residual %lld, ld_preact %lld",
                       io->ldx, io->ldy, io->ld_residual, io->ld_preact);
  if (!ops::aligned(io->x, 2) || !ops::aligned(io->y, ops::esize(io->y_dtype)) ||
      (io->residual && !ops::aligned(io->residual, ops::esize(io->residual_dtype))) || !ops::aligned(io->preact, 2))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element");
  DeviceGuard guard(c.device);
  const lin::Epilogue epi = {c.bias, io->residual, io->y, io->preact, io->ld_residual, io->ldy, io->ld_preact,
                             c.bias_dtype == APK_F32, io->residual_dtype == APK_F32, io->y_dtype == APK_F32, c.act};
  if (M <= STREAM_ROWS) return stream(h, io, epi);
  // fp32 results keep the weights as two bf16 terms: K is twice as long
  const bool low = io->y_dtype == APK_F32, copy = low || !ops::on16(io->x, io->ldx, M, APK_BF16);
  if (low && K > ops::MAX_SIZE / 2) return h->err.fail(APK_EINVAL, "an fp32 result of %d features: at most 2^29", K);
  const long long ld = low ? 2ll * K : K;
  APK_TRY(h->scratch.enter(s, &h->err));
  ScratchUse use(&h->scratch, &h->err);
  const size_t bw = ops::up256((size_t)N * ld * 2), bx = copy ? ops::up256((size_t)M * ld * 2) : 0;
  APK_TRY(use.begin(bw + bx, 0));
  lin4::Expand e{};
  e.w = static_cast<const uint8_t*>(c.W);
  e.s = c.scales;
  e.z = c.zeros;
  e.out = reinterpret_cast<uint16_t*>(h->scratch.data());
  e.x = static_cast<const uint16_t*>(io->x);
  e.xx = copy ? reinterpret_cast<uint16_t*>(h->scratch.data() + bw) : nullptr;
  e.ldw = c.ldw;
  e.ldx = io->ldx;
  e.n = N;
  e.k = K;
  e.group = c.group;
  e.groups = ops::ceil_div(K, c.group);
  e.s_f32 = c.scale_dtype == APK_F32;
  e.low = low;
  e.rows = M;
  const long long pieces = std::max<long long>((long long)N * (K / 32), copy ? (long long)M * (K / 8) : 0);
  Launch l(dim3((unsigned)std::min<long long>(ops::ceil_div(pieces, 256ll), h->sms * 8)), 256, 0, s);
  APK_TRY(cu_status(cudaLaunchKernelEx(&l.cfg, lin4::expand, e), "launching the weights' expansion", &h->err));
  lin::Product p{};
  p.P = {e.out, ld, N, (int)ld, false};
  p.Q = {copy ? (const void*)e.xx : io->x, copy ? ld : io->ldx, M, (int)ld, false};
  p.rows = M;
  p.cols = N;
  p.k = (int)ld;
  p.epi = epi;
  APK_TRY(lin::run_products(&p, 1, h->sms, c.device, h->scratch.status(), c.wait_limit_ns, s, &h->err.text));
  return use.end();
}

}  // namespace

extern "C" {

apk_status apk_linear4_create(const apk_linear4_config* cfg, apk_linear4** out) { return ops::make(cfg, out, create); }

apk_status apk_linear4_destroy(apk_linear4* h) {
  delete h;
  return APK_OK;
}

const char* apk_linear4_last_error(const apk_linear4* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_linear4_forward(apk_linear4* h, const apk_linear_io* io) {
  return ops::call(h, io, [&] { return forward(h, io); });
}

apk_status apk_linear4_status(apk_linear4* h, void* stream, int* device_status) {
  return ops::call(h, device_status, [&] {
    DeviceGuard guard(h->cfg.device);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    APK_TRY(cu_status(cudaMemcpyAsync(device_status, h->scratch.status(), sizeof(int), cudaMemcpyDeviceToHost, s), "status copy",
                      &h->err));
    APK_TRY(cu_status(cudaMemsetAsync(h->scratch.status(), 0, sizeof(int), s), "status clear", &h->err));
    return cu_status(cudaStreamSynchronize(s), "cudaStreamSynchronize", &h->err);
  });
}

}  // extern "C"
