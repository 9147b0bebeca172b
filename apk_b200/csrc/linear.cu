// A linear layer, y = act(x W + b) + r, and its gradients (apk_linear_* of
// include/apk.h): argument checks, scratch, and the two memory-bound kernels
// around the products of linear_gemm.cu.  No reference counterpart: the
// reference multiplies bare matrices (src/tcyield.cu:91-356).
#include <algorithm>
#include <mutex>
#include <new>

#include "act.cuh"
#include "common.cuh"
#include "linear.h"

namespace apk {

namespace lin {

__device__ __forceinline__ uint16_t f2bf(float v) {
  uint16_t r;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
  return r;
}

// Copies operands whose base or row stride is not a multiple of 16 bytes (TMA
// cannot address them) to rows of ld elements, ld a multiple of 8.  One
// thread per 8 elements.
struct Repack {
  const uint16_t* src;
  uint16_t* dst;
  long long lds;
  int rows, cols, ld;
  long long first;  // chunk index of this operand's first chunk
};
struct RepackParams {
  Repack op[2];
  int n;
  long long chunks;
};
__device__ __forceinline__ void repack_block(const RepackParams& p, int block, int blocks) {
  for (long long i = (long long)block * 256 + threadIdx.x; i < p.chunks; i += (long long)blocks * 256) {
    const Repack& o = p.op[p.n > 1 && i >= p.op[1].first ? 1 : 0];
    const long long at = i - o.first;
    const int per = o.ld / 8;
    const long long r = at / per;
    const int c = (int)(at - r * per) * 8;
    union {
      uint16_t h[8];
      uint4 v;
    } u;
    const uint16_t* s = o.src + r * o.lds + c;
#pragma unroll
    for (int j = 0; j < 8; ++j) u.h[j] = c + j < o.cols ? s[j] : (uint16_t)0;
    *reinterpret_cast<uint4*>(o.dst + r * o.ld + c) = u.v;
  }
}
__global__ void __launch_bounds__(256) repack(const __grid_constant__ RepackParams p) {
  pdl_launch();
  pdl_wait();
  repack_block(p, blockIdx.x, gridDim.x);
}

struct DzParams {
  const uint16_t* dy;
  const uint16_t* z;  // null: no activation
  uint16_t* dz;       // null: not wanted (it is dy)
  void* db;           // null: no bias
  float* part;        // [row blocks][cols rounded up to 8] partial column sums
  unsigned* count;    // one per column block, zero between launches
  long long ld_dy, ld_z, ld_dz;
  int rows, cols, rows_per_block, act, db_f32;
  int cblocks, rblocks;  // column ranges, row ranges; further blocks repack
};

constexpr int DZ_COLS = 256;  // columns of a block: 8 per lane
constexpr int DZ_BLOCKS = 4;  // of an SM

// dz = dy * act'(z), rounded to bf16 (the products' operand type), and the
// column sums of the unrounded dz.  One pass over dy and z.  A block sums its
// rows in registers and shared memory; the last block of a column range adds
// the row blocks' sums in their order, so db does not depend on the order of
// arrival.  VEC: rows of 16-byte aligned 8-element chunks.  The grid is one
// residency of four blocks an SM (64 registers), rounded down.  4096 x 8192
// with gelu_tanh, no dz: 34.0 us; rounded up, the 16 blocks over ran alone, 42.8;
// five blocks an SM at 48 registers, with spills, 35.4 in one residency and
// 40.0 with places left empty.  With dx of 256 columns behind it: 71, 84, 70, 75.
// Blocks past the first cblocks * rblocks copy operands for the products that
// follow (one launch for both).
template <bool VEC>
__global__ void __launch_bounds__(256, DZ_BLOCKS) dz_kernel(const __grid_constant__ DzParams p,
                                                         const __grid_constant__ RepackParams copies) {
  __shared__ float sum[8][DZ_COLS];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int own = p.cblocks * p.rblocks;
  if ((int)blockIdx.x >= own) {
    pdl_launch();
    pdl_wait();
    repack_block(copies, (int)blockIdx.x - own, (int)gridDim.x - own);
    return;
  }
  const int cb = (int)blockIdx.x % p.cblocks, rb = (int)blockIdx.x / p.cblocks;
  const int c0 = cb * DZ_COLS;
  const long long r1 = min((long long)p.rows, (long long)(rb + 1) * p.rows_per_block);
  float acc[8] = {};
  pdl_launch();
  pdl_wait();
  auto colof = [&](int i) { return VEC ? lane * 8 + i : lane + 32 * i; };
  struct Row {
    uint4 y, z;
  };
  const uint4 zero = make_uint4(0, 0, 0, 0);
  with_act(p.z ? p.act : APK_ACT_NONE, [&](auto tag) {
    constexpr int ACT = decltype(tag)::value;
    auto load = [&](long long r) {
      Row v = {zero, zero};
      if (r >= r1) return v;
      if constexpr (VEC) {
        if (c0 + lane * 8 < p.cols) {
          v.y = __ldcs(reinterpret_cast<const uint4*>(p.dy + r * p.ld_dy + c0 + lane * 8));
          if (ACT != APK_ACT_NONE) v.z = __ldcs(reinterpret_cast<const uint4*>(p.z + r * p.ld_z + c0 + lane * 8));
        }
      } else {
        union {
          uint16_t h[8];
          uint4 v;
        } y, z;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool in = c0 + colof(i) < p.cols;
          y.h[i] = in ? p.dy[r * p.ld_dy + c0 + colof(i)] : (uint16_t)0;
          z.h[i] = ACT != APK_ACT_NONE && in ? p.z[r * p.ld_z + c0 + colof(i)] : (uint16_t)0;
        }
        v = {y.v, z.v};
      }
      return v;
    };
    long long r = (long long)rb * p.rows_per_block + warp;
    Row now = load(r);
    for (; r < r1; r += 8) {
      const Row next = load(r + 8);  // in flight while this row is worked on
      uint4 out;
      const uint32_t* y = &now.y.x;
      const uint32_t* z = &now.z.x;
      uint32_t* o = &out.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float d0 = __uint_as_float(y[i] << 16) * act_grad_f<ACT>(__uint_as_float(z[i] << 16));
        const float d1 = __uint_as_float(y[i] & 0xFFFF0000u) * act_grad_f<ACT>(__uint_as_float(z[i] & 0xFFFF0000u));
        acc[2 * i] += d0;
        acc[2 * i + 1] += d1;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(d1), "f"(d0));
      }
      if (p.dz) {
        if constexpr (VEC) {
          if (c0 + lane * 8 < p.cols) *reinterpret_cast<uint4*>(p.dz + r * p.ld_dz + c0 + lane * 8) = out;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c0 + colof(i) < p.cols)
              p.dz[r * p.ld_dz + c0 + colof(i)] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
        }
      }
      now = next;
    }
  });
  if (!p.db) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[warp][colof(i)] = acc[i];
  __syncthreads();
  const int c = c0 + (int)threadIdx.x;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += sum[w][threadIdx.x];
  if (p.rblocks > 1) {
    const int ldp = (p.cols + 7) / 8 * 8;
    if (c < p.cols) p.part[(long long)rb * ldp + c] = s;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      last = atomicAdd(&p.count[cb], 1u) == (unsigned)p.rblocks - 1;
      if (last) p.count[cb] = 0;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    // warp w adds the row blocks w, w + 8, ..., then the warps are added in order
    float t[8] = {};
    if (c0 + lane * 8 < ldp) {
#pragma unroll 4
      for (int b = warp; b < p.rblocks; b += 8) {
        const float4* q = reinterpret_cast<const float4*>(p.part + (long long)b * ldp + c0 + lane * 8);
        const float4 lo = __ldcg(q), hi = __ldcg(q + 1);
        t[0] += lo.x;
        t[1] += lo.y;
        t[2] += lo.z;
        t[3] += lo.w;
        t[4] += hi.x;
        t[5] += hi.y;
        t[6] += hi.z;
        t[7] += hi.w;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[warp][lane * 8 + i] = t[i];
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sum[w][threadIdx.x];
  }
  if (c < p.cols) {
    if (p.db_f32) static_cast<float*>(p.db)[c] = s;
    else static_cast<uint16_t*>(p.db)[c] = f2bf(s);
  }
}

}  // namespace lin
}  // namespace apk

using namespace apk;

struct apk_linear {
  apk_linear_config cfg{};
  Err err;
  int sms = 0;
  Scratch scratch;
  std::mutex mu;  // calls from several host threads are taken one at a time
};

namespace {

// Sizes up to here leave the kernels' 32-bit counts room to step past the end.
constexpr int MAX_SIZE = 1 << 30;

bool tma_ok(const void* p, long long ld, int outer) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld % 8 == 0 || outer == 1);
}
int up8(int n) { return (n + 7) / 8 * 8; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// an operand as TMA can address it; one row needs no stride
lin::Operand operand(const void* p, long long ld, int outer, int inner, bool mn) {
  return {p, outer == 1 ? (long long)up8(inner) : ld, outer, inner, mn};
}
// The operands of one launch of the repack kernel.
struct RepackList {
  lin::RepackParams p{};
  // `*src` becomes the copy at dst
  void add(const void** src, long long* ld, int rows, int cols, void* dst) {
    lin::Repack& o = p.op[p.n++];
    o = {static_cast<const uint16_t*>(*src), static_cast<uint16_t*>(dst), *ld, rows, cols, up8(cols), p.chunks};
    p.chunks += (long long)rows * (o.ld / 8);
    *src = dst;
    *ld = o.ld;
  }
  unsigned blocks(int sms) const { return (unsigned)std::min<long long>((p.chunks + 255) / 256, sms * 16); }
  apk_status run(int sms, cudaStream_t s, Err* err) const {
    if (p.n == 0) return APK_OK;
    Launch l(dim3(blocks(sms)), 256, 0, s);
    return cu_status(cudaLaunchKernelEx(&l.cfg, lin::repack, p), "launching the repack kernel", err);
  }
};

#define APK_TRY(x)                    \
  do {                                \
    const apk_status st_ = (x);       \
    if (st_ != APK_OK) return st_;    \
  } while (0)

bool valid_dtype(int d) { return d == APK_F32 || d == APK_BF16; }
const size_t esize[2] = {4, 2};  // APK_F32, APK_BF16
bool aligned_to(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % esize[dtype] == 0; }

apk_status forward(apk_linear* h, const apk_linear_io* io) {
  const apk_linear_config& c = h->cfg;
  const int K = c.in_features, N = c.out_features, M = io->rows;
  const cudaStream_t s = static_cast<cudaStream_t>(io->stream);
  if (M < 0 || M > MAX_SIZE) return h->err.fail(APK_EINVAL, "rows is %d: at most 2^30", M);
  if (M == 0) return APK_OK;
  if (!io->x || !io->y) return h->err.fail(APK_EINVAL, "x or y is NULL");
  if (!valid_dtype(io->y_dtype)) return h->err.fail(APK_EINVAL, "y_dtype %d", io->y_dtype);
  if (io->residual && !valid_dtype(io->residual_dtype))
    return h->err.fail(APK_EINVAL, "residual_dtype %d", io->residual_dtype);
  if (io->ldx < K || io->ldy < N || (io->residual && io->ld_residual < N) || (io->preact && io->ld_preact < N))
    return h->err.fail(APK_EINVAL, "a row stride is below its row: ldx %lld, ldy %lld, ld_residual %lld, ld_preact %lld",
                       io->ldx, io->ldy, io->ld_residual, io->ld_preact);
  if (!aligned_to(io->x, APK_BF16) || !aligned_to(io->y, io->y_dtype) ||
      (io->residual && !aligned_to(io->residual, io->residual_dtype)) || !aligned_to(io->preact, APK_BF16))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element");
  DeviceGuard guard(c.device);
  const int w_outer = c.w_layout == APK_W_KN ? K : N, w_inner = c.w_layout == APK_W_KN ? N : K;
  const lin::Epilogue epi = {c.bias, io->residual, io->y, io->preact, io->ld_residual, io->ldy, io->ld_preact,
                             c.bias_dtype == APK_F32, io->residual_dtype == APK_F32, io->y_dtype == APK_F32, c.act};
  if (lin::streams(M, (long long)K * N * 2, c.w_layout == APK_W_NK, tma_ok(c.W, c.ldw, w_outer)))
    return cu_status(lin::run_stream(io->x, io->ldx, c.W, c.ldw, c.w_layout == APK_W_NK, M, N, K, epi, h->sms, s),
                     "launching the streaming kernel", &h->err);
  APK_TRY(h->scratch.enter(s, &h->err));
  const void* x = io->x;
  const void* w = c.W;
  long long ldx = io->ldx, ldw = c.ldw;
  const bool px = !tma_ok(x, ldx, M), pw = !tma_ok(w, ldw, w_outer);
  ScratchUse use(&h->scratch, &h->err);
  if (px || pw) {
    const size_t bx = px ? up256((size_t)M * up8(K) * 2) : 0, bw = pw ? up256((size_t)w_outer * up8(w_inner) * 2) : 0;
    const size_t zeroed = up256((size_t)(N + lin::DZ_COLS - 1) / lin::DZ_COLS * 4);
    APK_TRY(use.begin(zeroed + bx + bw, zeroed));
    RepackList list;
    if (px) list.add(&x, &ldx, M, K, h->scratch.data() + zeroed);
    if (pw) list.add(&w, &ldw, w_outer, w_inner, h->scratch.data() + zeroed + bx);
    APK_TRY(list.run(h->sms, s, &h->err));
  }
  lin::Product p{};
  p.P = operand(w, ldw, w_outer, w_inner, c.w_layout == APK_W_KN);
  p.Q = operand(x, ldx, M, K, false);
  p.rows = M;
  p.cols = N;
  p.k = K;
  p.epi = epi;
  APK_TRY(lin::run_products(&p, 1, h->sms, c.device, h->scratch.status(), c.wait_limit_ns, s, &h->err.text));
  return use.end();
}

apk_status backward(apk_linear* h, const apk_linear_grads* g) {
  const apk_linear_config& c = h->cfg;
  const int K = c.in_features, N = c.out_features, M = g->rows;
  const cudaStream_t s = static_cast<cudaStream_t>(g->stream);
  const bool kn = c.w_layout == APK_W_KN;
  const int w_outer = kn ? K : N, w_inner = kn ? N : K;
  if (M < 0 || M > MAX_SIZE) return h->err.fail(APK_EINVAL, "rows is %d: at most 2^30", M);
  if (!g->dx && !g->dw && !g->db) return h->err.fail(APK_EINVAL, "no gradient is asked for");
  if (g->db && !c.bias) return h->err.fail(APK_EINVAL, "db of a layer without a bias");
  if (g->dw && !valid_dtype(g->dw_dtype)) return h->err.fail(APK_EINVAL, "dw_dtype %d", g->dw_dtype);
  if (M > 0 && (!g->dy || (g->dw && !g->x) || (c.act != APK_ACT_NONE && !g->preact)))
    return h->err.fail(APK_EINVAL, "dy, x (for dw) or preact (with an activation) is NULL");
  if (g->ld_dy < N || (g->dw && (g->ldx < K || g->ld_dw < w_inner)) || (g->dx && g->ld_dx < K) ||
      (c.act != APK_ACT_NONE && g->ld_preact < N))
    return h->err.fail(APK_EINVAL, "a row stride is below its row: ldx %lld, ld_dy %lld, ld_preact %lld, ld_dx %lld, ld_dw %lld",
                       g->ldx, g->ld_dy, g->ld_preact, g->ld_dx, g->ld_dw);
  if (!aligned_to(g->dy, APK_BF16) || !aligned_to(g->x, APK_BF16) || !aligned_to(g->preact, APK_BF16) ||
      !aligned_to(g->dx, APK_BF16) || (g->dw && !aligned_to(g->dw, g->dw_dtype)) ||
      (g->db && !aligned_to(g->db, c.bias_dtype)))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element");
  DeviceGuard guard(c.device);
  if (M == 0) {  // sums over no rows
    if (g->dw)
      APK_TRY(cu_status(cudaMemset2DAsync(g->dw, (size_t)g->ld_dw * esize[g->dw_dtype], 0,
                                          (size_t)w_inner * esize[g->dw_dtype], w_outer, s),
                        "clearing dw", &h->err));
    if (g->db) APK_TRY(cu_status(cudaMemsetAsync(g->db, 0, (size_t)N * esize[c.bias_dtype], s), "clearing db", &h->err));
    return APK_OK;
  }
  APK_TRY(h->scratch.enter(s, &h->err));
  const bool act = c.act != APK_ACT_NONE;
  const bool products = g->dx || g->dw;
  const bool own_dz = products && (act || !tma_ok(g->dy, g->ld_dy, M));
  const bool px = g->dw && !tma_ok(g->x, g->ldx, M), pw = g->dx && !tma_ok(c.W, c.ldw, w_outer);
  // blocks of the elementwise pass: one residency at most, at least 16 rows each
  const int cblocks = (N + lin::DZ_COLS - 1) / lin::DZ_COLS;
  int rblocks = std::max(1, std::min((M + 15) / 16, lin::DZ_BLOCKS * h->sms / cblocks));
  const int per = ((M + rblocks - 1) / rblocks + 7) / 8 * 8;
  rblocks = (M + per - 1) / per;
  const size_t zeroed = up256((size_t)cblocks * 4);
  const size_t bpart = g->db ? up256((size_t)rblocks * up8(N) * 4) : 0;
  const size_t bdz = own_dz ? up256((size_t)M * up8(N) * 2) : 0;
  const size_t bx = px ? up256((size_t)M * up8(K) * 2) : 0, bw = pw ? up256((size_t)w_outer * up8(w_inner) * 2) : 0;
  ScratchUse use(&h->scratch, &h->err);
  if (g->db || own_dz || px || pw) APK_TRY(use.begin(zeroed + bpart + bdz + bx + bw, zeroed));
  uint8_t* base = h->scratch.data();
  const void* x = g->x;
  const void* w = c.W;
  long long ldx = g->ldx, ldw = c.ldw;
  RepackList list;
  if (px) list.add(&x, &ldx, M, K, base + zeroed + bpart + bdz);
  if (pw) list.add(&w, &ldw, w_outer, w_inner, base + zeroed + bpart + bdz + bx);
  const void* dz = g->dy;
  long long ld_dz = g->ld_dy;
  if (!g->db && !own_dz) {
    APK_TRY(list.run(h->sms, s, &h->err));
  } else {
    lin::DzParams d{};
    d.dy = static_cast<const uint16_t*>(g->dy);
    d.z = act ? static_cast<const uint16_t*>(g->preact) : nullptr;
    d.ld_dy = g->ld_dy;
    d.ld_z = g->ld_preact;
    if (own_dz) {
      d.dz = reinterpret_cast<uint16_t*>(base + zeroed + bpart);
      d.ld_dz = ld_dz = up8(N);
      dz = d.dz;
    }
    d.db = g->db;
    d.db_f32 = c.bias_dtype == APK_F32;
    d.part = reinterpret_cast<float*>(base + zeroed);
    d.count = reinterpret_cast<unsigned*>(base);
    d.rows = M;
    d.cols = N;
    d.rows_per_block = per;
    d.act = c.act;
    // (the last chunk of a row may reach past N: only within an 8-multiple row)
    const bool vec = N % 8 == 0 && tma_ok(g->dy, g->ld_dy, M) && (!act || tma_ok(g->preact, g->ld_preact, M));
    d.cblocks = cblocks;
    d.rblocks = rblocks;
    Launch l(dim3(cblocks * rblocks + list.blocks(h->sms)), 256, 0, s);
    APK_TRY(cu_status(cudaLaunchKernelEx(&l.cfg, vec ? lin::dz_kernel<true> : lin::dz_kernel<false>, d, list.p),
                      "launching the dz kernel", &h->err));
  }
  lin::Product p[2] = {};
  int n = 0;
  if (g->dx) {  // dx[m][k] = sum_n dz[m][n] W[k][n]
    lin::Product& a = p[n++];
    a.P = operand(w, ldw, w_outer, w_inner, !kn);
    a.Q = operand(dz, ld_dz, M, N, false);
    a.rows = M;
    a.cols = K;
    a.k = N;
    a.epi = {nullptr, nullptr, g->dx, nullptr, 0, g->ld_dx, 0, 0, 0, 0, APK_ACT_NONE};
  }
  if (g->dw) {  // dW in W's layout: rows of x^T by columns of dz, or the reverse
    lin::Product& a = p[n++];
    const lin::Operand ox = operand(x, ldx, M, K, true), oz = operand(dz, ld_dz, M, N, true);
    a.P = kn ? oz : ox;
    a.Q = kn ? ox : oz;
    a.rows = w_outer;
    a.cols = w_inner;
    a.k = M;
    a.epi = {nullptr, nullptr, g->dw, nullptr, 0, g->ld_dw, 0, 0, 0, g->dw_dtype == APK_F32, APK_ACT_NONE};
  }
  if (n) APK_TRY(lin::run_products(p, n, h->sms, c.device, h->scratch.status(), c.wait_limit_ns, s, &h->err.text));
  return use.end();
}

apk_status create(const apk_linear_config* cfg, apk_linear* h) {
  if (!cfg) return h->err.fail(APK_EINVAL, "cfg is NULL");
  h->cfg = *cfg;
  const apk_linear_config& c = h->cfg;
  if (c.in_features < 1 || c.out_features < 1 || c.in_features > MAX_SIZE || c.out_features > MAX_SIZE)
    return h->err.fail(APK_EINVAL, "in_features %d, out_features %d: 1 to 2^30", c.in_features, c.out_features);
  if (c.w_layout != APK_W_KN && c.w_layout != APK_W_NK) return h->err.fail(APK_EINVAL, "w_layout %d", (int)c.w_layout);
  if (c.act < APK_ACT_NONE || c.act > APK_ACT_SILU) return h->err.fail(APK_EINVAL, "act %d", (int)c.act);
  if (!c.W) return h->err.fail(APK_EINVAL, "W is NULL");
  if (c.ldw < (c.w_layout == APK_W_KN ? c.out_features : c.in_features))
    return h->err.fail(APK_EINVAL, "ldw %lld is below W's row", c.ldw);
  if (c.bias && !valid_dtype(c.bias_dtype)) return h->err.fail(APK_EINVAL, "bias_dtype %d", (int)c.bias_dtype);
  if (!aligned_to(c.W, APK_BF16) || (c.bias && !aligned_to(c.bias, c.bias_dtype)))
    return h->err.fail(APK_EINVAL, "W or bias is not aligned to its element");
  if (c.wait_limit_ns < 0) return h->err.fail(APK_EINVAL, "wait_limit_ns is negative");
  if (c.wait_limit_ns == 0) h->cfg.wait_limit_ns = 2000000000ll;
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || c.device < 0 || c.device >= ndev) {
    cudaGetLastError();
    return h->err.fail(APK_ECUDA, "no CUDA device %d", c.device);
  }
  DeviceGuard guard(c.device);
  int major = 0, sms = 0;
  APK_TRY(cu_status(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, c.device), "device query", &h->err));
  APK_TRY(cu_status(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c.device), "device query", &h->err));
  if (major != 10) return h->err.fail(APK_EUNSUPPORTED, "the kernels are built for sm_100a");
  APK_TRY(cu_status(lin::prepare(), "preparing the linear kernels", &h->err));
  h->sms = sms;
  if (c.sms < 0 || c.sms > sms) return h->err.fail(APK_EINVAL, "sms %d of %d", c.sms, sms);
  if (c.sms > 0) h->sms = c.sms;
  return h->scratch.open(c.device, &h->err);
}

}  // namespace

extern "C" {

apk_status apk_linear_create(const apk_linear_config* cfg, apk_linear** out) {
  if (!out) return APK_EINVAL;
  *out = new (std::nothrow) apk_linear;
  if (!*out) return APK_ENOMEM;
  try {
    return create(cfg, *out);  // *out is set on failure too: its last_error says why
  } catch (...) {
    return APK_ENOMEM;
  }
}

apk_status apk_linear_destroy(apk_linear* h) {
  if (!h) return APK_OK;
  delete h;
  return APK_OK;
}

const char* apk_linear_last_error(const apk_linear* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_linear_forward(apk_linear* h, const apk_linear_io* io) {
  if (!h || !h->scratch.status() || !io) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    return forward(h, io);
  } catch (...) {
    return APK_ENOMEM;
  }
}

apk_status apk_linear_backward(apk_linear* h, const apk_linear_grads* g) {
  if (!h || !h->scratch.status() || !g) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    return backward(h, g);
  } catch (...) {
    return APK_ENOMEM;
  }
}

apk_status apk_linear_status(apk_linear* h, void* stream, int* device_status) {
  if (!h || !h->scratch.status() || !device_status) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    DeviceGuard guard(h->cfg.device);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    APK_TRY(cu_status(cudaMemcpyAsync(device_status, h->scratch.status(), sizeof(int), cudaMemcpyDeviceToHost, s), "status copy",
                      &h->err));
    APK_TRY(cu_status(cudaMemsetAsync(h->scratch.status(), 0, sizeof(int), s), "status clear", &h->err));
    return cu_status(cudaStreamSynchronize(s), "cudaStreamSynchronize", &h->err);
  } catch (...) {
    return APK_ENOMEM;
  }
}

}  // extern "C"
