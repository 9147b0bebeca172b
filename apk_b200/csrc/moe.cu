// A routed mixture-of-experts layer for up to 64 tokens in one kernel
// (apk_moe_* of include/apk.h): router, top-k, the chosen experts' two
// products and the weighted sum.  No reference counterpart: the reference
// multiplies bare matrices (src/tcyield.cu:91-356).
//
// What bounds it is reading the chosen experts' weights once, so every
// product streams weight rows from global memory straight into MMA fragments
// (stream.cuh; the tokens are the MMA's N axis, gathered by index) and the
// layer is one persistent cooperative kernel, one CTA of 16 warps per SM, whose
// phases meet at grid barriers instead of kernel boundaries:
//   0  partial router logits: 16 experts x a slice of d_model per item
//   1  every CTA picks the experts of all tokens for itself (T x E logits are
//      cheaper to read 148 times from L2 than to pass through another
//      barrier), then hidden = act(gate) * up, 8 gate and 8 up rows per item,
//      so both halves of a product sit in one thread's accumulator
//   2  each (token, choice) pair's output row in fp32
//   3  y[t] = sum over the choices, in their order, of p * row
// An item's rows are read by 1-16 warps of a CTA that split k: many when
// there are few items (a token or two), one when there are many.  Sums across
// warps go through shared memory in warp order.  Nothing depends on the order
// of arrival: an expert's tokens are a bit mask, so their columns are ordered
// by token.
//
// Rounding: the hidden values are rounded to bf16 once as the second
// product's operand; logits, softmax, both products and the sum are fp32.
#include <algorithm>
#include <mutex>
#include <new>

#include "act.cuh"
#include "common.cuh"
#include "linear.h"
#include "stream.cuh"

namespace apk {
namespace moe {

constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int MAX_TOKENS = 64, MAX_EXPERTS = 512, MAX_TOPK = 16;
constexpr int ROUND = 128;  // k of one warp's round: 8 16-byte weight loads a lane

struct Params {
  const uint16_t* x;
  const uint16_t* router;
  const uint16_t* w_in;
  const uint16_t* w_out;
  void* y;
  int* ids;      // [tokens][top_k] or null
  float* probs;  // [tokens][top_k] or null
  long long ldx, ldy;
  int tokens, experts, top_k, d, f, act, gated, renorm, y_f32;
  int red_stride;  // floats of a warp's place in the shared sums
  int rsplit;    // slices of d_model in phase 0
  unsigned* barrier;  // {arrived, generation}
  int* status;
  long long limit;
  float* logits;  // [rsplit][tokens][experts]
  uint16_t* hid;  // [tokens * top_k][f], rows grouped by expert
  float* out;     // [tokens * top_k][d]
};

struct Shared {
  unsigned long long mask[MAX_EXPERTS];  // the tokens that chose an expert
  short active[MAX_EXPERTS];             // experts with tokens, ascending
  short base[MAX_EXPERTS];               // an active expert's first row
  short sel[MAX_TOKENS * MAX_TOPK];      // expert, then row, of (token, choice)
  float prob[MAX_TOKENS * MAX_TOPK];
  unsigned char tok[MAX_TOKENS * MAX_TOPK];  // token of a row
  int warp_n[WARPS], warp_rows[WARPS];
  int n_active;
  int abort;
};

// Every CTA of the grid has arrived (and its earlier writes are visible).
// The last to arrive clears the count and advances the generation, so the
// words need no reset between launches.
__device__ __forceinline__ bool grid_barrier(const Params& p, Shared& sh) {
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned gen, old;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(gen) : "l"(p.barrier + 1) : "memory");
    __threadfence();
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(p.barrier) : "memory");
    if (old == gridDim.x - 1) {
      asm volatile("st.relaxed.gpu.global.u32 [%0], 0;" ::"l"(p.barrier) : "memory");
      asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p.barrier + 1), "r"(gen + 1) : "memory");
    } else {
      const long long t0 = globaltimer_ns();
      int n = 0;
      while (true) {
        unsigned now;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(p.barrier + 1) : "memory");
        if (now != gen) break;
        if (++n == 64) {
          n = 0;
          if (globaltimer_ns() - t0 > p.limit) {
            report_status(p.status, DEV_WAIT_TIMEOUT_SPIN, nullptr);
            sh.abort = 1;
            break;
          }
        }
      }
    }
    __threadfence();
  }
  __syncthreads();
  return sh.abort == 0;
}

struct Frag {
  uint4 a[4], b[4];
};
// One round of weight rows w0 (MMA rows g) and w1 (g + 8) at k0 + 32 u + 8 t.
__device__ __forceinline__ void load_round(Frag& f, const uint16_t* w0, const uint16_t* w1, int k0, int t, int k) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int at = k0 + 32 * u + 8 * t;
    const bool in = at < k;
    f.a[u] = in ? stream::ld_weights(w0 + at) : make_uint4(0, 0, 0, 0);
    f.b[u] = in ? stream::ld_weights(w1 + at) : make_uint4(0, 0, 0, 0);
  }
}
// acc += rows (w0 | w1) times the NT8 x 8 token rows xr, over the rounds
// first, first + step, ... of k.  The next round's weights are in flight while
// one is multiplied.
// `Load` reads 16 bytes of a token row.
template <int NT8, class Load>
__device__ __forceinline__ void stream_rows(float (&acc)[NT8][4], const uint16_t* w0, const uint16_t* w1,
                                            const uint16_t* const (&xr)[NT8], int k, int first, int step, int t,
                                            Load ld) {
  int k0 = first * ROUND;
  if (k0 >= k) return;
  Frag f;
  load_round(f, w0, w1, k0, t, k);
  while (true) {
    const int next = k0 + step * ROUND;
    Frag n;
    if (NT8 <= 2) load_round(n, w0, w1, next, t, k);  // (past the end: zero, nothing read)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = k0 + 32 * u + 8 * t;
      uint4 c[NT8];
#pragma unroll
      for (int i = 0; i < NT8; ++i) c[i] = at < k ? ld(xr[i] + at) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NT8; ++i) {
        stream::mma_bf16(acc[i], f.a[u].x, f.b[u].x, f.a[u].y, f.b[u].y, c[i].x, c[i].y);
        stream::mma_bf16(acc[i], f.a[u].z, f.b[u].z, f.a[u].w, f.b[u].w, c[i].z, c[i].w);
      }
    }
    k0 = next;
    if (k0 >= k) break;
    if (NT8 <= 2) f = n;
    else load_round(f, w0, w1, k0, t, k);
  }
}

struct LdConst {  // the layer's input: not written during the kernel
  __device__ uint4 operator()(const uint16_t* p) const { return __ldg(reinterpret_cast<const uint4*>(p)); }
};
struct LdWritten {  // written by other CTAs in an earlier phase: from L2
  __device__ uint4 operator()(const uint16_t* p) const { return __ldcg(reinterpret_cast<const uint4*>(p)); }
};

// The `ws` warps of a group add their accumulators into the first one's.  A
// warp's place in `red` has the same size for every group of the CTA (groups
// may be at items with different numbers of tokens).
template <int NT8>
__device__ __forceinline__ void join_warps(float (&acc)[NT8][4], float* red, int stride, int ws, int warp, int lane) {
  if (ws == 1) return;
  red += warp * stride + lane;
  const int j = warp & (ws - 1), id = 1 + warp / ws;
#pragma unroll
  for (int i = 0; i < NT8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) red[(i * 4 + c) * 32] = acc[i][c];
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(32 * ws) : "memory");
  if (j == 0)
    for (int w = 1; w < ws; ++w)
#pragma unroll
      for (int i = 0; i < NT8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] += red[w * stride + (i * 4 + c) * 32];
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(32 * ws) : "memory");  // red is free again
}

// Warps that share an item: enough that every warp of the grid has one,
// within the rounds that k has.
__device__ __forceinline__ int warps_per_item(long long items, int k) {
  int ws = 1;
  while (ws < WARPS && items * ws < (long long)gridDim.x * WARPS && ws * ROUND < k) ws *= 2;
  return ws;
}

template <int NT8>
__device__ __forceinline__ void item_in(const Params& p, const Shared& sh, float* red, int a, int tile, int n, int ws) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int e = sh.active[a], base = sh.base[a];
  const int rows_e = p.gated ? 2 * p.f : p.f;
  const int f0 = tile * (p.gated ? 8 : 16);
  const uint16_t* w = p.w_in + (long long)e * rows_e * p.d;
  // gated: MMA row g is gate f0 + g, row g + 8 its up; else features f0 + g and f0 + g + 8
  const int r0 = min(f0 + g, p.f - 1), r1 = p.gated ? p.f + r0 : min(f0 + g + 8, p.f - 1);
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.x + sh.tok[base + min(8 * i + g, n - 1)] * p.ldx;
  float acc[NT8][4] = {};
  stream_rows<NT8>(acc, w + (long long)r0 * p.d, w + (long long)r1 * p.d, xr, p.d, warp & (ws - 1), ws, t, LdConst());
  join_warps<NT8>(acc, red, p.red_stride, ws, warp, lane);
  if (warp & (ws - 1)) return;
  with_act(p.act, [&](auto tag) {
    constexpr int ACT = decltype(tag)::value;
#pragma unroll
    for (int i = 0; i < NT8; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 8 * i + 2 * t + c;
        if (col >= n) continue;
        uint16_t* h = p.hid + (long long)(base + col) * p.f;
        auto put = [&](int f, float v) {
          uint16_t r;
          asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
          if (f < p.f) h[f] = r;
        };
        if (p.gated) {
          put(f0 + g, act_f<ACT>(acc[i][c]) * acc[i][c + 2]);
        } else {
          put(f0 + g, act_f<ACT>(acc[i][c]));
          put(f0 + g + 8, act_f<ACT>(acc[i][c + 2]));
        }
      }
  });
}

template <int NT8>
__device__ __forceinline__ void item_out(const Params& p, const Shared& sh, float* red, int a, int tile, int n, int ws) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int e = sh.active[a], base = sh.base[a], d0 = tile * 16;
  const uint16_t* w = p.w_out + (long long)e * p.d * p.f;
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.hid + (long long)(base + min(8 * i + g, n - 1)) * p.f;
  float acc[NT8][4] = {};
  stream_rows<NT8>(acc, w + (long long)min(d0 + g, p.d - 1) * p.f, w + (long long)min(d0 + g + 8, p.d - 1) * p.f, xr, p.f,
                   warp & (ws - 1), ws, t, LdWritten());
  join_warps<NT8>(acc, red, p.red_stride, ws, warp, lane);
  if (warp & (ws - 1)) return;
#pragma unroll
  for (int i = 0; i < NT8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = 8 * i + 2 * t + (c & 1), d = d0 + g + 8 * (c >> 1);
      if (col < n && d < p.d) p.out[(long long)(base + col) * p.d + d] = acc[i][c];
    }
}

// Partial logits of 16 experts for all tokens, 64 at a time in NT8 = 8 tiles.
template <int NT8>
__device__ __forceinline__ void item_router(const Params& p, float* red, int tile, int slice) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int e0 = tile * 16;
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.x + min(8 * i + g, p.tokens - 1) * p.ldx;
  float acc[NT8][4] = {};
  stream_rows<NT8>(acc, p.router + (long long)min(e0 + g, p.experts - 1) * p.d,
                   p.router + (long long)min(e0 + g + 8, p.experts - 1) * p.d, xr, p.d, slice * WARPS + warp,
                   p.rsplit * WARPS, t, LdConst());
  join_warps<NT8>(acc, red, p.red_stride, WARPS, warp, lane);
  if (warp) return;
#pragma unroll
  for (int i = 0; i < NT8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int tok = 8 * i + 2 * t + (c & 1), e = e0 + g + 8 * (c >> 1);
      if (tok < p.tokens && e < p.experts) p.logits[((long long)slice * p.tokens + tok) * p.experts + e] = acc[i][c];
    }
}

// Order of the logits as unsigned integers; a NaN comes first, as in a
// descending sort.
__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  v += 0.f;  // -0 and 0 tie
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// One warp picks a token's experts: top_k rounds of "largest key, lowest
// index", then their softmax over all experts.
__device__ __forceinline__ void route_token(const Params& p, Shared& sh, int tok) {
  const int lane = threadIdx.x & 31;
  constexpr int PER = MAX_EXPERTS / 32;
  float v[PER];
  unsigned key[PER];
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    v[i] = 0.f;
    key[i] = 0;  // below every logit's key: -inf has key 0x007FFFFF
    if (e < p.experts) {
      for (int s = 0; s < p.rsplit; ++s) v[i] += __ldcg(p.logits + ((long long)s * p.tokens + tok) * p.experts + e);
      key[i] = order_key(v[i]);
      best = v[i] != v[i] ? v[i] : fmaxf(best, v[i]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float other = __shfl_xor_sync(~0u, best, o);
    best = (best != best || other != other) ? NAN : fmaxf(best, other);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 32 * i < p.experts) sum += __expf(v[i] - best);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  float chosen = 0.f;
  for (int j = 0; j < p.top_k; ++j) {
    unsigned k = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) k = max(k, key[i]);
    k = __reduce_max_sync(~0u, k);
    int at = MAX_EXPERTS;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == k && lane + 32 * i < p.experts) at = lane + 32 * i;
    at = __reduce_min_sync(~0u, at);
    float pj = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == lane + 32 * i) {
        key[i] = 0;
        pj = __fdividef(__expf(v[i] - best), sum);
      }
    pj = __shfl_sync(~0u, pj, at & 31);
    chosen += pj;
    if (lane == 0) {
      sh.sel[tok * p.top_k + j] = (short)at;
      sh.prob[tok * p.top_k + j] = pj;
      atomicOr(&sh.mask[at], 1ull << tok);
    }
  }
  __syncwarp();
  if (p.renorm && lane < p.top_k)
    sh.prob[tok * p.top_k + lane] = __fdividef(sh.prob[tok * p.top_k + lane], chosen);
}

__global__ void __launch_bounds__(THREADS, 1) moe_layer(const __grid_constant__ Params p) {
  extern __shared__ float red[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) sh.abort = 0;

  // -------- 0: partial logits --------
  const int etiles = (p.experts + 15) / 16;
  for (int it = blockIdx.x; it < etiles * p.rsplit; it += gridDim.x) {
    const int tile = it % etiles, slice = it / etiles;
    if (p.tokens <= 8) item_router<1>(p, red, tile, slice);
    else if (p.tokens <= 16) item_router<2>(p, red, tile, slice);
    else if (p.tokens <= 32) item_router<4>(p, red, tile, slice);
    else item_router<8>(p, red, tile, slice);
  }
  for (int e = tid; e < p.experts; e += THREADS) sh.mask[e] = 0;
  if (!grid_barrier(p, sh)) return;

  // -------- 1: routing (by every CTA), then the hidden values --------
  for (int tok = warp; tok < p.tokens; tok += WARPS) route_token(p, sh, tok);
  __syncthreads();
  {
    // thread e: rank of expert e among those with tokens, and its first row
    const int n = tid < p.experts ? __popcll(sh.mask[tid]) : 0;
    const unsigned some = __ballot_sync(~0u, n > 0);
    int rows = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(~0u, rows, o);
      if (lane >= o) rows += up;
    }
    if (lane == 31) {
      sh.warp_n[warp] = __popc(some);
      sh.warp_rows[warp] = rows;
    }
    __syncthreads();
    int a = __popc(some & ((1u << lane) - 1)), r = rows - n;
    for (int w = 0; w < warp; ++w) {
      a += sh.warp_n[w];
      r += sh.warp_rows[w];
    }
    if (n > 0) {
      sh.active[a] = (short)tid;
      sh.base[a] = (short)r;
      unsigned long long m = sh.mask[tid];
      for (int i = 0; m; ++i, m &= m - 1) sh.tok[r + i] = (unsigned char)(__ffsll((long long)m) - 1);
    }
    if (tid == THREADS - 1) sh.n_active = a + (n > 0);
  }
  __syncthreads();
  const int n_active = sh.n_active;
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.tokens * p.top_k; i += THREADS) {
      if (p.ids) p.ids[i] = sh.sel[i];
      if (p.probs) p.probs[i] = sh.prob[i];
    }
  }
  // f(a, tile, columns): an item of active expert a's `tiles` row tiles, by warps_per_item warps
  auto for_items = [&](int tiles, int k, auto f) {
    const long long items = (long long)n_active * tiles;
    const int ws = warps_per_item(items, k), slots = gridDim.x * (WARPS / ws);
    for (long long it = (long long)(warp / ws) * gridDim.x + blockIdx.x; it < items; it += slots) {
      const int a = (int)(it / tiles);
      f(a, (int)(it - (long long)a * tiles), __popcll(sh.mask[sh.active[a]]), ws);
    }
  };
  for_items((p.f + (p.gated ? 7 : 15)) / (p.gated ? 8 : 16), p.d, [&](int a, int tile, int n, int ws) {
    if (n <= 8) item_in<1>(p, sh, red, a, tile, n, ws);
    else if (n <= 16) item_in<2>(p, sh, red, a, tile, n, ws);
    else if (n <= 32) item_in<4>(p, sh, red, a, tile, n, ws);
    else item_in<8>(p, sh, red, a, tile, n, ws);
  });
  if (!grid_barrier(p, sh)) return;

  // -------- 2: output rows of the pairs --------
  for_items((p.d + 15) / 16, p.f, [&](int a, int tile, int n, int ws) {
    if (n <= 8) item_out<1>(p, sh, red, a, tile, n, ws);
    else if (n <= 16) item_out<2>(p, sh, red, a, tile, n, ws);
    else if (n <= 32) item_out<4>(p, sh, red, a, tile, n, ws);
    else item_out<8>(p, sh, red, a, tile, n, ws);
  });
  // the row of each (token, choice), in place of its expert
  __syncthreads();
  for (int a = tid; a < n_active; a += THREADS) {
    const int e = sh.active[a];
    unsigned long long m = sh.mask[e];
    for (int i = 0; m; ++i, m &= m - 1) {
      const int tok = __ffsll((long long)m) - 1;
      for (int j = 0; j < p.top_k; ++j)
        if (sh.sel[tok * p.top_k + j] == e) {
          sh.sel[tok * p.top_k + j] = (short)(-1 - (sh.base[a] + i));  // (negative: not an expert)
          break;
        }
    }
  }
  if (!grid_barrier(p, sh)) return;

  // -------- 3: weighted sum --------
  const int quads = p.d / 4;
  for (int i = blockIdx.x * THREADS + tid; i < p.tokens * quads; i += gridDim.x * THREADS) {
    const int tok = i / quads, d = (i - tok * quads) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < p.top_k; ++j) {
      const int row = -1 - sh.sel[tok * p.top_k + j];
      const float w = sh.prob[tok * p.top_k + j];
      const float4 o = __ldcg(reinterpret_cast<const float4*>(p.out + (long long)row * p.d + d));
      s.x += w * o.x;
      s.y += w * o.y;
      s.z += w * o.z;
      s.w += w * o.w;
    }
    const long long at = tok * p.ldy + d;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (p.y_f32) {
        static_cast<float*>(p.y)[at + c] = v[c];
      } else {
        uint16_t r;
        asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v[c]));
        static_cast<uint16_t*>(p.y)[at + c] = r;
      }
    }
  }
}

constexpr int red_bytes(int nt8) { return WARPS * nt8 * 4 * 32 * 4; }

}  // namespace moe
}  // namespace apk

using namespace apk;

struct apk_moe {
  apk_moe_config cfg{};
  Err err;
  int sms = 0;
  int* status = nullptr;
  Scratch scratch;
  std::mutex mu;
};

#define APK_TRY(x)                    \
  do {                                \
    const apk_status st_ = (x);       \
    if (st_ != APK_OK) return st_;    \
  } while (0)

namespace {

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

apk_status create(const apk_moe_config* cfg, apk_moe* h) {
  if (!cfg) return h->err.fail(APK_EINVAL, "cfg is NULL");
  h->cfg = *cfg;
  const apk_moe_config& c = h->cfg;
  if (c.experts < 1 || c.experts > moe::MAX_EXPERTS)
    return h->err.fail(APK_EINVAL, "experts is %d: 1 to %d", c.experts, moe::MAX_EXPERTS);
  if (c.top_k < 1 || c.top_k > moe::MAX_TOPK || c.top_k > c.experts)
    return h->err.fail(APK_EINVAL, "top_k is %d: 1 to %d, of %d experts", c.top_k, moe::MAX_TOPK, c.experts);
  if (c.d_model < 8 || c.d_ff < 8 || c.d_model % 8 || c.d_ff % 8)
    return h->err.fail(APK_EINVAL, "d_model %d and d_ff %d have to be multiples of 8", c.d_model, c.d_ff);
  if (c.act < APK_ACT_NONE || c.act > APK_ACT_SILU) return h->err.fail(APK_EINVAL, "act %d", (int)c.act);
  if (!c.router || !c.w_in || !c.w_out) return h->err.fail(APK_EINVAL, "router, w_in or w_out is NULL");
  if (!aligned(c.router, 16) || !aligned(c.w_in, 16) || !aligned(c.w_out, 16))
    return h->err.fail(APK_EINVAL, "router, w_in and w_out have to be aligned to 16 bytes");
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
  if (c.sms < 0 || c.sms > sms) return h->err.fail(APK_EINVAL, "sms %d of %d", c.sms, sms);
  h->sms = c.sms ? c.sms : sms;
  APK_TRY(cu_status(cudaFuncSetAttribute(moe::moe_layer, cudaFuncAttributeMaxDynamicSharedMemorySize, moe::red_bytes(8)),
                    "preparing the expert kernel", &h->err));
  int per_sm = 0;
  APK_TRY(cu_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, moe::moe_layer, moe::THREADS, moe::red_bytes(8)),
                    "preparing the expert kernel", &h->err));
  if (per_sm < 1) return h->err.fail(APK_EUNSUPPORTED, "the expert kernel does not fit an SM");
  void* st = nullptr;
  APK_TRY(cu_status(cudaMalloc(&st, 256), "cudaMalloc", &h->err));
  h->status = static_cast<int*>(st);
  APK_TRY(cu_status(cudaMemset(st, 0, 256), "cudaMemset", &h->err));
  return cu_status(cudaStreamSynchronize(nullptr), "cudaStreamSynchronize", &h->err);
}

apk_status forward(apk_moe* h, const apk_moe_io* io) {
  const apk_moe_config& c = h->cfg;
  if (io->tokens < 0 || io->tokens > moe::MAX_TOKENS)
    return h->err.fail(APK_EINVAL, "tokens is %d: at most %d", io->tokens, moe::MAX_TOKENS);
  if (io->tokens == 0) return APK_OK;
  if (!io->x || !io->y) return h->err.fail(APK_EINVAL, "x or y is NULL");
  if (io->y_dtype != APK_F32 && io->y_dtype != APK_BF16) return h->err.fail(APK_EINVAL, "y_dtype %d", (int)io->y_dtype);
  if (io->ldx < c.d_model || io->ldy < c.d_model)
    return h->err.fail(APK_EINVAL, "a row stride is below its row: ldx %lld, ldy %lld", io->ldx, io->ldy);
  if (!aligned(io->x, 16) || io->ldx % 8)
    return h->err.fail(APK_EINVAL, "the rows of x have to start on 16 bytes (ldx %lld)", io->ldx);
  if (!aligned(io->y, io->y_dtype == APK_F32 ? 4 : 2) || !aligned(io->ids, 4) || !aligned(io->probs, 4))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element");
  DeviceGuard guard(c.device);
  const cudaStream_t s = static_cast<cudaStream_t>(io->stream);
  moe::Params p{};
  // phase 0: slices of d_model so that the SMs share the router, one round of 16 warps at least each
  const int etiles = (c.experts + 15) / 16;
  p.rsplit = std::max(1, std::min({h->sms / etiles, (c.d_model + moe::WARPS * moe::ROUND - 1) / (moe::WARPS * moe::ROUND), 8}));
  const size_t pairs = (size_t)io->tokens * c.top_k;
  const size_t b_log = up256((size_t)p.rsplit * io->tokens * c.experts * 4), b_hid = up256(pairs * c.d_ff * 2);
  const size_t b_out = up256(pairs * c.d_model * 4);
  APK_TRY(h->scratch.begin(256 + b_log + b_hid + b_out, 256, s, &h->err));
  uint8_t* b = h->scratch.data();
  p.x = static_cast<const uint16_t*>(io->x);
  p.router = static_cast<const uint16_t*>(c.router);
  p.w_in = static_cast<const uint16_t*>(c.w_in);
  p.w_out = static_cast<const uint16_t*>(c.w_out);
  p.y = io->y;
  p.ids = io->ids;
  p.probs = io->probs;
  p.ldx = io->ldx;
  p.ldy = io->ldy;
  p.tokens = io->tokens;
  p.experts = c.experts;
  p.top_k = c.top_k;
  p.d = c.d_model;
  p.f = c.d_ff;
  p.act = c.act;
  p.gated = c.gated != 0;
  p.renorm = c.renormalize != 0;
  p.y_f32 = io->y_dtype == APK_F32;
  p.barrier = reinterpret_cast<unsigned*>(b);
  p.status = h->status;
  p.limit = c.wait_limit_ns;
  p.logits = reinterpret_cast<float*>(b + 256);
  p.hid = reinterpret_cast<uint16_t*>(b + 256 + b_log);
  p.out = reinterpret_cast<float*>(b + 256 + b_log + b_hid);
  const int nt8 = io->tokens <= 8 ? 1 : io->tokens <= 16 ? 2 : io->tokens <= 32 ? 4 : 8;
  p.red_stride = nt8 * 128;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.gridDim = dim3(h->sms);
  cfg.blockDim = dim3(moe::THREADS);
  cfg.dynamicSmemBytes = moe::red_bytes(nt8);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  APK_TRY(cu_status(cudaLaunchKernelEx(&cfg, moe::moe_layer, p), "launching the expert kernel", &h->err));
  return h->scratch.end(s, &h->err);
}

}  // namespace

extern "C" {

apk_status apk_moe_create(const apk_moe_config* cfg, apk_moe** out) {
  if (!out) return APK_EINVAL;
  *out = new (std::nothrow) apk_moe;
  if (!*out) return APK_ENOMEM;
  try {
    return create(cfg, *out);
  } catch (...) {
    return APK_ENOMEM;
  }
}

apk_status apk_moe_destroy(apk_moe* h) {
  if (!h) return APK_OK;
  if (h->status) {
    DeviceGuard guard(h->cfg.device);
    h->scratch.release();
    cudaFree(h->status);
  }
  delete h;
  return APK_OK;
}

const char* apk_moe_last_error(const apk_moe* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_moe_forward(apk_moe* h, const apk_moe_io* io) {
  if (!h || !h->status || !io) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    return forward(h, io);
  } catch (...) {
    return APK_ENOMEM;
  }
}

apk_status apk_moe_status(apk_moe* h, void* stream, int* device_status) {
  if (!h || !h->status || !device_status) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    DeviceGuard guard(h->cfg.device);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    APK_TRY(cu_status(cudaMemcpyAsync(device_status, h->status, sizeof(int), cudaMemcpyDeviceToHost, s), "status copy",
                      &h->err));
    APK_TRY(cu_status(cudaMemsetAsync(h->status, 0, sizeof(int), s), "status clear", &h->err));
    APK_TRY(cu_status(cudaStreamSynchronize(s), "cudaStreamSynchronize", &h->err));
    // a barrier that was given up has left its words half counted
    if (*device_status != 0 && h->scratch.data()) {
      APK_TRY(cu_status(cudaMemsetAsync(h->scratch.data(), 0, 256, s), "barrier clear", &h->err));
      APK_TRY(cu_status(cudaStreamSynchronize(s), "cudaStreamSynchronize", &h->err));
    }
    return APK_OK;
  } catch (...) {
    return APK_ENOMEM;
  }
}

}  // extern "C"
