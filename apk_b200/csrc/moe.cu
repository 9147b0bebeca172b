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
//   1  the tokens' experts (up to 16 tokens: every CTA picks them for itself,
//      which is cheaper than passing them through another barrier), then hidden = act(gate) * up, 8 gate and 8 up rows per item,
//      so both halves of a product sit in one thread's accumulator
//   2  each (token, choice) pair's output row in fp32 (one token: its output,
//      and no phase 3)
//   3  y[t] = sum over the choices, in their order, of p * row
// An item's rows are read by 1-16 warps of a CTA that split k: many when
// there are few items (a token or two), one when there are many.  Sums across
// warps go through shared memory in warp order.  Nothing depends on the order
// of arrival: an expert's tokens are a bit mask, so their columns are ordered
// by token.
//
// Rounding: logits, softmax, both products and the sum are fp32.  For a bf16
// result the hidden values, the second product's operand, are rounded to bf16
// once (2.3e-3 from 64 bits in the 2-norm, 1.7e-3 with the result's rounding
// alone; 64 tokens on 4 ungated experts of 2048 x 4096 87 us).  For an fp32
// result they are the sum of two bf16 values, 2^-17 of themselves off, and both
// products take 512 k at a time, as the linear layer does (that case 117 us).
#include <algorithm>
#include <mutex>
#include <new>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "linear.h"
#include "stream.cuh"

namespace apk {
namespace moe {

constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int MAX_TOKENS = 64, MAX_EXPERTS = 512, MAX_TOPK = 16;
constexpr int MAX_WIDTH = 1 << 26;  // of d_model and d_ff: a row index times one stays within 32 bits
constexpr int LOCAL_LOGITS = 2048, LOCAL_BYTES = 96 << 10;
constexpr int ROUND = 128;  // k of one warp's round: 8 16-byte weight loads a lane
constexpr int PIECE = 4;    // rounds that an accumulator of an fp32 result takes

struct Params {
  const uint16_t* x;
  const uint16_t* router;
  const uint16_t* w_in;
  const uint16_t* w_out;
  void* y;
  int* ids;      // [tokens][top_k] or null
  float* probs;  // [tokens][top_k] or null
  long long ldx, ldy;
  int tokens, experts, top_k, d, f, act, gated, renorm;
  int red_stride;  // floats of a warp's place in the shared sums
  int rsplit;    // slices of d_model in phase 0
  int local;     // every CTA computes all logits itself
  unsigned* barrier;  // [0] arrivals, [32] their number when this launch began, [33] whether one ran out
  int* status;
  long long limit;
  float* logits;  // [rsplit][tokens][experts]
  float2* choice; // [tokens][top_k] expert (as bits), weight
  uint16_t* hid;  // [tokens * top_k][f], rows grouped by expert; F32: [f / 8][2][8], both terms
  float* out;     // [tokens * top_k][d]
};

struct Shared {
  unsigned long long mask[MAX_EXPERTS];  // the tokens that chose an expert
  short active[MAX_EXPERTS];             // experts with tokens, ascending
  short base[MAX_EXPERTS];               // an active expert's first row
  short sel[MAX_TOKENS * MAX_TOPK];      // expert of (token, choice)
  short row[MAX_TOKENS * MAX_TOPK];      // and its row
  float prob[MAX_TOKENS * MAX_TOPK];
  unsigned char tok[MAX_TOKENS * MAX_TOPK];  // token of a row
  float logits[LOCAL_LOGITS];            // p.local: all of them
  int warp_n[WARPS], warp_rows[WARPS];
  int n_active;
  int abort;
  unsigned target;  // thread 0: the arrivals that the current barrier waits for
};

// A grid barrier in two halves, so that loads which do not depend on it can
// be issued between them (issued before the first, they would delay its
// fence).  After the second every CTA has arrived, and what it wrote before is
// visible.  One word counts arrivals and is never reset: a barrier is passed
// when it has grown by the grid's size, so the last arrival itself releases
// the others.  Another word holds the count at which a launch begins; it is
// moved on when the launch's last barrier lies behind every CTA.
__device__ __forceinline__ void grid_arrive(const Params& p, Shared& sh) {
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.target += gridDim.x;
    __threadfence();
    asm volatile("red.relaxed.gpu.global.add.u32 [%0], 1;" ::"l"(p.barrier) : "memory");
  }
}
// False: a barrier of this launch, or of one before it with these words that
// apk_moe_status has not been asked about, ran out.  The count is of no use then, and a CTA that
// went on by it could read what others have yet to write.
__device__ __forceinline__ bool grid_wait(const Params& p, Shared& sh) {
  if (threadIdx.x == 0 && !sh.abort) {
    long long t0 = 0;
    for (int n = 1;; ++n) {
      unsigned now;
      asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(p.barrier) : "memory");
      if ((int)(now - sh.target) >= 0) break;
      if ((n & 63) == 0) {
        const long long t = globaltimer_ns();
        if (t0 == 0) t0 = t;
        if (t - t0 > p.limit) {
          report_status(p.status, DEV_WAIT_TIMEOUT_SPIN, nullptr);
          *reinterpret_cast<volatile unsigned*>(p.barrier + 33) = 1;
          sh.abort = 1;
          break;
        }
      }
    }
    __threadfence();
  }
  __syncthreads();
  return sh.abort == 0;
}
__device__ __forceinline__ bool grid_barrier(const Params& p, Shared& sh) {
  grid_arrive(p, sh);
  return grid_wait(p, sh);
}
// The next launch begins where this one's last barrier ended.
__device__ __forceinline__ void grid_done(const Params& p, const Shared& sh) {
  if (blockIdx.x == 0 && threadIdx.x == 0) p.barrier[32] = sh.target;
}

struct Frag {
  uint4 a[4], b[4];
};
// One round of weight rows w0 (MMA rows g) and w1 (g + 8) at k0 + 32 u + 8 t.
template <bool BOTH = true>
__device__ __forceinline__ void load_round(Frag& f, const uint16_t* w0, const uint16_t* w1, int k0, int t, int k) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int at = k0 + 32 * u + 8 * t;
    const bool in = at < k;
    f.a[u] = in ? stream::ld_weights(w0 + at) : make_uint4(0, 0, 0, 0);
    f.b[u] = BOTH && in ? stream::ld_weights(w1 + at) : make_uint4(0, 0, 0, 0);
  }
}
// The two weight rows of a lane (MMA rows g and g + 8); null: none.
struct Rows {
  const uint16_t* w0;
  const uint16_t* w1;
};
// acc += `w` rows times the NT8 x 8 token rows xr, over the rounds first,
// first + step, ... of k.  On entry f holds round `first`; the next round's
// weights are in flight while one is multiplied, and at the end the first
// round of the next item's rows, so that the loads do not pause between items.
// Load reads 16 bytes of a token row, whose values have TERMS bf16 terms.
// EXACT: the tensor core truncates as it adds, a bias of about 1e-9 per k of
// the result; so every 512 k are added with rounding to a total in the shared
// memory given.  (The accumulators of 64 tokens twice would not fit the
// registers.)
template <int NT8, bool EXACT = false, class Load>
__device__ __forceinline__ void stream_rows(float (&acc)[NT8][4], Frag& f, const Rows w, const Rows next_item,
                                            const uint16_t* const (&xr)[NT8], int k, int first, int step, int t,
                                            Load ld, float* total = nullptr) {
  const int begin = first * ROUND;
  auto flush = [&](bool back) {
#pragma unroll
    for (int i = 0; i < NT8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float& sum = total[(i * 4 + c) * 32];
        const float s = sum + acc[i][c];
        if (back) acc[i][c] = s;
        else sum = s, acc[i][c] = 0.f;
      }
  };
  if constexpr (EXACT)
#pragma unroll
    for (int i = 0; i < NT8 * 4; ++i) total[i * 32] = 0.f;
  int left = PIECE;
#pragma unroll 1
  for (int k0 = begin; k0 < k; k0 += step * ROUND) {
    const int next = k0 + step * ROUND;
    Frag n;
    if (NT8 <= 2) load_round(n, w.w0, w.w1, next, t, k);  // (past the end: zero, nothing read)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = k0 + 32 * u + 8 * t;
      uint4 c[NT8];
#pragma unroll
      for (int v = 0; v < Load::TERMS; ++v) {
#pragma unroll
        for (int i = 0; i < NT8; ++i)
          c[i] = at < k ? ld(xr[i] + Load::TERMS * at + 8 * v) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NT8; ++i) {
          stream::mma_bf16(acc[i], f.a[u].x, f.b[u].x, f.a[u].y, f.b[u].y, c[i].x, c[i].y);
          stream::mma_bf16(acc[i], f.a[u].z, f.b[u].z, f.a[u].w, f.b[u].w, c[i].z, c[i].w);
        }
      }
    }
    if (NT8 <= 2) f = n;
    else if (next < k) load_round(f, w.w0, w.w1, next, t, k);
    if (EXACT && --left == 0) {
      flush(false);
      left = PIECE;
    }
  }
  if constexpr (EXACT) flush(true);
  if (next_item.w0) load_round(f, next_item.w0, next_item.w1, begin, t, k);
}

struct LdConst {  // the layer's input: not written during the kernel
  static constexpr int TERMS = 1;
  __device__ uint4 operator()(const uint16_t* p) const { return __ldg(reinterpret_cast<const uint4*>(p)); }
};
template <int N>
struct LdWritten {  // written by other CTAs in an earlier phase: from L2
  static constexpr int TERMS = N;
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

// Warps that share an item: 1, 2, ... 16, by the least time of a warp in
// rounds: its items times the rounds of one and about three more for the join
// and what the loads lose at an item's end.
__device__ __forceinline__ int warps_per_item(unsigned items, int k) {
  int best = 1;
  unsigned least = ~0u;
  const unsigned rounds = (k + ROUND - 1) / ROUND;
#pragma unroll
  for (int lg = 0; lg <= 4; ++lg) {
    const unsigned slots = gridDim.x * (WARPS >> lg);
    const unsigned cost = (items + slots - 1) / slots * (((rounds + (1u << lg) - 1) >> lg) + 3);
    if (cost < least) {
      least = cost;
      best = 1 << lg;
    }
  }
  return best;
}

// A phase's items in two parts: full sweeps of one item per warp, then the
// rest, shared by more warps each.
struct Walk {
  struct Part {
    int ws, first, end, step;
  };
  int bulk, items, ws;
  __device__ Walk(int n, int k) : items(n) {
    const int warps = gridDim.x * WARPS;
    ws = warps_per_item(n, k);
    bulk = 0;
    if (n > warps && ws == 1) {
      bulk = n / warps * warps;
      ws = warps_per_item(n - bulk, k);
    }
  }
  __device__ Part part(int i, int warp) const {
    if (i == 0) return {1, warp * (int)gridDim.x + (int)blockIdx.x, bulk, (int)gridDim.x * WARPS};
    return {ws, bulk + warp / ws * (int)gridDim.x + (int)blockIdx.x, items, (int)gridDim.x * (WARPS / ws)};
  }
};

// Rows of expert a's tile in the first product.  Gated: MMA row g is gate
// f0 + g and row g + 8 its up; else features f0 + g and f0 + g + 8.
__device__ __forceinline__ Rows rows_in(const Params& p, const Shared& sh, int a, int tile, int g) {
  const uint16_t* w = p.w_in + (long long)sh.active[a] * (p.gated ? 2 * p.f : p.f) * p.d;
  const int f0 = tile * (p.gated ? 8 : 16);
  const int r0 = min(f0 + g, p.f - 1), r1 = p.gated ? p.f + r0 : min(f0 + g + 8, p.f - 1);
  return {w + (long long)r0 * p.d, w + (long long)r1 * p.d};
}
__device__ __forceinline__ Rows rows_out(const Params& p, const Shared& sh, int a, int tile, int g) {
  const uint16_t* w = p.w_out + (long long)sh.active[a] * p.d * p.f;
  const int d0 = tile * 16;
  return {w + (long long)min(d0 + g, p.d - 1) * p.f, w + (long long)min(d0 + g + 8, p.d - 1) * p.f};
}

// F32 of these and of the kernel: the result's type.
template <int NT8, bool F32>
__device__ __forceinline__ void item_in(const Params& p, const Shared& sh, float* red, Frag& f, Rows w, Rows next, int a,
                                        int tile, int n, int ws) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int base = sh.base[a], f0 = tile * (p.gated ? 8 : 16);
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.x + sh.tok[base + min(8 * i + g, n - 1)] * p.ldx;
  float acc[NT8][4] = {};
  // (totals in the warp's place in the shared sums, which join_warps takes after this)
  stream_rows<NT8, F32>(acc, f, w, next, xr, p.d, warp & (ws - 1), ws, t, LdConst(), red + warp * p.red_stride + lane);
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
        uint16_t* h = p.hid + ((long long)(base + col) * p.f * (1 + F32));
        auto put = [&](int at, float v) {
          uint16_t r;
          asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
          if (at >= p.f) return;
          if constexpr (!F32) {
            h[at] = r;
          } else {
            uint16_t* const two = h + 2 * at - (at & 7);
            two[0] = r;
            const bool finite = (r & 0x7F80) != 0x7F80;  // (an infinity stays one)
            const float rest = finite ? v - __uint_as_float((uint32_t)r << 16) : 0.f;
            asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(rest));
            two[8] = r;
          }
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

template <int NT8, bool F32>
__device__ __forceinline__ void item_out(const Params& p, const Shared& sh, float* red, Frag& f, Rows w, Rows next,
                                         int a, int tile, int n, int ws) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int base = sh.base[a], d0 = tile * 16;
  const uint16_t* xr[NT8];
#pragma unroll
  for (int i = 0; i < NT8; ++i) xr[i] = p.hid + ((long long)(base + min(8 * i + g, n - 1)) * p.f * (1 + F32));
  float acc[NT8][4] = {};
  stream_rows<NT8, F32>(acc, f, w, next, xr, p.f, warp & (ws - 1), ws, t, LdWritten<1 + F32>(),
                        red + warp * p.red_stride + lane);
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

// Partial logits of 16 experts for the 16 tokens from t0, into dst[token][experts].
__device__ __forceinline__ void item_router(const Params& p, float* red, int tile, int slice, int slices, int t0,
                                            float* dst) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int e0 = tile * 16;
  const uint16_t* xr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) xr[i] = p.x + min(t0 + 8 * i + g, p.tokens - 1) * p.ldx;
  float acc[2][4] = {};
  const Rows w = {p.router + (long long)min(e0 + g, p.experts - 1) * p.d,
                  p.router + (long long)min(e0 + g + 8, p.experts - 1) * p.d};
  Frag f;
  load_round(f, w.w0, w.w1, (slice * WARPS + warp) * ROUND, t, p.d);
  stream_rows<2>(acc, f, w, Rows{}, xr, p.d, slice * WARPS + warp, slices * WARPS, t, LdConst());
  join_warps<2>(acc, red, p.red_stride, WARPS, warp, lane);
  if (warp) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int tok = t0 + 8 * i + 2 * t + (c & 1), e = e0 + g + 8 * (c >> 1);
      if (tok < p.tokens && e < p.experts) dst[tok * p.experts + e] = acc[i][c];
    }
}

template <bool F32>
__device__ __forceinline__ void put_y(const Params& p, long long at, float v) {
  if constexpr (F32) {
    static_cast<float*>(p.y)[at] = v;
  } else {
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
    static_cast<uint16_t*>(p.y)[at] = r;
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

// One warp picks a token's experts from its logits: top_k rounds of "largest
// key, lowest index", then their softmax over all experts.  Lane j of the
// first top_k gets the j-th choice and its weight.  PER experts a lane.
template <int PER, class Load>
__device__ __forceinline__ void route_token(const Params& p, Load logit, int& my_e, float& my_p) {
  const int lane = threadIdx.x & 31;
  float v[PER];
  unsigned key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < p.experts ? logit(lane + 32 * i) : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = lane + 32 * i < p.experts ? order_key(v[i]) : 0;  // 0: below any logit's key
  float my_v = 0.f;
  my_e = 0;
  for (int j = 0; j < p.top_k; ++j) {
    unsigned k = key[0];
    int i0 = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > k) {
        k = key[i];
        i0 = i;
      }
    const unsigned top = __reduce_max_sync(~0u, k);
    const int at = (int)__reduce_min_sync(~0u, k == top ? (unsigned)(lane + 32 * i0) : ~0u);
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == lane + 32 * i) {
        key[i] = 0;
        mine = v[i];
      }
    mine = __shfl_sync(~0u, mine, at & 31);
    if (lane == j) {
      my_e = at;
      my_v = mine;
    }
  }
  // the first choice has the largest logit (or is a NaN, as every probability then is)
  const float best = __shfl_sync(~0u, my_v, 0);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 32 * i < p.experts) sum += __expf(v[i] - best);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  my_p = lane < p.top_k ? __fdividef(__expf(my_v - best), sum) : 0.f;
  if (p.renorm) {
    float chosen = my_p;
#pragma unroll
    for (int o = MAX_TOPK / 2; o; o >>= 1) chosen += __shfl_xor_sync(~0u, chosen, o);
    my_p = __fdividef(my_p, chosen);
  }
}
template <class Load>
__device__ __forceinline__ void route_token(const Params& p, Load logit, int& my_e, float& my_p) {
  if (p.experts <= 32) route_token<1>(p, logit, my_e, my_p);
  else if (p.experts <= 64) route_token<2>(p, logit, my_e, my_p);
  else if (p.experts <= 128) route_token<4>(p, logit, my_e, my_p);
  else if (p.experts <= 256) route_token<8>(p, logit, my_e, my_p);
  else route_token<16>(p, logit, my_e, my_p);
}

// One token: the output without the sum's barrier.  A CTA takes `ROWS` (8 or
// 16) of the output's rows over all chosen experts, its warps splitting the
// (expert, round) pairs; the probabilities are applied per expert.
template <int ROWS, bool F32>
__device__ __forceinline__ bool one_token_out(const Params& p, Shared& sh, float* red) {
  constexpr int TERMS = 1 + F32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rounds = (p.f + ROUND - 1) / ROUND, units = p.top_k * rounds;
  auto load = [&](Frag& f, int tile, int u) {
    const long long r0 = min(tile * ROWS + g, p.d - 1), r1 = min(tile * ROWS + g + 8, p.d - 1);
    const int j = u / rounds;
    const uint16_t* w = p.w_out + (long long)sh.sel[j] * p.d * p.f;
    load_round<ROWS == 16>(f, w + r0 * p.f, w + r1 * p.f, (u - j * rounds) * ROUND, t, p.f);
  };
  Frag f;
  grid_arrive(p, sh);
  if (warp < units && (int)blockIdx.x * ROWS < p.d) load(f, blockIdx.x, warp);
  if (!grid_wait(p, sh)) return false;
  for (int tile = blockIdx.x; tile * ROWS < p.d; tile += gridDim.x) {
    float s0 = 0.f, s1 = 0.f;
    for (int u = warp; u < units; u += WARPS) {
      const int j = u / rounds, k0 = (u - j * rounds) * ROUND;
      const uint16_t* h = p.hid + sh.row[j] * p.f * TERMS;
      Frag n;  // the next unit, of this tile or the next one
      if (u + WARPS < units) load(n, tile, u + WARPS);
      else if ((tile + (int)gridDim.x) * ROWS < p.d) load(n, tile + gridDim.x, warp);
      float acc[4] = {};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = k0 + 32 * v + 8 * t;
#pragma unroll
        for (int i = 0; i < TERMS; ++i) {
          const uint4 c = at < p.f ? LdWritten<TERMS>()(h + TERMS * at + 8 * i) : make_uint4(0, 0, 0, 0);
          stream::mma_bf16(acc, f.a[v].x, f.b[v].x, f.a[v].y, f.b[v].y, c.x, c.y);
          stream::mma_bf16(acc, f.a[v].z, f.b[v].z, f.a[v].w, f.b[v].w, c.z, c.w);
        }
      }
      s0 += sh.prob[j] * acc[0];
      s1 += sh.prob[j] * acc[2];
      f = n;
    }
    // every column holds the same token: column 0 is lane 4g's
    if (t == 0) {
      red[warp * 16 + g] = s0;
      red[warp * 16 + g + 8] = s1;
    }
    __syncthreads();
    const int d = tile * ROWS + (int)threadIdx.x;
    if (threadIdx.x < ROWS && d < p.d) {
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) y += red[w * 16 + threadIdx.x];
      put_y<F32>(p, d, y);
    }
    __syncthreads();
  }
  return true;
}

template <bool F32>
__global__ void __launch_bounds__(THREADS, 1) moe_layer(const __grid_constant__ Params p) {
  extern __shared__ float red[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint2 begun = {};
  if (tid == 0)
    asm volatile("ld.volatile.global.v2.u32 {%0, %1}, [%2];" : "=r"(begun.x), "=r"(begun.y) : "l"(p.barrier + 32));
  auto begin = [&]() {  // (behind the first loads of weights, so that these do not wait for the two words)
    if (tid != 0) return;
    sh.target = begun.x;
    sh.abort = begun.y != 0;
  };
  for (int e = tid; e < p.experts; e += THREADS) sh.mask[e] = 0;

  // -------- 0: logits --------
  const int etiles = (p.experts + 15) / 16;
  if (p.local) {
    for (int tile = 0; tile < etiles; ++tile) item_router(p, red, tile, 0, 1, 0, sh.logits);
    begin();
    __syncthreads();
  } else {
    const int tgroups = (p.tokens + 15) / 16;
    for (int it = blockIdx.x; it < etiles * p.rsplit * tgroups; it += gridDim.x) {
      const int slice = it / etiles % p.rsplit;
      item_router(p, red, it % etiles, slice, p.rsplit, it / (etiles * p.rsplit) * 16,
                  p.logits + (long long)slice * p.tokens * p.experts);
    }
    begin();
    if (!grid_barrier(p, sh)) return;
  }

  // -------- 1: routing (by every CTA), then the hidden values --------
  // A logit is the sum of its slices.  Up to 16 tokens: warp w of every CTA
  // routes token w.  More: warp 0 of CTA b routes token b for all, and another
  // barrier passes the choices on (64 tokens of 128 experts: 8 us instead of 15).
  const bool shared_out = p.tokens > WARPS;
  auto each_token = [&](int tok) {
    int my_e;
    float my_p;
    route_token(
        p,
        [&](int e) {
          if (p.local) return sh.logits[tok * p.experts + e];
          float v[8];
#pragma unroll
          for (int s = 0; s < 8; ++s)
            v[s] = s < p.rsplit ? __ldcg(p.logits + ((long long)s * p.tokens + tok) * p.experts + e) : 0.f;
          return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        },
        my_e, my_p);
    if (lane < p.top_k) {
      if (shared_out) {
        p.choice[tok * p.top_k + lane] = make_float2(__int_as_float(my_e), my_p);
      } else {
        sh.sel[tok * p.top_k + lane] = (short)my_e;
        sh.prob[tok * p.top_k + lane] = my_p;
        atomicOr(&sh.mask[my_e], 1ull << tok);
      }
    }
  };
  if (shared_out) {
    if (warp == 0)
      for (int tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) each_token(tok);
    if (!grid_barrier(p, sh)) return;
    for (int i = tid; i < p.tokens * p.top_k; i += THREADS) {
      const float2 c = __ldcg(p.choice + i);
      // (an index even if, against the rules, another launch uses this buffer at the same time)
      const int e = (int)min(__float_as_uint(c.x), (unsigned)p.experts - 1);
      sh.sel[i] = (short)e;
      sh.prob[i] = c.y;
      atomicOr(&sh.mask[e], 1ull << (i / p.top_k));
    }
  } else if (warp < p.tokens) {
    each_token(warp);
  }
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
    if (n > 0 || tid == THREADS - 1) {
      const int before = min(warp, (p.experts + 31) / 32);  // warps with experts below this one
      for (int w = 0; w < before; ++w) {
        a += sh.warp_n[w];
        r += sh.warp_rows[w];
      }
    }
    if (n > 0) {
      sh.active[a] = (short)tid;
      sh.base[a] = (short)r;
      unsigned long long m = sh.mask[tid];
      for (int i = 0; m; ++i, m &= m - 1) {
        const int tok = __ffsll((long long)m) - 1;
        sh.tok[r + i] = (unsigned char)tok;
        for (int j = 0; j < p.top_k; ++j)
          if (sh.sel[tok * p.top_k + j] == tid) sh.row[tok * p.top_k + j] = (short)(r + i);
      }
    }
    if (tid == THREADS - 1) sh.n_active = a + (n > 0);
  }
  __syncthreads();
  const int n_active = sh.n_active;
  if (blockIdx.x == 0 && !sh.abort) {
    for (int i = tid; i < p.tokens * p.top_k; i += THREADS) {
      if (p.ids) p.ids[i] = sh.sel[i];
      if (p.probs) p.probs[i] = sh.prob[i];
    }
  }
  // the tokens of a warp's item, as the MMA's N axis
  auto by_columns = [&](int n, auto f) {
    if (n <= 8) f(std::integral_constant<int, 1>());
    else if (n <= 16) f(std::integral_constant<int, 2>());
    else if (n <= 32) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, 8>());
  };
  Frag frag;
  {
    const int tiles = (p.f + (p.gated ? 7 : 15)) / (p.gated ? 8 : 16);
    const Walk walk(n_active * tiles, p.d);
    for (int part = walk.bulk ? 0 : 1; part < 2; ++part) {
      const Walk::Part q = walk.part(part, warp);
      Rows w = {};
      if (q.first < q.end) {
        w = rows_in(p, sh, q.first / tiles, q.first % tiles, g);
        load_round(frag, w.w0, w.w1, (warp & (q.ws - 1)) * ROUND, t, p.d);
      }
      for (int it = q.first; it < q.end; it += q.step) {
        const int a = it / tiles, next = it + q.step;
        const Rows wn = next < q.end ? rows_in(p, sh, next / tiles, next % tiles, g) : Rows{};
        const int n = __popcll(sh.mask[sh.active[a]]);
        by_columns(n, [&](auto c) { item_in<decltype(c)::value, F32>(p, sh, red, frag, w, wn, a, it % tiles, n, q.ws); });
        w = wn;
      }
      __syncthreads();  // the second part's groups are others
    }
  }

  // -------- 2: output rows of the pairs --------
  if (p.tokens == 1) {
    const bool ok =
        (p.d + 7) / 8 <= 2 * (int)gridDim.x ? one_token_out<8, F32>(p, sh, red) : one_token_out<16, F32>(p, sh, red);
    if (ok) grid_done(p, sh);
    return;
  }
  {
    const int tiles = (p.d + 15) / 16;
    const Walk walk(n_active * tiles, p.f);
    const int start = walk.bulk ? 0 : 1;
    grid_arrive(p, sh);
    for (int part = start; part < 2; ++part) {
      const Walk::Part q = walk.part(part, warp);
      Rows w = {};
      if (q.first < q.end) {  // (the first part's weights travel while the barrier is waited for)
        w = rows_out(p, sh, q.first / tiles, q.first % tiles, g);
        load_round(frag, w.w0, w.w1, (warp & (q.ws - 1)) * ROUND, t, p.f);
      }
      if (part == start && !grid_wait(p, sh)) return;
      for (int it = q.first; it < q.end; it += q.step) {
        const int a = it / tiles, next = it + q.step;
        const Rows wn = next < q.end ? rows_out(p, sh, next / tiles, next % tiles, g) : Rows{};
        const int n = __popcll(sh.mask[sh.active[a]]);
        by_columns(n, [&](auto c) { item_out<decltype(c)::value, F32>(p, sh, red, frag, w, wn, a, it % tiles, n, q.ws); });
        w = wn;
      }
      __syncthreads();
    }
  }
  if (!grid_barrier(p, sh)) return;
  grid_done(p, sh);

  // -------- 3: weighted sum --------
  const int quads = p.d / 4;
  for (int i = blockIdx.x * THREADS + tid; i < p.tokens * quads; i += gridDim.x * THREADS) {
    const int tok = i / quads, d = (i - tok * quads) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < p.top_k; ++j) {
      const float w = sh.prob[tok * p.top_k + j];
      const float4 o = __ldcg(reinterpret_cast<const float4*>(p.out + (long long)sh.row[tok * p.top_k + j] * p.d + d));
      s.x += w * o.x;
      s.y += w * o.y;
      s.z += w * o.z;
      s.w += w * o.w;
    }
    const long long at = tok * p.ldy + d;
    put_y<F32>(p, at, s.x);
    put_y<F32>(p, at + 1, s.y);
    put_y<F32>(p, at + 2, s.z);
    put_y<F32>(p, at + 3, s.w);
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
  if (c.d_model > moe::MAX_WIDTH || c.d_ff > moe::MAX_WIDTH)
    return h->err.fail(APK_EINVAL, "d_model %d, d_ff %d: at most 2^26", c.d_model, c.d_ff);
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
  for (auto kernel : {moe::moe_layer<false>, moe::moe_layer<true>}) {
    APK_TRY(cu_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, moe::red_bytes(8)),
                      "preparing the expert kernel", &h->err));
    int per_sm = 0;
    APK_TRY(cu_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, moe::THREADS, moe::red_bytes(8)),
                      "preparing the expert kernel", &h->err));
    if (per_sm < 1) return h->err.fail(APK_EUNSUPPORTED, "the expert kernel does not fit an SM");
  }
  return h->scratch.open(c.device, &h->err);
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
  const size_t b_log = up256((size_t)p.rsplit * io->tokens * c.experts * 4), b_hid = up256((pairs * c.d_ff * 2) << (io->y_dtype == APK_F32));
  const size_t b_out = up256(pairs * c.d_model * 4), b_choice = up256(pairs * 8);
  APK_TRY(h->scratch.enter(s, &h->err));
  ScratchUse use(&h->scratch, &h->err);
  APK_TRY(use.begin(256 + b_log + b_hid + b_out + b_choice, 256));
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
  p.barrier = reinterpret_cast<unsigned*>(b);
  p.status = h->scratch.status();
  p.limit = c.wait_limit_ns;
  p.logits = reinterpret_cast<float*>(b + 256);
  p.hid = reinterpret_cast<uint16_t*>(b + 256 + b_log);
  p.out = reinterpret_cast<float*>(b + 256 + b_log + b_hid);
  p.choice = reinterpret_cast<float2*>(b + 256 + b_log + b_hid + b_out);
  // a small router (16 tokens, 96 KB of weights at most) is read by every CTA
  // from L2 in less time than a grid barrier takes
  p.local = io->tokens <= 16 && io->tokens * c.experts <= moe::LOCAL_LOGITS &&
            (long long)c.experts * c.d_model * 2 <= moe::LOCAL_BYTES;
  const int nt8 = io->tokens <= 8 ? 1 : io->tokens <= 16 ? 2 : io->tokens <= 32 ? 4 : 8;
  p.red_stride = std::max(nt8, 2) * 128;  // (the router's items have two tiles of tokens)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.gridDim = dim3(h->sms);
  cfg.blockDim = dim3(moe::THREADS);
  cfg.dynamicSmemBytes = moe::red_bytes(std::max(nt8, 2));
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  APK_TRY(cu_status(cudaLaunchKernelEx(&cfg, io->y_dtype == APK_F32 ? moe::moe_layer<true> : moe::moe_layer<false>, p),
                    "launching the expert kernel", &h->err));
  return use.end();
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
  delete h;
  return APK_OK;
}

const char* apk_moe_last_error(const apk_moe* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_moe_forward(apk_moe* h, const apk_moe_io* io) {
  if (!h || !h->scratch.status() || !io) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    return forward(h, io);
  } catch (...) {
    return APK_ENOMEM;
  }
}

apk_status apk_moe_status(apk_moe* h, void* stream, int* device_status) {
  if (!h || !h->scratch.status() || !device_status) return APK_EINVAL;
  try {
    std::lock_guard<std::mutex> lock(h->mu);
    DeviceGuard guard(h->cfg.device);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    APK_TRY(cu_status(cudaMemcpyAsync(device_status, h->scratch.status(), sizeof(int), cudaMemcpyDeviceToHost, s), "status copy",
                      &h->err));
    APK_TRY(cu_status(cudaMemsetAsync(h->scratch.status(), 0, sizeof(int), s), "status clear", &h->err));
    APK_TRY(cu_status(cudaStreamSynchronize(s), "cudaStreamSynchronize", &h->err));
    // a barrier that was given up has left its words half counted, a graph's in
    // the buffer that it was captured with
    return *device_status != 0 ? h->scratch.clear(256, s, &h->err) : APK_OK;
  } catch (...) {
    return APK_ENOMEM;
  }
}

}  // extern "C"
