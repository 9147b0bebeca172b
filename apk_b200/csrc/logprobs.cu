// Log probabilities of given tokens, entropy and the largest alternatives of
// rows of logits, and their gradient (apk_logprobs_* of include/apk.h).  No
// counterpart in the reference, which multiplies bare matrices
// (src/tcyield.cu:91-356).
//
//   m = max x,  S = sum exp(x - m),  l = (x - m) - log S,  p = exp(l)
//   entropy H = log S - sum exp(x - m) (x - m) / S
//   dx_j = dlogprob ([j = token] - p_j) - dentropy p_j (l_j + H)
//
// Bound by memory: the logits are read once, with a running maximum and sums
// that are scaled where it grows.  A value costs one multiply-add,
//   t = x L - c,  c = m L rounded,  L = log2(e) rounded,
// one 2^t and the two sums, of 2^t and of 2^t t, in pairs (f32x2).  What c's
// and L's roundings move is taken back at the end, once a row in 64 bits: the
// sums belong to the exact reference c / L in place of m.  Masked values (-inf)
// are raised to -1e9, which leaves them 2^t = 0 without a 0 * inf; rows whose
// maximum is not between -1e8 and 1e8 are taken again, step by step.
//
// The alternatives come out of the same pass.  The first rounds of 2048 values,
// as many as are on their way, give a bound that their k-th largest value reaches; a value that reaches the
// bound is put into a buffer in shared memory.  As rounds go by, one warp at a
// time raises the bound by what the buffer holds, while the others go on: any
// bound that k values reach is right, so nobody waits for anybody.  Between n
// and 2 n values about k pass (the n-th value is among the k largest so far
// with chance k / n).  At the end the buffer is cut to its k largest.  Rows in
// which far more pass, ascending ones, fill it up: they are taken again, cut
// after every round.
#include <algorithm>

#include "act.cuh"
#include "ops.cuh"
#include "ops.h"

namespace apk {
namespace logp {

constexpr int THREADS = 256, ROUND = THREADS * 8;  // values of a block's round
constexpr int MAX_TOP = 32, MAX_SPLIT = 16;
constexpr int ROOM = ROUND + MAX_TOP;              // of the buffer: the list, and a whole round
template <bool F32>
constexpr int AHEAD = F32 ? 2 : 4;                 // eights of a thread on their way
constexpr float LOWEST = -1e9f;                    // (as bf16: 0xCE6E)
// The running maximum before the first value, and where it ends: there c is
// rounded to steps of 16, and 2^t of the maximum itself stays below 2^8.
constexpr float NONE = -1e8f, MOST = 1e8f;
static_assert(MAX_SPLIT * MAX_TOP <= ROOM, "the parts' lists fit the buffer");

struct Params {
  const uint8_t* x;
  long long ld;      // bytes
  const void* tokens;
  float* logprob;
  float* entropy;
  int* ids;
  float* tops;
  float2* stats;
  int rows, vocabulary, top, split, tokens_64;
};

// What orders alternatives: the value (a NaN above all, -0 as 0), then the
// lower index; larger is better, 0 is none.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);  // (of a NaN: a NaN)
}
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  return (unsigned long long)order_of(x) << 32 | ~(uint32_t)i;
}
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp_of(float d) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * LOG2E));
  return e;
}

// A row's values by eights, from the aligned place at or before its first.
template <bool F32>
struct Row {
  const uint8_t* base;
  int shift, n;
  unsigned lo, whole;  // the eights that lie in the row whole: `whole` from `lo` on
  __device__ __forceinline__ Row(const uint8_t* p, int n_) : n(n_) {
    const int bytes = (int)(reinterpret_cast<uintptr_t>(p) & (F32 ? 31 : 15));
    base = p - bytes;
    shift = bytes / (F32 ? 4 : 2);
    lo = shift ? 1 : 0;
    const unsigned hi = (unsigned)(n + shift) / 8;
    whole = hi > lo ? hi - lo : 0;
  }
  __device__ __forceinline__ int eights() const { return (int)((unsigned)(n + shift + 7) / 8); }
  __device__ __forceinline__ int first(int v) const { return v * 8 - shift; }
  static __device__ __forceinline__ void none(ops::Raw<F32>& r) {
    const uint32_t w = F32 ? 0xFF800000u : 0xFF80FF80u;
    r.a = make_uint4(w, w, w, w);
    if constexpr (F32) r.b = r.a;
  }
  // one that lies in the row whole
  __device__ __forceinline__ void load_whole(int v, ops::Raw<F32>& r) const {
    const uint8_t* q = base + (long long)v * (F32 ? 32 : 16);
    if constexpr (F32)
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
                   : "l"(q)
                   : "memory");
    else
      r.a = __ldcs(reinterpret_cast<const uint4*>(q));
  }
  // into a row that starts at `out`, at the same place within the alignment
  __device__ __forceinline__ void store(int v, uint8_t* out, const ops::Raw<F32>& o) const {
    const int e = first(v);
    uint8_t* q = out + (long long)e * (F32 ? 4 : 2);
    if ((unsigned)v - lo < whole) {
      __stcs(reinterpret_cast<uint4*>(q), o.a);
      if constexpr (F32) __stcs(reinterpret_cast<uint4*>(q) + 1, o.b);
      return;
    }
    float y[8];
    ops::unpack(o, y);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i >= 0 && e + i < n) ops::st_any(out, e + i, y[i], F32);
  }
  // -inf where the row does not reach
  __device__ __forceinline__ void load(int v, ops::Raw<F32>& r) const {
    if ((unsigned)v - lo < whole) {
      load_whole(v, r);
      return;
    }
    const uint8_t* q = base + (long long)v * (F32 ? 32 : 16);
    none(r);
    const int e = first(v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i >= 0 && e + i < n) ops::set1(r, i, q, i);
  }
};

using ops::add2;
using ops::fma2;
using ops::pair2;
using ops::unpair2;
__device__ __forceinline__ float ex2(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// Eight values raised to LOWEST, in pairs; the largest of them as they were (a
// NaN stays, and is the largest).
__device__ __forceinline__ float raised(const ops::Raw<false>& r, unsigned long long (&x)[4]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
  uint32_t m, n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(w[i]), "r"(0xCE6ECE6Eu));
    x[i] = pair2(ops::bf_lo(v), ops::bf_hi(v));
  }
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(w[0]), "r"(w[1]));
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(n) : "r"(w[2]), "r"(w[3]));
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(n));
  return max_nan(ops::bf_lo(m), ops::bf_hi(m));
}
__device__ __forceinline__ float raised(const ops::Raw<true>& r, unsigned long long (&x)[4]) {
  float v[8];
  ops::unpack(r, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pair2(max_nan(v[2 * i], LOWEST), max_nan(v[2 * i + 1], LOWEST));
  return max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])), max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
}

// Sums of 2^t and 2^t t, t = x L - c, c = m L.
struct Soft {
  float m = NONE, s = 0.f, u = 0.f;
  // (never contracted into a multiply-add: what is added up goes by the rounded product)
  static __device__ __forceinline__ float c_of(float m) { return __fmul_rn(m, LOG2E); }
  __device__ __forceinline__ void raise(float to) {
    const float d = c_of(m) - c_of(to), f = ex2(d);
    u = f * fmaf(s, fmaxf(d, -2000.f), u);  // (f is 0 there: no 0 * inf)
    s *= f;
    m = to;
  }
};
// A thread's sums, over two accumulators each.  The reference follows the
// maximum in steps of more than STEP: with every new maximum in any lane, a
// warp would scale in nearly every round.  (What the entropy's sum is rounded
// by grows with the distance: 16 was as fast and cost a digit.)
constexpr float STEP = 2.f;
struct Sums {
  float m = NONE, most = NONE;
  unsigned long long s = 0, u = 0, minus_c;
  __device__ __forceinline__ Sums() { minus_c = pair2(-Soft::c_of(NONE), -Soft::c_of(NONE)); }
  __device__ __forceinline__ void add(const unsigned long long (&x)[4], float top) {
    most = fmaxf(most, top);
    if (top > m + STEP) {
      Soft a = sums();
      a.raise(top);
      m = top;
      s = pair2(a.s, 0.f);
      u = pair2(a.u, 0.f);
      minus_c = pair2(-Soft::c_of(m), -Soft::c_of(m));
    }
    const unsigned long long l = pair2(LOG2E, LOG2E);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long t = fma2(x[i], l, minus_c);
      float t0, t1;
      unpair2(t, t0, t1);
      const unsigned long long e = pair2(ex2(t0), ex2(t1));
      s = add2(s, e);
      u = fma2(e, t, u);
    }
  }
  __device__ __forceinline__ Soft sums() const {
    Soft a;
    float x, y;
    unpair2(s, x, y);
    a.s = x + y;
    unpair2(u, x, y);
    a.u = x + y;
    a.m = m;
    return a;
  }
  __device__ __forceinline__ Soft soft() const {
    Soft a = sums();
    a.raise(most);
    return a;
  }
};

struct Shared {
  unsigned long long buf[ROOM];  // 0: not written
  unsigned long long limit;      // k values reach it
  unsigned long long group[32];
  unsigned long long list[MAX_TOP];
  float m[8], s[8], u[8];
  int count;
  // of a row's first block: the parts' results
  unsigned long long lists[MAX_SPLIT * MAX_TOP];
  float4 parts[MAX_SPLIT];
};

// A row's maximum, log of the sum of exp(x - m), and entropy.
struct Result {
  float m, log_s, entropy;
};
__device__ __forceinline__ Result result_of(const Soft& a) {
  // sum 2^(x L - c): its reference is c / L
  constexpr double per_l = 1.0 / (double)LOG2E;
  const float log_s = logf(a.s);
  return {a.m, (float)(log_s + ((double)Soft::c_of(a.m) * per_l - a.m)), log_s - a.u / a.s * (float)per_l};
}
// The same by the definition, for a row whose maximum is far out: x - m, and
// exp of it, value by value.  All threads.
template <bool F32>
__device__ __noinline__ Result far_out(const uint8_t* x, int n, Shared& sh) {
  float m = -INFINITY, s = 0.f, u = 0.f;
  bool nan = false;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const float v = ops::ld_any(x, i, F32);
    nan |= v != v;
    m = fmaxf(m, v);
  }
  auto over_all = [&](float v, auto f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.m[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.m[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) v = f(v, sh.m[w]);
    return v;
  };
  m = over_all(m, [](float a, float b) { return fmaxf(a, b); });
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const float d = max_nan(ops::ld_any(x, i, F32) - m, -1000.f), e = exp_of(d);
    s += e;
    u = fmaf(e, d, u);
  }
  s = over_all(nan ? NAN : s, [](float a, float b) { return a + b; });
  u = over_all(u, [](float a, float b) { return a + b; });
  const float log_s = logf(s);
  return {m, log_s, log_s - u / s};
}

// The k-th largest of a warp's keys; 0 if fewer lanes have any.
__device__ __forceinline__ unsigned long long kth_of(unsigned long long key, int k) {
  if (k > 8) {  // by every lane's rank: 32 steps that do not wait for one another
    const int lane = threadIdx.x & 31;
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
      const unsigned long long other = __shfl_sync(0xFFFFFFFFu, key, i);
      rank += other > key || (other == key && i < lane);  // (equal ones are 0s)
    }
    return __shfl_sync(0xFFFFFFFFu, key, __ffs(__ballot_sync(0xFFFFFFFFu, rank == k - 1)) - 1);
  }
  const uint32_t low = (uint32_t)key;
  uint32_t left = (uint32_t)(key >> 32), top;
  while (true) {  // values from above, those that are equal at once
    top = __reduce_max_sync(0xFFFFFFFFu, left);
    if (top == 0) return 0;
    const int n = __popc(__ballot_sync(0xFFFFFFFFu, left == top));
    if (n >= k) break;
    k -= n;
    if (left == top) left = 0;
  }
  uint32_t tied = left == top ? low : 0, at;
  while (true) {  // (~index: no two are equal)
    at = __reduce_max_sync(0xFFFFFFFFu, tied);
    if (--k == 0) break;
    if (tied == at) tied = 0;
  }
  return (unsigned long long)top << 32 | at;
}
// The k-th largest of the bests of 32 groups of 8 threads: a bound that at
// least k of what the threads hold reach (0 if fewer than k groups hold any).
__device__ __forceinline__ unsigned long long bound_of(unsigned long long best, int k, Shared& sh) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
    best = other > best ? other : best;
  }
  if ((threadIdx.x & 7) == 0) sh.group[threadIdx.x >> 3] = best;
  __syncthreads();
  return kth_of(sh.group[threadIdx.x & 31], k);
}
__device__ __forceinline__ void put(unsigned long long key, Shared& sh) {
  const int at = atomicAdd(&sh.count, 1);
  if (at < ROOM) sh.buf[at] = key;
}
// Those of eight values, the first of index e, that reach the bound `limit`,
// whose value is `value`.  (One at a time: few do, and the loop that this
// stands in has to stay short.)
template <bool F32, class Put>
__device__ __forceinline__ void put_from(const ops::Raw<F32>& raw, int e, int n, unsigned long long limit, float value, Put put) {
  float x[8];
  ops::unpack(raw, x);
  unsigned which = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) which |= !(x[i] < value) ? 1u << i : 0u;  // (a NaN reaches it)
#pragma unroll 1
  for (; which; which &= which - 1) {
    const int i = __ffs(which) - 1;
    const float a = i & 4 ? x[4] : x[0], b = i & 4 ? x[5] : x[1], c = i & 4 ? x[6] : x[2], d = i & 4 ? x[7] : x[3];
    const float v = i & 2 ? (i & 1 ? d : c) : i & 1 ? b : a;
    const unsigned long long key = key_of(v, e + i);
    if (key >= limit && e + i >= 0 && e + i < n) put(key);
  }
}
// The best of eight values, the first of index e; 0 if none lies in the row.
template <bool F32>
__device__ __forceinline__ unsigned long long best_of(const ops::Raw<F32>& raw, int e, int n) {
  float x[8];
  ops::unpack(raw, x);
  const float most =
      max_nan(max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3])), max_nan(max_nan(x[4], x[5]), max_nan(x[6], x[7])));
  unsigned which = 0, in = 0xFF;
#pragma unroll
  for (int i = 0; i < 8; ++i) which |= x[i] == most || x[i] != x[i] ? 1u << i : 0u;  // (a NaN is the largest)
  if (e < 0) in &= 0xFFu << -e;
  if (e + 8 > n) in &= e < n ? 0xFFu >> (e + 8 - n) : 0u;
  which &= in;  // (behind the row's ends are -infs: where they are the largest, all in the row are)
  return which ? key_of(most, e + __ffs(which) - 1) : 0;
}
// One warp: the bound raised to the k-th largest of what its lanes see, each
// the largest of every 32nd value in the buffer (fewer than k lanes with any: not).
__device__ __forceinline__ void raise_limit(int k, Shared& sh) {
  const int lane = threadIdx.x & 31;
  const int c = min(*(volatile int*)&sh.count, ROOM);
  unsigned long long best = 0;
  for (int i = lane; i < c; i += 32) {
    const unsigned long long key = *(volatile unsigned long long*)&sh.buf[i];
    best = key > best ? key : best;
  }
  const unsigned long long bound = kth_of(best, k);
  if (lane == 0 && bound) atomicMax(&sh.limit, bound);
}
// Cuts the buffer to its k largest, sorted; returns their smallest, or 0 if
// there are fewer.  All threads; barriers before and behind.
__device__ __noinline__ unsigned long long cut(int k, Shared& sh) {
  __syncthreads();
  int c = min(sh.count, ROOM);
  if (c > 96) {  // first what the bound leaves
    constexpr int EACH = (ROOM + THREADS - 1) / THREADS;
    unsigned long long mine[EACH], best = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = i * THREADS + (int)threadIdx.x;
      mine[i] = at < c ? sh.buf[at] : 0;
      best = mine[i] > best ? mine[i] : best;
    }
    const unsigned long long bound = bound_of(best, k, sh);  // (its barrier is behind all reads of buf and count)
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (mine[i] && mine[i] >= bound) put(mine[i], sh);
    __syncthreads();
    c = sh.count;
  }
  for (int i = threadIdx.x; i < c; i += THREADS) {
    const unsigned long long mine = sh.buf[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < c; ++j) rank += sh.buf[j] > mine;
    if (rank < k) sh.list[rank] = mine;
  }
  __syncthreads();
  const int kept = min(c, k);
  if ((int)threadIdx.x < kept) sh.buf[threadIdx.x] = sh.list[threadIdx.x];
  if (threadIdx.x == 0) sh.count = kept;
  __syncthreads();
  return c >= k ? sh.list[k - 1] : 0;
}

// The same by one warp, for the end of a row: lane i gets the i-th largest, or
// 0 where there are fewer.
// (The block's way costs four barriers with all warps behind them.)
__device__ __forceinline__ unsigned long long cut_by_warp(int k, Shared& sh) {
  const int lane = threadIdx.x & 31, c = sh.count;
  unsigned long long best = 0;
  for (int i = lane; i < c; i += 32) best = sh.buf[i] > best ? sh.buf[i] : best;
  const unsigned long long bound = kth_of(best, k);
  int n = 0;
  for (int i = 0; i < c; i += 32) {
    const unsigned long long key = i + lane < c ? sh.buf[i + lane] : 0;
    const bool in = key && key >= bound;
    const unsigned all = __ballot_sync(0xFFFFFFFFu, in);
    const int at = n + __popc(all & ((1u << lane) - 1));
    __syncwarp();  // (survivors go over what has been read)
    if (in) sh.buf[at] = key;
    n += __popc(all);
  }
  __syncwarp();
  for (int i = lane; i < n; i += 32) {
    const unsigned long long mine = sh.buf[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += sh.buf[j] > mine;
    if (rank < k) sh.list[rank] = mine;
  }
  __syncwarp();
  return lane < min(n, k) ? sh.list[lane] : 0;
}

__device__ __forceinline__ long long token_of(const Params& p, long long row) {
  return p.tokens_64 ? static_cast<const long long*>(p.tokens)[row] : (long long)static_cast<const int*>(p.tokens)[row];
}

// One warp: a row's results.  Lane 0 has its token, lane i its i-th alternative.
template <bool TOP>
__device__ __forceinline__ void finish(const Params& p, long long row, long long token, float at_token, const Result& res,
                                       unsigned long long key) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    if (p.logprob)
      p.logprob[row] = token < 0 ? 0.f : token < p.vocabulary ? (at_token - res.m) - res.log_s : __int_as_float(0x7FC00000);
    if (p.entropy) p.entropy[row] = res.entropy;
    if (p.stats) p.stats[row] = make_float2(res.m, res.log_s);
  }
  if constexpr (TOP)
    if (lane < p.top) {
      p.ids[row * p.top + lane] = index_of(key);
      p.tops[row * p.top + lane] = (value_of(key) - res.m) - res.log_s;
    }
}

// Short rows, a warp each: all of a row is in registers.  No thread waits for
// another warp; the alternatives' buffer is the warp's own, and where too many
// values reach the bound (rows of equal values) the largest is taken k times.
constexpr int SHORT = 2048, SHORT_ROOM = 192;
template <bool F32, bool TOP, int EIGHTS>
__global__ void __launch_bounds__(THREADS) short_rows(const __grid_constant__ Params p) {
  __shared__ unsigned long long bufs[TOP ? 8 : 1][SHORT_ROOM], lists[TOP ? 8 : 1][MAX_TOP];
  __shared__ int counts[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * 8 + warp;
  pdl_launch();
  pdl_wait();
  if (row >= p.rows) return;
  const uint8_t* px = p.x + row * p.ld;
  const Row<F32> r(px, p.vocabulary);
  const int eights = r.eights();
  ops::Raw<F32> raw[EIGHTS];
#pragma unroll
  for (int j = 0; j < EIGHTS; ++j) {
    if (lane + 32 * j < eights) r.load(lane + 32 * j, raw[j]);
    else Row<F32>::none(raw[j]);
  }
  long long token = -1;
  float at_token = 0.f;
  if (p.tokens && lane == 0) {
    token = token_of(p, row);
    if (token >= 0 && token < p.vocabulary) at_token = ops::ld_any(px, token, F32);
  }
  Sums sums;
#pragma unroll
  for (int j = 0; j < EIGHTS; ++j) {
    unsigned long long x[4];
    const float most = raised(raw[j], x);
    sums.add(x, most);
  }
  Soft soft = sums.soft();
  float m = soft.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  soft.raise(m);
  soft.s = ops::warp_sum(soft.s);
  soft.u = ops::warp_sum(soft.u);
  Result res;
  if (m > NONE && m < MOST) {
    res = result_of(soft);
  } else {  // by the definition
    float top = -INFINITY, s = 0.f, u = 0.f;
    bool nan = false;
    for (int i = lane; i < p.vocabulary; i += 32) {
      const float v = ops::ld_any(px, i, F32);
      nan |= v != v;
      top = fmaxf(top, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    for (int i = lane; i < p.vocabulary; i += 32) {
      const float d = max_nan(ops::ld_any(px, i, F32) - top, -1000.f), e = exp_of(d);
      s += e;
      u = fmaf(e, d, u);
    }
    s = ops::warp_sum(nan ? NAN : s);
    u = ops::warp_sum(u);
    const float log_s = logf(s);
    res = {top, log_s, log_s - u / s};
  }
  unsigned long long key = 0;
  if constexpr (TOP) {
    unsigned long long* buf = bufs[warp];
    unsigned long long* list = lists[warp];
    unsigned long long best = 0;
#pragma unroll
    for (int j = 0; j < EIGHTS; ++j) {
      const unsigned long long b = best_of(raw[j], r.first(lane + 32 * j), p.vocabulary);
      best = b > best ? b : best;
    }
    const unsigned long long bound = kth_of(best, p.top);
    const float value = bound ? value_of(bound) : -INFINITY;
    if (lane == 0) counts[warp] = 0;
    __syncwarp();
    if (best >= bound)
#pragma unroll
      for (int j = 0; j < EIGHTS; ++j)
        put_from<F32>(raw[j], r.first(lane + 32 * j), p.vocabulary, bound, value, [&](unsigned long long k) {
          const int to = atomicAdd(&counts[warp], 1);
          if (to < SHORT_ROOM) buf[to] = k;
        });
    __syncwarp();
    const int c = counts[warp];
    if (c <= SHORT_ROOM) {
      for (int i = lane; i < c; i += 32) {
        const unsigned long long mine = buf[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < c; ++j) rank += buf[j] > mine;
        if (rank < p.top) list[rank] = mine;
      }
      __syncwarp();
      if (lane < p.top) key = list[lane];
    } else {
      unsigned long long last = 0;
      for (int k = 0; k < p.top; ++k) {
        unsigned long long most = 0;
        for (int i = lane; i < p.vocabulary; i += 32) {
          const unsigned long long v = key_of(ops::ld_any(px, i, F32), i);
          // (at first nothing lies above: a NaN at index 0 has the largest key there is)
          most = (k == 0 || v < last) && v > most ? v : most;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, most, o);
          most = other > most ? other : most;
        }
        last = most;
        if (lane == k) key = most;
      }
    }
  }
  finish<TOP>(p, row, token, at_token, res, key);
}

// One row, or one of p.split parts of it, a block: few rows have a cluster each.
template <bool F32, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) forward(const __grid_constant__ Params p) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / p.split;
  const int part = blockIdx.x - (int)(row * p.split);
  // (the parts write into the first one's shared memory: it has to have begun by then)
  if (p.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch();
  pdl_wait();
  const uint8_t* px = p.x + row * p.ld;
  const Row<F32> r(px, p.vocabulary);
  const int per = (r.eights() + p.split - 1) / p.split;
  const int v0 = part * per, v1 = min(v0 + per, r.eights());
  const int rounds = max(0, v1 - v0 + THREADS - 1) / THREADS;
  long long token = -1;
  float at_token = 0.f;
  if (p.tokens && tid == 0) {  // (its value is in flight beside the row's)
    token = token_of(p, row);
    if (token >= 0 && token < p.vocabulary) at_token = ops::ld_any(px, token, F32);
  }

  Sums sums;
  const int mine = v0 + tid;
  // rounds of whole eights, but for the first, which may hold the row's first
  const int inner = (min(v1, (int)(r.lo + r.whole)) - v0) / THREADS;
  auto get = [&](int round, ops::Raw<F32>& raw) {
    const int v = mine + round * THREADS;
    if (round > 0 && round < inner) r.load_whole(v, raw);
    else if (v < v1) r.load(v, raw);
    else Row<F32>::none(raw);
  };
  constexpr int N = AHEAD<F32>;
  ops::Raw<F32> ring[N];
#pragma unroll
  for (int i = 0; i < N; ++i) get(i, ring[i]);
  unsigned long long bound = 0;  // everything reaches it
  float limit = -INFINITY;       // its value and index
  int limit_at = 0x7FFFFFFF;
  auto follow = [&](unsigned long long key) {
    if (!key) return;
    bound = key;
    limit = value_of(key);
    limit_at = index_of(key);
  };
  auto put_here = [&](unsigned long long key) { put(key, sh); };
  if constexpr (TOP) {
    for (int i = tid; i < ROOM; i += THREADS) sh.buf[i] = 0;
    if (tid == 0) {
      sh.count = 0;
      sh.limit = 0;
    }
    // the first rounds' own bound (a barrier is in it, behind the clearing)
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int v = mine + i * THREADS;
      const unsigned long long one = v < v1 ? best_of(ring[i], r.first(v), p.vocabulary) : 0;
      best = one > best ? one : best;
    }
    follow(bound_of(best, p.top, sh));
    if (tid == 0) atomicMax(&sh.limit, bound);
  }
  int until = N;  // the round at which a warp raises the bound
  for (int round0 = 0; round0 < rounds; round0 += N) {
    if constexpr (TOP) {
      if (round0 == until) {
        if (tid >> 5 == (__ffs(until) & 7)) raise_limit(p.top, sh);
        until *= 2;
      }
      if (round0) follow(*(volatile unsigned long long*)&sh.limit);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int round = round0 + i;
      if (round >= rounds) break;
      unsigned long long x[4];
      const float most = raised(ring[i], x);
      // (the order that the compiler makes most of: 114 and 79 us the other way
      // for 2048 x 100003 with 5 alternatives and none, 108 and 75 this)
      if constexpr (TOP) {
        sums.add(x, most);
        if (__builtin_expect(!(most < limit), 0)) {  // (equal values up to the bound's index; a NaN)
          const int v = mine + round * THREADS, e = r.first(v);
          if ((most != limit || e <= limit_at) && v < v1) put_from<F32>(ring[i], e, p.vocabulary, bound, limit, put_here);
        }
        get(round + N, ring[i]);
      } else {
        get(round + N, ring[i]);
        sums.add(x, most);
      }
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    if (sh.count > ROOM) {  // too many: round by round
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
      bound = 0;
      for (int round = 0; round < rounds; ++round) {
        ops::Raw<F32> raw;
        get(round, raw);
        if (mine + round * THREADS < v1)
          put_from<F32>(raw, r.first(mine + round * THREADS), p.vocabulary, bound, bound ? value_of(bound) : -INFINITY, put_here);
        bound = cut(p.top, sh);
      }
      __syncthreads();
    }
  }
  // the rest is one warp's: the block's sums and its k largest
  Soft soft = sums.soft();
  float m = soft.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  soft.raise(m);
  soft.s = ops::warp_sum(soft.s);
  soft.u = ops::warp_sum(soft.u);
  if ((tid & 31) == 0) {
    sh.m[tid >> 5] = soft.m;
    sh.s[tid >> 5] = soft.s;
    sh.u[tid >> 5] = soft.u;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, sh.m[w]);
  Soft all;
  unsigned long long key = 0;
  if (tid < 32) {
    if (tid < 8) {
      all.m = sh.m[tid];
      all.s = sh.s[tid];
      all.u = sh.u[tid];
    }
    all.raise(m);
    all.s = ops::warp_sum(all.s);
    all.u = ops::warp_sum(all.u);
    if constexpr (TOP) key = cut_by_warp(p.top, sh);
  }
  if (p.split > 1) {  // the parts meet in the first one's shared memory
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < 32) {
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&sh.parts[part])), "r"(0));
      if (tid == 0)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(all.m), "f"(all.s), "f"(all.u), "f"(0.f) : "memory");
      if constexpr (TOP) {
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&sh.lists[part * p.top])), "r"(0));
        if (tid < p.top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + tid * 8), "l"(key) : "memory");
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (part != 0) return;
    for (int i = 0; i < p.split; ++i) m = fmaxf(m, sh.parts[i].x);
    if (tid < 32) {
      all = Soft();
      if (tid < p.split) {
        all.m = sh.parts[tid].x;
        all.s = sh.parts[tid].y;
        all.u = sh.parts[tid].z;
      }
      all.raise(m);
      all.s = ops::warp_sum(all.s);
      all.u = ops::warp_sum(all.u);
      if constexpr (TOP) {
        const int n = p.split * p.top;  // (0s, of parts with fewer values, are below every bound)
        for (int i = tid; i < n; i += 32) sh.buf[i] = sh.lists[i];
        if (tid == 0) sh.count = n;
        __syncwarp();
        key = cut_by_warp(p.top, sh);
      }
    }
  }
  const bool usual = m > NONE && m < MOST;
  Result res = {};
  if (!usual) {
    __syncthreads();  // (it uses sh.m)
    res = far_out<F32>(px, p.vocabulary, sh);
  }
  if (tid >= 32) return;
  if (usual) res = result_of(all);
  finish<TOP>(p, row, token, at_token, res, key);
}

struct Grads {
  const uint8_t* x;
  uint8_t* dx;
  long long ld, ld_d;  // bytes
  const void* tokens;
  const float* dlogprob;
  const float* dentropy;
  const float* entropy;
  const float2* stats;
  int rows, vocabulary, tokens_64, pieces;
};
constexpr int EIGHTS = 4;  // of a thread

// A block takes 8192 values of a row.  SAME: logits and gradient start at the
// same place within 16 (32) bytes, so that both go by eights.
//   t = ((x - m) - log S) L,  -dx = 2^t (dlogprob + dentropy (entropy + t ln 2))
// in pairs of values; masked ones are raised to -1e9 as in the forward pass,
// and the token's own term is added by the thread that has it.  Rows far out
// (|m| of 1e8 and more) have x - m limited instead.
// p.pieces of 0: rows are short, and a warp's each.  Not SAME: value by value
// (2048 x 50257 bf16 in rows of 50304: 75 us, into rows of 50257 217).
template <bool F32, bool SAME>
__global__ void __launch_bounds__(THREADS, 4) backward(const __grid_constant__ Grads p) {
  const int T = p.pieces ? THREADS : 32, t = threadIdx.x & (T - 1);
  const long long row = p.pieces ? blockIdx.x / p.pieces : (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  const int piece = p.pieces ? blockIdx.x - (int)(row * p.pieces) : 0;
  pdl_launch();
  pdl_wait();
  if (row >= p.rows) return;
  long long token = -1;
  if (p.tokens) token = p.tokens_64 ? static_cast<const long long*>(p.tokens)[row] : (long long)static_cast<const int*>(p.tokens)[row];
  float a = p.dlogprob && token >= 0 ? p.dlogprob[row] : 0.f;
  if (token >= p.vocabulary && a != 0.f) a = __int_as_float(0x7FC00000);
  const float h = p.dentropy ? p.dentropy[row] : 0.f;
  const bool zero = a == 0.f && h == 0.f;  // a padded row, say: nothing is read
  const float2 st = p.stats[row];
  const float ah = h != 0.f ? fmaf(h, p.entropy[row], a) : a;
  const Row<F32> r(p.x + row * p.ld, p.vocabulary);
  uint8_t* out = p.dx + row * p.ld_d;
  const bool usual = st.x > NONE && st.x < MOST;
  const float s_l = st.y * LOG2E, h_l = h * 0.69314718f;
  auto grad = [&](float x, long long i) {  // one value, by the same steps
    float d;
    if (usual) {
      const float t = fmaf(max_nan(x, LOWEST) - st.x, LOG2E, -s_l);
      d = ex2(t) * fmaf(t, -h_l, -ah);
    } else {
      const float l = max_nan((x - st.x) - st.y, -1000.f);
      d = -exp_of(l) * fmaf(h, l, ah);
    }
    return i == token ? d + a : d;
  };
  if constexpr (SAME) {
    const int first = piece * EIGHTS * THREADS + t, end = p.pieces ? min(first + EIGHTS * THREADS, r.eights()) : r.eights();
    if (zero) {
      for (int v = first; v < end; v += T) r.store(v, out, ops::Raw<F32>{});
      return;
    }
    const ops::f32x2 minus_m = ops::both(-st.x), l2 = ops::both(LOG2E), minus_s = ops::both(-s_l);
    const ops::f32x2 ht = ops::both(-h_l), minus_a = ops::both(-ah);
    for (int v0 = first; v0 < end; v0 += EIGHTS * T) {
      ops::Raw<F32> raw[EIGHTS];
#pragma unroll
      for (int j = 0; j < EIGHTS; ++j)
        if (v0 + j * T < end) r.load(v0 + j * T, raw[j]);
#pragma unroll
      for (int j = 0; j < EIGHTS; ++j) {
        const int v = v0 + j * T;
        if (v >= end) continue;
        const int e = r.first(v);
        float y[8];
        if (usual) {
          ops::f32x2 x[4];
          raised(raw[j], x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const ops::f32x2 t2 = fma2(add2(x[i], minus_m), l2, minus_s);
            float t0, t1;
            unpair2(t2, t0, t1);
            unpair2(ops::mul2(pair2(ex2(t0), ex2(t1)), fma2(t2, ht, minus_a)), y[2 * i], y[2 * i + 1]);
          }
          if (token >= e && token < e + 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (token == e + i) y[i] += a;
          }
        } else {
          ops::unpack(raw[j], y);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = grad(y[i], e + i);
        }
        ops::Raw<F32> o;
        ops::pack(y, o);
        r.store(v, out, o);
      }
    }
  } else {
    const long long e0 = (long long)piece * EIGHTS * ROUND, e1 = min(e0 + EIGHTS * ROUND, (long long)p.vocabulary);
    for (long long e = e0 + t; e < e1; e += T)
      ops::st_any(out, e, zero ? 0.f : grad(ops::ld_any(p.x + row * p.ld, e, F32), e), F32);
  }
}

}  // namespace logp
}  // namespace apk

using namespace apk;

struct apk_logprobs {
  apk_logprobs_config cfg{};
  Err err;
  bool opened = false;
  int sms = 0, most_split = 8;
  std::mutex mu;
};

namespace {

apk_status create(const apk_logprobs_config* cfg, apk_logprobs* h) {
  h->cfg = *cfg;
  if (h->cfg.top < 0 || h->cfg.top > logp::MAX_TOP)
    return h->err.fail(APK_EINVAL, "top is %d: 0 to %d", h->cfg.top, logp::MAX_TOP);
  APK_TRY(ops::open_device(h->cfg.device, &h->sms, &h->err));
  DeviceGuard guard(h->cfg.device);
  // clusters of 16, where the device has room for one
  int fit = 1 << 20;
  for (const void* f : {reinterpret_cast<const void*>(&logp::forward<false, false>), reinterpret_cast<const void*>(&logp::forward<false, true>),
                        reinterpret_cast<const void*>(&logp::forward<true, false>), reinterpret_cast<const void*>(&logp::forward<true, true>)}) {
    APK_TRY(cu_status(cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "preparing the log probabilities", &h->err));
    Launch l(dim3(logp::MAX_SPLIT), logp::THREADS, 0, nullptr, logp::MAX_SPLIT);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, f, &l.cfg) != cudaSuccess) cudaGetLastError();
    fit = std::min(fit, n);
  }
  if (fit >= 1) h->most_split = logp::MAX_SPLIT;
  return APK_OK;
}

apk_status check_logits(const void* x, long long ld, int rows, int vocabulary, int dtype, Err* err) {
  if (rows < 0 || rows > ops::MAX_SIZE) return err->fail(APK_EINVAL, "rows is %d: at most 2^30", rows);
  if (vocabulary < 1 || vocabulary > ops::MAX_SIZE) return err->fail(APK_EINVAL, "vocabulary is %d: 1 to 2^30", vocabulary);
  if (!ops::valid_dtype(dtype)) return err->fail(APK_EINVAL, "dtype %d", dtype);
  if (rows > 0 && !x) return err->fail(APK_EINVAL, "logits is NULL");
  if (ld < vocabulary) return err->fail(APK_EINVAL, "a row stride is below its row: %lld", ld);
  if (!ops::aligned(x, ops::esize(dtype))) return err->fail(APK_EINVAL, "logits is not aligned to its element");
  return APK_OK;
}

template <bool F32, bool TOP>
auto short_of(int vocabulary) {
  return vocabulary <= 249 ? logp::short_rows<F32, TOP, 1> : vocabulary <= 1017 ? logp::short_rows<F32, TOP, 4> : logp::short_rows<F32, TOP, 8>;
}

apk_status forward(apk_logprobs* h, const apk_logprobs_io* io) {
  const int V = io->vocabulary, M = io->rows, k = h->cfg.top;
  const cudaStream_t s = static_cast<cudaStream_t>(io->stream);
  APK_TRY(check_logits(io->logits, io->ld, M, V, io->dtype, &h->err));
  if (k > V) return h->err.fail(APK_EINVAL, "top %d of a vocabulary of %d", k, V);
  if (M == 0) return APK_OK;
  if (k > 0 && (!io->top_ids || !io->top_logprobs)) return h->err.fail(APK_EINVAL, "top_ids or top_logprobs is NULL");
  if (io->logprob && !io->tokens) return h->err.fail(APK_EINVAL, "logprob without tokens");
  if (!ops::aligned(io->tokens, io->tokens_64 ? 8 : 4) || !ops::aligned(io->logprob, 4) || !ops::aligned(io->entropy, 4) ||
      !ops::aligned(io->top_ids, 4) || !ops::aligned(io->top_logprobs, 4) || !ops::aligned(io->stats, 8))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element (stats: to its pair)");
  DeviceGuard guard(h->cfg.device);
  const size_t es = ops::esize(io->dtype);
  logp::Params p{};
  p.x = static_cast<const uint8_t*>(io->logits);
  p.ld = io->ld * (long long)es;
  p.tokens = io->logprob ? io->tokens : nullptr;
  p.tokens_64 = io->tokens_64;
  p.logprob = io->logprob;
  p.entropy = io->entropy;
  p.ids = io->top_ids;
  p.tops = io->top_logprobs;
  p.stats = reinterpret_cast<float2*>(io->stats);
  p.rows = M;
  p.vocabulary = V;
  p.top = k;
  // parts of at least a round each, while the rows alone leave places empty
  p.split = 1;
  while (2 * p.split <= h->most_split && 2ll * p.split * M <= 2 * h->sms && 2 * p.split <= V / logp::ROUND) p.split *= 2;
  const bool f = io->dtype == APK_F32;
  if (V <= logp::SHORT - 7) {  // (and up to 7 places before the row)
    const auto rows = k ? (f ? short_of<true, true>(V) : short_of<false, true>(V))
                        : (f ? short_of<true, false>(V) : short_of<false, false>(V));
    Launch l(dim3(ops::ceil_div(M, 8)), logp::THREADS, 0, s);
    return cu_status(cudaLaunchKernelEx(&l.cfg, rows, p), "launching the log probabilities", &h->err);
  }
  const auto kernel = k ? (f ? logp::forward<true, true> : logp::forward<false, true>)
                        : (f ? logp::forward<true, false> : logp::forward<false, false>);
  Launch l(dim3(M * p.split), logp::THREADS, 0, s, p.split);
  return cu_status(cudaLaunchKernelEx(&l.cfg, kernel, p), "launching the log probabilities", &h->err);
}

apk_status backward(apk_logprobs* h, const apk_logprobs_grads* g) {
  const int V = g->vocabulary, M = g->rows;
  APK_TRY(check_logits(g->logits, g->ld, M, V, g->dtype, &h->err));
  if (M == 0) return APK_OK;
  const size_t es = ops::esize(g->dtype);
  if (!g->dlogits || !g->stats) return h->err.fail(APK_EINVAL, "dlogits or stats is NULL");
  if (!g->dlogprob && !g->dentropy) return h->err.fail(APK_EINVAL, "no output's gradient is given");
  if ((g->dlogprob && !g->tokens) || (g->dentropy && !g->entropy))
    return h->err.fail(APK_EINVAL, "dlogprob without tokens, or dentropy without entropy");
  if (g->ld_d < V) return h->err.fail(APK_EINVAL, "a row stride is below its row: %lld", g->ld_d);
  if (!ops::aligned(g->dlogits, es) || !ops::aligned(g->tokens, g->tokens_64 ? 8 : 4) || !ops::aligned(g->dlogprob, 4) ||
      !ops::aligned(g->dentropy, 4) || !ops::aligned(g->entropy, 4) || !ops::aligned(g->stats, 8))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element (stats: to its pair)");
  DeviceGuard guard(h->cfg.device);
  const int align = g->dtype == APK_F32 ? 32 : 16;
  logp::Grads p{};
  p.x = static_cast<const uint8_t*>(g->logits);
  p.dx = static_cast<uint8_t*>(g->dlogits);
  p.ld = g->ld * (long long)es;
  p.ld_d = g->ld_d * (long long)es;
  p.tokens = g->dlogprob ? g->tokens : nullptr;
  p.tokens_64 = g->tokens_64;
  p.dlogprob = g->dlogprob;
  p.dentropy = g->dentropy;
  p.entropy = g->entropy;
  p.stats = reinterpret_cast<const float2*>(g->stats);
  p.rows = M;
  p.vocabulary = V;
  // (rows that start on an alignment have no places before them)
  const bool on = reinterpret_cast<uintptr_t>(p.x) % align == 0 && (M == 1 || p.ld % align == 0);
  p.pieces = (int)(((long long)V + (on ? 0 : 7) + logp::EIGHTS * logp::ROUND - 1) / (logp::EIGHTS * logp::ROUND));
  const bool rows = V <= logp::SHORT;
  if (rows) p.pieces = 0;
  if ((long long)M * p.pieces > 0x7FFFFFFFll) return h->err.fail(APK_EINVAL, "%d rows of %d are too many for a launch", M, V);
  const bool same = (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.dx)) % align == 0 &&
                    (M == 1 || (p.ld - p.ld_d) % align == 0);
  const bool f = g->dtype == APK_F32;
  const auto kernel = same ? (f ? logp::backward<true, true> : logp::backward<false, true>)
                           : (f ? logp::backward<true, false> : logp::backward<false, false>);
  Launch l(dim3(rows ? ops::ceil_div(M, logp::THREADS / 32) : M * p.pieces), logp::THREADS, 0, static_cast<cudaStream_t>(g->stream));
  return cu_status(cudaLaunchKernelEx(&l.cfg, kernel, p), "launching the log probabilities' gradient", &h->err);
}

}  // namespace

extern "C" {

apk_status apk_logprobs_create(const apk_logprobs_config* cfg, apk_logprobs** out) { return ops::make(cfg, out, create); }

apk_status apk_logprobs_destroy(apk_logprobs* h) {
  delete h;
  return APK_OK;
}

const char* apk_logprobs_last_error(const apk_logprobs* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_logprobs_forward(apk_logprobs* h, const apk_logprobs_io* io) {
  return ops::call(h, io, [&] { return forward(h, io); });
}

apk_status apk_logprobs_backward(apk_logprobs* h, const apk_logprobs_grads* g) {
  return ops::call(h, g, [&] { return backward(h, g); });
}

}  // extern "C"
