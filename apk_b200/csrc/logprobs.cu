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
// that are scaled where it grows.  x - m is taken before it is multiplied by
// log2(e), so that large logits cost no digits.
//
// The alternatives come out of the same pass.  The first round of 2048 values
// gives a bound that its k-th largest value reaches; a value above the bound
// is put into a buffer in shared memory; after 1, 2, 4, 8, ... rounds the
// buffer is cut to its k largest, whose smallest is the new bound.  Between
// two cuts about k values pass (the chance of the n-th value to be among the
// k largest so far is k / n).  Rows in which far more pass, ascending ones,
// fill the buffer up: their rounds are taken again one by one.
#include <algorithm>

#include "act.cuh"
#include "ops.cuh"
#include "ops.h"

namespace apk {
namespace logp {

constexpr int THREADS = 256, ROUND = THREADS * 8;  // values of a block's round
constexpr int MAX_TOP = 32, MAX_SPLIT = 64;
constexpr int ROOM = ROUND + MAX_TOP;              // of the buffer: the list, and a whole round
constexpr float NONE = -3.402823466e38f;           // the running maximum before the first value
static_assert(MAX_SPLIT * MAX_TOP <= ROOM, "the splits' lists fit the buffer");

struct Params {
  const uint8_t* x;
  long long ld;      // bytes
  const void* tokens;
  float* logprob;
  float* entropy;
  int* ids;
  float* tops;
  float2* stats;
  float4* part;      // [row][split] m, S, sum e d
  unsigned long long* lists;  // [row][split][top]
  unsigned* arrived; // [row], zero between launches
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
  __device__ __forceinline__ Row(const uint8_t* p, int n_) : n(n_) {
    const int bytes = (int)(reinterpret_cast<uintptr_t>(p) & (F32 ? 31 : 15));
    base = p - bytes;
    shift = bytes / (F32 ? 4 : 2);
  }
  __device__ __forceinline__ int eights() const { return (int)(((long long)n + shift + 7) / 8); }
  __device__ __forceinline__ long long first(int v) const { return (long long)v * 8 - shift; }
  // -inf where the row does not reach
  __device__ __forceinline__ void load(int v, ops::Raw<F32>& r) const {
    const long long e = first(v);
    const uint8_t* q = base + (long long)v * (F32 ? 32 : 16);
    if (e >= 0 && e + 8 <= n) {
      if constexpr (F32)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
                     : "l"(q)
                     : "memory");
      else
        r.a = __ldcs(reinterpret_cast<const uint4*>(q));
      return;
    }
    const uint32_t none = F32 ? 0xFF800000u : 0xFF80FF80u;
    r.a = make_uint4(none, none, none, none);
    if constexpr (F32) r.b = r.a;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i >= 0 && e + i < n) ops::set1(r, i, q, i);
  }
};

struct Soft {
  float m = NONE, s = 0.f, u = 0.f;
  // m grows to to: what was summed is scaled.  (What is more than e^1000
  // smaller is gone, and -inf * 0 does not arise.)
  __device__ __forceinline__ void raise(float to) {
    const float d = fmaxf(m - to, -1000.f), f = exp_of(d);
    u = f * fmaf(s, d, u);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(const float (&x)[8], float most) {
    if (most > m) raise(most);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = max_nan(x[i] - m, -1000.f), e = exp_of(d);
      s += e;
      u = fmaf(e, d, u);
    }
  }
};

struct Shared {
  unsigned long long buf[ROOM];
  unsigned long long group[32];
  unsigned long long list[MAX_TOP];
  float m[8], s[8], u[8];
  int count;
  bool last;
};

// Over the block: every thread gets the row's m, s and u.
__device__ __forceinline__ Soft join(Soft a, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  __syncthreads();  // (who reads an earlier result is done)
  if (lane == 0) sh.m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, sh.m[w]);
  a.raise(m);
  a.s = ops::warp_sum(a.s);
  a.u = ops::warp_sum(a.u);
  if (lane == 0) {
    sh.s[warp] = a.s;
    sh.u[warp] = a.u;
  }
  __syncthreads();
  a.s = a.u = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    a.s += sh.s[w];
    a.u += sh.u[w];
  }
  return a;
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
  const unsigned long long mine = sh.group[threadIdx.x & 31];
  int rank = 0;
#pragma unroll 8
  for (int i = 0; i < 32; ++i) {
    const unsigned long long other = sh.group[i];
    // (equal ones are 0s: any order)
    rank += other > mine || (other == mine && i < (int)(threadIdx.x & 31));
  }
  const int at = __ffs(__ballot_sync(0xFFFFFFFFu, rank == k - 1)) - 1;
  return __shfl_sync(0xFFFFFFFFu, mine, at);
}
__device__ __forceinline__ void put(unsigned long long key, Shared& sh) {
  const int at = atomicAdd(&sh.count, 1);
  if (at < ROOM) sh.buf[at] = key;
}
// Cuts the buffer to its k largest, sorted; returns their smallest, or 0 if
// there are fewer.  All threads; barriers before and behind.
__device__ __forceinline__ unsigned long long cut(int k, Shared& sh) {
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

__device__ __forceinline__ long long token_of(const Params& p, long long row) {
  return p.tokens_64 ? static_cast<const long long*>(p.tokens)[row] : (long long)static_cast<const int*>(p.tokens)[row];
}

// One row, or one of p.split parts of it, a block.
template <bool F32, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) forward(const __grid_constant__ Params p) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / p.split;
  const int part = blockIdx.x - (int)(row * p.split);
  pdl_launch();
  pdl_wait();
  const uint8_t* px = p.x + row * p.ld;
  const Row<F32> r(px, p.vocabulary);
  const int per = (r.eights() + p.split - 1) / p.split;
  const int v0 = part * per, v1 = min(v0 + per, r.eights());
  const int rounds = max(0, v1 - v0 + THREADS - 1) / THREADS;
  long long token = -1;
  float at_token = 0.f;
  if (p.tokens && tid == 0) {
    token = token_of(p, row);
    if (token >= 0 && token < p.vocabulary) at_token = ops::ld_any(px, token, F32);
  }
  if (TOP && tid == 0) sh.count = 0;

  Soft soft;
  float limit = 0.f;       // the k-th largest so far
  uint32_t limit_order = 0;
  auto get = [&](int round, ops::Raw<F32>& raw) {
    const int v = v0 + round * THREADS + tid;
    if (round < rounds && v < v1) {
      r.load(v, raw);
    } else {
      const uint32_t none = F32 ? 0xFF800000u : 0xFF80FF80u;
      raw.a = make_uint4(none, none, none, none);
      if constexpr (F32) raw.b = raw.a;
    }
  };
  auto above = [&](int round, const float (&x)[8], float most) {
    if (!(most <= limit)) {  // (a NaN is above)
      const int e = (int)r.first(v0 + round * THREADS + tid);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (order_of(x[i]) > limit_order && e + i >= 0 && e + i < p.vocabulary) put(key_of(x[i], e + i), sh);
    }
  };
  auto cut_now = [&]() {
    const unsigned long long key = cut(p.top, sh);
    limit_order = (uint32_t)(key >> 32);
    limit = value_of(key);
  };
  ops::Raw<F32> now, next;
  get(0, now);
  get(1, next);
  int from = 1, until = 2;  // rounds between two cuts
  for (int round = 0; round < rounds; ++round) {
    float x[8];
    ops::unpack(now, x);
    now = next;
    get(round + 2, next);
    const float most = max_nan(max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3])), max_nan(max_nan(x[4], x[5]), max_nan(x[6], x[7])));
    soft.add(x, most);
    if constexpr (TOP) {
      if (round == 0) {
        const long long e = r.first(v0 + tid);
        const bool mine = v0 + tid < v1;
        unsigned long long key[8], best = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          key[i] = mine && e + i >= 0 && e + i < p.vocabulary ? key_of(x[i], (int)e + i) : 0;
          best = key[i] > best ? key[i] : best;
        }
        const unsigned long long bound = bound_of(best, p.top, sh);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key[i] && key[i] >= bound) put(key[i], sh);
        cut_now();
      } else {
        above(round, x, most);
        if (round + 1 == until || round + 1 == rounds) {
          __syncthreads();
          if (sh.count > ROOM) {  // too many: the rounds since the last cut again, one by one
            __syncthreads();
            if (tid == 0) sh.count = p.top;
            __syncthreads();
            for (int again = from; again <= round; ++again) {
              ops::Raw<F32> raw;
              get(again, raw);
              ops::unpack(raw, x);
              float top = x[0];
#pragma unroll
              for (int i = 1; i < 8; ++i) top = max_nan(top, x[i]);
              above(again, x, top);
              cut_now();
            }
          } else {
            cut_now();
          }
          from = until;
          until *= 2;
        }
      }
    }
  }
  soft = join(soft, sh);
  if (p.split > 1) {
    const long long at = row * p.split + part;
    if constexpr (TOP)
      if (tid < p.top) p.lists[at * p.top + tid] = tid < sh.count ? sh.list[tid] : 0;
    if (tid == 0) p.part[at] = make_float4(soft.m, soft.s, soft.u, 0.f);
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      sh.last = atomicAdd(&p.arrived[row], 1u) == (unsigned)p.split - 1;
      if (sh.last) p.arrived[row] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    Soft mine;
    if (tid < p.split) {
      const float4 v = __ldcg(p.part + row * p.split + tid);
      mine.m = v.x;
      mine.s = v.y;
      mine.u = v.z;
    }
    soft = join(mine, sh);
    if constexpr (TOP) {
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int i = tid; i < p.split * p.top; i += THREADS) {
        const unsigned long long key = __ldcg(p.lists + row * p.split * p.top + i);
        if (key) put(key, sh);
      }
      cut(p.top, sh);
    }
  }
  const float log_s = logf(soft.s);
  if (tid == 0) {
    if (p.logprob)
      p.logprob[row] = token < 0 ? 0.f : token < p.vocabulary ? (at_token - soft.m) - log_s : __int_as_float(0x7FC00000);
    if (p.entropy) p.entropy[row] = log_s - soft.u / soft.s;
    if (p.stats) p.stats[row] = make_float2(soft.m, log_s);
  }
  if constexpr (TOP)
    if (tid < p.top) {
      p.ids[row * p.top + tid] = index_of(sh.list[tid]);
      p.tops[row * p.top + tid] = (value_of(sh.list[tid]) - soft.m) - log_s;
    }
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
template <bool F32, bool SAME>
__global__ void __launch_bounds__(THREADS, 4) backward(const __grid_constant__ Grads p) {
  const long long row = blockIdx.x / p.pieces;
  const int piece = blockIdx.x - (int)(row * p.pieces);
  pdl_launch();
  pdl_wait();
  long long token = -1;
  if (p.tokens) token = p.tokens_64 ? static_cast<const long long*>(p.tokens)[row] : (long long)static_cast<const int*>(p.tokens)[row];
  float a = p.dlogprob && token >= 0 ? p.dlogprob[row] : 0.f;
  if (token >= p.vocabulary) a = __int_as_float(0x7FC00000);
  const float h = p.dentropy ? p.dentropy[row] : 0.f;
  const bool zero = a == 0.f && h == 0.f;  // a padded row, say: nothing is read
  const float2 st = p.stats[row];
  const float ah = h != 0.f ? fmaf(h, p.entropy[row], a) : a;
  const Row<F32> r(p.x + row * p.ld, p.vocabulary);
  uint8_t* out = p.dx + row * p.ld_d;
  auto grad = [&](float x, long long i) {
    const float l = max_nan((x - st.x) - st.y, -1000.f), e = exp_of(l);
    const float d = -e * fmaf(h, l, ah);
    return zero ? 0.f : i == token ? d + a : d;
  };
  if constexpr (SAME) {
    const int v0 = piece * EIGHTS * THREADS + (int)threadIdx.x, nv = r.eights();
    ops::Raw<F32> raw[EIGHTS];
#pragma unroll
    for (int j = 0; j < EIGHTS; ++j)
      if (!zero && v0 + j * THREADS < nv) r.load(v0 + j * THREADS, raw[j]);
#pragma unroll
    for (int j = 0; j < EIGHTS; ++j) {
      const int v = v0 + j * THREADS;
      if (v >= nv) continue;
      const long long e = r.first(v);
      float x[8];
      ops::unpack(raw[j], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = grad(x[i], e + i);
      if (e >= 0 && e + 8 <= r.n) {
        ops::Raw<F32> o;
        ops::pack(x, o);
        uint4* q = reinterpret_cast<uint4*>(out + e * (F32 ? 4 : 2));
        __stcs(q, o.a);
        if constexpr (F32) __stcs(q + 1, o.b);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i >= 0 && e + i < r.n) ops::st_any(out, e + i, x[i], F32);
      }
    }
  } else {
    const long long e0 = (long long)piece * EIGHTS * ROUND, e1 = min(e0 + EIGHTS * ROUND, (long long)p.vocabulary);
    for (long long e = e0 + threadIdx.x; e < e1; e += THREADS)
      ops::st_any(out, e, grad(zero ? 0.f : ops::ld_any(p.x + row * p.ld, e, F32), e), F32);
  }
}

}  // namespace logp
}  // namespace apk

using namespace apk;

struct apk_logprobs {
  apk_logprobs_config cfg{};
  Err err;
  int sms = 0;
  Scratch scratch;
  std::mutex mu;
};

namespace {

apk_status create(const apk_logprobs_config* cfg, apk_logprobs* h) {
  h->cfg = *cfg;
  if (h->cfg.top < 0 || h->cfg.top > logp::MAX_TOP)
    return h->err.fail(APK_EINVAL, "top is %d: 0 to %d", h->cfg.top, logp::MAX_TOP);
  APK_TRY(ops::open_device(h->cfg.device, &h->sms, &h->err));
  DeviceGuard guard(h->cfg.device);
  return h->scratch.open(h->cfg.device, &h->err);
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
  p.split = std::max(1, std::min({logp::MAX_SPLIT, V / logp::ROUND, 2 * h->sms / M}));
  APK_TRY(h->scratch.enter(s, &h->err));
  ScratchUse use(&h->scratch, &h->err);
  if (p.split > 1) {
    const size_t zeroed = ops::up256((size_t)2 * h->sms * 4), parts = (size_t)M * p.split;
    APK_TRY(use.begin(zeroed + ops::up256(parts * 16) + parts * k * 8, zeroed));
    p.arrived = reinterpret_cast<unsigned*>(h->scratch.data());
    p.part = reinterpret_cast<float4*>(h->scratch.data() + zeroed);
    p.lists = reinterpret_cast<unsigned long long*>(h->scratch.data() + zeroed + ops::up256(parts * 16));
  }
  const bool f = io->dtype == APK_F32;
  const auto kernel = k ? (f ? logp::forward<true, true> : logp::forward<false, true>)
                        : (f ? logp::forward<true, false> : logp::forward<false, false>);
  Launch l(dim3(M * p.split), logp::THREADS, 0, s);
  APK_TRY(cu_status(cudaLaunchKernelEx(&l.cfg, kernel, p), "launching the log probabilities", &h->err));
  return use.end();
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
  p.pieces = (int)(((long long)V + 7 + logp::EIGHTS * logp::ROUND - 1) / (logp::EIGHTS * logp::ROUND));
  if ((long long)M * p.pieces > 0x7FFFFFFFll) return h->err.fail(APK_EINVAL, "%d rows of %d are too many for a launch", M, V);
  const bool same = (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.dx)) % align == 0 &&
                    (M == 1 || (p.ld - p.ld_d) % align == 0);
  const bool f = g->dtype == APK_F32;
  const auto kernel = same ? (f ? logp::backward<true, true> : logp::backward<false, true>)
                           : (f ? logp::backward<true, false> : logp::backward<false, false>);
  Launch l(dim3(M * p.pieces), logp::THREADS, 0, static_cast<cudaStream_t>(g->stream));
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
