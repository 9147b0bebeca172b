// bf16 products with a fused epilogue, out = act(Q P + bias) + res, at any
// size: the layer operators' GEMM (forward, and both gradients in one
// launch).
//
// The MMA's M axis (the TMEM lanes) is the output's columns and its N axis
// the output's rows, so an epilogue warp holds 32 consecutive columns of a
// row in one register: stores, residual loads and the pre-activation are
// contiguous along a warp whatever the row stride or the base's alignment,
// the bias is one register per lane, and a call with few rows takes an MMA
// with a small N (16, 32, 64) instead of padding them to 128.
//
// Kernel<CG, FM, NT, S, SPLIT>: CG CTAs (a pair for CG = 2) compute 128 CG FM
// columns by NT rows.  Warp 0 feeds a ring of S TMA stages of 64 k, warp 1
// issues the MMAs into one of two TMEM accumulators, warps 2-9 drain the
// other: persistent CTAs walk the tiles of up to two products, so a launch
// has one tail.  Edges are TMA's zero fill on load and a predicate on store.
//
// FM = 2 (512 columns by 256 rows a pair): both accumulators belong to one
// tile, whose rows are loaded once for both.  What bounds the largest
// products is the operands' way into the SMs (37 bytes a clock and SM, 885
// clocks for a stage whose MMAs take 512); this tile loads 48 KB for two such
// steps instead of 64.  Its epilogue hides less, so the MMAs are reordered at
// both ends of a tile: the first stages feed accumulator 0 while 1 is still
// being drained, and the last ones finish 0 before 1.
//
// SPLIT: a tile's K range is shared by a cluster of 2-8 CTAs, for calls with
// fewer tiles than SMs.  Rank r owns the rows r, r + split, ...: each CTA
// stores its fp32 accumulator's rows into their owners' shared memory (stores
// need not be waited for one by one, as loads from there would), and past one
// cluster barrier the owners sum them in rank order and finish.  Nothing goes
// through global memory, and the order of the sum is fixed.
//
// EXACT: for fp32 results of long sums.  The tensor core adds each product of
// 16 k to the accumulator with truncation, a bias of about 1e-9 k of the
// result (1e-6 at 1024 k, 9e-6 at 8192); an fp32 result would show it, a bf16
// one does not.  So K is taken 512 at a time in alternating accumulators, and
// the epilogue warps add the pieces in registers with rounding.
//
// Every wait is bounded; one that runs out raises the status word and lets
// every role unwind: nothing leaves (shared memory, TMEM) before the loads and
// MMAs in flight have ended, whichever role gave up.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "linear.h"
#include "tcgen05.cuh"

namespace apk {
namespace lin {

constexpr int BK = 64;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr int P_BYTES = 128 * BK * 2;
constexpr int RASTER_GROUP = 8;
constexpr int EXACT_KB = 8;  // k-blocks of one accumulator under EXACT

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, uint32_t bits) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(bits) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(tm), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(tm), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    tc::mma_bf16(d, a, b, idesc, acc);
}
// One arrival on `bar` (a shared::cluster address) once this thread's MMAs are done.
template <int CG>
__device__ __forceinline__ void commit_to(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

template <int S>
struct __align__(16) Shared {
  uint64_t full[S], empty[S];
  uint64_t tfull[2], tempty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

// The CTA that gives up tells the other one of its pair, whose waits depend on it.
template <int CG, int S>
__device__ __forceinline__ void give_up(Shared<S>& sh) {
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
  if constexpr (CG == 2)
    asm volatile("st.volatile.shared::cluster.u32 [%0], %1;" ::"r"(map_rank(smem_u32(&sh.abort), cluster_rank() ^ 1)),
                 "r"(1)
                 : "memory");
}
template <int CG, int S>
__device__ __forceinline__ bool bwait(uint64_t* bar, uint32_t parity, const GemmParams& p, Shared<S>& sh, int code) {
  if (try_wait_cluster(bar, parity)) return true;
  const long long t0 = globaltimer_ns();
  int n = 0;
  while (true) {
    if (try_wait_cluster(bar, parity)) return true;
    if (++n == 64) {
      n = 0;
      if (*reinterpret_cast<volatile int*>(&sh.abort)) return false;
      if (globaltimer_ns() - t0 > p.limit) {
        give_up<CG>(sh);
        report_status(p.status, code, nullptr);
        return false;
      }
    }
  }
}
// At a role's end, for what it has in flight: until a second after t0, however
// short the caller's limit is.
__device__ __forceinline__ void bwait_end(uint64_t* bar, uint32_t parity, long long t0) {
  while (!try_wait_cluster(bar, parity))
    if (globaltimer_ns() - t0 > 1000000000ll) return;
}

__device__ __forceinline__ float load_elem(const void* p, long long i, int f32) {
  return f32 ? static_cast<const float*>(p)[i]
             : __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
__device__ __forceinline__ uint16_t to_bf16(float v) {
  uint16_t r;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void store_elem(void* p, long long i, float v, int f32) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = to_bf16(v);
}

// The fields in registers.  The compiler would rather load them again from
// the indexed kernel parameter at every use.
__device__ __forceinline__ Epilogue pinned(const Epilogue& c) {
  Epilogue e = c;
  asm volatile("" : "+l"(e.bias), "+l"(e.res), "+l"(e.out), "+l"(e.pre));
  asm volatile("" : "+l"(e.ld_res), "+l"(e.ld_out), "+l"(e.ld_pre));
  asm volatile("" : "+r"(e.bias_f32), "+r"(e.res_f32), "+r"(e.out_f32), "+r"(e.act));
  return e;
}

// W rows of one output column: bias, pre-activation, activation, residual,
// stores.  out and pre point at the first row's element; so and sp are the
// bytes to the next one.  The types and the presence of the pre-activation
// are fixed per call of this function: with run-time flags in the element
// loop and an address product per element the epilogue took 51 instructions a
// row and twice the time of the MMAs of 2048 k.
template <int ACT, bool PRE, bool F32, bool RES, int W>
__device__ __forceinline__ void finish_full(const uint32_t (&v)[W], const uint32_t (&raw)[W], int shift, float bias,
                                            uint8_t* out, uint8_t* pre, long long so, long long sp) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float z = __uint_as_float(v[i]) + bias;
    if (PRE) {
      *reinterpret_cast<uint16_t*>(pre) = to_bf16(z);
      pre += sp;
    }
    float y = act_f<ACT>(z);
    if (RES) y += __uint_as_float(raw[i] << shift);
    if (F32) *reinterpret_cast<float*>(out) = y;
    else *reinterpret_cast<uint16_t*>(out) = to_bf16(y);
    out += so;
  }
}
// The same for n < W rows.
template <int ACT, int W>
__device__ __forceinline__ void finish_part(const Epilogue& e, const uint32_t (&v)[W], const uint32_t (&raw)[W],
                                            int shift, float bias, uint8_t* out, uint8_t* pre, long long so,
                                            long long sp, int n) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i < n) {
      const float z = __uint_as_float(v[i]) + bias;
      if (e.pre) store_elem(pre + i * sp, 0, z, 0);
      const float res = e.res ? __uint_as_float(raw[i] << shift) : 0.f;
      store_elem(out + i * so, 0, act_f<ACT>(z) + res, e.out_f32);
    }
  }
}
// min(n, W) rows r, r + step, ... of column c; raw: their residual's bits, if
// any.  SMALL: only the code with run-time flags (where it is inlined often).
template <int W, bool SMALL = false>
__device__ __forceinline__ void finish(const Epilogue& e, const uint32_t (&v)[W], const uint32_t (&raw)[W], float bias,
                                       int r, int step, int n, long long c) {
  const int es = e.out_f32 ? 4 : 2, shift = e.res_f32 ? 0 : 16;
  uint8_t* out = static_cast<uint8_t*>(e.out) + (r * e.ld_out + c) * es;
  uint8_t* pre = static_cast<uint8_t*>(e.pre) + (r * e.ld_pre + c) * 2;
  const long long so = e.ld_out * step * es, sp = e.ld_pre * step * 2;
  with_act(e.act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    auto full = [&](auto pre_, auto f32_, auto res_) {
      finish_full<ACT, decltype(pre_)::value, decltype(f32_)::value, decltype(res_)::value, W>(v, raw, shift, bias, out,
                                                                                               pre, so, sp);
    };
    const std::true_type yes;
    const std::false_type no;
    if (SMALL || n < W) finish_part<ACT, W>(e, v, raw, shift, bias, out, pre, so, sp, n);
    else if (e.res) e.out_f32 ? (e.pre ? full(yes, yes, yes) : full(no, yes, yes))
                              : (e.pre ? full(yes, no, yes) : full(no, no, yes));
    else e.out_f32 ? (e.pre ? full(yes, yes, no) : full(no, yes, no)) : (e.pre ? full(yes, no, no) : full(no, no, no));
  });
}
// The residual of the rows r, r + step, ... (W, of which n exist), as loaded
// bits.  With a condition on every load the loads went out one by one: a full
// block has none.
template <int W>
__device__ __forceinline__ void load_residual(const Epilogue& e, uint32_t (&res)[W], int r, int step, int n,
                                              long long c) {
  const long long ld = e.ld_res * step;
  if (e.res_f32) {
    const uint32_t* p = static_cast<const uint32_t*>(e.res) + r * e.ld_res + c;
    if (n >= W) {
#pragma unroll
      for (int i = 0; i < W; ++i) res[i] = p[i * ld];
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) res[i] = i < n ? p[i * ld] : 0u;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(e.res) + r * e.ld_res + c;
    if (n >= W) {
#pragma unroll
      for (int i = 0; i < W; ++i) res[i] = p[i * ld];
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) res[i] = i < n ? p[i * ld] : 0u;
    }
  }
}

// The split K's sum for this thread's column c of the rows this rank owns
// (`own` of them, the i-th is row rank + SPLIT i of n), i = i0, i0 + 2, ...
// part: shared address of [rank][own][128] floats, at the column.
template <int SPLIT>
__device__ __forceinline__ void sum_ranks(const Epilogue& e, uint32_t part, int own, int rank, int i0, int n, int r0,
                                          long long c, float bias) {
  constexpr int U = 8, STEP = 2 * SPLIT;
  for (int i = i0; rank + SPLIT * i < n; i += 2 * U) {
    const int row = rank + SPLIT * i, left = (n - row + STEP - 1) / STEP;
    uint32_t raw[U], v[U];
    if (e.res) load_residual<U>(e, raw, r0 + row, STEP, left, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float z = 0.f;
#pragma unroll
      for (int s = 0; s < SPLIT; ++s) {
        float w;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(w) : "r"(part + (s * own + min(i + 2 * u, own - 1)) * 512));
        z += w;
      }
      v[u] = __float_as_uint(z);
    }
    finish<U>(e, v, raw, bias, r0 + row, STEP, left, c);
  }
}

template <int CG, int FM, int NT, int S, bool SPLIT, bool EXACT>
struct Cfg {
  static constexpr int QROWS = NT / CG;
  static constexpr int Q_BYTES = QROWS * BK * 2;
  static constexpr int Q_AT = FM * P_BYTES;
  static constexpr int STAGE = Q_AT + Q_BYTES;
  static constexpr int COLS = 128 * CG * FM;  // of a tile
  static constexpr int NBUF = SPLIT && !EXACT ? 1 : 2;
  static constexpr int TMEM_COLS = NBUF * NT < 32 ? 32 : NBUF * NT;
  static constexpr int SMEM = S * STAGE + (SPLIT ? NT * 512 : 0) + 1024;
  static_assert(FM == 1 || (CG == 2 && !SPLIT && !EXACT), "");
  static_assert((TMEM_COLS & (TMEM_COLS - 1)) == 0 && TMEM_COLS <= 512, "");
};

// The q-th tile of group `g` of G, or -1.  Of two products the one with the
// longer tiles comes first; groups that get one of those fewer take `extra`
// of the shorter ones each before the rest is dealt out (to them first), so
// that all end together.
__device__ __forceinline__ int tile_of(const GemmParams& p, int g, int G, int q) {
  const int n0 = p.tiles0, n1 = p.tiles - n0;
  const int mine = g < n0 ? (n0 - g + G - 1) / G : 0;
  if (q < mine) return g + q * G;
  q -= mine;
  const int rem = n0 % G, extra = rem ? p.extra : 0, others = rem ? G - rem : 0;
  const int head = min(n1, others * extra);
  if (extra && g >= rem) {
    if (q < extra) {
      const int j = g - rem + q * others;
      return j < head ? n0 + j : -1;
    }
    q -= extra;
  }
  const int j = head + (g >= rem ? g - rem : g - rem + G) + q * G;
  return j < n1 ? n0 + j : -1;
}

template <int CG, int FM, int NT, int S, bool SPLIT, bool EXACT>
__global__ void __launch_bounds__(THREADS, 1) lin_gemm(const __grid_constant__ GemmParams p) {
  using C = Cfg<CG, FM, NT, S, SPLIT, EXACT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Shared<S> sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t crank = (CG == 2 || SPLIT) ? cluster_rank() : 0;
  const uint32_t prank = CG == 2 ? crank : 0;   // rank in the MMA pair
  const int krank = SPLIT ? (int)crank : 0;     // rank in the K split
  const bool leader = prank == 0;

  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh.tfull[b], 1);
      mbar_init(&sh.tempty[b], CG * EPI_WARPS);
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbar_init();
    for (int i = 0; i < p.nprob; ++i) {
      tma_prefetch_desc(&p.pr[i].tmP);
      tma_prefetch_desc(&p.pr[i].tmQ);
    }
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)),
                   "r"(C::TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tc::tmem_alloc(&sh.tmem_base, C::TMEM_COLS);
      tc::tmem_relinquish();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2 || SPLIT) cluster_sync();
  tc::fence_after_sync();
  pdl_launch();
  pdl_wait();
  const uint32_t tbase = sh.tmem_base;

  // The tiles of this CTA (pair, cluster): tile_of(q), q = 0, 1, ...
  const int group = CG == 2 ? 2 : SPLIT ? p.split : 1;
  const int gi = (int)blockIdx.x / group, groups = (int)gridDim.x / group;
  auto tile = [&](int q) { return tile_of(p, gi, groups, q); };
  // tile t: its product, and its first row and column (this CTA's column in a pair)
  auto locate = [&](int t, int& r0, int& c0) -> const Problem& {
    const Problem& pr = p.pr[t < p.tiles0 ? 0 : 1];
    int tr, tc_;
    tile_coords(t < p.tiles0 ? t : t - p.tiles0, pr.tiles_r, pr.tiles_c, RASTER_GROUP, tr, tc_);
    r0 = tr * NT;
    c0 = tc_ * C::COLS + 128 * (int)prank;
    return pr;
  };
  auto k_range = [&](const Problem& pr, int& kb, int& ke) {
    kb = SPLIT ? pr.nkb * krank / p.split : 0;
    ke = SPLIT ? pr.nkb * (krank + 1) / p.split : pr.nkb;
  };

  // accumulators that a tile's n k-blocks are spread over
  auto pieces = [](int n) { return EXACT ? max(1, (n + EXACT_KB - 1) / EXACT_KB) : 1; };

  if (warp == 0 && lane == 0) {
    // ================================ producer ================================
    uint32_t P = 0;
    bool ok = true;
    for (int q = 0, t; ok && (t = tile(q)) >= 0; ++q) {
      int r0, c0, kb, ke;
      const Problem& pr = locate(t, r0, c0);
      k_range(pr, kb, ke);
      r0 += C::QROWS * (int)prank;
      for (; kb < ke; ++kb, ++P) {
        const int s = P % S;
        ok = bwait<CG>(&sh.empty[s], ((P / S) & 1) ^ 1, p, sh, DEV_WAIT_TIMEOUT_FULL);
        if (!ok) break;
        // both CTAs' loads of a pair complete on the leader's barrier
        uint32_t bar = smem_u32(&sh.full[s]);
        if constexpr (CG == 2) bar = map_rank(bar, 0);
        if (leader) mbar_arrive_expect_tx(&sh.full[s], CG * C::STAGE);
        const uint32_t d = smem_u32(ring + s * C::STAGE);
        const int k = kb * BK;
#pragma unroll
        for (int h = 0; h < FM; ++h) {
          const uint32_t at = d + h * P_BYTES;
          const int c = c0 + 128 * CG * h;
          if (pr.p_mn) {
            load_box<CG>(at, &pr.tmP, c, k, bar);
            load_box<CG>(at + 8192, &pr.tmP, c + 64, k, bar);
          } else {
            load_box<CG>(at, &pr.tmP, k, c, bar);
          }
        }
        if (NT >= 64 && pr.q_mn) {
#pragma unroll
          for (int b = 0; b < C::QROWS / 64; ++b)
            load_box<CG>(d + C::Q_AT + b * 8192, &pr.tmQ, r0 + 64 * b, k, bar);
        } else {
          load_box<CG>(d + C::Q_AT, &pr.tmQ, k, r0, bar);
        }
      }
    }
    // The loads in flight land before the shared memory goes away.  They have
    // landed already unless another role gave up, which this one may not have
    // noticed.  (A pair's loads complete on the leader's barriers.)
    if (leader) {
      const long long t0 = globaltimer_ns();
      for (uint32_t q = P > (uint32_t)S ? P - S : 0; q < P; ++q) bwait_end(&sh.full[q % S], (q / S) & 1, t0);
    }
  } else if (warp == 1 && lane == 0 && leader) {
    // =================================== MMA ===================================
    uint32_t Q = 0, U = 0;  // stages and accumulators used
    bool ok = true;
    // an arrival in every CTA of the pair once the MMAs issued so far are done
    auto commit_all = [&](uint64_t* bar) {
      const uint32_t a = smem_u32(bar);
      if constexpr (CG == 2) {
        commit_to<CG>(map_rank(a, 0));
        commit_to<CG>(map_rank(a, 1));
      } else {
        commit_to<CG>(a);
      }
    };
    for (int T = 0, t; ok && (t = tile(T)) >= 0; ++T) {
      int r0, c0, kb, ke;
      const Problem& pr = locate(t, r0, c0);
      k_range(pr, kb, ke);
      const uint32_t idesc = pr.idesc;
      const uint32_t p_step = pr.p_mn ? 2048 : 32, q_step = pr.q_mn ? 2048 : 32;
      const uint32_t p_lbo = pr.p_mn ? 8192 : 16, q_lbo = pr.q_mn ? 8192 : 16;
      auto full = [&](uint32_t i) { return bwait<CG>(&sh.full[i % S], (i / S) & 1, p, sh, DEV_WAIT_TIMEOUT_FULL); };
      // stage i's MMAs with the h-th 128 columns of each CTA into accumulator buf
      auto mmas = [&](uint32_t i, int h, int buf, bool first) {
        const uint32_t sp = smem_u32(ring + (i % S) * C::STAGE) + h * P_BYTES, sq = smem_u32(ring + (i % S) * C::STAGE) + C::Q_AT;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          mma<CG>(tbase + (uint32_t)buf * NT, tc::smem_desc(sp + kk * p_step, p_lbo, 1024, tc::LAYOUT_SW128),
                  tc::smem_desc(sq + kk * q_step, q_lbo, 1024, tc::LAYOUT_SW128), idesc, (!first || kk > 0) ? 1u : 0u);
      };
      const int n = ke - kb;
      if constexpr (FM == 1) {
        for (int c = 0; c < pieces(n) && ok; ++c, ++U) {
          const int buf = U % C::NBUF, i0 = EXACT ? c * EXACT_KB : 0, i1 = EXACT ? min(n, i0 + EXACT_KB) : n;
          ok = bwait<CG>(&sh.tempty[buf], ((U / C::NBUF) & 1) ^ 1, p, sh, DEV_WAIT_TIMEOUT_TMEM);
          if (!ok) break;
          tc::fence_after_sync();
          for (int i = i0; i < i1; ++i, ++Q) {
            ok = full(Q);
            if (!ok) break;
            mmas(Q, 0, buf, i == i0);
            commit_all(&sh.empty[Q % S]);
          }
          if (ok) commit_all(&sh.tfull[buf]);
        }
      } else {
        // stages i = 0 .. w: accumulator 0 first; n - l .. n: 0 before 1
        const int w = n < S - 1 ? n : S - 1, l = n - w < S - 1 ? n - w : S - 1;
        ok = bwait<CG>(&sh.tempty[0], (T & 1) ^ 1, p, sh, DEV_WAIT_TIMEOUT_TMEM);
        if (!ok) break;
        tc::fence_after_sync();
        for (int i = 0; i < w && ok; ++i) {
          ok = full(Q + i);
          if (ok) mmas(Q + i, 0, 0, i == 0);
        }
        ok = ok && bwait<CG>(&sh.tempty[1], (T & 1) ^ 1, p, sh, DEV_WAIT_TIMEOUT_TMEM);
        if (!ok) break;
        tc::fence_after_sync();
        if (l == 0) commit_all(&sh.tfull[0]);
        for (int i = 0; i < w; ++i) {
          mmas(Q + i, 1, 1, i == 0);
          commit_all(&sh.empty[(Q + i) % S]);
        }
        for (int i = w; i < n - l && ok; ++i) {
          ok = full(Q + i);
          if (!ok) break;
          mmas(Q + i, 0, 0, false);
          mmas(Q + i, 1, 1, false);
          commit_all(&sh.empty[(Q + i) % S]);
        }
        for (int i = n - l; i < n && ok; ++i) {
          ok = full(Q + i);
          if (ok) mmas(Q + i, 0, 0, false);
        }
        if (!ok) break;
        if (l > 0) commit_all(&sh.tfull[0]);
        for (int i = n - l; i < n; ++i) {
          mmas(Q + i, 1, 1, false);
          commit_all(&sh.empty[(Q + i) % S]);
        }
        commit_all(&sh.tfull[1]);
        Q += n;
      }
    }
    // The MMAs in flight end before the tensor memory and the operands go
    // away.  The epilogue has waited for them, unless it gave up.
    commit_to<CG>(smem_u32(&sh.drain));
    bwait_end(&sh.drain, 0, globaltimer_ns());
  } else if (warp >= 2) {
    // ================================ epilogue ================================
    constexpr int W = NT >= 64 ? 32 : 8;  // rows of one TMEM load
    const int q = warp & 3, g = (warp - 2) >> 2;
    // i: tiles, or half tiles of FM = 2; U: accumulators drained
    uint32_t U = 0;
    for (int i = 0, t; (t = tile(i / FM)) >= 0; ++i) {
      int r0, c0, kb, ke;
      const Problem& pr = locate(t, r0, c0);
      k_range(pr, kb, ke);
      c0 += 128 * CG * (i % FM);
      const Epilogue e = pinned(pr.epi);
      const int col = 32 * q + lane;
      const bool in = c0 + col < pr.cols;
      const long long c = c0 + col;
      float bias = 0.f;
      if (!SPLIT && in && e.bias) bias = load_elem(e.bias, c, e.bias_f32);
      const bool has_res = !SPLIT && e.res && in;
      uint32_t raw[W];
      if (has_res && r0 + g * W < pr.rows) load_residual<W>(e, raw, r0 + g * W, 1, pr.rows - r0 - g * W, c);
      const uint32_t tcol = tbase + ((uint32_t)(32 * q) << 16);
      auto wait_acc = [&]() {
        const bool ok = bwait<CG>(&sh.tfull[U % C::NBUF], (U / C::NBUF) & 1, p, sh, DEV_WAIT_TIMEOUT_TMEM);
        tc::fence_after_sync();
        return ok;
      };
      auto free_acc = [&]() {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) arrive_cluster(map_rank(smem_u32(&sh.tempty[U % C::NBUF]), 0));
          else mbar_arrive(&sh.tempty[U % C::NBUF]);
        }
        ++U;
      };
      // a split tile's rows to their owners; a CTA whose share of K is empty sends zeros
      auto push = [&](int b, const uint32_t(&v)[W]) {
        const uint32_t at = smem_u32(ring + S * C::STAGE) + (uint32_t)(krank * (NT / p.split) * 512 + col * 4);
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const int row = b * W + k;
          st_cluster_f32(map_rank(at, row & (p.split - 1)) + (row / p.split) * 512, kb < ke ? v[k] : 0u);
        }
      };
      if constexpr (EXACT) {
        constexpr int NB = NT / W / 2;  // this warp's blocks
        uint32_t acc[NB][W] = {};
        bool ok = true;
        for (int k = pieces(ke - kb); k > 0; --k) {
          ok = wait_acc();
          if (!ok) break;
          const uint32_t ta = tcol + (U % C::NBUF) * NT;
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            uint32_t v[W];
            tc::ld_32x32b<W>(ta + (g + 2 * j) * W, v);
            tc::wait_ld();
#pragma unroll
            for (int x = 0; x < W; ++x) acc[j][x] = __float_as_uint(__uint_as_float(acc[j][x]) + __uint_as_float(v[x]));
          }
          free_acc();
        }
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int b = g + 2 * j, r = r0 + b * W, n = pr.rows - r;
          if constexpr (SPLIT) {
            push(b, acc[j]);
          } else if (in && n > 0) {
            if (has_res && j > 0) load_residual<W>(e, raw, r, 1, n, c);
            finish<W, true>(e, acc[j], raw, bias, r, 1, n, c);
          }
        }
        continue;
      }
      if (!wait_acc()) break;
      const uint32_t ta = tcol + (U % C::NBUF) * NT;
#pragma unroll 1
      for (int b = g; b < NT / W; b += 2) {
        const int r = r0 + b * W, n = pr.rows - r;
        uint32_t v[W];
        if constexpr (SPLIT) {
          tc::ld_32x32b<W>(ta + b * W, v);
          tc::wait_ld();
          push(b, v);
        } else {
          if (n <= 0) break;  // (uniform; later blocks lie further out)
          tc::ld_32x32b<W>(ta + b * W, v);
          uint32_t res[W];
          if (e.res) {
#pragma unroll
            for (int k = 0; k < W; ++k) res[k] = raw[k];
          }
          if (has_res && b + 2 < NT / W && n > 2 * W) load_residual<W>(e, raw, r + 2 * W, 1, n - 2 * W, c);
          tc::wait_ld();
          if (in) finish<W>(e, v, res, bias, r, 1, n, c);
          __syncwarp();
        }
      }
      if constexpr (SPLIT) break;  // one tile a cluster
      free_acc();
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if constexpr (SPLIT) {
    cluster_sync();  // every rank's rows have arrived
    int r0, c0;
    const Problem& pr = locate(gi, r0, c0);
    const Epilogue e = pr.epi;  // in registers: a field of an indexed kernel parameter costs 80 cycles a use
    if (tid < 256 && !sh.abort) {
      const int col = tid & 127;
      const long long c = c0 + col;
      if (c < pr.cols) {
        const float bias = e.bias ? load_elem(e.bias, c, e.bias_f32) : 0.f;
        const uint32_t part = smem_u32(ring + S * C::STAGE) + col * 4;
        const int n = min(NT, pr.rows - r0), i0 = tid >> 7, own = NT / p.split;
        if (p.split == 2) sum_ranks<2>(e, part, own, krank, i0, n, r0, c, bias);
        else if (p.split == 4) sum_ranks<4>(e, part, own, krank, i0, n, r0, c, bias);
        else sum_ranks<8>(e, part, own, krank, i0, n, r0, c, bias);
      }
    }
  }
  if constexpr (CG == 2) {
    cluster_sync();  // no access reaches a CTA that has left
    // After a wait ran out the leader may have stopped before it expected the
    // other CTA's last loads, so that no barrier tells when they have landed: a
    // millisecond is a thousand times what a load takes.
    if (warp == 0 && *reinterpret_cast<volatile int*>(&sh.abort)) {
      const long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000) __nanosleep(1000);
    }
  }
  if (warp == 1) {
    __syncwarp();
    tc::fence_after_sync();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(C::TMEM_COLS) : "memory");
    else
      tc::tmem_dealloc(tbase, C::TMEM_COLS);
  }
  if constexpr (CG == 2) cluster_sync();
}

// ------------------------------------------------------------------- host side

namespace {

struct Variant {
  int cg, fm, nt, stages;
  bool split, exact;
  const void* fn;
  int smem;
};
template <int CG, int FM, int NT, int S, bool SPLIT, bool EXACT = false>
Variant variant() {
  return {CG,    FM, NT, S, SPLIT, EXACT, reinterpret_cast<const void*>(&lin_gemm<CG, FM, NT, S, SPLIT, EXACT>),
          Cfg<CG, FM, NT, S, SPLIT, EXACT>::SMEM};
}
const Variant* variants(int* n) {
  static const Variant v[] = {
      variant<2, 2, 256, 4, false>(), variant<2, 1, 256, 6, false>(), variant<1, 1, 128, 6, false>(),
      variant<1, 1, 64, 8, false>(),  variant<1, 1, 32, 8, false>(),  variant<1, 1, 16, 8, false>(),
      variant<1, 1, 128, 4, true>(),  variant<1, 1, 64, 7, true>(),   variant<1, 1, 32, 8, true>(),
      variant<1, 1, 16, 8, true>(),   variant<2, 1, 128, 8, false, true>(), variant<1, 1, 64, 8, false, true>(),
      variant<1, 1, 64, 7, true, true>()};
  *n = (int)(sizeof v / sizeof v[0]);
  return v;
}

PFN_cuTensorMapEncodeTiled_v12000 g_enc = nullptr;
std::mutex g_mu;
bool g_ready[64] = {};

apk_status encode(CUtensorMap* tm, const Operand& o, int box_inner, int box_outer, std::string* why) {
  cuuint64_t dims[2] = {(cuuint64_t)o.inner, (cuuint64_t)o.outer};
  cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(o.p), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return APK_OK;
  char buf[160];
  snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed (%d) for a %d x %d operand, row stride %lld", (int)r,
           o.outer, o.inner, o.ld);
  *why = buf;
  return APK_ECUDA;
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

struct Choice {
  const Variant* v;
  int split;
  int slots;  // CTAs, pairs or clusters that are resident at once
  double cost;
};

// Clusters of 2, 4 and 8 CTAs (index log2) that can be resident at once: an
// SM cluster lies within one GPC, so eight CTAs find fewer places than 148 / 8.
int g_clusters[64][4];

// The variant with the least estimated time for these products on `sms` SMs,
// in SM clocks.  Per 64-deep k-block and tile: the MMA's own time (128 x NT x
// 64 at 4096 MAC per clock and SM) or the time a stage takes to arrive at an
// SM (37 bytes a clock measured for the pairs, 45 for single CTAs: the widest
// tile is bound by this); for the whole: its bytes at the memory's
// rate (3300 a clock).  A tile's epilogue takes 8500 clocks per 256 rows of a
// CTA's 128 columns (measured without residual or activation; they add about
// 4000 and 3000); a second accumulator hides it behind the next tile, or half
// of it where both belong to one tile.  A split adds its barrier and sum.
Choice choose(const Product* pr, int n, int sms, int dev) {
  int nv;
  const Variant* vs = variants(&nv);
  double bytes = 0, epi = 0;
  for (int j = 0; j < n; ++j)
    epi = std::max(epi, 8500.0 + (pr[j].epi.act != APK_ACT_NONE ? 3000 : 0) + (pr[j].epi.res ? 4000 : 0));
  for (int j = 0; j < n; ++j)
    bytes += 2.0 * ((double)pr[j].rows * pr[j].k + (double)pr[j].cols * pr[j].k + (double)pr[j].rows * pr[j].cols);
  bool exact = false;  // a long sum that is not rounded to bf16
  for (int j = 0; j < n; ++j) exact = exact || (pr[j].epi.out_f32 && pr[j].k > EXACT_KB * BK);
  Choice best{nullptr, 1, 1, 0};
  for (int i = 0; i < nv; ++i) {
    const Variant& v = vs[i];
    bool fits = v.exact == exact;
    for (int j = 0; j < n; ++j) fits = fits && !(pr[j].Q.mn && v.nt < 64);
    if (!fits) continue;
    const double per_kb = std::max(v.nt * 2.0 * v.fm, (v.fm * P_BYTES + v.nt / v.cg * 128) / (v.cg == 2 ? 37.0 : 45.0));
    for (int lg = v.split ? 1 : 0; lg <= (v.split ? 3 : 0); ++lg) {
      const int sp = 1 << lg, per = v.cg * sp;
      if (per > sms) continue;
      int slots = std::max(1, sms / per);
      if (per > 1) slots = std::max(1, std::min(slots, g_clusters[dev][per == 2 ? 1 : lg]));
      long long tiles = 0;
      double work = 0, longest = 0;
      for (int j = 0; j < n; ++j) {
        const long long t = (long long)ceil_div(pr[j].rows, v.nt) * ceil_div(pr[j].cols, 128 * v.cg * v.fm);
        const double mma = ceil_div(ceil_div(pr[j].k, BK), sp) * per_kb, drain = epi * v.nt / 256;
        const double one = v.fm == 2 ? mma + 1.5 * drain : v.split ? mma : std::max(mma, drain) + 150;
        tiles += t;
        work += t * one;
        longest = std::max(longest, one);
      }
      if (v.split && tiles > slots) continue;  // one tile per cluster, all resident
      // one product runs in whole sweeps; two are dealt out evenly but for half a tile
      const double sweeps = n == 1 ? (double)((tiles + slots - 1) / slots) * longest : work / slots + longest / 2;
      double cost = 6000 + std::max(bytes / 3300, std::max(longest, sweeps));
      if (v.fm == 1) cost += v.nt * 20.0;  // the last tile's epilogue
      if (v.split) cost += 1500 + v.nt / sp * 6.0;
      if (!best.v || cost < best.cost) best = {&v, sp, slots, cost};
    }
  }
  return best;
}

}  // namespace

cudaError_t prepare() {
  std::lock_guard<std::mutex> lock(g_mu);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int nv;
  const Variant* vs = variants(&nv);
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!g_ready[dev]) {
    if (!g_enc) {
      cudaDriverEntryPointQueryResult q;
      void* fn = nullptr;
      e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q);
      if (e != cudaSuccess) return e;
      if (q != cudaDriverEntryPointSuccess || !fn) return cudaErrorSymbolNotFound;
      g_enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
    for (int i = 0; i < nv; ++i) {
      e = cudaFuncSetAttribute(vs[i].fn, cudaFuncAttributeMaxDynamicSharedMemorySize, vs[i].smem);
      if (e != cudaSuccess) return e;
    }
    // the largest shared memory of each cluster size decides
    for (int lg = 1; lg <= 3; ++lg) {
      g_clusters[dev][lg] = 1 << 20;
      for (int i = 0; i < nv; ++i) {
        if (!(vs[i].split || (vs[i].cg == 2 && lg == 1))) continue;
        Launch l(dim3(1 << lg), THREADS, vs[i].smem, nullptr, 1 << lg);
        int c = 0;
        e = cudaOccupancyMaxActiveClusters(&c, vs[i].fn, &l.cfg);
        if (e != cudaSuccess) return e;
        g_clusters[dev][lg] = std::min(g_clusters[dev][lg], c);
      }
    }
    g_ready[dev] = true;
  }
  return cudaSuccess;
}

apk_status run_products(const Product* pr, int n, int sms, int dev, int* status, long long limit, cudaStream_t stream,
                        std::string* why) {
  Product longer_first[2];
  if (n == 2 && pr[0].k < pr[1].k) {
    longer_first[0] = pr[1];
    longer_first[1] = pr[0];
    pr = longer_first;
  }
  const Choice ch = choose(pr, n, sms, dev);
  if (n == 2) {
    // products that want different tiles run one after the other
    const double apart = choose(pr, 1, sms, dev).cost + choose(pr + 1, 1, sms, dev).cost;
    if (apart + 8000 < ch.cost) {  // (a second launch, and a second tail)
      const apk_status st = run_products(pr, 1, sms, dev, status, limit, stream, why);
      return st != APK_OK ? st : run_products(pr + 1, 1, sms, dev, status, limit, stream, why);
    }
  }
  const Variant& v = *ch.v;
  GemmParams p;
  p.nprob = n;
  p.tiles = 0;
  p.tiles0 = 0;
  p.split = ch.split;
  p.extra = n == 2 && !v.split ? ceil_div(pr[0].k, BK) / ceil_div(pr[1].k, BK) : 0;
  p.status = status;
  p.limit = limit;
  for (int j = 0; j < n; ++j) {
    Problem& q = p.pr[j];
    q.epi = pr[j].epi;
    q.rows = pr[j].rows;
    q.cols = pr[j].cols;
    q.nkb = ceil_div(pr[j].k, BK);
    q.tiles_r = ceil_div(q.rows, v.nt);
    q.tiles_c = ceil_div(q.cols, 128 * v.cg * v.fm);
    q.p_mn = pr[j].P.mn;
    q.q_mn = pr[j].Q.mn;
    q.idesc = tc::idesc_bf16_f32(128 * v.cg, v.nt, q.p_mn, q.q_mn);
    apk_status st = encode(&q.tmP, pr[j].P, 64, q.p_mn ? 64 : 128, why);
    if (st == APK_OK) st = encode(&q.tmQ, pr[j].Q, 64, q.q_mn ? 64 : v.nt / v.cg, why);
    if (st != APK_OK) return st;
    if ((long long)q.tiles_r * q.tiles_c + p.tiles > (1 << 28)) {
      *why = "too many output tiles";
      return APK_EINVAL;
    }
    p.tiles += q.tiles_r * q.tiles_c;
    if (j == 0) p.tiles0 = p.tiles;
  }
  const int cl = v.split ? ch.split : v.cg;
  const int groups = v.split ? p.tiles : std::min(p.tiles, ch.slots);
  Launch l(dim3(groups * cl), THREADS, v.smem, stream, cl);
  void* args[] = {&p};
  const cudaError_t e = cudaLaunchKernelExC(&l.cfg, v.fn, args);
  if (e != cudaSuccess) {
    *why = std::string("launching the linear kernel: ") + cudaGetErrorString(e);
    return APK_ECUDA;
  }
  return APK_OK;
}

}  // namespace lin
}  // namespace apk
