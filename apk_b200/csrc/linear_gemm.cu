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
// Kernel<CG, NT, S, SPLIT>: CG CTAs (a pair for CG = 2) compute 128 CG columns
// by NT rows.  Warp 0 feeds a ring of S TMA stages of 64 k, warp 1 issues
// the MMAs into one of two TMEM accumulators, warps 2-9 drain the other:
// persistent CTAs walk the tiles of up to two products, so a launch has one
// tail.  Edges are TMA's zero fill on load and a predicate on store.
//
// SPLIT: a tile's K range is shared by a cluster of 2-8 CTAs, for calls with
// fewer tiles than SMs.  Each leaves its fp32 accumulator in its own shared
// memory (the drained ring) and, past a cluster barrier, sums every
// p.split-th row over the cluster in rank order: nothing goes through global
// memory, and the order of the sum is fixed.
//
// Every wait is bounded; one that runs out raises the status word and lets
// every role unwind.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

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
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
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

template <int S>
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
        *reinterpret_cast<volatile int*>(&sh.abort) = 1;
        report_status(p.status, code, nullptr);
        return false;
      }
    }
  }
}
__device__ __forceinline__ void bwait_unwind(uint64_t* bar, uint32_t parity, long long limit) {
  const long long t0 = globaltimer_ns();
  while (!try_wait_cluster(bar, parity))
    if (globaltimer_ns() - t0 > limit) return;
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

// W rows of one output column: bias, pre-activation, activation, residual,
// stores.  out and pre point at the first row's element.  The types and the
// presence of the pre-activation are fixed per call of this function: with
// run-time flags in the element loop and an address product per element the
// epilogue took 51 instructions a row and twice the time of the MMAs of 2048 k.
template <int ACT, bool PRE, bool F32, int W>
__device__ __forceinline__ void finish_full(const Epilogue& e, const uint32_t (&v)[W], const float (&res)[W],
                                            float bias, uint8_t* out, uint8_t* pre) {
  const long long so = e.ld_out * (F32 ? 4 : 2), sp = e.ld_pre * 2;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float z = __uint_as_float(v[i]) + bias;
    if (PRE) {
      *reinterpret_cast<uint16_t*>(pre) = to_bf16(z);
      pre += sp;
    }
    const float y = act_f<ACT>(z) + res[i];
    if (F32) *reinterpret_cast<float*>(out) = y;
    else *reinterpret_cast<uint16_t*>(out) = to_bf16(y);
    out += so;
  }
}
// The same for a block that reaches past the last row.
template <int ACT, int W>
__device__ __forceinline__ void finish_part(const Epilogue& e, const uint32_t (&v)[W], const float (&res)[W],
                                            float bias, uint8_t* out, uint8_t* pre, int n) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i < n) {
      const float z = __uint_as_float(v[i]) + bias;
      if (e.pre) store_elem(pre, i * e.ld_pre, z, 0);
      store_elem(out, i * e.ld_out, act_f<ACT>(z) + res[i], e.out_f32);
    }
  }
}
template <int W>
__device__ __forceinline__ void load_residual(const Epilogue& e, float (&res)[W], int r, int n, long long c) {
  if (e.res_f32) {
    const float* p = static_cast<const float*>(e.res) + r * e.ld_res + c;
#pragma unroll
    for (int i = 0; i < W; ++i, p += e.ld_res) res[i] = i < n ? *p : 0.f;
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(e.res) + r * e.ld_res + c;
    uint16_t h[W];
#pragma unroll
    for (int i = 0; i < W; ++i, p += e.ld_res) h[i] = i < n ? *p : (uint16_t)0;
#pragma unroll
    for (int i = 0; i < W; ++i) res[i] = __uint_as_float((uint32_t)h[i] << 16);
  }
}

template <int CG, int NT, int S, bool SPLIT>
struct Cfg {
  static constexpr int QROWS = NT / CG;
  static constexpr int Q_BYTES = QROWS * BK * 2;
  static constexpr int STAGE = P_BYTES + Q_BYTES;
  static constexpr int NBUF = SPLIT ? 1 : 2;
  static constexpr int TMEM_COLS = NBUF * NT < 32 ? 32 : NBUF * NT;
  static constexpr int SMEM = S * STAGE + 1024;
  static_assert(!SPLIT || S * STAGE >= NT * 512, "the split sum reuses the ring");
  static_assert((TMEM_COLS & (TMEM_COLS - 1)) == 0 && TMEM_COLS <= 512, "");
};

template <int CG, int NT, int S, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) lin_gemm(const __grid_constant__ GemmParams p) {
  using C = Cfg<CG, NT, S, SPLIT>;
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

  // The tiles of this CTA (pair, cluster): t0, t0 + step, ...
  const int group = CG == 2 ? 2 : SPLIT ? p.split : 1;
  const int t0 = (int)blockIdx.x / group, step = (int)gridDim.x / group;
  // tile t: its product, and its first row and column (this CTA's column in a pair)
  auto locate = [&](int t, int& r0, int& c0) -> const Problem& {
    const Problem& pr = p.pr[t < p.tiles0 ? 0 : 1];
    int tr, tc_;
    tile_coords(t < p.tiles0 ? t : t - p.tiles0, pr.tiles_r, pr.tiles_c, RASTER_GROUP, tr, tc_);
    r0 = tr * NT;
    c0 = tc_ * 128 * CG + 128 * (int)prank;
    return pr;
  };
  auto k_range = [&](const Problem& pr, int& kb, int& ke) {
    kb = SPLIT ? pr.nkb * krank / p.split : 0;
    ke = SPLIT ? pr.nkb * (krank + 1) / p.split : pr.nkb;
  };

  if (warp == 0 && lane == 0) {
    // ================================ producer ================================
    uint32_t P = 0;
    bool ok = true;
    for (int t = t0; t < p.tiles && ok; t += step) {
      int r0, c0, kb, ke;
      const Problem& pr = locate(t, r0, c0);
      k_range(pr, kb, ke);
      r0 += C::QROWS * (int)prank;
      for (; kb < ke; ++kb, ++P) {
        const int s = P % S;
        ok = bwait(&sh.empty[s], ((P / S) & 1) ^ 1, p, sh, DEV_WAIT_TIMEOUT_FULL);
        if (!ok) break;
        // both CTAs' loads of a pair complete on the leader's barrier
        uint32_t bar = smem_u32(&sh.full[s]);
        if constexpr (CG == 2) bar = map_rank(bar, 0);
        if (leader) mbar_arrive_expect_tx(&sh.full[s], CG * C::STAGE);
        const uint32_t d = smem_u32(ring + s * C::STAGE);
        const int k = kb * BK;
        if (pr.p_mn) {
          load_box<CG>(d, &pr.tmP, c0, k, bar);
          load_box<CG>(d + 8192, &pr.tmP, c0 + 64, k, bar);
        } else {
          load_box<CG>(d, &pr.tmP, k, c0, bar);
        }
        if (NT >= 64 && pr.q_mn) {
#pragma unroll
          for (int b = 0; b < C::QROWS / 64; ++b)
            load_box<CG>(d + P_BYTES + b * 8192, &pr.tmQ, r0 + 64 * b, k, bar);
        } else {
          load_box<CG>(d + P_BYTES, &pr.tmQ, k, r0, bar);
        }
      }
    }
    if (!ok && leader) {
      // unwinding: the loads in flight land before the shared memory goes away
      for (uint32_t q = P > (uint32_t)S ? P - S : 0; q < P; ++q)
        bwait_unwind(&sh.full[q % S], (q / S) & 1, p.limit);
    }
  } else if (warp == 1 && lane == 0 && leader) {
    // =================================== MMA ===================================
    uint32_t Q = 0, T = 0;
    bool ok = true;
    for (int t = t0; t < p.tiles && ok; t += step, ++T) {
      int r0, c0, kb, ke;
      const Problem& pr = locate(t, r0, c0);
      k_range(pr, kb, ke);
      const int buf = T % C::NBUF;
      ok = bwait(&sh.tempty[buf], ((T / C::NBUF) & 1) ^ 1, p, sh, DEV_WAIT_TIMEOUT_TMEM);
      if (!ok) break;
      tc::fence_after_sync();
      const uint32_t d = tbase + (uint32_t)buf * NT;
      const uint32_t idesc = pr.idesc;
      const uint32_t p_step = pr.p_mn ? 2048 : 32, q_step = pr.q_mn ? 2048 : 32;
      const uint32_t p_lbo = pr.p_mn ? 8192 : 16, q_lbo = pr.q_mn ? 8192 : 16;
      for (int k = kb; k < ke; ++k, ++Q) {
        const int s = Q % S;
        ok = bwait(&sh.full[s], (Q / S) & 1, p, sh, DEV_WAIT_TIMEOUT_FULL);
        if (!ok) break;
        const uint32_t sp = smem_u32(ring + s * C::STAGE), sq = sp + P_BYTES;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          mma<CG>(d, tc::smem_desc(sp + kk * p_step, p_lbo, 1024, tc::LAYOUT_SW128),
                  tc::smem_desc(sq + kk * q_step, q_lbo, 1024, tc::LAYOUT_SW128), idesc, (k > kb || kk > 0) ? 1u : 0u);
        const uint32_t e = smem_u32(&sh.empty[s]);
        if constexpr (CG == 2) {
          commit_to<CG>(map_rank(e, 0));
          commit_to<CG>(map_rank(e, 1));
        } else {
          commit_to<CG>(e);
        }
      }
      if (!ok) break;
      const uint32_t f = smem_u32(&sh.tfull[buf]);
      if constexpr (CG == 2) {
        commit_to<CG>(map_rank(f, 0));
        commit_to<CG>(map_rank(f, 1));
      } else {
        commit_to<CG>(f);
      }
    }
    if (!ok) {
      commit_to<CG>(smem_u32(&sh.drain));
      bwait_unwind(&sh.drain, 0, p.limit);
    }
  } else if (warp >= 2) {
    // ================================ epilogue ================================
    constexpr int W = NT >= 64 ? 32 : 8;  // rows of one TMEM load
    const int q = warp & 3, g = (warp - 2) >> 2;
    uint32_t T = 0;
    for (int t = t0; t < p.tiles; t += step, ++T) {
      int r0, c0;
      const Problem& pr = locate(t, r0, c0);
      const Epilogue& e = pr.epi;
      const int buf = T % C::NBUF;
      const int col = 32 * q + lane;
      const bool in = c0 + col < pr.cols;
      const long long c = c0 + col;
      float bias = 0.f;
      if (!SPLIT && in && e.bias) bias = load_elem(e.bias, c, e.bias_f32);
      if (!bwait(&sh.tfull[buf], (T / C::NBUF) & 1, p, sh, DEV_WAIT_TIMEOUT_TMEM)) break;
      tc::fence_after_sync();
      const uint32_t ta = tbase + ((uint32_t)(32 * q) << 16) + (uint32_t)buf * NT;
      if constexpr (SPLIT) {
        // the accumulator, [row][128 columns] in the drained ring; a CTA
        // whose share of K is empty holds zero
        int kb, ke;
        k_range(pr, kb, ke);
        float* part = reinterpret_cast<float*>(ring);
#pragma unroll 1
        for (int b = g; b < NT / W; b += 2) {
          uint32_t v[W];
          tc::ld_32x32b<W>(ta + b * W, v);
          tc::wait_ld();
#pragma unroll
          for (int i = 0; i < W; ++i) part[(b * W + i) * 128 + col] = kb < ke ? __uint_as_float(v[i]) : 0.f;
        }
      } else {
#pragma unroll 1
        for (int b = g; b < NT / W; b += 2) {
          const int r = r0 + b * W;
          if (r >= pr.rows) break;  // (uniform; later blocks lie further out)
          uint32_t v[W];
          float res[W];
          tc::ld_32x32b<W>(ta + b * W, v);
          const int n = pr.rows - r;
          if (e.res && in) {
            load_residual<W>(e, res, r, n, c);
          } else {
#pragma unroll
            for (int i = 0; i < W; ++i) res[i] = 0.f;
          }
          tc::wait_ld();
          if (in) {
            uint8_t* out = static_cast<uint8_t*>(e.out) + (r * e.ld_out + c) * (e.out_f32 ? 4 : 2);
            uint8_t* pre = static_cast<uint8_t*>(e.pre) + (r * e.ld_pre + c) * 2;
            with_act(e.act, [&](auto a) {
              constexpr int ACT = decltype(a)::value;
              if (n < W) finish_part<ACT, W>(e, v, res, bias, out, pre, n);
              else if (e.out_f32 && e.pre) finish_full<ACT, true, true, W>(e, v, res, bias, out, pre);
              else if (e.out_f32) finish_full<ACT, false, true, W>(e, v, res, bias, out, pre);
              else if (e.pre) finish_full<ACT, true, false, W>(e, v, res, bias, out, pre);
              else finish_full<ACT, false, false, W>(e, v, res, bias, out, pre);
            });
          }
          __syncwarp();
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) arrive_cluster(map_rank(smem_u32(&sh.tempty[buf]), 0));
          else mbar_arrive(&sh.tempty[buf]);
        }
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if constexpr (SPLIT) {
    cluster_sync();  // every rank's partial tile is in its shared memory
    int r0, c0;
    const Problem& pr = locate(t0, r0, c0);
    const Epilogue& e = pr.epi;
    if (tid < 256 && !sh.abort) {
      const int col = tid & 127;
      const long long c = c0 + col;
      if (c < pr.cols) {
        const float bias = e.bias ? load_elem(e.bias, c, e.bias_f32) : 0.f;
        const uint32_t base = smem_u32(ring) + col * 4;
        for (int j = krank + p.split * (tid >> 7); j < NT && r0 + j < pr.rows; j += 2 * p.split) {
          float part[8];
#pragma unroll
          for (int s = 0; s < 8; ++s)
            part[s] = s < p.split ? ld_cluster_f32(map_rank(base, s) + j * 512) : 0.f;
          float z = part[0];
#pragma unroll
          for (int s = 1; s < 8; ++s) z += part[s];
          z += bias;
          const long long r = r0 + j;
          const float res = e.res ? load_elem(e.res, r * e.ld_res + c, e.res_f32) : 0.f;
          if (e.pre) store_elem(e.pre, r * e.ld_pre + c, z, 0);
          with_act(e.act, [&](auto a) {
            store_elem(e.out, r * e.ld_out + c, act_f<decltype(a)::value>(z) + res, e.out_f32);
          });
        }
      }
    }
    __syncthreads();
  }
  if constexpr (CG == 2 || SPLIT) cluster_sync();  // no access reaches a CTA that has left
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
  int cg, nt, stages;
  bool split;
  const void* fn;
  int smem;
};
template <int CG, int NT, int S, bool SPLIT>
Variant variant() {
  return {CG, NT, S, SPLIT, reinterpret_cast<const void*>(&lin_gemm<CG, NT, S, SPLIT>), Cfg<CG, NT, S, SPLIT>::SMEM};
}
const Variant* variants(int* n) {
  static const Variant v[] = {variant<2, 256, 6, false>(), variant<1, 128, 6, false>(), variant<1, 64, 8, false>(),
                              variant<1, 32, 8, false>(),  variant<1, 16, 8, false>(),  variant<1, 128, 6, true>(),
                              variant<1, 64, 8, true>(),   variant<1, 32, 8, true>(),   variant<1, 16, 8, true>()};
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
  double cost;
};

// The variant with the least estimated time for these products on `sms` SMs.
// In SM clocks per 64-deep k-block of one tile: the MMA's own time (128 x NT
// x 64 at 4096 MAC per clock and SM) or, for narrow tiles, the time its
// stage takes to arrive; and per tile the ring's fill and the epilogue's
// drain, which two accumulators hide behind the next tile.
Choice choose(const Product* pr, int n, int sms) {
  int nv;
  const Variant* vs = variants(&nv);
  Choice best{nullptr, 1, 0};
  for (int i = 0; i < nv; ++i) {
    const Variant& v = vs[i];
    bool fits = true;
    for (int j = 0; j < n; ++j) fits = fits && !(pr[j].Q.mn && v.nt < 64);
    if (!fits) continue;
    const double per_kb = std::max(v.nt / v.cg * 2.0 * v.cg, (P_BYTES + v.nt / v.cg * 128) / 60.0);
    for (int sp = v.split ? 2 : 1; sp <= (v.split ? 8 : 1); sp *= 2) {
      long long tiles = 0;
      double work = 0, longest = 0;
      for (int j = 0; j < n; ++j) {
        const long long t = (long long)ceil_div(pr[j].rows, v.nt) * ceil_div(pr[j].cols, 128 * v.cg);
        const double one = ceil_div(ceil_div(pr[j].k, BK), sp) * per_kb + (v.nt >= 128 ? 300 : 150);
        tiles += t;
        work += t * one;
        longest = std::max(longest, one);
      }
      const int slots = std::max(1, sms / (v.cg * sp));
      if (v.split && (tiles > slots || tiles * sp > 65535 * 32ll)) continue;
      double cost = 2500 + (tiles <= slots ? longest : std::max(longest, work / slots * (double)(ceil_div((int)std::min<long long>(tiles, 1 << 30), slots) * (double)slots / tiles)));
      cost += v.nt * 6.0;                         // the last tile's epilogue
      if (v.split) cost += 1200 + v.nt * 4.0;     // cluster barriers and the sum
      if (!best.v || cost < best.cost) best = {&v, sp, cost};
    }
  }
  return best;
}

}  // namespace

cudaError_t prepare(int* pairs) {
  std::lock_guard<std::mutex> lock(g_mu);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int nv;
  const Variant* vs = variants(&nv);
  if (dev >= 64 || !g_ready[dev]) {
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
    if (dev < 64) g_ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = vs[0].smem;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(pairs, vs[0].fn, &cfg);
}

apk_status run_products(const Product* pr, int n, int sms, int* status, long long limit, cudaStream_t stream,
                        std::string* why) {
  const Choice ch = choose(pr, n, sms);
  const Variant& v = *ch.v;
  GemmParams p;
  p.nprob = n;
  p.tiles = 0;
  p.tiles0 = 0;
  p.split = ch.split;
  p.status = status;
  p.limit = limit;
  for (int j = 0; j < n; ++j) {
    Problem& q = p.pr[j];
    q.epi = pr[j].epi;
    q.rows = pr[j].rows;
    q.cols = pr[j].cols;
    q.nkb = ceil_div(pr[j].k, BK);
    q.tiles_r = ceil_div(q.rows, v.nt);
    q.tiles_c = ceil_div(q.cols, 128 * v.cg);
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
  const int groups = v.split ? p.tiles : std::min(p.tiles, std::max(1, sms / v.cg));
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
