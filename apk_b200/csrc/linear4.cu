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
// are written out as bf16 first.  For a bf16 result they are rounded to it, by up
// to 2^-8 of a weight, as the result itself is (4096 x 8192: 128 rows are 0.0022 of
// their size off, 64 rows, whose weights are not rounded, 0.0017); a second term
// for the rest, which an fp32 result has, makes K twice as long (128 x 4096 x 8192
// 41 us, so 74).
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
  int rows, n, k, group, groups, s_f32;
  int group_shift;  // log2 of the chunks of a group, or -1
  int split;  // CTAs of a cluster that share K
  int kw;     // warps that share a tile's K; 16 / kw tiles are worked on at once
  int tiles;  // of 16 features
  int slice;  // chunks of x in shared memory at once
  lin::Epilogue epi;
};

constexpr int WARPS = 16, FT = 16, CHUNK = 128;
constexpr int PART_LD = 20;  // a token's 16 sums, apart by 20: no two of a warp's stores meet in a bank
constexpr int SMEM = 226 << 10;
constexpr int part_bytes(int tokens) { return WARPS * tokens * PART_LD * 4; }

// Weights are read once.  A warp's load takes 64 bytes of eight rows; past L1
// the two halves of a line are fetched each for itself, which costs where they
// come out of L2 and pays where they come out of memory (1 x 4096 x 8192 out of
// L2 9.3 us past L1 and 7.9 through it, out of memory 9.6 and 9.8; 64 rows 32.3
// and 30.9, 32.7 and 37.7).  So: through L1 for up to 8 rows.  (KEEP)
template <bool KEEP, class T>
__device__ __forceinline__ T ld_w(const uint8_t* q, bool in) {
  T v{};
  if (!in) return v;
  if constexpr (KEEP || sizeof(T) == 4) return *reinterpret_cast<const T*>(q);
  else if constexpr (sizeof(T) == 16) return stream::ld_late(q);
  else return stream::ld_late8(q);
}
// Eight weights less their zero point: h[i] is the pair (i, i + 4).
__device__ __forceinline__ void dequant(uint32_t w, uint32_t minus_zero, uint32_t (&h)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)));
    // (v - (128 + z), as the multiply-add by one that there is an instruction for)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(h[i]) : "r"(v), "r"(0x3F803F80u), "r"(minus_zero));
  }
}
// Eight values of x in the same order.
__device__ __forceinline__ void pairs(const uint4& v, uint32_t (&h)[4]) {
  h[0] = __byte_perm(v.x, v.z, 0x5410);
  h[1] = __byte_perm(v.x, v.z, 0x7632);
  h[2] = __byte_perm(v.y, v.w, 0x5410);
  h[3] = __byte_perm(v.y, v.w, 0x7632);
}
// P: groups that a chunk of 128 k has (1 for groups of 128 and more).  A
// warp's lane (g, t) holds weights of the features g and g + 8; a group's
// 32 / P k-values of a lane lie together.
//
// One CTA of 16 warps an SM (two of 8 were slower).  It lays x out in shared memory as the B fragments that its
// warps will want, already in the nibbles' order, once for all features that
// it takes: read from global memory, x cost more of L1 than the weights did
// (32 rows of 4096 x 8192: 37 us).  Warps share tiles of 16 features by K;
// a warp has AHEAD chunks of weights, 32 bytes a lane, on their way, its
// neighbours the chunks between.
template <int NT8>
constexpr int AHEAD = NT8 <= 4 ? 4 : 2;
// Scales and zero points of a chunk: lane t has its t-th group's and hands them
// round; or with WIDE (P of 4, bf16 scales, whole chunks) every lane has all
// four of both features, which costs no exchanges (16 x 8192 x 4096: 18.9 us
// without).
template <bool WIDE>
struct Chunk {
  uint32_t w[2][4];
  float s[2];
  uint32_t z;  // -(128 + zero point), of feature g in the low half
};
template <>
struct Chunk<true> {
  uint32_t w[2][4];
  uint2 s[2];
  uint32_t z[2];  // a byte each
};
// XA: pieces of x that a thread has on their way while x is laid out.  (One each:
// 32 x 4096 x 4096 14.6 us, eight 13.5; up to 8 rows, 8 x 4096 x 8192 10.1, four
// 9.7; but the one piece of a single row 8.1 in that code and 7.9 in its own.)
template <int NT8, int P, bool ZEROS, bool VEC, bool WIDE, int XA>
__global__ void __launch_bounds__(32 * WARPS, 1) stream4(const __grid_constant__ Params p) {
  constexpr int TOK = 8 * NT8, WORDS = 4 / P, A = AHEAD<NT8>;  // WORDS: 32-bit words of a lane and group
  extern __shared__ uint4 xs[];  // [chunk][word][row][t]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = (int)blockIdx.x % p.split;
  const int kept = NT8 == 1 ? p.rows : TOK;  // rows in shared memory
  float* part = reinterpret_cast<float*>(xs + p.slice * 4 * kept * 4);  // [warp][token][PART_LD]
  const int kw = warp % p.kw, tw = warp / p.kw, at_once = WARPS / p.kw;
  const int chunks = (p.k + CHUNK - 1) / CHUNK, per = (chunks + p.split - 1) / p.split;
  const int c_begin = rank * per, c_end = min(c_begin + per, chunks);
  const int sets = (p.tiles + at_once - 1) / at_once, set_step = (int)gridDim.x / p.split;
  pdl_launch();
  pdl_wait();
  // A lane's weights of a tile: k = chunk * 128 + h * 128 / P + t * 32 / P and
  // what follows; and the index of the scale it loads, the chunk's t-th
  // group's (with fewer groups: one of them), without the chunk's part.
  const uint8_t* w_of[2];
  long long s_of[2];
  auto go_to = [&](int tile) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int f = min(tile * FT + g + 8 * m, p.n - 1);
      w_of[m] = p.w + f * p.ldw + t * (16 / P);
      s_of[m] = (long long)f * p.groups + (WIDE ? 0 : t & (P - 1));
    }
  };
  auto load = [&](Chunk<WIDE>& c, int chunk) {
    const bool whole = (chunk + 1) * CHUNK <= p.k;  // (K ends inside the last chunk, perhaps)
#pragma unroll
    for (int h = 0; h < P; ++h) {
      const bool in = whole || chunk * CHUNK + h * (CHUNK / P) + t * (32 / P) < p.k;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* q = w_of[m] + (long long)chunk * (CHUNK / 2) + h * (CHUNK / 2 / P);
        if constexpr (P == 1) {
          const uint4 v = ld_w<NT8 == 1, uint4>(q, in);
          c.w[m][0] = v.x, c.w[m][1] = v.y, c.w[m][2] = v.z, c.w[m][3] = v.w;
        } else if constexpr (P == 2) {
          const uint2 v = ld_w<NT8 == 1, uint2>(q, in);
          c.w[m][2 * h] = v.x, c.w[m][2 * h + 1] = v.y;
        } else {
          c.w[m][h] = ld_w<NT8 == 1, uint32_t>(q, in);
        }
      }
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        c.s[m] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.s) + s_of[m] + chunk * P);
        if (ZEROS) c.z[m] = *reinterpret_cast<const uint32_t*>(p.z + s_of[m] + chunk * P) & 0x0F0F0F0Fu;
      }
      return;
    } else {
      const bool in = whole || chunk * CHUNK + (t & (P - 1)) * (CHUNK / P) < p.k;
      const int gr = P > 1 ? chunk * P : p.group_shift >= 0 ? chunk >> p.group_shift : chunk / (p.group / CHUNK);
      c.s[0] = in ? ops::ld_any(p.s, s_of[0] + gr, p.s_f32) : 0.f;
      c.s[1] = in ? ops::ld_any(p.s, s_of[1] + gr, p.s_f32) : 0.f;
      if (ZEROS) c.z = 0xC300C300u | (in ? (uint32_t)(p.z[s_of[0] + gr] & 15) | (uint32_t)(p.z[s_of[1] + gr] & 15) << 16 : 0u);
    }
  };
  // x of `n` chunks from `chunk` on; a thread's piece is eight contiguous k
  auto stage = [&](int chunk, int n) {
    const int rows = min(p.rows, kept), all = n * 16 * kept;
    for (int i0 = tid; i0 < all; i0 += XA * 32 * WARPS) {
      uint4 v[XA];
#pragma unroll
      for (int u = 0; u < XA; ++u) {
        // the 16 pieces of a row's chunk go to neighbouring threads
        const int i = i0 + u * 32 * WARPS, row = (i >> 4) % kept, k = (chunk + (i >> 4) / kept) * CHUNK + (i & 15) * 8;
        v[u] = make_uint4(0, 0, 0, 0);
        if (i < all && row < rows) {
          const uint16_t* q = p.x + row * p.ldx + k;
          if (VEC) v[u] = k < p.k ? stream::ld_rows(q) : v[u];
          else v[u] = stream::ld8_any(q, p.k - k);
        }
      }
#pragma unroll
      for (int u = 0; u < XA; ++u) {
        const int i = i0 + u * 32 * WARPS, e = i & 15, row = (i >> 4) % kept, c = (i >> 4) / kept;
        if (i >= all) break;
        uint32_t h[4];
        pairs(v[u], h);
        // piece e is word j of group h for lane t: e = (h * 4 + t) * (4 / P) + j
        const int j = e % WORDS, tt = e / WORDS % 4, hh = e / (WORDS * 4), word = hh * WORDS + j;
        xs[((c * 4 + word) * kept + row) * 4 + tt] = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
  };
  const int my_row = NT8 == 1 ? min(g, p.rows - 1) : g;
  float total[NT8][4];
  auto multiply = [&](const Chunk<WIDE>& c, int chunk) {  // chunk: of the slice
#pragma unroll
    for (int h = 0; h < P; ++h) {
      float acc[NT8][4] = {};
      float s[2];
      uint32_t z[2];
      if constexpr (WIDE) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint32_t two = h < 2 ? c.s[m].x : c.s[m].y;
          s[m] = h & 1 ? ops::bf_hi(two) : ops::bf_lo(two);
          z[m] = ZEROS ? __byte_perm(c.z[m], 0xC3, 0x4040 | h * 0x0101) : 0xC308C308u;
        }
      } else {
        const uint32_t zz = !ZEROS ? 0xC308C308u : P == 1 ? c.z : __shfl_sync(0xFFFFFFFFu, c.z, (lane & ~3) | h);
        z[0] = ZEROS ? __byte_perm(zz, 0, 0x1010) : zz;
        z[1] = ZEROS ? __byte_perm(zz, 0, 0x3232) : zz;
#pragma unroll
        for (int m = 0; m < 2; ++m) s[m] = P == 1 ? c.s[m] : __shfl_sync(0xFFFFFFFFu, c.s[m], (lane & ~3) | h);
      }
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        uint32_t a[4], b[4];
        dequant(c.w[0][h * WORDS + j], z[0], a);
        dequant(c.w[1][h * WORDS + j], z[1], b);
        const uint4* x = xs + ((chunk * 4 + h * WORDS + j) * kept + my_row) * 4 + t;
#pragma unroll
        for (int i = 0; i < NT8; ++i) {
          const uint4 v = x[i * 32];
          stream::mma_bf16(acc[i], a[0], b[0], a[1], b[1], v.x, v.y);
          stream::mma_bf16(acc[i], a[2], b[2], a[3], b[3], v.z, v.w);
        }
      }
#pragma unroll
      for (int i = 0; i < NT8; ++i) {
        total[i][0] = fmaf(s[0], acc[i][0], total[i][0]);
        total[i][1] = fmaf(s[0], acc[i][1], total[i][1]);
        total[i][2] = fmaf(s[1], acc[i][2], total[i][2]);
        total[i][3] = fmaf(s[1], acc[i][3], total[i][3]);
      }
    }
  };
  Chunk<WIDE> ring[A];
  auto prime = [&](int set, int begin) {
#pragma unroll
    for (int i = 0; i < A; ++i)
      if (set * at_once + tw < p.tiles && begin + kw + i * p.kw < min(begin + p.slice, c_end)) load(ring[i], begin + kw + i * p.kw);
  };
  int set = (int)blockIdx.x / p.split;
  go_to(set * at_once + tw);
  prime(set, c_begin);
  const bool once = c_end - c_begin <= p.slice;  // x stays where it is
  for (bool first = true; set < sets; set += set_step, first = false) {
    const int tile = set * at_once + tw;
#pragma unroll
    for (int i = 0; i < NT8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) total[i][j] = 0.f;
    for (int begin = c_begin; begin < c_end; begin += p.slice) {
      const int end = min(begin + p.slice, c_end);
      if (!once || first) {
        if (!once) __syncthreads();
        stage(begin, end - begin);
        __syncthreads();
      }
      if (tile < p.tiles) {
#pragma unroll 1
        for (int c0 = begin + kw; c0 < end; c0 += A * p.kw) {
#pragma unroll
          for (int i = 0; i < A; ++i) {
            const int c = c0 + i * p.kw;
            if (c >= end) break;
            multiply(ring[i], c - begin);
            if (c + A * p.kw < end) load(ring[i], c + A * p.kw);
          }
        }
      }
      // the next weights travel while this tile is finished
      if (end < c_end) {
        prime(set, end);
      } else {
        go_to((set + set_step) * at_once + tw);
        prime(set + set_step, c_begin);
      }
    }
#pragma unroll
    for (int i = 0; i < NT8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[(warp * TOK + 8 * i + 2 * t + (j & 1)) * PART_LD + g + 8 * (j >> 1)] = total[i][j];
    __syncthreads();
    if (p.split > 1)
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int o = rank * 32 * WARPS + tid; o < at_once * TOK * FT; o += p.split * 32 * WARPS) {
      const int c = o % FT, tok = o / FT % TOK, which = o / (FT * TOK);
      const long long col = (long long)(set * at_once + which) * FT + c;
      if (tok >= p.rows || col >= p.n) continue;
      const float* from = part + (which * p.kw * TOK + tok) * PART_LD + c;
      float y = 0.f;
      for (int r = 0; r < p.split; ++r) {  // in the order of ranks and warps
        if (p.split == 1) {
          for (int w = 0; w < p.kw; ++w) y += from[w * TOK * PART_LD];
        } else {
          uint32_t q;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(q) : "r"(smem_u32(from)), "r"(r));
          for (int w = 0; w < p.kw; ++w) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(q + w * TOK * PART_LD * 4) : "memory");
            y += v;
          }
        }
      }
      const lin::Epilogue& e = p.epi;
      if (e.bias) y += ops::ld_any(e.bias, col, e.bias_f32);
      const float res = e.res ? ops::ld_any(e.res, tok * e.ld_res + col, e.res_f32) : 0.f;
      if (e.pre) ops::st_any(e.pre, tok * e.ld_pre + col, y, false);
      with_act(e.act, [&](auto a) { ops::st_any(e.out, tok * e.ld_out + col, act_f<decltype(a)::value>(y) + res, e.out_f32); });
    }
    // the sums are written again, and no read reaches a CTA that has left
    __syncthreads();
    if (p.split > 1)
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// The weights as bf16, [n][ld]; with `low` also what that rounds away, in the
// next k columns, and x twice beside each other to go with it.  Of a value that
// is not finite nothing is left over, and the second x has 0 in the place of
// its own: inf times a rest of 0 would make a NaN of an infinite sum.
struct Expand {
  const uint8_t* w;
  const void* s;
  const uint8_t* z;
  uint16_t* out;
  const uint16_t* x;
  uint16_t* xx;
  long long ldw, ldx;
  int n, k, group, groups, group_log, s_f32, low, rows;
};
// Two bf16 values, 0 where one is not finite.
__device__ __forceinline__ uint32_t finite(uint32_t v) {
  if ((v & 0x7F80u) == 0x7F80u) v &= 0xFFFF0000u;
  return (v & 0x7F800000u) == 0x7F800000u ? v & 0xFFFFu : v;
}
__global__ void __launch_bounds__(256) expand(const __grid_constant__ Expand p) {
  pdl_launch();
  pdl_wait();
  // a block takes two rows at once, a thread eight k of 2048, and of the next 2048
  const long long ld = p.low ? 2ll * p.k : p.k;
  for (long long f0 = blockIdx.x; f0 < p.n; f0 += 2ll * gridDim.x) {
    for (int k0 = (int)threadIdx.x * 8; k0 < p.k; k0 += 4096) {
      uint32_t w[4];
      float s[4], z[4];
      uint16_t* to[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long f = f0 + (j >> 1) * (long long)gridDim.x;
        const int k = k0 + (j & 1) * 2048;
        to[j] = nullptr;
        if (f >= p.n || k >= p.k) continue;
        const long long at = f * p.groups + (p.group_log >= 0 ? k >> p.group_log : k / p.group);
        s[j] = ops::ld_any(p.s, at, p.s_f32);
        z[j] = 128.f + (p.z ? (float)(p.z[at] & 15) : 8.f);
        w[j] = *reinterpret_cast<const uint32_t*>(p.w + f * p.ldw + k / 2);
        to[j] = p.out + f * ld + k;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!to[j]) continue;
        float q[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // 128 + q again: an integer's conversion is slower
          uint32_t v;
          asm("lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;" : "=r"(v) : "r"(w[j] >> (4 * e)));
          q[e] = s[j] * (ops::bf_lo(v) - z[j]);
          q[e + 4] = s[j] * (ops::bf_hi(v) - z[j]);
        }
        ops::Raw<false> r;
        ops::pack(q, r);
        *reinterpret_cast<uint4*>(to[j]) = r.a;
        if (p.low) {
          float hi[8];
          ops::unpack(r, hi);
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = isfinite(hi[e]) ? q[e] - hi[e] : 0.f;
          ops::pack(q, r);
          *reinterpret_cast<uint4*>(to[j] + p.k) = r.a;
        }
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
    if (p.low) *reinterpret_cast<uint4*>(p.xx + r * ld + p.k + k) = make_uint4(finite(v.x), finite(v.y), finite(v.z), finite(v.w));
  }
}

template <int NT8, int P, bool WIDE, int XA>
const void* fn(bool zeros, bool vec) {
  return zeros ? (vec ? reinterpret_cast<const void*>(&stream4<NT8, P, true, true, WIDE, XA>)
                      : reinterpret_cast<const void*>(&stream4<NT8, P, true, false, WIDE, XA>))
               : (vec ? reinterpret_cast<const void*>(&stream4<NT8, P, false, true, WIDE, XA>)
                      : reinterpret_cast<const void*>(&stream4<NT8, P, false, false, WIDE, XA>));
}
// The kernel for a layer's group, scales and zero points, and x that is (vec) or is not on 16 bytes.
template <int NT8, int XA>
const void* fn(const apk_linear4_config& c, bool vec) {
  const bool wide = c.scale_dtype == APK_BF16 && c.in_features % CHUNK == 0 && ops::aligned(c.scales, 8) && ops::aligned(c.zeros, 4);
  return c.group == 32   ? (wide ? fn<NT8, 4, true, XA>(c.zeros, vec) : fn<NT8, 4, false, XA>(c.zeros, vec))
         : c.group == 64 ? fn<NT8, 2, false, XA>(c.zeros, vec)
                         : fn<NT8, 1, false, XA>(c.zeros, vec);
}
// nt: tiles of 8 rows; many: more pieces of x than threads
const void* fn(const apk_linear4_config& c, bool vec, int nt, bool many) {
  return nt == 1 ? (many ? fn<1, 4>(c, vec) : fn<1, 1>(c, vec)) : nt == 2 ? fn<2, 8>(c, vec) : nt == 4 ? fn<4, 8>(c, vec) : fn<8, 8>(c, vec);
}

}  // namespace lin4
}  // namespace apk

using namespace apk;

struct apk_linear4 {
  apk_linear4_config cfg{};
  Err err;
  bool opened = false;
  int sms = 0;
  int clusters[9] = {};  // of 2, 4 and 8 CTAs that run at once
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
  // (a layer's group and zero points leave ten kernels that it may launch)
  for (const bool vec : {false, true})
    for (const bool many : {false, true})
      for (int nt = 1; nt <= (many ? 8 : 1); nt *= 2)
        APK_TRY(cu_status(cudaFuncSetAttribute(lin4::fn(c, vec, nt, many), cudaFuncAttributeMaxDynamicSharedMemorySize, lin4::SMEM),
                          "preparing the 4-bit product", &h->err));
  for (int split = 2; split <= 8; split *= 2) {
    Launch l(dim3(split), 32 * lin4::WARPS, lin4::SMEM, nullptr, split);
    APK_TRY(cu_status(cudaOccupancyMaxActiveClusters(&h->clusters[split], lin4::fn(c, true, 1, false), &l.cfg),
                      "preparing the 4-bit product", &h->err));
  }
  return h->scratch.open(c.device, &h->err);
}

// Rows up to here stream the weights.
constexpr int STREAM_ROWS = 64;

apk_status stream(apk_linear4* h, const apk_linear_io* io, const lin::Epilogue& epi) {
  const apk_linear4_config& c = h->cfg;
  lin4::Params p{};
  int grid = 0;
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
  p.group_shift = -1;
  for (int i = 0; i < 24; ++i)
    if (c.group == lin4::CHUNK << i) p.group_shift = i;
  p.epi = epi;
  const bool vec = ops::on16(io->x, io->ldx, io->rows, APK_BF16);
  const int nt = io->rows <= 8 ? 1 : io->rows <= 16 ? 2 : io->rows <= 32 ? 4 : 8;
  p.tiles = ops::ceil_div(p.n, lin4::FT);
  const int chunks = ops::ceil_div(p.k, lin4::CHUNK), kept = nt == 1 ? io->rows : 8 * nt;
  const int room = (lin4::SMEM - lin4::part_bytes(8 * nt)) / (kept * lin4::CHUNK * 2);  // chunks of x
  // What a launch takes, in chunks of a warp: rounds of tiles, each with its
  // chunks and 4 for its end (of a cluster 8, of eight CTAs 11), and x laid out once where it
  // fits (half a chunk's time each), else again in every round.  Where warps
  // would idle, more of them share a tile, which leaves fewer to finish
  // (50 x 1184 x 80: 11.5 us with 8 for all clusters and few warps a tile, now 8.9).
  long long best = -1;
  for (int split = 1; split <= 8; split *= 2) {
    if (split > 1 && (split > chunks || h->clusters[split] == 0)) break;
    const int places = split == 1 ? h->sms : std::min(h->clusters[split], h->sms / split);
    const int mine = ops::ceil_div(chunks, split);
    for (int kw = 1; kw <= lin4::WARPS && places > 0; kw *= 2) {
      const int sets = ops::ceil_div(p.tiles, lin4::WARPS / kw), rounds = ops::ceil_div(sets, places);
      const long long x = (long long)mine * kept / 64 * (mine <= room ? 1 : rounds);
      const long long cost = (long long)rounds * (ops::ceil_div(mine, kw) * std::max(2, nt) / 2 + (split == 1 ? 4 : split < 8 ? 8 : 11)) + x;
      if (best >= 0 && (cost > best || (cost == best && split != p.split))) continue;
      best = cost;
      p.split = split;
      p.kw = kw;
      p.slice = std::min(mine, room);
      grid = std::min(sets, places) * split;
    }
  }
  const void* f = lin4::fn(c, vec, nt, p.slice * 16 * kept > 32 * lin4::WARPS);
  Launch l(dim3(grid), 32 * lin4::WARPS, p.slice * kept * lin4::CHUNK * 2 + lin4::part_bytes(8 * nt),
           static_cast<cudaStream_t>(io->stream), p.split);
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
  e.group_log = -1;
  for (int i = 5; i < 31; ++i)
    if (c.group == 1 << i) e.group_log = i;
  e.groups = ops::ceil_div(K, c.group);
  e.s_f32 = c.scale_dtype == APK_F32;
  e.low = low;
  e.rows = M;
  const long long blocks = std::max<long long>((N + 1) / 2, copy ? (long long)M * (K / 8) / 256 + 1 : 0);
  Launch l(dim3((unsigned)std::min<long long>(blocks, h->sms * 8)), 256, 0, s);
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
