// Layer norm over the last axis, forward and backward (apk_norm_* of
// include/apk.h).  No counterpart in the reference, which multiplies bare
// matrices (src/tcyield.cu:91-356).
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   n = (x - mean) rstd,  y = n w + b
//   g = dy w,  dx = rstd (g - mean(g) - n mean(g n)) + residual_grad
//   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Both passes are bound by memory: every row is read once into registers and
// all sums over it are taken from there, in fp32.  The variance is taken from
// the differences d = x - m.  Far from zero m is off by the roundings of a sum
// of large values (a row of 5000.3s, eps 1e-5, would get up to 0.3 w + b in
// place of b): where it is larger than the deviation, mean(d) corrects it,
//   mean = m + mean(d),  sum (x - mean)^2 = sum d^2 - mean(d) sum d.
// Elsewhere the values are hardly larger than their differences, and so are the
// sum's roundings.  (Both sums in one pass for every row: 8192 x 4096 bf16 31.1
// us; so 28.3, without any of it 27.6.)
#include <algorithm>
#include <vector>

#include "ops.cuh"
#include "ops.h"

namespace apk {
namespace norm {

constexpr int MAX_FEATURES = 16384;  // 1024 threads of two pieces

// Rows on their way, this one among them: 98 KB of shared memory (196 KB for
// more than 512 threads, of which an SM takes one block) hold them.
template <bool XF>
constexpr int FWD_STAGES = XF ? 3 : 6;
template <bool XF, bool DF, int T>
constexpr int BWD_STAGES = 24 / ((XF ? 8 : 4) + (DF ? 4 : 2)) / (T > 512 ? 2 : 1);
// Rows that start anywhere go by their threads together through shared memory.
// Not so the largest blocks, which have a row or few each, and short rows, a
// warp each (forward 1537 x 1001 fp32: 4.2 us, so 5.1, 16384 x 333 bf16 9.6 and
// 9.7; backward 500 x 111 6.0 and 7.4, 16384 x 333 23.7 and 23.4).
template <bool VEC, bool WARP, int T>
constexpr bool SHARED = !VEC && !WARP && T <= 512;

struct Params {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  const void* r;     // residual gradient, or null
  void* y;           // y, or dx (null: not wanted)
  float2* stats;
  float* part;       // [blocks][dw, db][cols rounded up to 8], or null
  void* dw;          // few rows: written by blocks of their own, from row_blocks on
  void* db;
  int row_blocks;
  long long ldx, ld_dy, ld_r, ldy;
  int rows, cols;
  float eps, per_col;  // 1 / cols
  int w_f32, b_f32;
};

// A row's thread t of T holds V pieces of eight columns: contiguous ones
// where rows can be read 16 bytes at a time (VEC), else every T-th column, so
// that a warp's loads are contiguous.
template <bool VEC>
__device__ __forceinline__ int column(int j, int i, int t, int T) {
  return VEC ? (j * T + t) * 8 + i : (j * 8 + i) * T + t;
}
template <bool VEC, bool F32, int V>
__device__ __forceinline__ void load_row(const void* p, long long row, ops::Raw<F32> (&raw)[V], int cols, int t, int T) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    raw[j] = {};
    if constexpr (VEC) {
      if ((j * T + t) * 8 < cols) ops::ld8(p, row + (j * T + t) * 8, raw[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (column<false>(j, i, t, T) < cols) ops::set1(raw[j], i, p, row + column<false>(j, i, t, T));
    }
  }
}
template <bool VEC, bool F32>
__device__ __forceinline__ void store_piece(void* p, long long row, const float (&v)[8], int j, int cols, int t, int T) {
  if constexpr (VEC) {
    ops::Raw<F32> raw;
    ops::pack(v, raw);
    if ((j * T + t) * 8 < cols) ops::st8(p, row + (j * T + t) * 8, raw);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (column<false>(j, i, t, T) < cols) ops::st_any(p, row + column<false>(j, i, t, T), v[i], F32);
  }
}
// weight or bias, kept in L1 by its reuse from row to row
template <bool VEC>
__device__ __forceinline__ void load_weight(const void* p, int f32, float (&v)[8], int j, int cols, int t, int T) {
  if (VEC && (j * T + t) * 8 < cols) {
    if (f32) {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + (j * T + t) * 8);
      const float4 lo = q[0], hi = q[1];
      v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
    } else {
      ops::Raw<false> r{*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + (j * T + t) * 8)};
      ops::unpack(r, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = !VEC && column<false>(j, i, t, T) < cols ? ops::ld_any(p, column<false>(j, i, t, T), f32) : 0.f;
  }
}

// The same of rows that go through shared memory: T is a constant, and where a
// pair of columns lies in the row for all threads nothing is compared.
template <bool F32>
__device__ __forceinline__ void store_odd(void* p, long long row, const float (&v)[8], int j, int cols, int t, int T) {
  uint8_t* q = static_cast<uint8_t*>(p) + (row + t) * (F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const int k = j * 8 + i;
    if ((k + 2) * T <= cols) {
      if constexpr (F32) {
        *reinterpret_cast<float*>(q + k * T * 4) = v[i];
        *reinterpret_cast<float*>(q + (k + 1) * T * 4) = v[i + 1];
      } else {
        const uint32_t two = ops::pack_bf16(v[i], v[i + 1]);
        *reinterpret_cast<uint16_t*>(q + k * T * 2) = (uint16_t)two;
        *reinterpret_cast<uint16_t*>(q + (k + 1) * T * 2) = (uint16_t)(two >> 16);
      }
    } else {
      if (k * T + t < cols) ops::st_any(q, k * T, v[i], F32);
      if ((k + 1) * T + t < cols) ops::st_any(q, (k + 1) * T, v[i + 1], F32);
    }
  }
}

// Sums of a and b over the T threads of a row: a warp, or the block.  `buf` is
// another one than in the call before, so that one barrier a call is enough: who
// writes a buffer again has passed the barrier behind its last reads.
template <bool WARP, int T_>
__device__ __forceinline__ float2 row_sums(float a, float b, float4 (*sh)[16], int buf, int T) {
  // two sums in five exchanges: from here the lower half of the warp has a, the upper b
  const bool upper = threadIdx.x & 16;
  float v = upper ? b : a;
  v += __shfl_xor_sync(0xFFFFFFFFu, upper ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if constexpr (WARP) {
    const float other = __shfl_xor_sync(0xFFFFFFFFu, v, 16);
    return upper ? make_float2(other, v) : make_float2(v, other);
  }
  float2* pair = reinterpret_cast<float2*>(sh[buf]);
  if ((threadIdx.x & 15) == 0) reinterpret_cast<float*>(pair + (threadIdx.x >> 5))[upper] = v;
  __syncthreads();
  if constexpr (T_ <= 256) {  // up to 8 warps: every thread adds them
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < T_ / 32; w += 2) {
      if (w * 32 >= T) break;
      const float4 q = sh[buf][w / 2];
      s.x += q.x;
      s.y += q.y;
      if ((w + 1) * 32 < T) {
        s.x += q.z;
        s.y += q.w;
      }
    }
    return s;
  } else {
    const int lane = threadIdx.x & 31;
    const float2 q = lane < T / 32 ? pair[lane] : make_float2(0.f, 0.f);
    return make_float2(ops::warp_sum(q.x), ops::warp_sum(q.y));
  }
}
template <bool WARP, int T_>
__device__ __forceinline__ float row_sum(float a, float4 (*sh)[16], int buf, int T) {
  a = ops::warp_sum(a);
  if constexpr (WARP) return a;
  float* one = reinterpret_cast<float*>(sh[buf]);
  const int lane = threadIdx.x & 31;
  if (lane == 0) one[threadIdx.x >> 5] = a;
  __syncthreads();
  if constexpr (T_ <= 256) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < T_ / 32; ++w)
      if (w * 32 < T) s += one[w];
    return s;
  } else {
    return ops::warp_sum(lane < T / 32 ? one[lane] : 0.f);
  }
}

// A thread's own pieces of the rows ahead, on their way into shared memory:
// stage, array and piece lie 16 bytes a thread apart, so that no other thread
// reads them and no barrier is needed.  What registers could hold of the next
// row alone left too little in flight (8192 x 4096 bf16 forward 56 us, backward
// 68).  S stages; every row is one group of copies, an empty one behind the last.
template <int V, bool F32, int S>
struct Ahead {
  uint32_t at;  // this thread's place in shared memory
  int threads;
  static constexpr int HALVES = F32 ? 2 : 1, SLOTS = V * HALVES;
  // `q`: this thread's first piece of the row; `pieces` of the V are in the row
  __device__ __forceinline__ void fetch(int stage, const uint8_t* q, int pieces, int T) const {
    const uint32_t to = at + stage * SLOTS * threads * 16;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < pieces)
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (j * HALVES + h) * threads * 16),
                       "l"(q + (j * T * HALVES + h) * 16ll)
                       : "memory");
  }
  __device__ __forceinline__ ops::Raw<F32> get(int stage, int j, int pieces) const {
    ops::Raw<F32> r = {};
    if (j < pieces) {
      const uint32_t from = at + (stage * SLOTS + j * HALVES) * threads * 16;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w) : "r"(from) : "memory");
      if constexpr (F32)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
                     : "r"(from + threads * 16)
                     : "memory");
    }
    return r;
  }
};
// Rows that start anywhere: the aligned 16-byte pieces that a row touches, one
// after the other, copied by the row's T threads and read by all of them, so
// that a barrier stands between (`arrived`, then the barrier; behind it the
// stage that was read last may be filled again).  T is a constant, and what lies
// behind a row's end are zeros, so that an element costs a load and a shift:
// with a comparison each and addresses by a running T it took 45 instructions.
// (8192 x 4001 bf16, element by element out of global memory: 66 us forward,
// 157 backward; so, 41 and 75.)
template <int V, bool F32, int T>
struct Odd {
  static constexpr int ES = F32 ? 4 : 2, BYTES = T * V * 8 * ES + 16;  // of a stage: a piece more, for the shift
  uint32_t at;  // the row's ring
  int end;      // of what every row writes of a stage: its pieces wherever it starts
  __device__ __forceinline__ Odd(uint32_t at_, int cols) : at(at_), end((cols * ES + 16 - ES + 15) / 16 * 16) {}
  // zeros behind it, once
  __device__ __forceinline__ void clear(int stages, int t) const {
    for (int s = 0; s < stages; ++s)
      for (int b = end + t * 16; b < BYTES; b += T * 16)
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at + s * BYTES + b), "r"(0) : "memory");
  }
  // `row`: its first byte, in memory that begins at `base`
  __device__ __forceinline__ void fetch(int stage, const uint8_t* row, const void* base, int cols, int t) const {
    const int shift = (int)(reinterpret_cast<uintptr_t>(row) & 15), bytes = shift + cols * ES;
    const uint8_t* q = row - shift;
    const uint32_t to = at + stage * BYTES;
    for (int b = t * 16; b < end; b += T * 16) {
      if (q + b < static_cast<const uint8_t*>(base)) {  // nothing in front of the first row is touched
        for (int e = 0; e < 16; e += ES) {
          const bool in = e >= shift && e < bytes;
          if constexpr (F32) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + e), "r"(in ? *reinterpret_cast<const uint32_t*>(q + e) : 0u) : "memory");
          else asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + e), "h"(in ? *reinterpret_cast<const uint16_t*>(q + e) : (uint16_t)0) : "memory");
        }
      } else {  // of the last pieces, what lies in the row; zeros behind it
        const int n = max(0, min(16, bytes - b));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + b), "l"(n ? q + b : row - shift), "r"(n) : "memory");
      }
    }
  }
  // piece j of thread t, 0 behind the last column
  __device__ __forceinline__ void get(int stage, const uint8_t* row, int j, int t, ops::f32x2 (&v)[4]) const {
    const uint32_t from = at + stage * BYTES + (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15) + t * ES;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (F32) {
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[i]) : "r"(from + (j * 8 + i) * T * ES) : "memory");
      } else {
        uint16_t h;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(from + (j * 8 + i) * T * ES) : "memory");
        x[i] = ops::bf_lo(h);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ops::pair2(x[2 * i], x[2 * i + 1]);
  }
};
// The next rows of an operand as this thread fetches them.
template <bool F32>
__device__ __forceinline__ const uint8_t* piece_of(const void* p, long long row, long long ld, int t) {
  return static_cast<const uint8_t*>(p) + (row * ld + t * 8) * (F32 ? 4 : 2);
}
__device__ __forceinline__ void fetched() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int S>
__device__ __forceinline__ void arrived() {  // the oldest of S groups
  asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
}

// WARP: a row is a warp's and a block of 8 takes 8; else a row is a block's.
// Weight and bias stay in registers from row to row (read from L1 for every
// row, they kept it busier than the rows did); T_ is the most threads of a
// block, of which an SM takes 512.
template <int V, bool VEC, bool WARP, bool XF, bool YF, int T_>
__global__ void __launch_bounds__(T_, T_ <= 512 ? 512 / T_ : 1) forward(const __grid_constant__ Params p) {
  constexpr int S = FWD_STAGES<XF>;
  constexpr bool HELD = V <= 2 && T_ <= 512;
  extern __shared__ uint4 ring[];
  __shared__ float4 sh[3][16];
  const int T = WARP ? 32 : SHARED<VEC, WARP, T_> ? T_ : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int per = WARP ? 8 : 1;
  const Ahead<V, XF, S> ahead{smem_u32(ring + threadIdx.x), (int)blockDim.x};
  const int pieces = t * 8 < p.cols ? (p.cols - t * 8 - 1) / (T * 8) + 1 : 0;  // of the V, where rows go by eights
  const long long step = (long long)gridDim.x * per;
  long long r = (long long)blockIdx.x * per + (WARP ? threadIdx.x >> 5 : 0);
  pdl_launch();
  pdl_wait();
  using OddX = Odd<V, XF, T_>;
  const OddX odd(smem_u32(ring), p.cols);
  if constexpr (SHARED<VEC, WARP, T_>) odd.clear(S, t);
  const uint8_t* px = piece_of<XF>(p.x, r, p.ldx, VEC ? t : 0);
  const uint8_t* now = px;  // this row
  const long long next_x = step * p.ldx * (XF ? 4 : 2);
  int left = r < p.rows ? (int)((p.rows - r - 1) / step) + 1 : 0;  // rows to be fetched
  auto fetch = [&](int stage) {
    if (left > 0) {
      if constexpr (VEC) ahead.fetch(stage, px, pieces, T);
      else odd.fetch(stage, px, p.x, p.cols, t);
      px += next_x;
      --left;
    }
    fetched();
  };
  if constexpr (VEC || SHARED<VEC, WARP, T_>)
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch(i);
  ops::f32x2 w[V][4], b[V][4];
  auto weights = [&](int j) {
    float v[8], c[8] = {};
    load_weight<VEC>(p.w, p.w_f32, v, j, p.cols, t, T);
    if (p.b) load_weight<VEC>(p.b, p.b_f32, c, j, p.cols, t, T);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[j][i] = ops::pair2(v[2 * i], v[2 * i + 1]);
      b[j][i] = ops::pair2(c[2 * i], c[2 * i + 1]);
    }
  };
  if constexpr (HELD)
#pragma unroll
    for (int j = 0; j < V; ++j) weights(j);
  for (int stage = 0; r < p.rows; r += step, stage = stage + 1 == S ? 0 : stage + 1) {
    ops::f32x2 v[V][4], s = 0;
    if constexpr (SHARED<VEC, WARP, T_>) {
      arrived<S - 1>();
      __syncthreads();
      fetch(stage == 0 ? S - 1 : stage - 1);
#pragma unroll
      for (int j = 0; j < V; ++j) odd.get(stage, now, j, t, v[j]);
      now += next_x;
    } else {
      ops::Raw<XF> raw[V];
      if constexpr (VEC) {
        fetch(stage == 0 ? S - 1 : stage - 1);
        arrived<S>();
#pragma unroll
        for (int j = 0; j < V; ++j) raw[j] = ahead.get(stage, j, pieces);
      } else {
        load_row<VEC, XF, V>(p.x, r * p.ldx, raw, p.cols, t, T);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ops::unpack2(raw[j], v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s = ops::add2(s, v[j][i]);  // (zero behind the last column)
    }
    float mean = row_sum<WARP, T_>(ops::sum2(s), sh, 0, T) * p.per_col;
    const ops::f32x2 minus = ops::both(-mean);
    s = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ops::f32x2 d = ops::add2(v[j][i], minus);
        if (!VEC && !(SHARED<VEC, WARP, T_> && (j * 8 + 2 * i + 2) * T <= p.cols)) {
          float lo, hi;
          ops::unpair2(d, lo, hi);
          d = ops::pair2(column<false>(j, 2 * i, t, T) < p.cols ? lo : 0.f, column<false>(j, 2 * i + 1, t, T) < p.cols ? hi : 0.f);
        }
        v[j][i] = d;
        if (!VEC || j < pieces) s = ops::fma2(d, d, s);
      }
    }
    float squares = row_sum<WARP, T_>(ops::sum2(s), sh, 1, T);
    if (mean * mean > squares * p.per_col) {  // (the same in all of the row's threads)
      s = 0;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (!VEC || j < pieces)
#pragma unroll
          for (int i = 0; i < 4; ++i) s = ops::add2(s, v[j][i]);
      const float sum = row_sum<WARP, T_>(ops::sum2(s), sh, 2, T), off = sum * p.per_col;
      const ops::f32x2 minus_off = ops::both(-off);
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = ops::add2(v[j][i], minus_off);
      squares = fmaf(-off, sum, squares);
      if (squares < 0.f) squares = 0.f;  // (a NaN stays)
      mean += off;
    }
    const float rstd = rsqrtf(fmaf(squares, p.per_col, p.eps));
    if (p.stats && t == 0) p.stats[r] = make_float2(mean, rstd);
    const ops::f32x2 scale = ops::both(rstd);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (!HELD) weights(j);
      float y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) ops::unpair2(ops::fma2(ops::mul2(v[j][i], scale), w[j][i], b[j][i]), y[2 * i], y[2 * i + 1]);
      if constexpr (SHARED<VEC, WARP, T_>) store_odd<YF>(p.y, r * p.ldy, y, j, p.cols, t, T);
      else store_piece<VEC, YF>(p.y, r * p.ldy, y, j, p.cols, t, T);
    }
  }
}

// Few rows: eight columns of the weight's gradient a block, its threads deal the
// rows out by eights of lanes.  The statistics are given, so that this needs
// nothing of dx, and the whole pass is one launch without scratch.
template <bool XF, bool DF>
__device__ __forceinline__ void columns(const Params& p) {
  __shared__ float sh[2][32][8];
  const int t = threadIdx.x, c = ((int)blockIdx.x - p.row_blocks) * 8 + (t & 7), groups = blockDim.x >> 3;
  float w = 0.f, b = 0.f;
  if (c < p.cols)
#pragma unroll 8
    for (int r = t >> 3; r < p.rows; r += groups) {
      const float2 st = p.stats[r];
      const float d = ops::ld_any(p.dy, r * p.ld_dy + c, DF);
      w = fmaf(d, (ops::ld_any(p.x, r * p.ldx + c, XF) - st.x) * st.y, w);
      b += d;
    }
#pragma unroll
  for (int o = 16; o >= 8; o >>= 1) {
    w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
  }
  if ((t & 31) < 8) {
    sh[0][t >> 5][t & 7] = w;
    sh[1][t >> 5][t & 7] = b;
  }
  __syncthreads();
  if (t >= 16 || c >= p.cols) return;
  float s = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) s += sh[t >> 3][i][t & 7];
  if (t < 8 && p.dw) ops::st_any(p.dw, c, s, p.w_f32);
  if (t >= 8 && p.db) ops::st_any(p.db, c, s, p.b_f32);
}

// A block takes every row_blocks-th row (of eight, with WARP) and keeps its
// columns' sums of dy n and dy in registers; they are written once, for
// reduce().  T_: the most threads of a block, of which an SM takes 512.
template <int V, bool VEC, bool WARP, bool XF, bool DF, int T_>
__global__ void __launch_bounds__(T_, T_ <= 512 ? 512 / T_ : 1) backward(const __grid_constant__ Params p) {
  constexpr int S = BWD_STAGES<XF, DF, T_>;
  constexpr bool HELD = (VEC || !WARP) && T_ <= 512;  // the weight stays in registers
  extern __shared__ uint4 ring[];
  __shared__ float4 sh[2][16];
  const int T = WARP ? 32 : SHARED<VEC, WARP, T_> ? T_ : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int per = WARP ? 8 : 1;
  const Ahead<V, XF, S> ax{smem_u32(ring + threadIdx.x), (int)blockDim.x};
  const Ahead<V, DF, S> ad{ax.at + S * ax.SLOTS * blockDim.x * 16, (int)blockDim.x};
  const Ahead<V, XF, S> ar{ad.at + S * ad.SLOTS * blockDim.x * 16, (int)blockDim.x};
  const int pieces = t * 8 < p.cols ? (p.cols - t * 8 - 1) / (T * 8) + 1 : 0;
  ops::f32x2 dw[V][4] = {}, db[V][4] = {};
  const long long step = (long long)p.row_blocks * per;
  long long r = (long long)blockIdx.x * per + (WARP ? threadIdx.x >> 5 : 0);
  pdl_launch();
  pdl_wait();
  if constexpr (T_ > 512 && V == 1)
    if ((int)blockIdx.x >= p.row_blocks) {
      columns<XF, DF>(p);
      return;
    }
  using OddX = Odd<V, XF, T_>;
  using OddD = Odd<V, DF, T_>;
  const OddX ox(smem_u32(ring), p.cols);
  const OddD od(ox.at + S * OddX::BYTES, p.cols);
  const OddX orr(od.at + S * OddD::BYTES, p.cols);
  if constexpr (SHARED<VEC, WARP, T_>) {
    ox.clear(S, t);
    od.clear(S, t);
    orr.clear(S, t);
  }
  const uint8_t* px = piece_of<XF>(p.x, r, p.ldx, VEC ? t : 0);
  const uint8_t* pd = piece_of<DF>(p.dy, r, p.ld_dy, VEC ? t : 0);
  const uint8_t* pr = piece_of<XF>(p.r, r, p.ld_r, VEC ? t : 0);
  const uint8_t *now_x = px, *now_d = pd, *now_r = pr;  // this row
  const long long next_x = step * p.ldx * (XF ? 4 : 2), next_d = step * p.ld_dy * (DF ? 4 : 2), next_r = step * p.ld_r * (XF ? 4 : 2);
  int left = r < p.rows ? (int)((p.rows - r - 1) / step) + 1 : 0;  // rows to be fetched
  auto fetch = [&](int stage) {
    if (left > 0) {
      if constexpr (VEC) {
        ax.fetch(stage, px, pieces, T);
        ad.fetch(stage, pd, pieces, T);
        if (p.r) ar.fetch(stage, pr, pieces, T);
      } else {
        ox.fetch(stage, px, p.x, p.cols, t);
        od.fetch(stage, pd, p.dy, p.cols, t);
        if (p.r) orr.fetch(stage, pr, p.r, p.cols, t);
      }
      px += next_x;
      pd += next_d;
      pr += next_r;
      --left;
    }
    fetched();
  };
  if constexpr (VEC || SHARED<VEC, WARP, T_>)
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch(i);
  ops::f32x2 w[V][4];
  auto weights = [&](int j) {
    float v[8];
    load_weight<VEC>(p.w, p.w_f32, v, j, p.cols, t, T);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[j][i] = ops::pair2(v[2 * i], v[2 * i + 1]);
  };
  if constexpr (HELD)
#pragma unroll
    for (int j = 0; j < V; ++j) weights(j);
  int buf = 0;
  float2 st = r < p.rows ? p.stats[r] : make_float2(0.f, 0.f);
  for (int stage = 0; r < p.rows; r += step, stage = stage + 1 == S ? 0 : stage + 1) {
    ops::f32x2 n[V][4], g[V][4], s1 = 0, s2 = 0;
    ops::Raw<XF> rx[V];
    ops::Raw<DF> rd[V];
    if constexpr (SHARED<VEC, WARP, T_>) {
      arrived<S - 1>();
      __syncthreads();
      fetch(stage == 0 ? S - 1 : stage - 1);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ox.get(stage, now_x, j, t, n[j]);
        od.get(stage, now_d, j, t, g[j]);
      }
      now_x += next_x;
      now_d += next_d;
    } else {
      if constexpr (VEC) {
        fetch(stage == 0 ? S - 1 : stage - 1);
        arrived<S>();
#pragma unroll
        for (int j = 0; j < V; ++j) {
          rx[j] = ax.get(stage, j, pieces);
          rd[j] = ad.get(stage, j, pieces);
        }
      } else {
        load_row<VEC, XF, V>(p.x, r * p.ldx, rx, p.cols, t, T);
        load_row<VEC, DF, V>(p.dy, r * p.ld_dy, rd, p.cols, t, T);
      }
    }
    const float2 st_next = r + step < p.rows ? p.stats[r + step] : make_float2(0.f, 0.f);
    const ops::f32x2 minus = ops::both(-st.x), rstd = ops::both(st.y);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (!HELD) weights(j);
      if constexpr (!SHARED<VEC, WARP, T_>) {
        ops::unpack2(rx[j], n[j]);
        ops::unpack2(rd[j], g[j]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        n[j][i] = ops::mul2(ops::add2(n[j][i], minus), rstd);
        dw[j][i] = ops::fma2(g[j][i], n[j][i], dw[j][i]);
        db[j][i] = ops::add2(db[j][i], g[j][i]);
        g[j][i] = ops::mul2(g[j][i], w[j][i]);  // (zero behind the last column)
        s1 = ops::add2(s1, g[j][i]);
        s2 = ops::fma2(g[j][i], n[j][i], s2);
      }
    }
    if (p.y) {
      const float2 s = row_sums<WARP, T_>(ops::sum2(s1), ops::sum2(s2), sh, buf, T);
      buf ^= 1;
      const ops::f32x2 a = ops::both(-s.x * p.per_col), b = ops::both(-s.y * p.per_col);
      ops::Raw<XF> rr[V];
      if (!VEC && !SHARED<VEC, WARP, T_> && p.r) load_row<VEC, XF, V>(p.r, r * p.ld_r, rr, p.cols, t, T);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ops::f32x2 res[4] = {};
        if (p.r) {
          if constexpr (SHARED<VEC, WARP, T_>) {
            orr.get(stage, now_r, j, t, res);
          } else {
            if constexpr (VEC) rr[j] = ar.get(stage, j, pieces);
            ops::unpack2(rr[j], res);
          }
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ops::unpair2(ops::fma2(rstd, ops::fma2(n[j][i], b, ops::add2(g[j][i], a)), res[i]), y[2 * i], y[2 * i + 1]);
        if constexpr (SHARED<VEC, WARP, T_>) store_odd<XF>(p.y, r * p.ldy, y, j, p.cols, t, T);
        else store_piece<VEC, XF>(p.y, r * p.ldy, y, j, p.cols, t, T);
      }
    }
    now_r += next_r;
    st = st_next;
  }
  if (!p.part) return;
  const int ldp = (p.cols + 7) / 8 * 8;
  float* part = p.part + (long long)blockIdx.x * 2 * ldp;
  float vw[V][8], vb[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ops::unpair2(dw[j][i], vw[j][2 * i], vw[j][2 * i + 1]);
      ops::unpair2(db[j][i], vb[j][2 * i], vb[j][2 * i + 1]);
    }
  if constexpr (WARP) {
    float(*join)[256 * V] = reinterpret_cast<float(*)[256 * V]>(ring);  // (all rows have arrived)
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) join[threadIdx.x >> 5][column<VEC>(j, i, t, T)] = h ? vb[j][i] : vw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < p.cols; c += 256) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += join[w][c];
        part[h * ldp + c] = s;
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      store_piece<VEC, true>(part, 0, vw[j], j, p.cols, t, T);
      store_piece<VEC, true>(part, ldp, vb[j], j, p.cols, t, T);
    }
  }
}

// The blocks' sums added up, in a fixed order: 32 columns a block, its warps
// deal the partials out.  (With 8 warps for hundreds of partials, the loads of 37 or
// 148 partials in a row took longer than a third of the pass itself.)
struct Reduce {
  const float* part;
  void* dw;
  void* db;
  int blocks, cols, w_f32, b_f32;
};
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) reduce(const __grid_constant__ Reduce p) {
  __shared__ float sh[WARPS][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, ldp = (p.cols + 7) / 8 * 8;
  void* out = blockIdx.y ? p.db : p.dw;
  pdl_launch();
  pdl_wait();
  if (!out) return;
  float s = 0.f;
  if (c < p.cols) {
    const float* q = p.part + blockIdx.y * ldp + c;
#pragma unroll 16
    for (int b = warp; b < p.blocks; b += WARPS) s += __ldcg(q + (long long)b * 2 * ldp);
  }
  sh[warp][lane] = s;
  __syncthreads();
  // a warp adds the warps' sums of its columns
  for (int i = warp; i < 32; i += WARPS) {
    const int mine = blockIdx.x * 32 + i;
    s = ops::warp_sum(lane < WARPS ? sh[lane][i] : 0.f);
    if (lane == 0 && mine < p.cols) ops::st_any(out, mine, s, blockIdx.y ? p.b_f32 : p.w_f32);
  }
}

struct Kernel {
  void (*fn)(Params);
  int smem;  // of a thread
  int threads;  // at most
  int more;  // shared memory besides
};
template <int V, bool VEC, bool WARP, int T, bool XF, bool YF>
Kernel fwd() {
  constexpr int S = FWD_STAGES<XF>;
  return {&forward<V, VEC, WARP, XF, YF, T>, VEC || SHARED<VEC, WARP, T> ? S * V * (XF ? 32 : 16) : 0, T, SHARED<VEC, WARP, T> ? S * 16 : 0};
}
template <int V, bool VEC, bool WARP, int T, bool XF, bool DF>
Kernel bwd() {
  constexpr int S = BWD_STAGES<XF, DF, T>;
  constexpr int rings = S * V * ((XF ? 64 : 32) + (DF ? 32 : 16)), join = 32 * V;  // (the join of a block's 8 warps)
  static_assert(rings >= join, "the join lies where the rings were");
  return {&backward<V, VEC, WARP, XF, DF, T>, VEC || SHARED<VEC, WARP, T> ? rings : WARP ? join : 0, T,
          SHARED<VEC, WARP, T> ? S * 3 * 16 : 0};
}
template <int V, bool WARP, int T>
Kernel fwd_of(bool vec, bool xf, bool yf) {
  if constexpr (WARP || T > 64)  // (as few single elements as 64 threads hold go by warps, or by few's form)
    if (!vec)
      return xf ? (yf ? fwd<V, false, WARP, T, true, true>() : fwd<V, false, WARP, T, true, false>())
                : (yf ? fwd<V, false, WARP, T, false, true>() : fwd<V, false, WARP, T, false, false>());
  return xf ? (yf ? fwd<V, true, WARP, T, true, true>() : fwd<V, true, WARP, T, true, false>())
            : (yf ? fwd<V, true, WARP, T, false, true>() : fwd<V, true, WARP, T, false, false>());
}
template <int V, bool WARP, int T>
Kernel bwd_of(bool vec, bool xf, bool df) {
  return vec ? (xf ? (df ? bwd<V, true, WARP, T, true, true>() : bwd<V, true, WARP, T, true, false>())
                   : (df ? bwd<V, true, WARP, T, false, true>() : bwd<V, true, WARP, T, false, false>()))
             : (xf ? (df ? bwd<V, false, WARP, T, true, true>() : bwd<V, false, WARP, T, true, false>())
                   : (df ? bwd<V, false, WARP, T, false, true>() : bwd<V, false, WARP, T, false, false>()));
}

// How rows are laid over threads: the kernel, threads of a block, rows of a block.
struct Shape {
  Kernel k;
  int T, per;
};
// Threads of two pieces each; rows through shared memory have a kernel's most.
int threads_of(int cols, bool vec) {
  const int T = ops::ceil_div(ops::ceil_div(cols, 16), 32) * 32;
  return vec || T > 512 ? T : T <= 64 ? 64 : T <= 128 ? 128 : T <= 256 ? 256 : 512;
}
// Where there are fewer rows than blocks that run at once, a row has more
// threads: one piece each.  (Blocks of more than 512 threads have 64 registers a
// thread: of two pieces, the forward kernels spill 20 to 40 bytes, the gradient's
// 210 to 280, of one piece the gradient's up to 32, where rows go by single
// elements.  2048 x 16384 bf16 forward 45.2 us; gradients of 250 x 16384 30.8.)
Shape fwd_shape(int cols, bool few, bool vec, bool xf, bool yf) {
  if (cols <= 256) return {fwd_of<1, true, 256>(vec, xf, yf), 256, 8};
  if (cols <= 512) return {fwd_of<2, true, 256>(vec, xf, yf), 256, 8};
  // single elements: a warp's row needs no barrier (1537 x 1001 fp32 4.1 us, with a block's row 4.5; bf16 both 4.4.
  // Not so many more, or fewer: bf16 16384 x 1001 23.9 and 18.8, 4000 x 777 7.0 and 6.6, 600 x 1001 4.0 and 3.2)
  if (!vec && cols <= 1024 && !few)
    return {xf ? (yf ? fwd<4, false, true, 256, true, true>() : fwd<4, false, true, 256, true, false>())
               : (yf ? fwd<4, false, true, 256, false, true>() : fwd<4, false, true, 256, false, false>()),
            256, 8};
  if (few && cols <= 8192) return {fwd_of<1, false, 1024>(vec, xf, yf), ops::ceil_div(ops::ceil_div(cols, 8), 32) * 32, 1};
  const int T = threads_of(cols, vec);
  return {T <= 64    ? fwd_of<2, false, 64>(vec, xf, yf)
          : T <= 128 ? fwd_of<2, false, 128>(vec, xf, yf)
          : T <= 256 ? fwd_of<2, false, 256>(vec, xf, yf)
          : T <= 512 ? fwd_of<2, false, 512>(vec, xf, yf)
                     : fwd_of<2, false, 1024>(vec, xf, yf),
          T, 1};
}
Shape bwd_shape(int cols, bool few, bool vec, bool xf, bool df) {
  if (few) return {bwd_of<1, false, 1024>(vec, xf, df), std::max(128, ops::ceil_div(ops::ceil_div(cols, 8), 32) * 32), 1};
  if (cols <= 256) return {bwd_of<1, true, 256>(vec, xf, df), 256, 8};
  if (cols <= 512) return {bwd_of<2, true, 256>(vec, xf, df), 256, 8};
  const int T = threads_of(cols, vec);
  return {T <= 64    ? bwd_of<2, false, 64>(vec, xf, df)
          : T <= 128 ? bwd_of<2, false, 128>(vec, xf, df)
          : T <= 256 ? bwd_of<2, false, 256>(vec, xf, df)
          : T <= 512 ? bwd_of<2, false, 512>(vec, xf, df)
                     : bwd_of<2, false, 1024>(vec, xf, df),
          T, 1};
}

}  // namespace norm
}  // namespace apk

using namespace apk;

struct apk_norm {
  apk_norm_config cfg{};
  Err err;
  bool opened = false;
  int sms = 0;
  Scratch scratch;
  std::mutex mu;
  std::vector<const void*> ready;  // kernels that have been given their shared memory
};

namespace {

apk_status create(const apk_norm_config* cfg, apk_norm* h) {
  h->cfg = *cfg;
  const apk_norm_config& c = h->cfg;
  if (c.features < 1 || c.features > norm::MAX_FEATURES)
    return h->err.fail(APK_EINVAL, "features is %d: 1 to %d", c.features, norm::MAX_FEATURES);
  if (!(c.eps > 0.f) || !(c.eps < 1e30f)) return h->err.fail(APK_EINVAL, "eps is %g: above 0 and finite", c.eps);
  if (!c.weight) return h->err.fail(APK_EINVAL, "weight is NULL");
  if (!ops::valid_dtype(c.weight_dtype) || (c.bias && !ops::valid_dtype(c.bias_dtype)))
    return h->err.fail(APK_EINVAL, "weight_dtype %d, bias_dtype %d", (int)c.weight_dtype, (int)c.bias_dtype);
  if (!ops::aligned(c.weight, ops::esize(c.weight_dtype)) || (c.bias && !ops::aligned(c.bias, ops::esize(c.bias_dtype))))
    return h->err.fail(APK_EINVAL, "weight or bias is not aligned to its element");
  APK_TRY(ops::open_device(c.device, &h->sms, &h->err));
  DeviceGuard guard(c.device);
  return h->scratch.open(c.device, &h->err);
}

apk_status launch(apk_norm* h, const norm::Shape& sh, const norm::Params& p, int grid, cudaStream_t s, const char* what) {
  const int smem = sh.k.smem * sh.T + sh.k.more;
  const void* fn = reinterpret_cast<const void*>(sh.k.fn);
  // (a kernel's blocks differ in size: it is given what its largest need)
  if (smem > 40 << 10 && std::find(h->ready.begin(), h->ready.end(), fn) == h->ready.end()) {
    APK_TRY(cu_status(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, sh.k.smem * sh.k.threads + sh.k.more), what, &h->err));
    h->ready.push_back(fn);
  }
  Launch l(dim3(grid), sh.T, smem, s);
  return cu_status(cudaLaunchKernelEx(&l.cfg, sh.k.fn, p), what, &h->err);
}

apk_status forward(apk_norm* h, const apk_norm_io* io) {
  const apk_norm_config& c = h->cfg;
  const int D = c.features, M = io->rows;
  if (M < 0 || M > ops::MAX_SIZE) return h->err.fail(APK_EINVAL, "rows is %d: at most 2^30", M);
  if (M == 0) return APK_OK;
  if (!io->x || !io->y) return h->err.fail(APK_EINVAL, "x or y is NULL");
  if (!ops::valid_dtype(io->x_dtype) || !ops::valid_dtype(io->y_dtype))
    return h->err.fail(APK_EINVAL, "x_dtype %d, y_dtype %d", (int)io->x_dtype, (int)io->y_dtype);
  if (io->ldx < D || io->ldy < D)
    return h->err.fail(APK_EINVAL, "a row stride is below its row: ldx %lld, ldy %lld", io->ldx, io->ldy);
  if (!ops::aligned(io->x, ops::esize(io->x_dtype)) || !ops::aligned(io->y, ops::esize(io->y_dtype)) || !ops::aligned(io->stats, 8))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element (stats: to its pair)");
  DeviceGuard guard(c.device);
  norm::Params p{};
  p.x = io->x;
  p.ldx = io->ldx;
  p.w = c.weight;
  p.b = c.bias;
  p.w_f32 = c.weight_dtype == APK_F32;
  p.b_f32 = c.bias_dtype == APK_F32;
  p.y = io->y;
  p.ldy = io->ldy;
  p.stats = reinterpret_cast<float2*>(io->stats);
  p.rows = M;
  p.cols = D;
  p.eps = c.eps;
  p.per_col = 1.f / D;
  const bool vec = D % 8 == 0 && ops::on16(io->x, io->ldx, M, io->x_dtype) && ops::on16(io->y, io->ldy, M, io->y_dtype) &&
                   ops::aligned(c.weight, 16) && ops::aligned(c.bias, 16);
  const bool xf = io->x_dtype == APK_F32, yf = io->y_dtype == APK_F32;
  const norm::Shape sh = norm::fwd_shape(D, M <= h->sms, vec, xf, yf);
  const int grid = std::min(ops::ceil_div(M, sh.per), h->sms * std::max(1, (sh.k.threads > 512 ? 1024 : 512) / sh.T));
  return launch(h, sh, p, grid, static_cast<cudaStream_t>(io->stream), "launching the layer norm");
}

apk_status backward(apk_norm* h, const apk_norm_grads* g) {
  const apk_norm_config& c = h->cfg;
  const int D = c.features, M = g->rows;
  const cudaStream_t s = static_cast<cudaStream_t>(g->stream);
  if (M < 0 || M > ops::MAX_SIZE) return h->err.fail(APK_EINVAL, "rows is %d: at most 2^30", M);
  if (!g->dx && !g->dw && !g->db) return h->err.fail(APK_EINVAL, "no gradient is asked for");
  if (g->db && !c.bias) return h->err.fail(APK_EINVAL, "db of a norm without a bias");
  if (M > 0 && (!g->dy || !g->x || !g->stats)) return h->err.fail(APK_EINVAL, "dy, x or stats is NULL");
  if (!ops::valid_dtype(g->x_dtype) || !ops::valid_dtype(g->dy_dtype))
    return h->err.fail(APK_EINVAL, "x_dtype %d, dy_dtype %d", (int)g->x_dtype, (int)g->dy_dtype);
  if (g->ldx < D || g->ld_dy < D || (g->dx && g->ld_dx < D) || (g->residual_grad && g->ld_residual < D))
    return h->err.fail(APK_EINVAL, "a row stride is below its row: ldx %lld, ld_dy %lld, ld_dx %lld, ld_residual %lld", g->ldx,
                       g->ld_dy, g->ld_dx, g->ld_residual);
  const size_t ex = ops::esize(g->x_dtype);
  if (!ops::aligned(g->x, ex) || !ops::aligned(g->dy, ops::esize(g->dy_dtype)) || !ops::aligned(g->dx, ex) ||
      !ops::aligned(g->residual_grad, ex) || !ops::aligned(g->stats, 8) || !ops::aligned(g->dw, ops::esize(c.weight_dtype)) ||
      (g->db && !ops::aligned(g->db, ops::esize(c.bias_dtype))))
    return h->err.fail(APK_EINVAL, "a pointer is not aligned to its element (stats: to its pair)");
  DeviceGuard guard(c.device);
  if (M == 0) {  // sums over no rows
    if (g->dw) APK_TRY(cu_status(cudaMemsetAsync(g->dw, 0, D * ops::esize(c.weight_dtype), s), "clearing dw", &h->err));
    if (g->db) APK_TRY(cu_status(cudaMemsetAsync(g->db, 0, D * ops::esize(c.bias_dtype), s), "clearing db", &h->err));
    return APK_OK;
  }
  norm::Params p{};
  p.x = g->x;
  p.dy = g->dy;
  p.w = c.weight;
  p.w_f32 = c.weight_dtype == APK_F32;
  p.r = g->residual_grad;
  p.y = g->dx;
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(g->stats));
  p.ldx = g->ldx;
  p.ld_dy = g->ld_dy;
  p.ld_r = g->ld_residual;
  p.ldy = g->ld_dx;
  p.rows = M;
  p.cols = D;
  p.per_col = 1.f / D;
  const bool vec = D % 8 == 0 && ops::on16(g->x, g->ldx, M, g->x_dtype) && ops::on16(g->dy, g->ld_dy, M, g->dy_dtype) &&
                   (!g->dx || ops::on16(g->dx, g->ld_dx, M, g->x_dtype)) &&
                   (!g->residual_grad || ops::on16(g->residual_grad, g->ld_residual, M, g->x_dtype)) && ops::aligned(c.weight, 16);
  const bool xf = g->x_dtype == APK_F32, df = g->dy_dtype == APK_F32;
  // (1 x 8192 would take 9.1 us so, and takes 6.5, 64 x 8192 11.6 and 9.7; 128 x 4096 5.0 against 7.4, 333 x 1001 4.7
  // against 8.8, 444 x 4096 9.0 against 10.4.  It would still be the faster behind the border: 600 x 1024 takes 8.3, so
  // 5.8, 600 x 4096 10.6 and 9.7, 1184 x 1024 9.9 and 8.6)
  const bool few = M <= 3 * h->sms && D <= 4096;
  const norm::Shape sh = norm::bwd_shape(D, few, vec, xf, df);
  const int grid = std::min(ops::ceil_div(M, sh.per), h->sms * std::max(1, (sh.k.threads > 512 ? 1024 : 512) / sh.T));
  const bool sums = g->dw || g->db;
  p.row_blocks = g->dx || !few ? grid : 0;
  if (few) {
    p.dw = g->dw;
    p.db = g->db;
    p.b_f32 = c.bias_dtype == APK_F32;
    return launch(h, sh, p, p.row_blocks + (sums ? ops::ceil_div(D, 8) : 0), s, "launching the layer norm's gradient");
  }
  APK_TRY(h->scratch.enter(s, &h->err));
  ScratchUse use(&h->scratch, &h->err);
  if (sums) {
    APK_TRY(use.begin(ops::up256((size_t)grid * 2 * ops::ceil_div(D, 8) * 8 * 4), 0));
    p.part = reinterpret_cast<float*>(h->scratch.data());
  }
  APK_TRY(launch(h, sh, p, grid, s, "launching the layer norm's gradient"));
  if (sums) {
    const norm::Reduce q{p.part, g->dw, g->db, grid, D, c.weight_dtype == APK_F32, c.bias_dtype == APK_F32};
    Launch l(dim3(ops::ceil_div(D, 32), 2), grid > 64 ? 1024 : 256, 0, s);
    APK_TRY(cu_status(cudaLaunchKernelEx(&l.cfg, grid > 64 ? norm::reduce<32> : norm::reduce<8>, q), "launching the sum of the weight's gradient", &h->err));
  }
  return use.end();
}

}  // namespace

extern "C" {

apk_status apk_norm_create(const apk_norm_config* cfg, apk_norm** out) { return ops::make(cfg, out, create); }

apk_status apk_norm_destroy(apk_norm* h) {
  delete h;
  return APK_OK;
}

const char* apk_norm_last_error(const apk_norm* h) { return h ? h->err.text.c_str() : "NULL handle"; }

apk_status apk_norm_forward(apk_norm* h, const apk_norm_io* io) {
  return ops::call(h, io, [&] { return forward(h, io); });
}

apk_status apk_norm_backward(apk_norm* h, const apk_norm_grads* g) {
  return ops::call(h, g, [&] { return backward(h, g); });
}

}  // extern "C"
