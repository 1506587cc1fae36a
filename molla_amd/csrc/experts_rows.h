// experts_rows.h -- products of a few rows (up to kFewPairs) with stacked experts'
// quantized matrices, gfx950.  The arithmetic is that of the batch-1 kernels
// (matvec_units.h): a lane takes one unit of 64 values of a row, whose packed
// integers meet the activation's limbs in exact integer dots, with one rounding a
// block scale.
//
// Streaming the experts' weights is all the cost, and the batch-1 kernels' shape
// fits it: a lane's activation in registers, a wave's weights sent for at once.  SUB
// lanes (16, 32 or 64) share a row, so that a small expert's short rows fill a wave,
// and a wave takes R rows of each matrix a lane.
#pragma once

#include <algorithm>

#include "experts.h"
#include "matvec_q6k_unit.h"
#include "matvec_rows.h"

namespace mi {
namespace {

// One lane's unit u (64 values) of a row: its activation X, its bytes, its dot.
template <int KIND>
struct RowUnit {
  using X = rows::XUnitRegs<KIND == MI_Q4_0 || KIND == MI_Q5_0>;
  typename mv::UnitOf<KIND, 1>::type w;
  template <class XA>
  static __device__ __forceinline__ void load_x(X& x, const XA& xa, int u) {
    rows::load_x(x, xa, u);
  }
  __device__ __forceinline__ void load(const uint8_t* row, int u) { w.load(row, 0, 0, 0, u); }
  __device__ __forceinline__ float dot(const X& x, int u) const {
    float a[1][1] = {{0.0f}};
    w.template compute<1>(x, u, a);
    return a[0][0];
  }
};
template <>
struct RowUnit<MI_Q6_K> {
  using X = mv::XQ6Regs;
  mv::Q6Piece w;
  uint32_t sh;
  template <class XA>
  static __device__ __forceinline__ void load_x(X& x, const XA& xa, int u) {
    mv::load_x6(x, xa, 8 * (u >> 2) + 4 * ((u >> 1) & 1) + (u & 1));
  }
  __device__ __forceinline__ void load(const uint8_t* row, int u) {
    const uint8_t* p = row + (int64_t)(u >> 2) * 210;
    sh = (uint32_t)((uintptr_t)p & 3u);
    mv::load_piece(w, p - sh, sh, (u >> 1) & 1, u & 1);
  }
  __device__ __forceinline__ float dot(const X& x, int u) const { return mv::piece_dot(w, sh, u & 1, x); }
};

// Matrix rows a lane holds at a time (of both matrices together): what the registers
// take beside an activation.  (Two activations at once, so that a unit is unpacked once
// for two pairs, leave room for four rows: 16 pairs over eight 14336 x 4096 experts of
// Q4_K 96 us against 84.)
template <int KIND>
constexpr int kLaneRows = KIND == MI_Q6_K || KIND == MI_Q5_K ? 4 : 8;

// The sums of N values over each SUB lanes, in every lane of them.
template <int SUB, int N>
__device__ __forceinline__ void reduce_rows(float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; k++) v[k] = lanes::reduce<SUB>(v[k], lanes::Add{});
}

__device__ __forceinline__ mv::XAcc xacc(const uint8_t* xq, int64_t row, int cols) {
  return mv::XAcc{xq + row * xq_token_bytes(cols), 0, (int64_t)(cols >> 5) * 16};
}

// ---- products, and act(gate) * up -----------------------------------------------
// Block (x, p): rows of the expert of pair p, if no earlier pair has the same one,
// against every pair that has it, the weights kept in registers between them where a
// row is one unit a lane.  KS waves split a row (their sums meet in LDS, added in
// wave order).  GLU (KS = 1): a block is 32 rows of both matrices, in passes of what
// its waves hold, and writes act(w0) * w1 in matvec form, the next product's input,
// once every pair's 32 values are in LDS.
constexpr int kGluWaves = 4;
template <int KIND, int SUB, int KS, bool GLU>
struct RowsShape {
  static constexpr int NSUB = 64 / SUB, M = GLU ? 2 : 1, N = kLaneRows<KIND>, R = N / M;
  static constexpr int kFull = 32 / (NSUB * R);  // waves that hold a GLU block's rows at once
  static constexpr int WR = GLU ? (kFull < kGluWaves ? kFull : kGluWaves) : 4 / KS;
  static constexpr int kPass = WR * NSUB * R, kPasses = GLU ? 32 / kPass : 1, kRows = kPass * kPasses;
  static constexpr int kThreads = 64 * WR * KS;
};
// ONE: the input is one row of floats (a decoding token, whatever its pairs), which
// every block brings into matvec form in LDS while its first weights are on their way:
// no launch ahead of this one (and the same bits).
constexpr int kOneCols = 8192;  // of such a row: 32 KB
template <int KIND, int SUB, int KS, bool GLU, bool ONE>
__global__ __launch_bounds__((RowsShape<KIND, SUB, KS, GLU>::kThreads), 2) void experts_rows_kernel(
    const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1, int64_t expert_bytes, int64_t rb, int rows, int cols,
    const uint8_t* __restrict__ xq, int share, const int32_t* __restrict__ ids, int pairs, int experts, int act,
    float* __restrict__ y, uint8_t* __restrict__ xq_out) {
  using Unit = RowUnit<KIND>;
  using S = RowsShape<KIND, SUB, KS, GLU>;
  constexpr int NSUB = S::NSUB, M = S::M, N = S::N, R = S::R, kRows = S::kRows;
  extern __shared__ __align__(16) uint8_t one_row[];
  __shared__ float grp[GLU ? kFewPairs : 2][GLU ? 32 : (KS > 1 ? KS * kRows : 1)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ks = wave % KS, wr = wave / KS;
  const int first = blockIdx.y, id = lane < pairs ? ids[lane] : -1;
  const int e = __builtin_amdgcn_readlane(id, first);
  const uint64_t mine = __ballot(id == e);
  if ((uint32_t)e >= (uint32_t)experts || (mine & ((1ull << first) - 1))) return;  // (uniform over the block)
  const int sub = lane / SUB, sl = lane % SUB;
  const int units = cols >> 6;
  const int turns = (units + SUB * KS - 1) / (SUB * KS);
  const uint8_t* base[M] = {w0 + e * expert_bytes};
  if constexpr (GLU) base[1] = w1 + e * expert_bytes;
#pragma unroll 1
  for (int pass = 0; pass < S::kPasses; pass++) {
    const int local = pass * S::kPass + wr * R * NSUB + sub;  // row r of this lane: + r * NSUB
    const int row0 = blockIdx.x * kRows + local;
    Unit un[N];
    auto load = [&](int u) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < N; k++) un[k].load(base[k / R] + (int64_t)min(row0 + (k % R) * NSUB, rows - 1) * rb, u);
    };
    int it = 0;
    for (uint64_t todo = mine; todo; todo &= todo - 1, it++) {
      const int p = __builtin_ctzll(todo);
      float acc[N] = {};
      for (int s = 0; s < turns; s++) {
        const int u0 = (s * KS + ks) * SUB + sl, u = min(u0, units - 1);
        typename Unit::X x;
        if constexpr (ONE) {
          if (it == 0 || turns > 1) load(u);
          if (pass == 0 && it == 0 && s == 0) {
            __builtin_amdgcn_sched_barrier(0);
            const float* row = (const float*)xq;
            for (int i0 = 0; i0 < cols >> 3; i0 += S::kThreads) {
              const int i = i0 + (int)threadIdx.x, at = 8 * min(i, (cols >> 3) - 1);
              const float4 a = *(const float4*)(row + at), b = *(const float4*)(row + at + 4);
              const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
              quantize8_to_lds(v, i < cols >> 3, i, cols, one_row);
            }
            __syncthreads();
          }
          Unit::load_x(x, mv::XLds{one_row, 0, (cols >> 5) * 16}, u);
        } else {
          Unit::load_x(x, xacc(xq, p / share, cols), u);
          if (it == 0 || turns > 1) load(u);
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
          const float v = un[k].dot(x, u);
          acc[k] += u0 < units ? v : 0.0f;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      reduce_rows<SUB>(acc);
      if constexpr (GLU) {
        if (sl == 0) {
#pragma unroll
          for (int r = 0; r < R; r++)
            grp[it][local + r * NSUB] = ((act & MI_ACT_GELU) ? mv::gelu(acc[r]) : mv::silu(acc[r])) * acc[R + r];
        }
      } else {
        if constexpr (KS > 1) {
          // (buffers take turns: a wave that writes one again has passed the barrier
          // behind the last reading of it)
          float* part = grp[it & 1];
          if (ks > 0 && sl == 0) {
#pragma unroll
            for (int r = 0; r < R; r++) part[ks * kRows + local + r * NSUB] = acc[r];
          }
          __syncthreads();
          if (ks > 0) continue;
#pragma unroll
          for (int r = 0; r < R; r++)
#pragma unroll
            for (int k = 1; k < KS; k++) acc[r] += part[k * kRows + local + r * NSUB];
        }
#pragma unroll
        for (int r = 0; r < R; r++)
          if (sl == 0 && row0 + r * NSUB < rows) y[(int64_t)p * rows + row0 + r * NSUB] = acc[r];
      }
    }
  }
  if constexpr (GLU) {
    __syncthreads();
    int it = 0;
    for (uint64_t todo = mine; todo; todo &= todo - 1, it++) {
      if (it % S::WR != wave) continue;
      quantize_group32(grp[it][lane & 31], lane & 31, blockIdx.x, rows >> 5,
                       xq_out + (int64_t)__builtin_ctzll(todo) * xq_token_bytes(rows), lane < 32);
    }
  }
}

// ---- the weighted sum -------------------------------------------------------------
// Block (x, t): its waves share the units of all of token t's pairs laid end to end
// (short rows of several experts fill a wave, and there is no launch behind it to add
// them).  A lane keeps its unit's activation and walks the block's rows, kRing - 1 of
// them on their way; the waves' sums wait in LDS and are added in wave order.
constexpr int kRing = 4, kSumRows = 64, kSumWaves = 8;  // rows a block takes at most; waves
template <int KIND>
__global__ __launch_bounds__(64 * kSumWaves, 2) void experts_sum_rows_kernel(
    const uint8_t* __restrict__ w, int64_t expert_bytes, int64_t rb, int rows, int cols, const uint8_t* __restrict__ xq,
    const int32_t* __restrict__ ids, const float* __restrict__ weights, int used, int experts, int add, int block_rows,
    float* __restrict__ y) {
  using Unit = RowUnit<KIND>;
  __shared__ float part[kSumWaves][kSumRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int64_t t = blockIdx.y;
  const int row0 = blockIdx.x * block_rows, n = min(block_rows, rows - row0);
  const int units = cols >> 6, all = used * units;
  for (int f0 = 64 * wave; f0 < all; f0 += 64 * waves) {
    const int f = min(f0 + lane, all - 1), k = f / units, u = f - k * units;
    const int e = ids[t * used + k];
    const bool live = f0 + lane < all && (uint32_t)e < (uint32_t)experts;
    const float weight = weights[t * used + k];
    typename Unit::X x;
    Unit::load_x(x, xacc(xq, t * used + k, cols), u);
    const uint8_t* base = w + (live ? e : 0) * expert_bytes + (int64_t)row0 * rb;
    Unit un[kRing];
#pragma unroll
    for (int i = 0; i < kRing - 1; i++) un[i].load(base + (int64_t)min(i, n - 1) * rb, u);
    // row r, after sending for row r + kRing - 1 (past the end: the last one again)
    auto step = [&](int r, Unit& use, Unit& refill) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      refill.load(base + (int64_t)min(r + kRing - 1, n - 1) * rb, u);
      __builtin_amdgcn_sched_barrier(0);
      const float v = use.dot(x, u);
      const float sum = wave_sum(live ? weight * v : 0.0f);
      if (lane == 0) part[wave][r] = f0 < 64 * waves ? sum : part[wave][r] + sum;
    };
    for (int r = 0; r < n; r += kRing) {
#pragma unroll
      for (int i = 0; i < kRing; i++) step(r + i, un[i], un[(i + kRing - 1) % kRing]);  // (rows past n: into room)
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < n) {
    float v = part[0][threadIdx.x];
    for (int k = 1; k < waves; k++) v += part[k][threadIdx.x];
    float* o = y + t * rows + row0 + threadIdx.x;
    *o = add ? *o + v : v;
  }
}

template <int KIND, int SUB, int KS, bool GLU>
int launch_rows_as(hipStream_t s, const ExpertRows& a) {
#define MI_ROWS(ONE, X, LDS)                                                                                         \
  do {                                                                                                               \
    using S = RowsShape<KIND, SUB, KS, GLU>;                                                                    \
    hipLaunchKernelGGL((experts_rows_kernel<KIND, SUB, KS, GLU, ONE>), dim3((a.rows + S::kRows - 1) / S::kRows, a.pairs), \
                       dim3(S::kThreads), LDS, s, (const uint8_t*)a.w0, (const uint8_t*)a.w1, a.rows * a.row_bytes,  \
                       a.row_bytes, a.rows, a.cols, (const uint8_t*)X, a.share, a.ids, a.pairs, a.experts, a.act, a.y, \
                       (uint8_t*)a.xq_out);                                                                          \
  } while (0)
  if (a.x) MI_ROWS(true, a.x, xq_token_bytes(a.cols));
  else MI_ROWS(false, a.xq, 0);
#undef MI_ROWS
  return hip_check(hipGetLastError(), "experts rows launch");
}

template <int KIND>
int launch_sum(hipStream_t s, const ExpertRows& a) {
  const int tokens = a.pairs / a.used, all = (a.cols >> 6) * a.used;
  const int waves = std::min((all + 63) / 64, kSumWaves);
  // rows a block: two waves a SIMD of the chip in one round, where there are as many rows
  const int64_t blocks = std::max<int64_t>((int64_t)cu_count() * 8 / (waves * tokens), 1);
  const int64_t each = ((a.rows + blocks - 1) / blocks + kRing - 1) / kRing * kRing;
  const int n = (int)std::min<int64_t>(each, kSumRows);
  hipLaunchKernelGGL(experts_sum_rows_kernel<KIND>, dim3((a.rows + n - 1) / n, tokens), dim3(64 * waves), 0, s,
                     (const uint8_t*)a.w0, a.rows * a.row_bytes, a.row_bytes, a.rows, a.cols, (const uint8_t*)a.xq, a.ids,
                     a.weights, a.used, a.experts, a.add, n, a.y);
  return hip_check(hipGetLastError(), "experts sum launch");
}

template <int KIND>
int launch_rows_kind(hipStream_t s, const ExpertRows& a) {
  const int units = a.cols >> 6;
  if (a.weights) return launch_sum<KIND>(s, a);
  if (a.w1) {
    if (units <= 16) return launch_rows_as<KIND, 16, 1, true>(s, a);
    if (units <= 32) return launch_rows_as<KIND, 32, 1, true>(s, a);
    return launch_rows_as<KIND, 64, 1, true>(s, a);
  }
  if (units <= 16) return launch_rows_as<KIND, 16, 1, false>(s, a);
  if (units <= 32) return launch_rows_as<KIND, 32, 1, false>(s, a);
  if (units <= 64) return launch_rows_as<KIND, 64, 1, false>(s, a);
  if (units <= 128) return launch_rows_as<KIND, 64, 2, false>(s, a);
  return launch_rows_as<KIND, 64, 4, false>(s, a);
}

}  // namespace
}  // namespace mi
