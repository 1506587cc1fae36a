// experts.hip -- a sparse-expert MLP: which experts a token takes (the router),
// the lists that group a call's rows by expert, and products of a few rows with
// the experts' quantized matrices; gfx950.  (Many rows: experts_tile.hip.)
//
// A pair is one expert that one token takes: pair p of a call belongs to row
// p / share of its input.  Experts are stacked: expert e's matrix is rows
// e * rows .. of one GGUF tensor, as a file's ffn_*_exps holds them.
#include <math.h>

#include <algorithm>

#include "experts.h"
#include "matvec_rows.h"

namespace mi {
namespace {

// ---- router -----------------------------------------------------------------
// logits[t][e] = x[t] . router[e], products and sums in float64: which of two
// near scores is larger must not hang on the order of a sum.
constexpr int kRouteTok = 4;  // tokens a wave takes
__global__ __launch_bounds__(256) void router_logits_kernel(const float* __restrict__ x,
                                                            const float* __restrict__ router, int width, int experts,
                                                            int tokens, double* __restrict__ logits) {
  const int lane = threadIdx.x & 63, e = blockIdx.x * 4 + (threadIdx.x >> 6), t0 = blockIdx.y * kRouteTok;
  if (e >= experts) return;
  double acc[kRouteTok] = {};
  const float* w = router + (int64_t)e * width;
  for (int i = 4 * lane; i < width; i += 256) {
    const float4 a = *(const float4*)(w + i);
#pragma unroll
    for (int k = 0; k < kRouteTok; k++) {
      const float4 b = *(const float4*)(x + (int64_t)min(t0 + k, tokens - 1) * width + i);
      acc[k] = fma((double)a.x, (double)b.x, acc[k]);
      acc[k] = fma((double)a.y, (double)b.y, acc[k]);
      acc[k] = fma((double)a.z, (double)b.z, acc[k]);
      acc[k] = fma((double)a.w, (double)b.w, acc[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kRouteTok; k++) {
    const double v = lanes::reduce_sum<64>(acc[k]);
    if (lane == 0 && t0 + k < tokens) logits[(int64_t)(t0 + k) * experts + e] = v;
  }
}

__device__ __forceinline__ double swap_half(double v, int xor_lane) {
  const uint64_t b = __double_as_longlong(v);
  const uint32_t lo = __shfl_xor((int)(uint32_t)b, xor_lane), hi = __shfl_xor((int)(uint32_t)(b >> 32), xor_lane);
  return __longlong_as_double((long long)(lo | ((uint64_t)hi << 32)));
}

// A wave a token: its logits (expert lane + 64 k in place k), their scores, then
// the largest score `used` times over, the lowest expert of equal ones.  A score
// that is not a number counts as the least.
template <int PER>
__global__ __launch_bounds__(64) void router_pick_kernel(const double* __restrict__ logits,
                                                         const float* __restrict__ bias, int experts, int used,
                                                         int flags, float scale, int32_t* __restrict__ ids,
                                                         float* __restrict__ weights) {
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  const double* row = logits + t * experts;
  double p[PER], score[PER];
  double top = -INFINITY;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    p[k] = lane + 64 * k < experts ? row[lane + 64 * k] : -INFINITY;
    top = fmax(top, p[k]);
  }
  if (flags & MI_ROUTER_SIGMOID) {
#pragma unroll
    for (int k = 0; k < PER; k++) p[k] = 1.0 / (1.0 + exp(-p[k]));
  } else {
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmax(top, swap_half(top, o));
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      p[k] = exp(p[k] - top);
      sum += lane + 64 * k < experts ? p[k] : 0.0;
    }
    sum = lanes::reduce_sum<64>(sum);
#pragma unroll
    for (int k = 0; k < PER; k++) p[k] /= sum;
  }
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int e = lane + 64 * k;
    score[k] = e < experts ? p[k] + (bias ? (double)bias[e] : 0.0) : -INFINITY;
    if (!(score[k] == score[k])) score[k] = -INFINITY;
  }
  uint32_t taken = 0;  // bit k: this lane's expert of place k
  double mine = 0.0, total = 0.0;
  for (int u = 0; u < used; u++) {
    double best = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int k = PER - 1; k >= 0; k--) {
      const int e = lane + 64 * k;
      if (e < experts && !((taken >> k) & 1) && score[k] >= best) best = score[k], at = e;
    }
    for (int o = 32; o; o >>= 1) {
      const double b = swap_half(best, o);
      const int a = __shfl_xor(at, o);
      if (b > best || (b == best && a < at)) best = b, at = a;
    }
    // (at is an expert: fewer than `experts` are taken)
    double w = 0.0;
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (lane + 64 * k == at) taken |= 1u << k, w = p[k];
    const uint64_t b = __double_as_longlong(w);
    const uint32_t lo = __shfl((int)(uint32_t)b, at & 63), hi = __shfl((int)(uint32_t)(b >> 32), at & 63);
    w = __longlong_as_double((long long)(lo | ((uint64_t)hi << 32)));
    total += w;
    if (lane == u) mine = w;
    if (lane == 0) ids[t * used + u] = at;
  }
  if (lane < used) {
    if (flags & MI_ROUTER_NORM) mine = total != 0.0 ? mine / total : 0.0;
    weights[t * used + lane] = (float)(mine * (double)scale);
  }
}

// ---- a call's rows by expert -------------------------------------------------
// One block: counts, their starts in tiles of 32 slots, the blocks' lists, and
// each pair's slot.  Which of an expert's slots a pair gets changes nothing of
// its row (a row's products depend on its own values only).
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void group_plan_kernel(const int32_t* __restrict__ ids, int pairs, int experts,
                                                                  int tiles_a_block, int32_t* __restrict__ slot,
                                                                  int32_t* __restrict__ order,
                                                                  int4* __restrict__ tiles, int32_t* __restrict__ count) {
  __shared__ int cnt[kMaxExperts], at[kMaxExperts], wave_sum[2][kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e < experts; e += kPlanThreads) cnt[e] = 0;
  __syncthreads();
  for (int p = tid; p < pairs; p += kPlanThreads) {
    const int e = ids[p];
    if ((uint32_t)e < (uint32_t)experts) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  // (kMaxExperts <= kPlanThreads: an expert a thread)
  const int n = tid < experts ? cnt[tid] : 0;
  const int t32 = (n + 31) >> 5, blocks = (t32 + tiles_a_block - 1) / tiles_a_block;
  int a = t32, b = blocks;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int ua = __shfl_up(a, o), ub = __shfl_up(b, o);
    if (lane >= o) a += ua, b += ub;
  }
  if (lane == 63) wave_sum[0][wave] = a, wave_sum[1][wave] = b;
  __syncthreads();
  int a0 = 0, b0 = 0;
  for (int w = 0; w < wave; w++) a0 += wave_sum[0][w], b0 += wave_sum[1][w];
  const int first = a0 + a - t32, entry = b0 + b - blocks;
  if (tid == kPlanThreads - 1) *count = entry + blocks;
  if (tid < experts) {
    at[tid] = first * 32;
    for (int k = 0; k < blocks; k++)
      tiles[entry + k] = make_int4(tid, first + k * tiles_a_block, first * 32 + n, 0);
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kPlanThreads) {
    const int e = ids[p];
    int s = -1;
    if ((uint32_t)e < (uint32_t)experts) {
      s = atomicAdd(&at[e], 1);
      order[s] = p;
    }
    slot[p] = s;
  }
}

// ---- a few rows ----------------------------------------------------------------
// Up to 64 pairs: block (x, p) takes 32 rows of the expert of pair p, if no
// earlier pair has the same one, against every pair that has it.  SUB lanes share
// a row, a unit (64 values; 128 for Q6_K) each, in turns where there are more; R
// rows of each matrix a lane, so that an activation read serves them all.  The
// arithmetic is matvec_units.h's: exact integer dots of a unit, one rounding a
// block.
// GLU: act(w0) * w1 of the 32 rows, written in matvec form (a group of xq_out's
// row p), the input of the next product.
template <int KIND, int SUB, int R, bool GLU>
__global__ __launch_bounds__(32 * SUB / R) void experts_rows_kernel(
    const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1, int64_t expert_bytes, int64_t rb, int rows, int cols,
    const uint8_t* __restrict__ xq, int share, const int32_t* __restrict__ ids, int pairs, int experts, int act,
    float* __restrict__ y, uint8_t* __restrict__ xq_out) {
  using Unit = typename mv::UnitOf<KIND, 1>::type;
  constexpr int NSUB = 64 / SUB, M = GLU ? 2 : 1;
  __shared__ float grp[2][GLU ? 32 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = blockIdx.y, id = lane < pairs ? ids[lane] : -1;
  const int e = __builtin_amdgcn_readfirstlane(__shfl(id, first));
  uint64_t todo = __ballot(id == e);
  if ((uint32_t)e >= (uint32_t)experts || (todo & ((1ull << first) - 1))) return;  // (uniform over the block)
  const int sub = lane / SUB, sl = lane % SUB;
  const int local = wave * NSUB * R + sub;  // row r of this lane: + r * NSUB
  const int row0 = blockIdx.x * 32 + local, units = cols / Unit::kElems;
  const uint8_t* base[M] = {w0 + e * expert_bytes};
  if constexpr (GLU) base[1] = w1 + e * expert_bytes;
  Unit un[M * R];
  auto load = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int r = 0; r < R; r++) un[m * R + r].load(base[m], rb, min(row0 + r * NSUB, rows - 1), rows - 1, u);
  };
  const bool fits = units <= SUB;  // the weights stay for every pair
  load(min(sl, units - 1));
  for (int it = 0; todo; todo &= todo - 1, it ^= 1) {
    const int p = __builtin_ctzll(todo);
    const mv::XAcc xa{xq + (int64_t)(p / share) * xq_token_bytes(cols), 0, (int64_t)(cols >> 5) * 16};
    float acc[M * R] = {};
    for (int u0 = 0; u0 < units; u0 += SUB) {
      const int u = min(u0 + sl, units - 1);
      if (!fits) load(u);
      const bool live = u0 + sl < units;
#pragma unroll
      for (int k = 0; k < M * R; k++) {
        float a[1][1] = {{0.0f}};
        un[k].template compute<1>(xa, u, a);
        acc[k] += live ? a[0][0] : 0.0f;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int k = 0; k < M * R; k++) acc[k] = lanes::reduce<SUB>(acc[k], lanes::Add{});
    if constexpr (GLU) {
      if (sl == 0) {
#pragma unroll
        for (int r = 0; r < R; r++)
          grp[it][local + r * NSUB] = ((act & MI_ACT_GELU) ? mv::gelu(acc[r]) : mv::silu(acc[r])) * acc[R + r];
      }
      // (buffers take turns: a wave that writes one again has passed the barrier
      // behind wave 0's last reading of it)
      __syncthreads();
      if (wave == 0)
        quantize_group32(grp[it][lane & 31], lane & 31, blockIdx.x, rows >> 5, xq_out + (int64_t)p * xq_token_bytes(rows),
                         lane < 32);
    } else {
#pragma unroll
      for (int r = 0; r < R; r++)
        if (sl == 0 && row0 + r * NSUB < rows) y[(int64_t)p * rows + row0 + r * NSUB] = acc[r];
    }
  }
}

// out[t] (+)= sum over k of weights[t][k] * part[t * used + k], in the order of k;
// a pair without an expert takes no part.
__global__ __launch_bounds__(256) void experts_sum_kernel(const float* __restrict__ part, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ weights, int width, int used,
                                                          int experts, int add, float* __restrict__ out) {
  const int i = 4 * (blockIdx.x * 256 + threadIdx.x);
  const int64_t t = blockIdx.y;
  if (i >= width) return;
  typedef float f4 __attribute__((ext_vector_type(4)));
  f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = 0; k < used; k++) {
    if ((uint32_t)ids[t * used + k] >= (uint32_t)experts) continue;
    const float w = weights[t * used + k];
    const f4 a = *(const f4*)(part + (t * used + k) * width + i);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = fmaf(w, a[e], v[e]);
  }
  f4* o = (f4*)(out + t * width + i);
  *o = add ? *o + v : v;
}

template <int KIND, int SUB, bool GLU>
int launch_rows_sub(hipStream_t s, const ExpertRows& a) {
  constexpr int R = 4;
  hipLaunchKernelGGL((experts_rows_kernel<KIND, SUB, R, GLU>), dim3((a.rows + 31) / 32, a.pairs), dim3(32 * SUB / R), 0, s,
                     (const uint8_t*)a.w0, (const uint8_t*)a.w1, a.rows * a.row_bytes, a.row_bytes, a.rows, a.cols,
                     (const uint8_t*)a.xq, a.share, a.ids, a.pairs, a.experts, a.act, a.y, (uint8_t*)a.xq_out);
  return hip_check(hipGetLastError(), "experts rows launch");
}

template <int KIND>
int launch_rows_kind(hipStream_t s, const ExpertRows& a) {
  const int units = a.cols / mv::UnitOf<KIND, 1>::type::kElems;
  if (a.w1) {
    if (units <= 16) return launch_rows_sub<KIND, 16, true>(s, a);
    if (units <= 32) return launch_rows_sub<KIND, 32, true>(s, a);
    return launch_rows_sub<KIND, 64, true>(s, a);
  }
  if (units <= 16) return launch_rows_sub<KIND, 16, false>(s, a);
  if (units <= 32) return launch_rows_sub<KIND, 32, false>(s, a);
  return launch_rows_sub<KIND, 64, false>(s, a);
}

}  // namespace

int launch_expert_rows(hipStream_t s, int kind, const ExpertRows& a) {
  switch (kind) {
    case MI_Q4_K: return launch_rows_kind<MI_Q4_K>(s, a);
    case MI_Q5_K: return launch_rows_kind<MI_Q5_K>(s, a);
    case MI_Q6_K: return launch_rows_kind<MI_Q6_K>(s, a);
    case MI_Q8_0: return launch_rows_kind<MI_Q8_0>(s, a);
    case MI_Q4_0: return launch_rows_kind<MI_Q4_0>(s, a);
    case MI_Q4_1: return launch_rows_kind<MI_Q4_1>(s, a);
    case MI_Q5_0: return launch_rows_kind<MI_Q5_0>(s, a);
    case MI_Q5_1: return launch_rows_kind<MI_Q5_1>(s, a);
  }
  return fail(MI_ERR_KIND, "experts: ggml type %d has no device kernel", kind);
}

int launch_expert_sum(hipStream_t s, const float* part, const int32_t* ids, const float* weights, int32_t width,
                      int32_t tokens, int32_t used, int32_t experts, bool add, float* out) {
  hipLaunchKernelGGL(experts_sum_kernel, dim3((width / 4 + 255) / 256, tokens), dim3(256), 0, s, part, ids, weights, width,
                     used, experts, add ? 1 : 0, out);
  return hip_check(hipGetLastError(), "experts sum launch");
}

int launch_group_plan(hipStream_t s, const int32_t* ids, int32_t pairs, int32_t experts, int32_t tiles_a_block,
                      const GroupPlan& g) {
  hipLaunchKernelGGL(group_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, ids, pairs, experts, tiles_a_block, g.slot,
                     g.order, (int4*)g.tiles, g.count);
  return hip_check(hipGetLastError(), "group plan launch");
}

int launch_router(hipStream_t s, const float* x, const float* router, const float* bias, int32_t width, int32_t experts,
                  int32_t used, int32_t tokens, int32_t flags, float scale, int32_t* ids, float* weights, void* work) {
  double* logits = (double*)work;
  hipLaunchKernelGGL(router_logits_kernel, dim3((experts + 3) / 4, (tokens + kRouteTok - 1) / kRouteTok), dim3(256), 0, s, x,
                     router, width, experts, tokens, logits);
  int rc = hip_check(hipGetLastError(), "router launch");
  if (rc) return rc;
#define MI_PICK(P)                                                                                             \
  hipLaunchKernelGGL(router_pick_kernel<P>, dim3(tokens), dim3(64), 0, s, logits, bias, experts, used, flags, \
                     scale, ids, weights)
  if (experts <= 64) MI_PICK(1);
  else if (experts <= 128) MI_PICK(2);
  else if (experts <= 256) MI_PICK(4);
  else MI_PICK(8);
#undef MI_PICK
  return hip_check(hipGetLastError(), "router launch");
}

}  // namespace mi
