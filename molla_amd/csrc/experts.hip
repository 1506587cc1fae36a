// experts.hip -- a sparse-expert MLP: which experts a token takes (the router), the
// lists that group a call's rows by expert, and the weighted sum of their products;
// gfx950.  (Products of a few rows: experts_rows.h, of many: experts_tile.hip.)
//
// A pair is one expert that one token takes: pair p of a call belongs to row
// p / share of its input.  Experts are stacked: expert e's matrix is rows
// e * rows .. of one GGUF tensor, as a file's ffn_*_exps holds them.
#include <math.h>

#include <algorithm>

#include "experts.h"

namespace mi {
namespace {

// ---- router -----------------------------------------------------------------
// logits[t][e] = x[t] . router[e], products and sums in float64: which of two
// near scores is larger must not hang on the order of a sum.
constexpr int kRouteTok = 4;  // tokens a wave takes
// Scores (tokens times experts) of a call from which the matrix cores take it.  Both
// kernels' time grows with the width, a wave an expert's with the scores besides, the
// matrix cores' little before the chip is full.  us a call, a wave an expert / matrix
// cores, with the choice: 128 experts of 4096 values, 128 tokens 17.4 / 23.5, 192 22.4 /
// 23.4, 224 25.0 / 23.6, 256 28.5 / 23.9; 64 of 2048, 384 tokens 14.1 / 15.1, 448 15.9 /
// 15.2, 512 17.1 / 15.2; 8 of 4096, 2048 tokens 18.5 / 19.7, 3584 25.6 / 21.4; 128 of
// 8192, 224 tokens 41.6 / 37.0; of 1024, 256 tokens 12.6 / 13.2; of 512, 512 14.2 / 11.2.
constexpr int64_t kRouteTile = 28672;
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

// The same on the matrix cores (v_mfma_f64_16x16x4_f64), for many tokens: a wave takes
// 16 tokens x 16 NE experts, the block's W waves every W-th step of 32 values, and their
// sums meet in LDS, added in wave order (2048 tokens, 128 experts of 4096 values, NE = 4:
// four waves 47 us, eight 53, sixteen 103; 32 tokens a wave, K in two parts, 47; one or
// five steps ahead 49, 57).  Lane l holds row or column l % 16
// and four values in turn of its quarter of 16 (the order of K is the same for both);
// result j of lane l is row 4 j + l / 16, column l % 16.
typedef double rd4 __attribute__((ext_vector_type(4)));
template <int NE, int W>
__global__ __launch_bounds__(64 * W) void router_tile_kernel(const float* __restrict__ x,
                                                                      const float* __restrict__ router, int width,
                                                                      int experts, int tokens,
                                                                      double* __restrict__ logits) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  __shared__ double part[W][4 * NE][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, q = lane >> 4;
  const int t0 = blockIdx.y * 16, e0 = blockIdx.x * (16 * NE);
  const float* xr = x + (int64_t)min(t0 + n, tokens - 1) * width;
  const float* wr[NE];
#pragma unroll
  for (int k = 0; k < NE; k++) wr[k] = router + (int64_t)min(e0 + 16 * k + n, experts - 1) * width;
  const int steps = (width + 31) / 32;
  struct Step {
    f4 a[2], b[NE][2];
  };
  // (past the end of a row: the last values, and zeros where they are used)
  auto load = [&](Step& v, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int at = min(32 * s + 16 * h + 4 * q, width - 4);
      v.a[h] = *(const f4*)(xr + at);
#pragma unroll
      for (int k = 0; k < NE; k++) v.b[k][h] = *(const f4*)(wr[k] + at);
    }
  };
  rd4 acc[NE];
#pragma unroll
  for (int k = 0; k < NE; k++) acc[k] = rd4{0.0, 0.0, 0.0, 0.0};
  auto use = [&](Step& v, int s) __attribute__((always_inline)) {
    if (32 * s + 32 > width) {  // (uniform)
#pragma unroll
      for (int h = 0; h < 2; h++)
        if (32 * s + 16 * h + 4 * q >= width) {
          v.a[h] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < NE; k++) v.b[k][h] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int k = 0; k < NE; k++)
          acc[k] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)v.a[h][i], (double)v.b[k][h][i], acc[k], 0, 0, 0);
  };
  // two steps on their way (past the last one: it again, and its use is left out)
  Step st[3];
  load(st[0], min(wave, steps - 1));
  load(st[1], min(wave + W, steps - 1));
  for (int s = wave; s < steps; s += 3 * W) {
#pragma unroll
    for (int i = 0; i < 3; i++) {
      const int now = s + i * W;
      load(st[(i + 2) % 3], min(now + 2 * W, steps - 1));
      __builtin_amdgcn_sched_barrier(0);
      if (now < steps) use(st[i], now);
    }
  }
#pragma unroll
  for (int k = 0; k < NE; k++)
#pragma unroll
    for (int j = 0; j < 4; j++) part[wave][4 * k + j][lane] = acc[k][j];
  __syncthreads();
  for (int i = threadIdx.x; i < 256 * NE; i += 64 * W) {
    const int l = i & 63, j = (i >> 6) & 3, k = i >> 8;
    double v = part[0][4 * k + j][l];
#pragma unroll
    for (int w = 1; w < W; w++) v += part[w][4 * k + j][l];
    const int t = t0 + 4 * j + (l >> 4), e = e0 + 16 * k + (l & 15);
    if (t < tokens && e < experts) logits[(int64_t)t * experts + e] = v;
  }
}

// The largest of a float64 over the wave, in every lane.
template <int CTRL>
__device__ __forceinline__ double max_dpp(double v) {
  return fmax(v, lanes::dpp_d<CTRL>(v));
}
__device__ __forceinline__ double wave_max(double v) {
  v = max_dpp<lanes::kXor1>(v);
  v = max_dpp<lanes::kXor2>(v);
  v = max_dpp<lanes::kHalfMirror>(v);
  v = max_dpp<lanes::kMirror>(v);
  uint64_t b = __double_as_longlong(v);
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  v = fmax(__longlong_as_double((long long)(lo[0] | ((uint64_t)hi[0] << 32))),
           __longlong_as_double((long long)(lo[1] | ((uint64_t)hi[1] << 32))));
  b = __double_as_longlong(v);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
  hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  return fmax(__longlong_as_double((long long)(lo[0] | ((uint64_t)hi[0] << 32))),
              __longlong_as_double((long long)(lo[1] | ((uint64_t)hi[1] << 32))));
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
  float add[PER];
  double top = -INFINITY;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int e = lane + 64 * k;
    p[k] = e < experts ? row[e] : -INFINITY;
    add[k] = bias && e < experts ? bias[e] : 0.0f;
    top = fmax(top, p[k]);
  }
  if (flags & MI_ROUTER_SIGMOID) {
#pragma unroll
    for (int k = 0; k < PER; k++) p[k] = 1.0 / (1.0 + exp(-p[k]));
  } else {
    top = wave_max(top);
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
  uint32_t left = 0;  // bit k: this lane's expert of place k, not taken yet
#pragma unroll
  for (int k = 0; k < PER; k++) {
    score[k] = p[k] + (double)add[k];
    if (!(score[k] == score[k])) score[k] = -INFINITY;
    if (lane + 64 * k < experts) left |= 1u << k;
  }
  int mine = 0;  // lane u: pick u
  double weight = 0.0;
  for (int u = 0; u < used; u++) {
    double best = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; k++)
      if ((left >> k) & 1) best = fmax(best, score[k]);
    best = wave_max(best);
    int at = 0;
    double w = 0.0;
    bool found = false;
    // (fewer than `experts` are taken: one of what is left has the largest score)
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const uint64_t has = __ballot(((left >> k) & 1) && score[k] == best);
      if (!found && has) {
        found = true;
        const int l = __builtin_ctzll(has);
        at = l + 64 * k;
        const uint64_t b = __double_as_longlong(p[k]);
        w = __longlong_as_double((long long)((uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l) |
                                             ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l) << 32)));
        if (lane == l) left &= ~(1u << k);
      }
    }
    if (lane == u) mine = at, weight = w;
  }
  double total = 1.0;
  if (flags & MI_ROUTER_NORM) {
    total = lanes::reduce_sum<64>(weight);
    if (total == 0.0) total = 1.0;
  }
  if (lane < used) {
    ids[t * used + lane] = mine;
    weights[t * used + lane] = (float)(weight / total * (double)scale);
  }
}

// ---- a call's rows by expert -------------------------------------------------
// The first block: counts, their starts in tiles of 32 slots, the blocks' lists, and
// the pair of each slot (-1 behind an expert's last).  Which of an expert's slots a
// pair gets changes nothing of its row (a row's products depend on its own values
// only).  The others: the largest size in each row of x.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void group_plan_kernel(const int32_t* __restrict__ ids, int pairs, int experts,
                                                                  int tiles_a_block, int32_t* __restrict__ order,
                                                                  int4* __restrict__ tiles, int32_t* __restrict__ count,
                                                                  const float* __restrict__ x, int rows, int cols,
                                                                  float* __restrict__ xtop) {
  __shared__ int cnt[kMaxExperts], at[kMaxExperts], wave_sum[2][kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x > 0) {  // a wave a row
    for (int r = (blockIdx.x - 1) * (kPlanThreads / 64) + wave; r < rows; r += (gridDim.x - 1) * (kPlanThreads / 64)) {
      float m = 0.0f;
      for (int i = 4 * lane; i < cols; i += 256) {
        const float4 v = *(const float4*)(x + (int64_t)r * cols + i);
        m = fmaxf(fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
      }
      m = lanes::reduce<64>(m, lanes::Max{});
      if (lane == 0) xtop[r] = m;
    }
    return;
  }
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
  if (tid == kPlanThreads - 1) {
    count[0] = entry + blocks;
    count[1] = (first + t32) * 32;  // slots
  }
  if (tid < experts) {
    at[tid] = first * 32;
    for (int k = 0; k < blocks; k++)
      tiles[entry + k] = make_int4(tid, first + k * tiles_a_block, first * 32 + n, 0);
    for (int k = n; k < t32 * 32; k++) order[first * 32 + k] = -1;
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kPlanThreads) {
    const int e = ids[p];
    if ((uint32_t)e < (uint32_t)experts) order[atomicAdd(&at[e], 1)] = p;
  }
}

// ---- the weighted sum of many rows' products ------------------------------------
// out[t] (+)= sum over k of weights[t][k] * part[t * used + k], in the order of k, a
// pair's splits added up first; a pair without an expert takes no part.
__global__ __launch_bounds__(256) void experts_sum_kernel(const float* __restrict__ part, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ weights, int width, int used,
                                                          int experts, int add, int splits, int64_t split_stride,
                                                          float* __restrict__ out) {
  const int i = 4 * (blockIdx.x * 256 + threadIdx.x);
  const int64_t t = blockIdx.y;
  if (i >= width) return;
  typedef float f4 __attribute__((ext_vector_type(4)));
  f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = 0; k < used; k++) {
    if ((uint32_t)ids[t * used + k] >= (uint32_t)experts) continue;
    const float w = weights[t * used + k];
    const float* p = part + (t * used + k) * width + i;
    f4 a = *(const f4*)p;
    for (int z = 1; z < splits; z++) a += *(const f4*)(p + z * split_stride);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = fmaf(w, a[e], v[e]);
  }
  f4* o = (f4*)(out + t * width + i);
  *o = add ? *o + v : v;
}

}  // namespace

int launch_expert_sum(hipStream_t s, const float* part, const int32_t* ids, const float* weights, int32_t width,
                      int32_t tokens, int32_t used, int32_t experts, bool add, int32_t splits, float* out) {
  hipLaunchKernelGGL(experts_sum_kernel, dim3((width / 4 + 255) / 256, tokens), dim3(256), 0, s, part, ids, weights, width,
                     used, experts, add ? 1 : 0, splits, (int64_t)tokens * used * width, out);
  return hip_check(hipGetLastError(), "experts sum launch");
}

int launch_group_plan(hipStream_t s, const int32_t* ids, int32_t pairs, int32_t experts, int32_t tiles_a_block,
                      const GroupPlan& g, const float* x, int32_t rows, int32_t cols) {
  const int more = x ? std::min((rows + kPlanThreads / 64 - 1) / (kPlanThreads / 64), 4 * cu_count()) : 0;
  hipLaunchKernelGGL(group_plan_kernel, dim3(1 + more), dim3(kPlanThreads), 0, s, ids, pairs, experts, tiles_a_block,
                     g.order, (int4*)g.tiles, g.count, x, rows, cols, g.xtop);
  return hip_check(hipGetLastError(), "group plan launch");
}

int launch_router(hipStream_t s, const float* x, const float* router, const float* bias, int32_t width, int32_t experts,
                  int32_t used, int32_t tokens, int32_t flags, float scale, int32_t* ids, float* weights, void* work) {
  double* logits = (double*)work;
  const int tiles = (tokens + 15) / 16;
  if ((int64_t)tokens * experts < kRouteTile)
    hipLaunchKernelGGL(router_logits_kernel, dim3((experts + 3) / 4, (tokens + kRouteTok - 1) / kRouteTok), dim3(256), 0, s,
                       x, router, width, experts, tokens, logits);
  // (the widest blocks that give every compute unit one: 1024 tokens, 128 experts of 4096
  // values 42 us a call at NE = 1, 31 at 2; 2048 tokens, 64 of 2048 25, 20)
  else if (experts > 16 && (int64_t)tiles * ((experts + 63) / 64) < cu_count() &&
           (int64_t)tiles * ((experts + 31) / 32) >= cu_count())
    hipLaunchKernelGGL((router_tile_kernel<2, 4>), dim3((experts + 31) / 32, tiles), dim3(256), 0, s, x, router, width,
                       experts, tokens, logits);
  else if ((int64_t)tiles * ((experts + 63) / 64) < cu_count() || experts <= 16)
    hipLaunchKernelGGL((router_tile_kernel<1, 8>), dim3((experts + 15) / 16, tiles), dim3(512), 0, s, x, router, width,
                       experts, tokens, logits);
  else
    hipLaunchKernelGGL((router_tile_kernel<4, 4>), dim3((experts + 63) / 64, tiles), dim3(256), 0, s, x, router, width,
                       experts, tokens, logits);
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
