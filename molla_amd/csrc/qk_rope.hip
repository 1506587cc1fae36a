// qk_rope.hip -- each head of q and k RMS-normed and rotated, and keys and
// values stored, in one pass (mi_qk_norm_rope), gfx950: what gpu_block.mojo:678
// device_attention does between the projections and the attention in four
// launches (two head norms, rope, the cache store).
//
//   y = x * f32(1 / sqrt(mean(x^2) + eps)) * gain   (float64 sum, as head_norm_kernel)
//   (a, b) <- (a c - b s, a s + b c),  c, s of theta = f32(pos) step / factor
//
// A head is a group of 32 or 64 lanes of one wave.  Its values are held as
// slots of two: slot s < dim / 2 is rotary pair s, the slots above it are the
// two-value runs behind the rotary part, so that one lane holds both halves of
// every pair in either pairing and a head never leaves its registers.
#include <math.h>

#include <algorithm>

#include "kv_device.h"
#include "xq_device.h"

namespace mi {
namespace {

constexpr int kQkThreads = 256;

// A wave takes runs of `per` heads of one token (q's, then k's, then v's,
// numbered end to end), its cosines and sines kept in registers for all of them.
template <int LPH, int NS, bool Q8>
__global__ __launch_bounds__(kQkThreads) void qk_rope_kernel(QkRope a, int heads_all, int per, int runs) {
#pragma clang fp contract(off)
  constexpr int GROUPS = 64 / LPH;
  extern __shared__ float stage[];  // Q8: a head's values a lane group
  const mi_qk& d = a.d;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane % LPH, grp = lane / LPH;
  const int64_t job = (int64_t)blockIdx.x * (kQkThreads / 64) + wave;
  const int64_t t64 = job / runs;
  if (t64 >= d.tokens || (d.count && t64 >= *d.count)) return;
  const int t = (int)t64, first = (int)(job - t64 * runs) * per, last = min(first + per, heads_all);
  const int D = d.head_dim, half = d.rope_dim >> 1, slots = D >> 1;
  const int p = d.pos[t];
  float cs[NS], sn[NS], gq[NS][2], gk[NS][2];
  int lo[NS], hi[NS];
  bool live[NS];
#pragma unroll
  for (int i = 0; i < NS; i++) {
    const int s = l + LPH * i;
    live[i] = s < slots;
    const bool turn = s < half;
    lo[i] = !live[i] ? 0 : turn ? (d.neox ? s : 2 * s) : d.rope_dim + 2 * (s - half);
    hi[i] = !live[i] ? 0 : turn && d.neox ? s + half : lo[i] + 1;
    cs[i] = 1.0f;
    sn[i] = 0.0f;
    if (turn) {
      const float theta = rope_theta(p, d.rope_steps, d.rope_factors, s);
      cs[i] = (float)cos((double)theta);
      sn[i] = (float)sin((double)theta);
    }
    gq[i][0] = d.q_norm && live[i] ? d.q_norm[lo[i]] : 1.0f;
    gq[i][1] = d.q_norm && live[i] ? d.q_norm[hi[i]] : 1.0f;
    gk[i][0] = d.k_norm && live[i] ? d.k_norm[lo[i]] : 1.0f;
    gk[i][1] = d.k_norm && live[i] ? d.k_norm[hi[i]] : 1.0f;
  }
  const int kvw = d.kv_heads * D;
  int64_t cell = -1, base = 0;
  if (d.k_cache) {
    if (d.cells) cell = d.cells[t];
    else if (a.kv_index) cell = a.kv_index[(int64_t)t * a.index_stride + p];
    else cell = p, base = (int64_t)t * a.cache_stride;
  }
  const int64_t row = base + cell * cache_row(d.cache_form, kvw);
  // (every lane of the wave walks the same number of heads: the sums and the
  // 8-bit blocks exchange lanes)
  for (int h0 = first; h0 < last; h0 += GROUPS) {
    const int h = h0 + grp;
    const bool on = h < last;
    const bool isq = h < d.heads, isv = h >= d.heads + d.kv_heads;
    const int hk = isq ? 0 : isv ? h - d.heads - d.kv_heads : h - d.heads;
    const float* src = isq ? d.q + t * d.q_stride + (int64_t)h * D
                           : (isv ? d.v + t * d.v_stride : d.k + t * d.k_stride) + (int64_t)hk * D;
    float x[NS][2];
#pragma unroll
    for (int i = 0; i < NS; i++) {
      x[i][0] = on && live[i] ? src[lo[i]] : 0.0f;
      x[i][1] = on && live[i] ? src[hi[i]] : 0.0f;
    }
    if (d.q_norm) {
      double acc = 0.0;
#pragma unroll
      for (int i = 0; i < NS; i++) acc += (double)x[i][0] * (double)x[i][0] + (double)x[i][1] * (double)x[i][1];
      acc = lanes::reduce_sum<LPH>(acc);
      if (!isv) {
        const float scale = (float)(1.0 / sqrt(acc / (double)D + (double)d.eps));
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) x[i][e] = x[i][e] * scale * (isq ? gq[i][e] : gk[i][e]);
      }
    }
    if (!isv) {
#pragma unroll
      for (int i = 0; i < NS; i++) {
        const float u = x[i][0], w = x[i][1];
        if (l + LPH * i < half) {
          x[i][0] = u * cs[i] - w * sn[i];
          x[i][1] = u * sn[i] + w * cs[i];
        }
      }
    }
    float* dst = !on || isv ? nullptr
                 : isq      ? d.q_out + t * d.q_out_stride + (int64_t)h * D
                 : d.k_out  ? d.k_out + t * d.k_out_stride + (int64_t)hk * D
                            : nullptr;
    if (dst) {
#pragma unroll
      for (int i = 0; i < NS; i++)
        if (live[i]) {
          dst[lo[i]] = x[i][0];
          dst[hi[i]] = x[i][1];
        }
    }
    if (cell < 0) continue;  // (uniform)
    __half* rowp = (__half*)(isv ? d.v_cache : d.k_cache) + row;
    if constexpr (Q8) {
      float* mine = stage + (wave * GROUPS + grp) * D;
#pragma unroll
      for (int i = 0; i < NS; i++)
        if (live[i]) {
          mine[lo[i]] = x[i][0];
          mine[hi[i]] = x[i][1];
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (on && !isq) {
        for (int b = l >> 5; b < (D >> 5); b += LPH >> 5)
          q8_store_block(mine[b * 32 + (l & 31)], rowp, (hk * D >> 5) + b, kvw, l & 31);
      }
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else if (on && !isq) {
#pragma unroll
      for (int i = 0; i < NS; i++)
        if (live[i]) {
          rowp[hk * D + lo[i]] = __float2half_rn(x[i][0]);
          rowp[hk * D + hi[i]] = __float2half_rn(x[i][1]);
        }
    }
  }
}

}  // namespace

int launch_qk_rope(hipStream_t s, const QkRope& a) {
  const mi_qk& d = a.d;
  const int heads_all = d.heads + d.kv_heads * (d.k_cache ? 2 : 1);
  // runs of heads: enough waves for the chip, as few as keep a token's angles together
  const int64_t waves = (int64_t)cu_count() * 8;
  const int per = (int)std::max<int64_t>(2, std::min<int64_t>(heads_all, (heads_all * (int64_t)d.tokens + waves - 1) / waves));
  const int runs = (heads_all + per - 1) / per;
  const int64_t blocks = ((int64_t)runs * d.tokens + 3) / 4;
  if (blocks > 0x7fffffff) return fail(MI_ERR_SHAPE, "qk_norm_rope: %d tokens of %d heads", d.tokens, heads_all);
  const bool q8 = d.k_cache && d.cache_form == MI_CACHE_Q8;
#define MI_QK(LPH, NS)                                                                                              \
  if (q8)                                                                                                           \
    hipLaunchKernelGGL((qk_rope_kernel<LPH, NS, true>), dim3((uint32_t)blocks), dim3(kQkThreads),                   \
                       sizeof(float) * d.head_dim * (kQkThreads / LPH), s, a, heads_all, per, runs);                \
  else                                                                                                              \
    hipLaunchKernelGGL((qk_rope_kernel<LPH, NS, false>), dim3((uint32_t)blocks), dim3(kQkThreads), 0, s, a, heads_all, \
                       per, runs)
  if (d.head_dim <= 64) MI_QK(32, 1);
  else if (d.head_dim <= 128) MI_QK(64, 1);
  else if (d.head_dim <= 256) MI_QK(64, 2);
  else MI_QK(64, 4);
#undef MI_QK
  return hip_check(hipGetLastError(), "qk_norm_rope launch");
}

}  // namespace mi
