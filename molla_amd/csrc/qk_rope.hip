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
// Any shape: 4096 tokens of 32 + 2 x 8 heads of 160 82 us (230 MB: 49 at a copy's
// rate), over q8_0 101; of 128 over q8_0 with half-split pairs in half a head 82, where
// the kernel below takes 46 for whole heads (words of 4 bytes, one head's loads at a
// time, over q8_0 a trip through LDS).
template <int LPH, int NS, bool Q8>
__global__ __launch_bounds__(kQkThreads) void qk_rope_kernel(mi_qk d, int heads_all, int per, int runs) {
#pragma clang fp contract(off)
  constexpr int GROUPS = 64 / LPH;
  extern __shared__ float stage[];  // Q8: a head's values a lane group
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane % LPH, grp = lane / LPH;
  const int64_t job = (int64_t)grid_block() * (kQkThreads / 64) + wave;
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
      double sd, cd;
      sincos((double)theta, &sd, &cd);
      cs[i] = (float)cd;
      sn[i] = (float)sd;
    }
    gq[i][0] = d.q_norm && live[i] ? d.q_norm[lo[i]] : 1.0f;
    gq[i][1] = d.q_norm && live[i] ? d.q_norm[hi[i]] : 1.0f;
    gk[i][0] = d.k_norm && live[i] ? d.k_norm[lo[i]] : 1.0f;
    gk[i][1] = d.k_norm && live[i] ? d.k_norm[hi[i]] : 1.0f;
  }
  const int kvw = d.kv_heads * D;
  const int64_t cell = d.k_cache ? d.cells[t] : -1, row = cell * cache_row(d.cache_form, kvw);
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

// The same where a head is a multiple of 64 values up to 256 and everything lies
// on 16 bytes: two neighbouring slots a lane, so that a lane's values are two
// words of 8 bytes (half-split pairs) or one of 16 (adjacent pairs), and D / 4
// lanes a head.  The loads of kAhead heads are sent for together: 4096 tokens of
// 32 + 2 x 8 heads of 128 68 -> 41.6 us (184 MB, 4.4 TB/s), over q8_0 46 (43 adjacent).
constexpr int kAhead = 4;

struct QkRow {  // of a token, by kind of head
  const float* src;
  float* dst;
  __half* cache;
};

template <int LPH, bool NEOX, bool Q8>
__global__ __launch_bounds__(kQkThreads) void qk_rope_vec_kernel(mi_qk d, int heads_all, int per, int runs) {
#pragma clang fp contract(off)
  constexpr int GROUPS = 64 / LPH, D = 4 * LPH;
  const int lane = threadIdx.x & 63, l = lane % LPH, grp = lane / LPH;
  const int64_t job = (int64_t)grid_block() * (kQkThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t64 = job / runs;
  if (t64 >= d.tokens || (d.count && t64 >= *d.count)) return;
  const int t = (int)t64, first = (int)(job - t64 * runs) * per, last = min(first + per, heads_all);
  const int half = d.rope_dim >> 1, p = d.pos[t];
  // slots 2 l and 2 l + 1: values lo .. and hi .. (two each, or four from lo)
  const bool turn = 2 * l < half;
  const int lo = !NEOX ? 4 * l : turn ? 2 * l : d.rope_dim + 2 * (2 * l - half), hi = lo + (NEOX && turn ? half : 2);
  const int kvw = d.kv_heads * D;
  const int64_t cell = d.k_cache ? d.cells[t] : -1, row = cell * cache_row(d.cache_form, kvw);
  auto source = [&](int h) __attribute__((always_inline)) {
    const int hk = h - d.heads, hv = hk - d.kv_heads;
    return h < d.heads ? d.q + t * d.q_stride + (int64_t)h * D
           : hv < 0    ? d.k + t * d.k_stride + (int64_t)hk * D
                       : d.v + t * d.v_stride + (int64_t)hv * D;
  };
  float x[kAhead][4];
  auto load = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const float* src = source(min(h0 + j * GROUPS + grp, last - 1));
      if constexpr (NEOX) {
        const float2 u = *(const float2*)(src + lo), w = *(const float2*)(src + hi);
        x[j][0] = u.x, x[j][1] = u.y, x[j][2] = w.x, x[j][3] = w.y;
      } else {
        const float4 u = *(const float4*)(src + lo);
        x[j][0] = u.x, x[j][1] = u.y, x[j][2] = u.z, x[j][3] = u.w;
      }
    }
  };
  load(first);
  // value e of a lane: slot e % 2 (half-split) or e / 2 (adjacent) of its two, first or second of the pair
  float cs[2] = {1.0f, 1.0f}, sn[2] = {0.0f, 0.0f}, gq[4], gk[4];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if (turn) {
      double sd, cd;
      sincos((double)rope_theta(p, d.rope_steps, d.rope_factors, 2 * l + i), &sd, &cd);
      cs[i] = (float)cd;
      sn[i] = (float)sd;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int at = e < 2 ? lo + e : hi + e - 2;
    gq[e] = d.q_norm ? d.q_norm[at] : 1.0f;
    gk[e] = d.q_norm ? d.k_norm[at] : 1.0f;
  }
  for (int h0 = first; h0 < last; h0 += kAhead * GROUPS) {
    float y[kAhead][4];
#pragma unroll
    for (int j = 0; j < kAhead; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) y[j][e] = x[j][e];
    if (h0 + kAhead * GROUPS < last) load(h0 + kAhead * GROUPS);
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int h = h0 + j * GROUPS + grp;
      const bool on = h < last, isq = h < d.heads, isv = h >= d.heads + d.kv_heads;
      const int hk = isq ? 0 : isv ? h - d.heads - d.kv_heads : h - d.heads;
      if (d.q_norm) {
        double acc = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) acc += (double)y[j][e] * (double)y[j][e];
        acc = lanes::reduce_sum<LPH>(acc);
        const float scale = (float)(1.0 / sqrt(acc / (double)D + (double)d.eps));
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (!isv) y[j][e] = y[j][e] * scale * (isq ? gq[e] : gk[e]);
      }
      if (!isv && turn) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float &u = y[j][NEOX ? i : 2 * i], &w = y[j][NEOX ? 2 + i : 2 * i + 1];
          const float ru = u * cs[i] - w * sn[i], rw = u * sn[i] + w * cs[i];
          u = ru;
          w = rw;
        }
      }
      float* dst = !on || isv ? nullptr
                   : isq      ? d.q_out + t * d.q_out_stride + (int64_t)h * D
                   : d.k_out  ? d.k_out + t * d.k_out_stride + (int64_t)hk * D
                              : nullptr;
      if (dst) {
        if constexpr (NEOX) {
          *(float2*)(dst + lo) = make_float2(y[j][0], y[j][1]);
          *(float2*)(dst + hi) = make_float2(y[j][2], y[j][3]);
        } else {
          *(float4*)(dst + lo) = make_float4(y[j][0], y[j][1], y[j][2], y[j][3]);
        }
      }
      if (cell < 0) continue;  // (uniform)
      __half* rowp = (__half*)(isv ? d.v_cache : d.k_cache) + row;
      if constexpr (Q8) {
        // 32 values are 16 lanes' first or second two (half-split: the rotary part is the
        // whole head), or 8 lanes' four; the rule is q8_store_block's
        float amax[2];
#pragma unroll
        for (int w = 0; w < 2; w++) amax[w] = fmaxf(fabsf(y[j][2 * w]), fabsf(y[j][2 * w + 1]));
        if constexpr (NEOX) {
#pragma unroll
          for (int w = 0; w < 2; w++) amax[w] = lanes::reduce<16>(amax[w], lanes::Max{});
        } else {
          amax[0] = amax[1] = lanes::reduce<8>(fmaxf(amax[0], amax[1]), lanes::Max{});
        }
        uint32_t bytes[2];
#pragma unroll
        for (int w = 0; w < 2; w++) {
          const float inv = amax[w] == 0.0f ? 0.0f : 127.0f / amax[w];
          uint32_t b[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float z = y[j][2 * w + e] * inv, r = z >= 0.0f ? z + 0.5f : z - 0.5f;
            b[e] = (uint32_t)max(-127, min(127, (int)r)) & 0xffu;
          }
          bytes[w] = b[0] | (b[1] << 8);
        }
        if (on && !isq) {
          uint8_t* q8 = (uint8_t*)rowp + hk * D;
          if constexpr (NEOX) {
            *(uint16_t*)(q8 + lo) = (uint16_t)bytes[0];
            *(uint16_t*)(q8 + hi) = (uint16_t)bytes[1];
            if ((l & 15) == 0) {
              rowp[(kvw >> 1) + ((hk * D + lo) >> 5)] = __float2half_rn(amax[0] / 127.0f);
              rowp[(kvw >> 1) + ((hk * D + hi) >> 5)] = __float2half_rn(amax[1] / 127.0f);
            }
          } else {
            *(uint32_t*)(q8 + lo) = bytes[0] | (bytes[1] << 16);
            if ((l & 7) == 0) rowp[(kvw >> 1) + ((hk * D + lo) >> 5)] = __float2half_rn(amax[0] / 127.0f);
          }
        }
      } else if (on && !isq) {
        const __half2 u = __floats2half2_rn(y[j][0], y[j][1]), w = __floats2half2_rn(y[j][2], y[j][3]);
        if constexpr (NEOX) {
          *(__half2*)(rowp + hk * D + lo) = u;
          *(__half2*)(rowp + hk * D + hi) = w;
        } else {
          __half2 both[2] = {u, w};
          *(uint2*)(rowp + hk * D + lo) = *(uint2*)both;
        }
      }
    }
  }
}

}  // namespace

// Whether the vector kernel takes the shape: its words may not straddle a pair's
// halves, the rotary part's end or an 8-bit block, and every row starts on 16 bytes.
static bool qk_vec_fits(const mi_qk& d) {
  if (d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256) return false;
  if (d.rope_dim % 4) return false;
  if (d.k_cache && d.cache_form == MI_CACHE_Q8 && d.neox && (d.rope_dim != d.head_dim)) return false;
  const uintptr_t p = (uintptr_t)d.q | (uintptr_t)d.k | (uintptr_t)d.v | (uintptr_t)d.q_out | (uintptr_t)d.k_out;
  const int64_t st = d.q_stride | d.k_stride | (d.v ? d.v_stride : 0) | d.q_out_stride | (d.k_out ? d.k_out_stride : 0);
  return !(p & 15) && !(st & 3);
}

int launch_qk_rope(hipStream_t s, const mi_qk& d) {
  const int heads_all = d.heads + d.kv_heads * (d.k_cache ? 2 : 1);
  const bool q8 = d.k_cache && d.cache_form == MI_CACHE_Q8, vec = qk_vec_fits(d);
  // runs of heads: enough waves for the chip, as few as keep a token's angles together
  const int64_t waves = (int64_t)cu_count() * 16;
  const int least = vec ? 256 / d.head_dim : 2;
  const int per = (int)std::max<int64_t>(least, std::min<int64_t>(heads_all, (heads_all * (int64_t)d.tokens + waves - 1) / waves));
  const int runs = (heads_all + per - 1) / per;
  const int64_t blocks = ((int64_t)runs * d.tokens + 3) / 4;
  if (blocks > 0x7fffffff) return fail(MI_ERR_SHAPE, "qk_norm_rope: %d tokens of %d heads", d.tokens, heads_all);
  if (vec) {
#define MI_QKV(LPH, N, Q)                                                                                             \
  hipLaunchKernelGGL((qk_rope_vec_kernel<LPH, N, Q>), grid_of(blocks), dim3(kQkThreads), 0, s, d, heads_all, \
                     per, runs)
#define MI_QKV_F(LPH)                      \
  if (d.neox) {                            \
    if (q8) MI_QKV(LPH, true, true);       \
    else MI_QKV(LPH, true, false);         \
  } else {                                 \
    if (q8) MI_QKV(LPH, false, true);      \
    else MI_QKV(LPH, false, false);        \
  }
    if (d.head_dim == 64) { MI_QKV_F(16) }
    else if (d.head_dim == 128) { MI_QKV_F(32) }
    else { MI_QKV_F(64) }
#undef MI_QKV_F
#undef MI_QKV
    return hip_check(hipGetLastError(), "qk_norm_rope launch");
  }
#define MI_QK(LPH, NS)                                                                                              \
  if (q8)                                                                                                           \
    hipLaunchKernelGGL((qk_rope_kernel<LPH, NS, true>), grid_of(blocks), dim3(kQkThreads),                   \
                       sizeof(float) * d.head_dim * (kQkThreads / LPH), s, d, heads_all, per, runs);                \
  else                                                                                                              \
    hipLaunchKernelGGL((qk_rope_kernel<LPH, NS, false>), grid_of(blocks), dim3(kQkThreads), 0, s, d, heads_all, \
                       per, runs)
  if (d.head_dim <= 64) MI_QK(32, 1);
  else if (d.head_dim <= 128) MI_QK(64, 1);
  else if (d.head_dim <= 256) MI_QK(64, 2);
  else MI_QK(64, 4);
#undef MI_QK
  return hip_check(hipGetLastError(), "qk_norm_rope launch");
}

}  // namespace mi
