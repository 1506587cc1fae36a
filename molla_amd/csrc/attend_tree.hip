// attend_tree.hip -- attention of trees of drafted tokens over a cache
// (mi_attend_tree), gfx950: attention.mojo:144 attend for several tokens of each
// of several sequences, every token over the sequence's committed positions and
// the nodes of its own tree that its mask has, over an f16 or a q8_0 cache, GQA.
//
// A block takes a tile of one sequence's query rows (row = token, query head of
// one key head) and a share of the keys, walked in slices with a running maximum
// and sum, and writes one partial result a row; a second launch folds the
// shares.  Sizes of the sequences are device values: a block finds its tokens
// from starts and leaves when there are none.
#include <math.h>

#include <algorithm>

#include "mi_internal.h"

namespace mi {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// The tokens and keys of sequence b, each held to what the host has checked.
struct TreeSeq {
  int t0, nodes, len, count;
};
__device__ __forceinline__ TreeSeq tree_seq(const mi_tree& tr, int b) {
  TreeSeq s;
  const int a = min(max(tr.starts[b], 0), tr.tokens), e = min(max(tr.starts[b + 1], a), tr.tokens);
  s.t0 = a;
  s.nodes = min(e - a, tr.max_nodes);
  s.len = min(max(tr.lengths[b], 0), tr.max_count);
  s.count = min(s.len + s.nodes, tr.max_count);
  return s;
}

// ---- any head width: the products on the VALU --------------------------------
// 16 query rows a block, four a wave; a slice's keys and values in LDS as
// floats.  Lane = (key, part of the dims) for the scores, dims for the values.
constexpr int kRowsTile = 16, kRowsThreads = 256;

__host__ __device__ __forceinline__ int rows_slice(int head_dim) {
  return head_dim <= 64 ? 64 : head_dim <= 128 ? 32 : head_dim <= 256 ? 16 : 4;
}
__host__ __device__ __forceinline__ size_t rows_lds_bytes(int head_dim) {
  const int kk = rows_slice(head_dim);
  return sizeof(float) * ((size_t)kk * (head_dim + 4) + (size_t)kk * head_dim + (size_t)kRowsTile * head_dim +
                          (size_t)4 * kk * 4);
}

template <bool Q8, int ND>
__global__ __launch_bounds__(kRowsThreads) void attend_tree_rows_kernel(TreeAttend a, int tiles, int shares,
                                                                        float* __restrict__ part_acc,
                                                                        float* __restrict__ part_ml) {
  const int share = blockIdx.x % shares, rest = blockIdx.x / shares;
  const int kvh = rest % a.kv_heads, z = rest / a.kv_heads, b = z / tiles, tile = z % tiles;
  const TreeSeq sq = tree_seq(a.tree, b);
  const int group = a.heads / a.kv_heads, tq = kRowsTile / group, n0 = tile * tq;
  if (n0 >= sq.nodes) return;
  const int D = a.head_dim, kk = rows_slice(D), KS = D + 4;
  const int words = (a.tree.max_nodes + 31) >> 5;
  extern __shared__ float4 lds[];
  float* Ks = (float*)lds;
  float* Vs = Ks + kk * KS;
  float* Qs = Vs + kk * D;
  float* Ps = Qs + kRowsTile * D;  // [wave][key][its 4 rows]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kvw = a.kv_heads * D, crow = cache_row(a.form, kvw);
  const __half* kc = (const __half*)a.k_cache + (a.kv_index ? 0 : (int64_t)b * a.cache_stride);
  const __half* vc = (const __half*)a.v_cache + (a.kv_index ? 0 : (int64_t)b * a.cache_stride);
  const int32_t* index = a.kv_index ? a.kv_index + (int64_t)b * a.index_stride : nullptr;

  // queries; rows past the sequence repeat its last token (not written)
  for (int i = tid; i < kRowsTile * D; i += kRowsThreads) {
    const int r = i / D, e = i - r * D, node = min(n0 + r / group, sq.nodes - 1);
    Qs[i] = a.q[(int64_t)(sq.t0 + node) * a.q_stride + (int64_t)(kvh * group + r % group) * D + e];
  }
  const int r0 = 4 * wave;
  const uint32_t* mrow[4];
#pragma unroll
  for (int r = 0; r < 4; r++)
    mrow[r] = a.tree.mask + (int64_t)(sq.t0 + min(n0 + (r0 + r) / group, sq.nodes - 1)) * words;

  float m2[4], l[4], o[4][ND];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    m2[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; i++) o[r][i] = 0.0f;
  }
  const float c2 = a.scale * kLog2e;
  const int parts = 64 / kk, part = lane / kk, key = lane % kk;
  const int slices = (sq.count + kk - 1) / kk;
  for (int sl = share; sl < slices; sl += shares) {
    const int base = sl * kk;
    __syncthreads();
    for (int i = tid; i < kk * (D / 8); i += kRowsThreads) {
      const int k = i / (D / 8), e = 8 * (i - k * (D / 8)), j = min(base + k, sq.count - 1);
      const int64_t at = (int64_t)(index ? max(index[j], 0) : j) * crow;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        const __half* c = (w ? vc : kc) + at;
        float* dst = w ? Vs + k * D + e : Ks + k * KS + e;
        float f[8];
        if constexpr (Q8) {
          const uint2 raw = *(const uint2*)((const int8_t*)c + kvh * D + e);
          const int8_t* q8 = (const int8_t*)&raw;
          const float fac = __half2float(c[(kvw >> 1) + ((kvh * D + e) >> 5)]);
#pragma unroll
          for (int u = 0; u < 8; u++) f[u] = (float)q8[u] * fac;
        } else {
          const uint4 raw = *(const uint4*)(c + kvh * D + e);
          const __half2* h2 = (const __half2*)&raw;
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const float2 g = __half22float2(h2[u]);
            f[2 * u] = g.x;
            f[2 * u + 1] = g.y;
          }
        }
        *(float4*)dst = make_float4(f[0], f[1], f[2], f[3]);
        *(float4*)(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
      }
    }
    __syncthreads();
    // scores of key `key` for the wave's four rows, a part of the dims a lane
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int e = 4 * part; e < D; e += 4 * parts) {
      const float4 k4 = *(const float4*)(Ks + key * KS + e);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float4 q4 = *(const float4*)(Qs + (r0 + r) * D + e);
        s[r] = fmaf(q4.x, k4.x, s[r]);
        s[r] = fmaf(q4.y, k4.y, s[r]);
        s[r] = fmaf(q4.z, k4.z, s[r]);
        s[r] = fmaf(q4.w, k4.w, s[r]);
      }
    }
    const int j = base + key, node = j - sq.len;
    const bool there = j < sq.count && (!index || index[min(j, sq.count - 1)] >= 0);
    bool masked = false;
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      for (int x = kk; x < 64; x <<= 1) s[r] += __shfl_xor(s[r], x);
      const bool sees = there && (node < 0 || ((mrow[r][node >> 5] >> (node & 31)) & 1));
      masked |= !sees;
      const float sc = sees ? s[r] * c2 : -INFINITY;
      float top = sc;
      for (int x = 1; x < kk; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
      const float mn = fmaxf(m2[r], top);
      const float old = mn == m2[r] ? 1.0f : exp2f(m2[r] - mn);
      p[r] = sees ? exp2f(sc - mn) : 0.0f;
      m2[r] = mn;
      l[r] *= old;
#pragma unroll
      for (int i = 0; i < ND; i++) o[r][i] *= old;
      float sum = p[r];
      for (int x = 1; x < kk; x <<= 1) sum += __shfl_xor(sum, x);
      l[r] += sum;
      if (!sees) p[r] = -1.0f;  // (not a weight: what lies there is not read as a value)
    }
    float* pw = Ps + wave * kk * 4;
    if (part == 0) *(float4*)(pw + 4 * key) = make_float4(p[0], p[1], p[2], p[3]);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool some = __any(masked);
    for (int k = 0; k < kk; k++) {
      const float4 p4 = *(const float4*)(pw + 4 * k);
      const float pr[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
      for (int i = 0; i < ND; i++) {
        const int e = lane + 64 * i;
        const float v = e < D ? Vs[k * D + e] : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (!some || pr[r] >= 0.0f) o[r][i] = fmaf(pr[r], v, o[r][i]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int node = n0 + (r0 + r) / group;
    if ((r0 + r) / group >= tq || node >= sq.nodes) continue;
    const int64_t row = (int64_t)(sq.t0 + node) * a.heads + kvh * group + (r0 + r) % group;
    const int64_t slot = row * shares + share;
    if (lane == 0) *(float2*)(part_ml + 2 * slot) = make_float2(m2[r], l[r]);
#pragma unroll
    for (int i = 0; i < ND; i++)
      if (lane + 64 * i < D) part_acc[slot * D + lane + 64 * i] = o[r][i];
  }
}

// Folds the shares of each (token, head) row: thread = 4 dims.  A share that no
// key of the row fell in has sum 0 and is left out; a row without any is zero.
__global__ __launch_bounds__(256) void attend_tree_fold_kernel(const float* __restrict__ part_acc,
                                                               const float* __restrict__ part_ml, mi_tree tree,
                                                               int heads, int D, int shares, float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int tpr = D >> 2, d4 = (int)(i % tpr);
  const int64_t row = i / tpr;
  if (row >= (int64_t)min(max(tree.starts[tree.batch], 0), tree.tokens) * heads) return;
  const float2* ml = (const float2*)part_ml + row * shares;
  const float4* acc = (const float4*)(part_acc + row * shares * D) + d4;
  float m = -INFINITY;
  for (int s = 0; s < shares; s++) {
    const float2 v = ml[s];
    if (v.y != 0.0f) m = fmaxf(m, v.x);
  }
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
  for (int s = 0; s < shares; s++) {
    const float2 v = ml[s];
    if (v.y == 0.0f) continue;
    const float4 x = acc[(int64_t)s * tpr];
    const float w = v.x == m ? 1.0f : exp2f(v.x - m);
    l = fmaf(v.y, w, l);
    o.x = fmaf(x.x, w, o.x);
    o.y = fmaf(x.y, w, o.y);
    o.z = fmaf(x.z, w, o.z);
    o.w = fmaf(x.w, w, o.w);
  }
  const float w = l != 0.0f ? 1.0f / l : 0.0f;
  ((float4*)out)[row * tpr + d4] = make_float4(o.x * w, o.y * w, o.z * w, o.w * w);
}

struct TreeGrid {
  int tiles, shares;
  int64_t blocks;
};

TreeGrid tree_grid(int heads, int kv_heads, int head_dim, const mi_tree& t) {
  TreeGrid g;
  const int tq = kRowsTile / (heads / kv_heads);
  g.tiles = (t.max_nodes + tq - 1) / tq;
  const int64_t pairs = (int64_t)t.batch * g.tiles * kv_heads;
  const int64_t slices = ((int64_t)t.max_count + rows_slice(head_dim) - 1) / rows_slice(head_dim);
  g.shares = (int)std::max<int64_t>(1, std::min<int64_t>({4 * (int64_t)cu_count() / pairs, slices, 64}));
  g.blocks = pairs * g.shares;
  return g;
}

}  // namespace

static size_t part_acc_bytes(int heads, int head_dim, const mi_tree& t, int shares) {
  return ((size_t)t.tokens * heads * shares * head_dim * sizeof(float) + 255) & ~(size_t)255;
}

size_t tree_attend_workspace(int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t form, const mi_tree& t) {
  (void)form;
  const TreeGrid g = tree_grid(heads, kv_heads, head_dim, t);
  return part_acc_bytes(heads, head_dim, t, g.shares) + (size_t)t.tokens * heads * g.shares * 2 * sizeof(float);
}

int launch_tree_attend(hipStream_t s, const TreeAttend& a, void* work) {
  const TreeGrid g = tree_grid(a.heads, a.kv_heads, a.head_dim, a.tree);
  if (g.blocks > 0x7fffffff) return fail(MI_ERR_SHAPE, "attend_tree: %d sequences of %d nodes", a.tree.batch, a.tree.max_nodes);
  float* part_acc = (float*)work;
  float* part_ml = (float*)((char*)work + part_acc_bytes(a.heads, a.head_dim, a.tree, g.shares));
  const size_t lds = rows_lds_bytes(a.head_dim);
#define MI_TREE_ROWS(ND)                                                                                             \
  if (a.form == MI_CACHE_Q8)                                                                                         \
    hipLaunchKernelGGL((attend_tree_rows_kernel<true, ND>), dim3((uint32_t)g.blocks), dim3(kRowsThreads), lds, s, a,  \
                       g.tiles, g.shares, part_acc, part_ml);                                                        \
  else                                                                                                               \
    hipLaunchKernelGGL((attend_tree_rows_kernel<false, ND>), dim3((uint32_t)g.blocks), dim3(kRowsThreads), lds, s, a, \
                       g.tiles, g.shares, part_acc, part_ml)
  if (a.head_dim <= 64) MI_TREE_ROWS(1);
  else if (a.head_dim <= 128) MI_TREE_ROWS(2);
  else if (a.head_dim <= 256) MI_TREE_ROWS(4);
  else MI_TREE_ROWS(8);
#undef MI_TREE_ROWS
  if (int rc = hip_check(hipGetLastError(), "attend_tree launch")) return rc;
  const int64_t threads = (int64_t)a.tree.tokens * a.heads * (a.head_dim / 4), blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return fail(MI_ERR_SHAPE, "attend_tree: %d tokens of %d heads", a.tree.tokens, a.heads);
  hipLaunchKernelGGL(attend_tree_fold_kernel, dim3((uint32_t)blocks), dim3(256), 0, s, part_acc, part_ml, a.tree,
                     a.heads, a.head_dim, g.shares, a.out);
  return hip_check(hipGetLastError(), "attend_tree fold launch");
}

}  // namespace mi
