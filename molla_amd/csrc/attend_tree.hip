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

// ---- head widths 64, 128 and 256: the products on the matrix cores -----------
// v_mfma_f32_16x16x32_f16.  A block is 64 NC query rows, 16 NC to a wave, and
// stages slices of 64 keys (32 at D = 256) in LDS for its four waves, the next
// slice's words on their way in registers behind the present one's products.
//
//   S^T = K Q^T, keys as rows and queries as columns: a lane's 8 scores of 32
//   keys belong to its own query, the softmax takes two exchanges between lanes
//   and the weights are in place as the B operand of O^T = V^T P^T, whose values
//   lie by rows in LDS and are read transposed (ds_read_b64_tr_b16).  Slot i of
//   lane group g takes key 4 g + i % 4 + 16 (i / 4), the order in which S^T
//   leaves them.
//   Queries enter as two halves, each query scaled by a power of two so that its
//   largest value is in [2^14, 2^15): every value to 2^-23 of itself (its float
//   to 2^-24), down to 2^-39 of the largest.  Weights, lifted by 2^14, enter as
//   two halves as well: to 2^-24 of the largest weight.
//
// q8_0: keys and values enter as their integers, exact halves; a key block's
// factor multiplies its part of the score, a value block's the weights, which
// are then split into halves at 2^(15 - X), X the exponent of the column's
// largest product since its maximum last rose (as in attend_decode.hip): what a
// column does not see has no part in its X.
//
// A value that is not finite in a node that some query does not see would give
// 0 * inf there: such values are staged as zeros and added at the end to the
// queries that see them.
//
// MFMA fragments (16x16x32): lane l holds row / column l % 16 and values
// 8 (l / 16) .. +8 of the 32; result element i of lane l is row 4 (l / 16) + i,
// column l % 16.
typedef _Float16 th2 __attribute__((ext_vector_type(2)));
typedef _Float16 th8 __attribute__((ext_vector_type(8)));
typedef short ts4 __attribute__((ext_vector_type(4)));
typedef short ts8 __attribute__((ext_vector_type(8)));
typedef float tf4 __attribute__((ext_vector_type(4)));
typedef uint32_t tu4 __attribute__((ext_vector_type(4)));

constexpr float kLift = 16384.0f;

__device__ __forceinline__ tf4 mfma16(th8 a, th8 b, tf4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 16-byte piece pc of LDS row r lies at slot pc ^ swz(r), so that the lanes
// served together fall on distinct banks: keys are read one piece of 16 rows,
// values (transposed) 4 rows x 32 bytes per 16 lanes.
template <int D>
__device__ __forceinline__ int key_swz(int r) {
  return D >= 128 ? (r & 15) : ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int val_swz(int r) {
  return (D >= 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1)) | ((r >> 2) & 3);
}

// over the four lanes that share a column
template <class Op>
__device__ __forceinline__ float across(float v, Op op) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
  p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// (by value: a bit cast of a vector's element itself takes its first element)
__device__ __forceinline__ th2 as_th2(uint32_t u) { return __builtin_bit_cast(th2, u); }

// eight signed bytes as halves: 0x64 above byte + 128 is 1152 + byte
__device__ __forceinline__ th8 int8_halves(uint32_t x, uint32_t y) {
  const th2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  x ^= 0x80808080u;
  y ^= 0x80808080u;
  const tu4 m = {__builtin_amdgcn_perm(0x64646464u, x, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u),
                 __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u)};
  tu4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(uint32_t, as_th2(m[i]) + off);
  return __builtin_bit_cast(th8, r);
}

// Bit i: whether a token with this mask row sees the key of node first + i.
// Keys ahead of the nodes are seen, those behind them are not.
__device__ __forceinline__ uint32_t seen_bits(const uint32_t* __restrict__ row, int words, int first, int nodes) {
  if (first <= -32) return 0xffffffffu;
  uint32_t bits;
  if (first < 0) {
    bits = (row[0] << -first) | ((1u << -first) - 1u);
  } else {
    const int w = first >> 5;
    const uint64_t two = (w < words ? row[w] : 0u) | ((uint64_t)(w + 1 < words ? row[w + 1] : 0u) << 32);
    bits = (uint32_t)(two >> (first & 31));
  }
  const int left = nodes - first;
  return left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1u) : 0u;
}

__device__ __forceinline__ bool not_finite(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }
// the two halves of w, zero where they are not finite
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  return (not_finite(w) ? 0u : w & 0xffffu) | (not_finite(w >> 16) ? 0u : w & 0xffff0000u);
}

__host__ __device__ constexpr int mfma_slice(int D) { return D <= 128 ? 64 : 32; }

template <int D, int NC, bool Q8, bool PAGED>
__global__ __launch_bounds__(256, 2) void attend_tree_kernel(TreeAttend a, int tiles, int shares,
                                                             float* __restrict__ part_acc,
                                                             float* __restrict__ part_ml) {
  constexpr int SL = mfma_slice(D), KS = D / 32, NT = D / 16, PIECES = D / 8;
  constexpr int PER = Q8 ? SL * D / 16 / 256 : SL * PIECES / 256;  // 16-byte words of K (and of V) a thread
  constexpr int WPK = Q8 ? D / 16 : PIECES;                       // words a key
  constexpr int ROWS = 64 * NC;
  __shared__ __align__(16) _Float16 ks[2][SL * D];
  __shared__ __align__(16) _Float16 vs[2][SL * D];
  __shared__ __align__(16) float fac[Q8 ? 2 : 1][2][Q8 ? KS : 1][Q8 ? SL : 1];  // q8_0 factors of keys and values
  __shared__ int held[PAGED ? 2 : 1][PAGED ? SL : 1];
  __shared__ int spoilt;  // some value of a node was not finite
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lm = lane & 15, lk = lane >> 4;
  const int share = blockIdx.x % shares, rest = blockIdx.x / shares;
  const int kvh = rest % a.kv_heads, z = rest / a.kv_heads, b = z / tiles, tile = z % tiles;
  const TreeSeq sq = tree_seq(a.tree, b);
  const int group = a.heads / a.kv_heads;
  if (tile * ROWS >= sq.nodes * group) return;
  const int words = (a.tree.max_nodes + 31) >> 5;
  const int kvw = a.kv_heads * D, crow = cache_row(a.form, kvw);
  const __half* kc = (const __half*)a.k_cache + (PAGED ? 0 : (int64_t)b * a.cache_stride);
  const __half* vc = (const __half*)a.v_cache + (PAGED ? 0 : (int64_t)b * a.cache_stride);
  const int32_t* index = PAGED ? a.kv_index + (int64_t)b * a.index_stride : nullptr;
  const int slices = (sq.count + SL - 1) / SL;

  // this lane's columns: rows past the sequence's repeat its last one (not written)
  const int first_row = tile * ROWS + wave * 16 * NC;
  const bool busy = first_row < sq.nodes * group;  // (uniform over the wave)
  int node[NC];
#pragma unroll
  for (int c = 0; c < NC; c++) node[c] = (first_row + 16 * c + lm) / group;
  auto row_of = [&](int c) __attribute__((always_inline)) {
    return (int64_t)(sq.t0 + min(node[c], sq.nodes - 1)) * a.heads + kvh * group + (first_row + 16 * c + lm) % group;
  };

  // staging: words tid + 256 j of a slice's keys, and of its values
  tu4 kw[PER], vw[PER];
  int cells[PAGED ? PER : 1], fcell = 0;  // the next slice's (negative: not held)
  tu4 fw = {0, 0, 0, 0};                  // q8_0: thread = (key or value, key) of the first 2 SL
  auto cell_at = [&](int j) __attribute__((always_inline)) { return index[min(j, sq.count - 1)]; };
  auto find = [&](int sl) __attribute__((always_inline)) {
    if constexpr (PAGED) {
#pragma unroll
      for (int j = 0; j < PER; j++) cells[j] = cell_at(sl * SL + (tid + 256 * j) / WPK);
      if (Q8) fcell = cell_at(sl * SL + tid % SL);
    }
  };
  // (the cells of the slice that is loaded: what is staged where nothing is held is zero)
  uint32_t dead = 0;
  auto load = [&](int sl) __attribute__((always_inline)) {
    dead = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int i = tid + 256 * j, key = i / WPK, pc = i % WPK, at = sl * SL + key;
      const int cell = PAGED ? cells[j] : min(at, sq.count - 1);
      if (at >= sq.count || (PAGED && cell < 0)) dead |= 1u << j;
      const int64_t off = (int64_t)(PAGED ? max(cell, 0) : cell) * crow + (Q8 ? (kvh * D + 16 * pc) / 2 : kvh * D + 8 * pc);
      kw[j] = *(const tu4*)(kc + off);
      vw[j] = *(const tu4*)(vc + off);
    }
    if constexpr (Q8) {
      const int at = sl * SL + tid % SL, cell = PAGED ? fcell : min(at, sq.count - 1);
      if (at >= sq.count || (PAGED && cell < 0)) dead |= 1u << 31;
      if (tid < 2 * SL) {
        const __half* f = (tid < SL ? kc : vc) + (int64_t)(PAGED ? max(cell, 0) : cell) * crow + (kvw >> 1) + ((kvh * D) >> 5);
        if constexpr (KS == 2) fw.x = *(const uint32_t*)f;
        else if constexpr (KS == 4) { fw.x = ((const uint2*)f)->x; fw.y = ((const uint2*)f)->y; }
        else fw = *(const tu4*)f;
      }
    }
  };
  auto store = [&](int sl, int buf) __attribute__((always_inline)) {
    const bool nodes_in = (sl + 1) * SL > sq.len;  // (uniform)
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int i = tid + 256 * j, key = i / WPK, pc = i % WPK;
      tu4 v = vw[j];
      if ((dead >> j) & 1) v = tu4{0, 0, 0, 0};
      if constexpr (Q8) {
        *(th8*)(ks[buf] + key * D + 8 * ((2 * pc) ^ key_swz<D>(key))) = int8_halves(kw[j].x, kw[j].y);
        *(th8*)(ks[buf] + key * D + 8 * ((2 * pc + 1) ^ key_swz<D>(key))) = int8_halves(kw[j].z, kw[j].w);
        *(th8*)(vs[buf] + key * D + 8 * ((2 * pc) ^ val_swz<D>(key))) = int8_halves(v.x, v.y);
        *(th8*)(vs[buf] + key * D + 8 * ((2 * pc + 1) ^ val_swz<D>(key))) = int8_halves(v.z, v.w);
      } else {
        if (nodes_in && sl * SL + key >= sq.len) {
          const tu4 f = {finite_halves(v.x), finite_halves(v.y), finite_halves(v.z), finite_halves(v.w)};
          if ((f.x ^ v.x) | (f.y ^ v.y) | (f.z ^ v.z) | (f.w ^ v.w)) spoilt = 1;
          v = f;
        }
        *(tu4*)(ks[buf] + key * D + 8 * (pc ^ key_swz<D>(key))) = kw[j];
        *(tu4*)(vs[buf] + key * D + 8 * (pc ^ val_swz<D>(key))) = v;
      }
      if (PAGED && pc == 0) held[buf][key] = !((dead >> j) & 1);
    }
    if constexpr (Q8) {
      if (tid < 2 * SL) {
        const uint32_t w[4] = {fw.x, fw.y, fw.z, fw.w};
#pragma unroll
        for (int u = 0; u < KS; u++)
          fac[buf][tid / SL][u][tid % SL] = dead >> 31 ? 0.0f : half_bits_to_float(w[u >> 1] >> (16 * (u & 1)));
      }
    }
  };

  if (tid == 0) spoilt = 0;
  int sl = share;
  if (sl < slices) {
    find(sl);
    load(sl);
    if (sl + shares < slices) find(sl + shares);
  }
  __builtin_amdgcn_sched_barrier(0);

  // the queries as B fragments, each scaled by a power of two that c2 takes back
  th8 qf[2][NC][KS];
  float c2[NC];
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const float* qr = a.q + (int64_t)(sq.t0 + min(node[c], sq.nodes - 1)) * a.q_stride +
                      (int64_t)(kvh * group + (first_row + 16 * c + lm) % group) * D + 8 * lk;
    tf4 raw[KS][2];
    float mx = 0.0f;
#pragma unroll
    for (int u = 0; u < KS; u++)
#pragma unroll
      for (int w = 0; w < 2; w++) {
        raw[u][w] = *(const tf4*)(qr + 32 * u + 4 * w);
#pragma unroll
        for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(raw[u][w][e]));
      }
    mx = across(mx, lanes::Max{});
    const int e2 = mx > 0.0f ? max(__builtin_amdgcn_frexp_expf(mx) - 15, -126) : 0;
    c2[c] = ldexpf(fabsf(a.scale) * kLog2e, e2);
    const float sc = ldexpf(a.scale < 0.0f ? -1.0f : 1.0f, -e2);
#pragma unroll
    for (int u = 0; u < KS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float f = raw[u][e >> 2][e & 3] * sc;
        const _Float16 h = (_Float16)f;
        qf[0][c][u][e] = h;
        qf[1][c][u][e] = (_Float16)fmaf((float)h, -1.0f, f);
      }
  }

  tf4 o[NC][NT];
  float mc[NC], l[NC];  // running maximum (of the scores, before c2) and this lane's part of the sum
  int xo[NC][Q8 ? KS : 1];  // q8_0: the X that a 32-dim block of o is held at
#pragma unroll
  for (int c = 0; c < NC; c++) {
    mc[c] = -1e30f;
    l[c] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < NT; dt++) o[c][dt] = tf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < (Q8 ? KS : 1); u++) xo[c][u] = -100;
  }

  // lane addresses in bytes: a piece's slot is an exclusive or with bits that a
  // row's start leaves free
  typedef __attribute__((address_space(3))) const char* lds_ptr;
  typedef __attribute__((address_space(3))) const th8* lds_h8;
  const uint32_t kat = 2 * lm * D + 16 * (lk ^ key_swz<D>(lm));
  uint32_t vat[2];
#pragma unroll
  for (int v = 0; v < 2; v++) {
    const int row = 4 * lk + (lm >> 2) + 16 * v;
    vat[v] = 2 * row * D + 16 * (((lm & 3) >> 1) ^ val_swz<D>(row)) + 8 * (lm & 1);
  }

  // 32 keys of slice sl
  auto step = [&](int kt, int buf) __attribute__((always_inline)) {
    const int base = sl * SL + 32 * kt;
    const lds_ptr kp = (lds_ptr)&ks[buf][32 * kt * D], vp = (lds_ptr)&vs[buf][32 * kt * D];
    tf4 s[NC][2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int c = 0; c < NC; c++) s[c][h] = tf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < KS; u++) {
        const th8 k8 = *(lds_h8)(kp + ((kat + 2 * 16 * h * D) ^ (64 * u)));
        if constexpr (Q8) {
          const tf4 f = *(const tf4*)&fac[buf][0][u][32 * kt + 16 * h + 4 * lk];
#pragma unroll
          for (int c = 0; c < NC; c++) {
            const tf4 d = mfma16(k8, qf[1][c][u], mfma16(k8, qf[0][c][u], tf4{0.0f, 0.0f, 0.0f, 0.0f}));
#pragma unroll
            for (int i = 0; i < 4; i++) s[c][h][i] = fmaf(f[i], d[i], s[c][h][i]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < NC; c++) s[c][h] = mfma16(k8, qf[1][c][u], mfma16(k8, qf[0][c][u], s[c][h]));
        }
      }
    }
    uint32_t there = 0xffffffffu;
    if constexpr (PAGED) there = (uint32_t)__ballot(held[buf][32 * kt + (lane & 31)] != 0);
    const bool all = base + 32 <= sq.len && there == 0xffffffffu;  // (uniform)
    th8 ph[NC], pl[NC];
    float p[NC][8];
    bool rose[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
      uint32_t mine = 0xffu;
      if (!all) {
        const uint32_t* mrow = a.tree.mask + (int64_t)(sq.t0 + min(node[c], sq.nodes - 1)) * words;
        mine = (seen_bits(mrow, words, base - sq.len, sq.count - sq.len) & there) >> (4 * lk);
#pragma unroll
        for (int i = 0; i < 8; i++)
          s[c][i >> 2][i & 3] = (mine >> ((i & 3) + 16 * (i >> 2))) & 1 ? s[c][i >> 2][i & 3] : -INFINITY;
      }
      float m = s[c][0][0];
#pragma unroll
      for (int i = 1; i < 8; i++) m = fmaxf(m, s[c][i >> 2][i & 3]);
      m = across(m, lanes::Max{});
      const float mn = fmaxf(mc[c], m);
      rose[c] = mn != mc[c];
      if (__any(rose[c] && l[c] != 0.0f)) {  // (else there is nothing yet)
        const float f = __builtin_amdgcn_exp2f((mc[c] - mn) * c2[c]);
        l[c] *= f;
#pragma unroll
        for (int dt = 0; dt < NT; dt++) o[c][dt] *= f;
      }
      mc[c] = mn;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        // (the difference first: c2 mc of large scores is rounded by more than 1)
        const float e = __builtin_amdgcn_exp2f((s[c][i >> 2][i & 3] - mn) * c2[c]);
        p[c][i] = all || (mine >> ((i & 3) + 16 * (i >> 2))) & 1 ? e : -0.0f;
        l[c] += p[c][i];
      }
      if constexpr (!Q8) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          ph[c][i] = (_Float16)fmaf(p[c][i], kLift, 0.0f);  // (one instruction)
          pl[c][i] = (_Float16)fmaf(p[c][i], kLift, -(float)ph[c][i]);
        }
      }
    }
#pragma unroll
    for (int dt = 0; dt < NT; dt++) {
      if constexpr (Q8) {
        if (dt % 2 == 0) {
          const int u = dt / 2;
          const tf4 f0 = *(const tf4*)&fac[buf][1][u][32 * kt + 4 * lk], f1 = *(const tf4*)&fac[buf][1][u][32 * kt + 16 + 4 * lk];
#pragma unroll
          for (int c = 0; c < NC; c++) {
            float w[8], wm = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              // (-0: not seen, whatever its factor)
              w[i] = __float_as_uint(p[c][i]) != 0x80000000u ? p[c][i] * (i < 4 ? f0[i & 3] : f1[i & 3]) : 0.0f;
              wm = fmaxf(wm, fabsf(w[i]));
            }
            wm = across(wm, lanes::Max{});
            const int old = xo[c][u];
            // (an infinite factor: the finite products are below 2^31)
            const int xw = wm < INFINITY ? __builtin_amdgcn_frexp_expf(wm) : 31;
            const int x = wm > 0.0f ? max(max(xw, rose[c] ? old - 60 : old), -100) : old;
            if (__any(x != old)) {
              const float f = ldexpf(1.0f, old - x);
              o[c][dt] *= f;
              o[c][dt + 1] *= f;
            }
            xo[c][u] = x;
            const float unit = ldexpf(1.0f, 15 - x);
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float v = w[i] * unit;
              ph[c][i] = (_Float16)v;
              pl[c][i] = (_Float16)(v - (float)ph[c][i]);
            }
            if (__builtin_expect(__any(!(wm < INFINITY)), 0)) {
#pragma unroll
              for (int i = 0; i < 8; i++)
                if (!(fabsf(w[i]) < INFINITY)) pl[c][i] = 0;
            }
          }
        }
      }
      ts8 v;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        const ts4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ts4*)(vp + (vat[w] ^ (32 * dt))));
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * w + e] = x[e];
      }
#pragma unroll
      for (int c = 0; c < NC; c++)
        o[c][dt] = mfma16(__builtin_bit_cast(th8, v), pl[c], mfma16(__builtin_bit_cast(th8, v), ph[c], o[c][dt]));
    }
  };

  __syncthreads();  // (spoilt)
  if (sl < slices) store(sl, 0);
  __syncthreads();
  for (int buf = 0; sl < slices; sl += shares, buf ^= 1) {
    const int next = sl + shares;
    const bool more = next < slices;  // (uniform)
    if (more) {
      load(next);
      if (next + shares < slices) find(next + shares);
    }
    if (busy) {
#pragma unroll
      for (int kt = 0; kt < SL / 32; kt++)
        if (sl * SL + 32 * kt < sq.count) step(kt, buf);
    }
    if (more) store(next, buf ^ 1);
    __syncthreads();
  }

  if (!Q8 && __builtin_expect(spoilt, 0) && busy) {
    for (int s0 = share; s0 < slices; s0 += shares) {
      for (int j = max(s0 * SL, sq.len); j < min((s0 + 1) * SL, sq.count); j++) {
        const int cell = PAGED ? index[j] : j;
        if (cell < 0) continue;
        const __half* vr = vc + (int64_t)cell * crow + kvh * D + 4 * lk;
        const int i = j - sq.len;
#pragma unroll
        for (int c = 0; c < NC; c++) {
          const uint32_t* mrow = a.tree.mask + (int64_t)(sq.t0 + min(node[c], sq.nodes - 1)) * words;
          const bool sees = (mrow[i >> 5] >> (i & 31)) & 1;
#pragma unroll
          for (int dt = 0; dt < NT; dt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float v = __half2float(vr[16 * dt + e]);
              if (sees && !(fabsf(v) < INFINITY)) o[c][dt][e] += v;
            }
        }
      }
    }
  }
  if (!busy) return;
#pragma unroll
  for (int c = 0; c < NC; c++) {
    const float sum = across(l[c], lanes::Add{});
    if (node[c] >= sq.nodes) continue;
    const int64_t row = row_of(c);
    const float w = (shares > 1 ? 1.0f : sum != 0.0f ? 1.0f / sum : 0.0f) * (Q8 ? 1.0f : 1.0f / kLift);
    float* dst = shares > 1 ? part_acc + (row * shares + share) * D : a.out + row * D;
#pragma unroll
    for (int dt = 0; dt < NT; dt++) {
      const float f = Q8 ? w * ldexpf(1.0f, xo[c][dt / 2] - 15) : w;
      *(tf4*)(dst + 16 * dt + 4 * lk) = o[c][dt] * f;
    }
    if (shares > 1 && lk == 0)
      *(float2*)(part_ml + 2 * (row * shares + share)) = make_float2(sum != 0.0f ? mc[c] * c2[c] : -INFINITY, sum);
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
  bool mfma;
  int columns;  // NC of attend_tree_kernel
  int tiles, shares;
  int64_t blocks;
};

TreeGrid tree_grid(int heads, int kv_heads, int head_dim, const mi_tree& t) {
  TreeGrid g;
  const int group = heads / kv_heads;
  g.mfma = head_dim == 64 || head_dim == 128 || head_dim == 256;
  g.columns = head_dim <= 128 && t.max_nodes * group > 64 ? 2 : 1;
  const int rows = g.mfma ? 64 * g.columns : kRowsTile, slice = g.mfma ? mfma_slice(head_dim) : rows_slice(head_dim);
  g.tiles = (t.max_nodes * group + rows - 1) / rows;
  const int64_t pairs = (int64_t)t.batch * g.tiles * kv_heads, slices = ((int64_t)t.max_count + slice - 1) / slice;
  const int64_t room = (g.mfma ? 2 : 4) * (int64_t)cu_count();
  g.shares = 1;
  int64_t least = INT64_MAX;
  for (int n = 1; n <= std::min<int64_t>(slices, 64); n++) {
    const int64_t cost = 16 * ((n * pairs + room - 1) / room) * ((slices + n - 1) / n + 2) + n;
    if (cost < least) g.shares = n, least = cost;
  }
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
  const dim3 grid((uint32_t)g.blocks);
#define MI_TREE(D, NC, Q, P)                                                                                       \
  hipLaunchKernelGGL((attend_tree_kernel<D, NC, Q, P>), grid, dim3(256), 0, s, a, g.tiles, g.shares, part_acc, part_ml)
#define MI_TREE_F(D, NC)                            \
  if (a.form == MI_CACHE_Q8) {                      \
    if (a.kv_index) MI_TREE(D, NC, true, true);     \
    else MI_TREE(D, NC, true, false);               \
  } else {                                          \
    if (a.kv_index) MI_TREE(D, NC, false, true);    \
    else MI_TREE(D, NC, false, false);              \
  }
#define MI_TREE_ROWS(ND)                                                                                             \
  if (a.form == MI_CACHE_Q8)                                                                                         \
    hipLaunchKernelGGL((attend_tree_rows_kernel<true, ND>), grid, dim3(kRowsThreads), rows_lds_bytes(a.head_dim), s,  \
                       a, g.tiles, g.shares, part_acc, part_ml);                                                     \
  else                                                                                                               \
    hipLaunchKernelGGL((attend_tree_rows_kernel<false, ND>), grid, dim3(kRowsThreads), rows_lds_bytes(a.head_dim), s, \
                       a, g.tiles, g.shares, part_acc, part_ml)
  if (a.head_dim == 64) {
    if (g.columns == 1) { MI_TREE_F(64, 1) }
    else { MI_TREE_F(64, 2) }
  } else if (a.head_dim == 128) {
    if (g.columns == 1) { MI_TREE_F(128, 1) }
    else { MI_TREE_F(128, 2) }
  } else if (a.head_dim == 256) {
    MI_TREE_F(256, 1)
  } else if (a.head_dim < 64) {
    MI_TREE_ROWS(1);
  } else if (a.head_dim < 128) {
    MI_TREE_ROWS(2);
  } else if (a.head_dim < 256) {
    MI_TREE_ROWS(4);
  } else {
    MI_TREE_ROWS(8);
  }
#undef MI_TREE
#undef MI_TREE_F
#undef MI_TREE_ROWS
  if (int rc = hip_check(hipGetLastError(), "attend_tree launch")) return rc;
  if (g.mfma && g.shares == 1) return MI_OK;  // (the finished rows)
  const int64_t threads = (int64_t)a.tree.tokens * a.heads * (a.head_dim / 4), blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return fail(MI_ERR_SHAPE, "attend_tree: %d tokens of %d heads", a.tree.tokens, a.heads);
  hipLaunchKernelGGL(attend_tree_fold_kernel, dim3((uint32_t)blocks), dim3(256), 0, s, part_acc, part_ml, a.tree,
                     a.heads, a.head_dim, g.shares, a.out);
  return hip_check(hipGetLastError(), "attend_tree fold launch");
}

}  // namespace mi
