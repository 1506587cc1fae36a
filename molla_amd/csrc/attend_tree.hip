// attend_tree.hip -- attention of trees of drafted tokens over a cache
// (mi_attend_tree), gfx950: attention.mojo:144 attend for several tokens of each
// of several sequences, every token over the sequence's committed positions and
// the nodes of its own tree that its mask has, over an f16 or a q8_0 cache, GQA.
//
// The work is a line of units, one for each (sequence, key head, tile of query
// rows, slice of keys), slices innermost; a query row is a token and a query head
// of the key head.  Lengths are device values, so the blocks share the line among
// themselves: each scans the sequences and takes an equal run of units, walking
// its slices with a running maximum and sum.  Of the tiles in a run only the first
// and the last can be another block's too: those leave partial results, two a
// block, that a second launch folds; the others' rows are finished.  (With as many
// parts for every tile as the longest sequence needs, the fold of 13 nodes over
// 32768 positions took 46 us, that of 8 over 2048 14; so 5.6 and 4.1.)
//
// Measured, products + fold under the profiler, heads 32 over 8 (over 4 at width 64):
// 8 sequences of up to 64 nodes over 8192 down to 4608 positions at width 128 122 to
// 147 + 8.7 us, the whole call among others 119 (324 TFLOP/s of the formula's products,
// twice that of the matrix cores', whose steps take turns with the softmax on the VALU
// at two waves a SIMD); 8 x 48 over 3000 down to 1691 at width 64 29 + 5.5 (bound by a
// step's chain of latencies at three waves a SIMD); 1 x 13 over 32768 36.3 + 5.6 (3.7
// TB/s; 6 once the first slices are there); 4 x 25 over 4099 of q8_0 40.5 + 5.4 (a
// barrier and a chain of latencies every 32 keys at two waves a SIMD: the VALU issues
// for about 15 us of it, the matrix cores are busy for 11 %); 1 x 8 over 2048 11.5 + 4.2
// (launches and the first loads' latency).  The kernel for the other widths has its
// products on the VALU: at width 160 8 x 64 3480 + 18 us, 1 x 13 773 + 6, 4 x 25 459 + 8
// (q8_0 452); at width 96 with 16 over 4 heads 8 x 64 1127 + 9 (at width 128 70 + 8).
#include <math.h>

#include <algorithm>

#include "mi_internal.h"

namespace mi {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxParts = 128;  // blocks that share a tile: two for a lane of the fold

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

__device__ __forceinline__ int tree_tiles(const TreeSeq& s, int shift, int rows) {
  return ((s.nodes << shift) + rows - 1) / rows;
}
__device__ __forceinline__ int tree_slices(const TreeSeq& s, int slice) { return (s.count + slice - 1) / slice; }
// A tile's units: its slices behind kStart that stand for the start of a run in it
// (queries, first loads), so that a block with two starts gets less of the rest.  us at
// 0, 3 and 6: 1 x 8 over 2048 13.8, 11.2, 11.4; 1 x 13 over 5000 17.2, 14.4, 14.6, over
// 32768 38.7, 36.0, 36.1, at width 64 23.7, 23.1, 23.2; 4 x 25 over 4099 34.0, 29.7,
// 29.0, of q8_0 43.5, 40.4, 43.1; 8 x 48 over 12000 at width 64 86.6, 81.1, 83.6; 64 x 1
// over 4096 of q8_0 174, 172, 180; no difference for 8 x 48 over 3000, 64 x 1 of f16 and
// 8 x 8 over 16384 of q8_0.
constexpr int kStart = 3;
__device__ __forceinline__ int tree_units(const TreeSeq& s, int slice) { return kStart + tree_slices(s, slice); }

struct IMax {
  __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};
// the sum over lanes 0 .. this one
__device__ __forceinline__ int lane_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // lane 15 of rows 0 and 2 to the row behind
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
  return v;
}

// Hands this block's units to `take`, a tile's run of slices at a time:
// take(sequence, b, key head, tile, first slice, end, part), part -1 where the
// run is the whole tile, else the block's part it goes to.  Every wave finds them
// for itself, 64 sequences at a time in its lanes.  plan: units a block, then each
// sequence's first unit (written by the first wave, for the fold).
template <class F>
__device__ __forceinline__ void tree_walk(const TreeAttend& a, int rows, int slice, int32_t* __restrict__ plan,
                                          F take) {
  const int lane = threadIdx.x & 63, shift = a.group_shift, batch = a.tree.batch;
  TreeSeq sq;
  int units;
  auto look = [&](int b0) __attribute__((always_inline)) {
    const int b = b0 + lane;
    sq = tree_seq(a.tree, min(b, batch - 1));
    if (b >= batch || sq.nodes == 0) sq.count = 0;
    units = sq.count ? tree_tiles(sq, shift, rows) * a.kv_heads * tree_units(sq, slice) : 0;
  };
  int total = 0, top = 0, upto = 0;  // upto: of the lanes up to this one
  for (int b0 = 0; b0 < batch; b0 += 64) {
    look(b0);
    upto = lane_scan(units);
    total += __builtin_amdgcn_readlane(upto, 63);
    top = max(top, lanes::reduce<64>(sq.count ? tree_units(sq, slice) : 0, IMax{}));
  }
  top = __builtin_amdgcn_readfirstlane(top);  // (the same in every lane)
  const uint32_t blocks = gridDim.x;
  const int per = max(max((int)(((uint32_t)total + blocks - 1) / blocks), (top + kMaxParts - 3) / (kMaxParts - 2)), 1);
  // blocks go to the 8 XCDs in turn: neighbours in the line, which are one
  // sequence's tiles over the same keys, to the same L2
  const int xcd = blockIdx.x & 7, in = blockIdx.x >> 3, many = blocks >> 3, rest = blocks & 7;
  const int block = xcd * many + min(xcd, rest) + in;
  const int64_t first = (int64_t)block * per;
  const bool writes = blockIdx.x == 0 && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == 0;
  if (writes && lane == 0) plan[0] = per;
  int b = -1, at = 0, chunk = 0;
  for (int b0 = 0, ahead = 0; b0 < batch && (b < 0 || writes); b0 += 64) {
    if (batch > 64) {
      look(b0);
      upto = ahead + lane_scan(units);
    }
    if (writes && b0 + lane < batch) plan[1 + b0 + lane] = upto - units;
    const uint64_t hit = __ballot(first >= upto - units && first < upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      b = b0 + l;
      at = (int)first - __builtin_amdgcn_readlane(upto - units, l);
      chunk = b0;
    }
    ahead = __builtin_amdgcn_readlane(upto, 63);
  }
  if (b < 0) return;  // (no units left for this block)
  b = __builtin_amdgcn_readfirstlane(b);  // (the same in every lane)
  at = __builtin_amdgcn_readfirstlane(at);
  if (batch > 64) look(chunk);
  TreeSeq s;
  s.t0 = __builtin_amdgcn_readlane(sq.t0, b - chunk);
  s.nodes = __builtin_amdgcn_readlane(sq.nodes, b - chunk);
  s.len = __builtin_amdgcn_readlane(sq.len, b - chunk);
  s.count = __builtin_amdgcn_readlane(sq.count, b - chunk);
  int left = (int)min<int64_t>(per, total - first);
  while (true) {
    const int run = tree_units(s, slice), tiles = tree_tiles(s, shift, rows);
    while (at < run * tiles * a.kv_heads) {
      const int pair = (uint32_t)at / (uint32_t)run, u = at - pair * run, n = min(run - u, left);
      const int head = tiles == 1 ? pair : (uint32_t)pair / (uint32_t)tiles;
      const int s0 = max(u - kStart, 0), s1 = u + n - kStart;
      const int part = u <= kStart && u + n == run ? -1 : 2 * block + (u <= kStart ? 1 : 0);
      if (s0 < s1) take(s, b, head, pair - head * tiles, s0, s1, part);
      left -= n;
      if (left == 0) return;
      at += n;
    }
    at = 0;
    s = tree_seq(a.tree, ++b);
  }
}

// Where part `part` of a tile's row keeps its sum, and behind all of them its
// (maximum in base 2, sum).
struct TreeParts {
  float* acc;
  float* ml;
};

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
__global__ __launch_bounds__(kRowsThreads) void attend_tree_rows_kernel(TreeAttend a, TreeParts parts,
                                                                        int32_t* __restrict__ plan) {
  extern __shared__ float4 lds[];
  const int D = a.head_dim, kk = rows_slice(D), KS = D + 4;
  const int words = (a.tree.max_nodes + 31) >> 5, shift = a.group_shift, group = 1 << shift;
  float* Ks = (float*)lds;
  float* Vs = Ks + kk * KS;
  float* Qs = Vs + kk * D;
  float* Ps = Qs + kRowsTile * D;  // [wave][key][its 4 rows]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kvw = a.kv_heads * D, crow = cache_row(a.form, kvw);
  const float c2 = a.scale * kLog2e;
  const int split = 64 / kk, part_d = lane / kk, key = lane % kk;

  tree_walk(a, kRowsTile, kk, plan, [&](const TreeSeq& sq, int b, int kvh, int tile, int s0, int s1, int part) {
    const __half* kc = (const __half*)a.k_cache + (a.kv_index ? 0 : (int64_t)b * a.cache_stride);
    const __half* vc = (const __half*)a.v_cache + (a.kv_index ? 0 : (int64_t)b * a.cache_stride);
    const int32_t* index = a.kv_index ? a.kv_index + (int64_t)b * a.index_stride : nullptr;
    // queries; rows past the sequence repeat its last token (not written)
    __syncthreads();
    for (int i = tid; i < kRowsTile * D; i += kRowsThreads) {
      const int r = tile * kRowsTile + i / D, e = i % D, node = min(r >> shift, sq.nodes - 1);
      Qs[i] = a.q[(int64_t)(sq.t0 + node) * a.q_stride + (int64_t)(kvh * group + (r & (group - 1))) * D + e];
    }
    const int r0 = 4 * wave;
    const uint32_t* mrow[4];
    float m2[4], l[4], o[4][ND];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      mrow[r] = a.tree.mask + (int64_t)(sq.t0 + min((tile * kRowsTile + r0 + r) >> shift, sq.nodes - 1)) * words;
      m2[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < ND; i++) o[r][i] = 0.0f;
    }
    for (int sl = s0; sl < s1; sl++) {
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
      for (int e = 4 * part_d; e < D; e += 4 * split) {
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
      if (part_d == 0) *(float4*)(pw + 4 * key) = make_float4(p[0], p[1], p[2], p[3]);
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
      const int row = tile * kRowsTile + r0 + r;
      if (row >> shift >= sq.nodes) continue;
      const int64_t slot = (int64_t)part * kRowsTile + r0 + r;
      float* dst = part < 0 ? a.out + ((int64_t)(sq.t0 + (row >> shift)) * a.heads + kvh * group + (row & (group - 1))) * D
                            : parts.acc + slot * D;
      const float w = part >= 0 ? 1.0f : l[r] != 0.0f ? 1.0f / l[r] : 0.0f;
#pragma unroll
      for (int i = 0; i < ND; i++)
        if (lane + 64 * i < D) dst[lane + 64 * i] = o[r][i] * w;
      if (part >= 0 && lane == 0) *(float2*)(parts.ml + 2 * slot) = make_float2(m2[r], l[r]);
    }
  });
}

// ---- head widths 64, 128 and 256: the products on the matrix cores -----------
// v_mfma_f32_16x16x32_f16.  A block is 64 NC / KW query rows, 16 NC to a wave, and
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
//   to 2^-24), down to 2^-39 of the largest.  Weights enter as two halves as well:
//   to 2^-23 of themselves, down to 2^-35 of the largest.
//
//   A weight is 2^(s c2 - mk), mk = a maximum times c2 less 10, rounded once and then
//   taken as it is, so that the rounding is the same in every weight of a row and
//   falls out of its quotient, as the 10 does (where mk is so large that it could
//   reach a weight's own size, the difference is taken before the product).  The
//   exponent's own rounding, at most 2^-21, is a weight's 3.3e-7.  mk follows the
//   running maximum where that would make a weight above 2^14: a half holds 2^16, and
//   with the slack most slices leave the sums as they are (8 x 64 129 -> 126 us at
//   best, 8 x 48 at width 64 29.8 -> 29.4).
//
// q8_0: keys and values enter as their integers, exact halves; a key block's
// factor multiplies its part of the score, a value block's the weights, which
// are then split into halves (the factors' share of 4 x 25 over 4099: 40 us against
// 30 of f16; at D = 256 115 against 47, where they do not fit the registers).  The
// factors are staged times 2^(11 - X), X the exponent of the largest one so far
// among committed positions, which every row sees (a weight's lower half ends at
// 2^-24: with X held at 0 or above, values near 4e-6 whose weights are 2^-12 of the
// largest came out 6e-3 of their size off; so 3.6e-7).  In 32 keys that some row does not
// see whole each row's products are scaled to its own largest and summed apart: what
// a row does not see has no part in its result.
//
// A value that is not finite in a node that some query does not see would give
// 0 * inf there: such values are staged as zeros and added at the end to the
// queries that see them, as are those of committed positions.
//
// MFMA fragments (16x16x32): lane l holds row / column l % 16 and values
// 8 (l / 16) .. +8 of the 32; result element i of lane l is row 4 (l / 16) + i,
// column l % 16.
typedef _Float16 th2 __attribute__((ext_vector_type(2)));
typedef _Float16 th8 __attribute__((ext_vector_type(8)));
typedef short ts4 __attribute__((ext_vector_type(4)));
typedef short ts8 __attribute__((ext_vector_type(8)));
typedef float tf2 __attribute__((ext_vector_type(2)));
typedef float tf4 __attribute__((ext_vector_type(4)));
typedef uint32_t tu4 __attribute__((ext_vector_type(4)));

constexpr float kLift = 10.0f, kSlack = 4.0f;   // of a weight's exponent: its sum 14 at most
constexpr int kFactor = 15 - (int)kSlack;       // q8_0: the largest factor's, for weights up to 2^kSlack
constexpr int kNoFactor = -24;                  // X ahead of the first factor, which is 2^-24 (X = -23) or more

// w f as two halves (ONE: f is 1, in a scalar register that the compiler takes for
// any value): an instruction each or less, the higher halves opaque so that the
// lower ones are taken from them where they lie in their pair
template <bool ONE, class F>
__device__ __forceinline__ void split(const float (&w)[8], F f, th8& hi, th8& lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    th2 h;
    if constexpr (ONE) h = __builtin_convertvector((tf2{w[i], w[i + 1]}), th2);
    else h = th2{(_Float16)fmaf(w[i], f(i), 0.0f), (_Float16)fmaf(w[i + 1], f(i + 1), 0.0f)};
    asm("" : "+v"(h));
    const th2 l = {(_Float16)fmaf(w[i], f(i), -(float)h[0]), (_Float16)fmaf(w[i + 1], f(i + 1), -(float)h[1])};
    hi[i] = h[0];
    hi[i + 1] = h[1];
    lo[i] = l[0];
    lo[i + 1] = l[1];
  }
}

__device__ __forceinline__ tf4 mfma16(th8 a, th8 b, tf4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// LDS rows are padded, so that the lanes served together fall on distinct banks
// and every fragment is at a fixed distance from a lane's first: keys (16 rows,
// one 16-byte piece of each) by 16 bytes, values (read transposed, 4 rows x 32
// bytes per 16 lanes) by 32.  (Pieces permuted by an exclusive or, as in
// attend_flash.hip, cost an instruction and a register for each.)
__host__ __device__ constexpr int key_row(int D) { return D + 8; }   // halves
__host__ __device__ constexpr int val_row(int D) { return D + 16; }

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

// Sizes by head width: keys of a slice (32 at D = 128 and 256, where the words of 64
// on their way cost the registers of a second block's wave: 8 x 64 at D = 128 209
// us, so 165 at the time; 64 at D = 64), and blocks a compute unit (one more at D =
// 128: q8_0 62 us against 43 for the registers, f16 no faster and 1 us more to fold;
// at D = 64: no faster).
__host__ __device__ constexpr int mfma_slice(int D) { return D == 64 ? 64 : 32; }
__host__ __device__ constexpr int mfma_blocks(int D) { return D == 64 ? 3 : 2; }

template <int D, int NC, bool Q8, bool PAGED, int KW = 1>
__global__ __launch_bounds__(256, mfma_blocks(D)) void attend_tree_kernel(TreeAttend a, TreeParts parts,
                                                                              int32_t* __restrict__ plan) {
  constexpr int SL = KW == 2 ? 64 : mfma_slice(D), KS = D / 32, NT = D / 16, PIECES = D / 8;
  constexpr int PER = Q8 ? (SL * D / 16 + 255) / 256 : SL * PIECES / 256;  // 16-byte words of K (and of V) a thread
  constexpr int WPK = Q8 ? D / 16 : PIECES;                               // words a key
  constexpr int ROWS = 64 * NC / KW;
  constexpr int VG = 2;  // 16-dim tiles of values a group of reads
  constexpr int FPER = 2 * SL * KS / 256;                                 // q8_0 factors of K and V a thread
  static_assert(PER * 256 == SL * WPK && FPER * 256 == 2 * SL * KS, "a slice's words dealt evenly");
  constexpr int KR = key_row(D), VR = val_row(D);
  __shared__ __align__(16) _Float16 ks[2][SL * KR];
  __shared__ __align__(16) _Float16 vs[2][SL * VR];
  __shared__ __align__(16) float fac[Q8 ? 2 : 1][2][Q8 ? KS : 1][Q8 ? SL : 1];  // q8_0 factors of keys and values
  __shared__ __align__(16) int xs[Q8 ? 2 : 1][Q8 ? KS : 1];                                 // X that the values' factors are at
  __shared__ int holes[2];  // the step whose slice in this buffer has a cell that is not held
  __shared__ int spoilt[2]; // the last (even, odd) run in which some staged value was not finite
  const int tid = threadIdx.x, lane = tid & 63, wave_all = __builtin_amdgcn_readfirstlane(tid >> 6);
  // KW = 2 (few rows): waves 2 and 3 have the rows of 0 and 1, and each slice's other
  // 32 keys
  const int wave = wave_all % (4 / KW), half = wave_all / (4 / KW);
  const int lm = lane & 15, lk = lane >> 4;
  const int shift = a.group_shift, group = 1 << shift, words = (a.tree.max_nodes + 31) >> 5;
  const int kvw = a.kv_heads * D, crow = cache_row(a.form, kvw);
  if (tid == 0) holes[0] = holes[1] = spoilt[0] = spoilt[1] = 0;
  __syncthreads();
  int turn = 0, run = 0;  // slices that this block has staged, and runs that it has taken

  // a lane's place in a tile of 32 keys, in halves: key lm, values 8 lk .., and for
  // the transposed reads row 4 lk + lm / 4, dims 4 (lm % 4) ..
  const int kat = lm * KR + 8 * lk, vat = (4 * lk + (lm >> 2)) * VR + 4 * (lm & 3);

  tree_walk(a, ROWS, SL, plan, [&](const TreeSeq& sq, int b, int kvh, int tile, int s0, int s1, int part) {
    const __half* kc = (const __half*)a.k_cache + (PAGED ? 0 : (int64_t)b * a.cache_stride) + (Q8 ? kvh * D / 2 : kvh * D);
    const __half* vc = (const __half*)a.v_cache + (PAGED ? 0 : (int64_t)b * a.cache_stride) + (Q8 ? kvh * D / 2 : kvh * D);
    const int32_t* index = PAGED ? a.kv_index + (int64_t)b * a.index_stride : nullptr;
    run++;
    const int first_turn = turn + 1;

    // this lane's columns: rows past the sequence's repeat its last one (not written)
    const int first_row = tile * ROWS + wave * 16 * NC;
    const bool busy = first_row < sq.nodes << shift;  // (uniform over the wave)
    int node[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) node[c] = (first_row + 16 * c + lm) >> shift;
    auto mask_row = [&](int c) __attribute__((always_inline)) {
      return a.tree.mask + (int64_t)(sq.t0 + min(node[c], sq.nodes - 1)) * words;
    };

    // staging: words tid + 256 j of a slice's keys, and of its values
    struct Stage {
      tu4 kw[PER], vw[PER];
      int cells[PAGED ? PER : 1], fcell[PAGED && Q8 ? FPER : 1];  // (negative: not held)
      uint16_t f[Q8 ? FPER : 1];  // q8_0: factors
      bool dead;                  // nothing is held where some word was loaded
    };
    Stage st;
    int xrun[Q8 ? FPER : 1];  // q8_0: the X so far of the blocks whose values' factors this thread stages
#pragma unroll
    for (int j = 0; j < (Q8 ? FPER : 1); j++) xrun[j] = kNoFactor;
    // q8_0: factor tid + 256 j of a slice: the keys' first, then the values', the keys of
    // a 32-dim block in SL lanes, whose largest X takes.  With KW = 2, where loads are
    // what a step waits for, the keys' with a key's blocks in neighbouring lanes, so that
    // their line is asked for once (182 -> 173 us; elsewhere the registers cost more)
    auto fkey = [&](int j) __attribute__((always_inline)) {
      const int i = tid + 256 * j;
      return KW == 2 && i < SL * KS ? i / KS : i % SL;
    };
    auto fblock = [&](int j) __attribute__((always_inline)) {
      const int i = tid + 256 * j;
      return KW == 2 && i < SL * KS ? i % KS : i / SL % KS;
    };
    auto cell_at = [&](int j) __attribute__((always_inline)) { return index[min(j, sq.count - 1)]; };
    auto find = [&](int sl, Stage& st) __attribute__((always_inline)) {
      if constexpr (PAGED) {
#pragma unroll
        for (int j = 0; j < PER; j++) st.cells[j] = cell_at(sl * SL + (tid + 256 * j) / WPK);
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < FPER; j++) st.fcell[j] = cell_at(sl * SL + fkey(j));
        }
      }
    };
    auto load = [&](int sl, Stage& st) __attribute__((always_inline)) {
      st.dead = false;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const int i = tid + 256 * j, at = sl * SL + i / WPK;
        int cell = PAGED ? st.cells[j] : min(at, sq.count - 1);
        // (opaque: an address formed ahead of the products would wait for its cell there)
        if (PAGED) asm volatile("" : "+v"(cell));
        st.dead |= PAGED && cell < 0;
        const int64_t off = (int64_t)(PAGED ? max(cell, 0) : cell) * crow + 8 * (i % WPK);
        st.kw[j] = *(const tu4*)(kc + off);
        st.vw[j] = *(const tu4*)(vc + off);
      }
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < FPER; j++) {
          const int i = tid + 256 * j, at = sl * SL + fkey(j);
          int cell = PAGED ? st.fcell[j] : min(at, sq.count - 1);
          if (PAGED) asm volatile("" : "+v"(cell));
          st.f[j] = *(const uint16_t*)((i < SL * KS ? kc : vc) + (int64_t)(PAGED ? max(cell, 0) : cell) * crow + (kvw >> 1) -
                                       kvh * D / 2 + ((kvh * D) >> 5) + fblock(j));
          if (at >= sq.count || (PAGED && cell < 0)) st.f[j] = 0;
        }
      }
    };
    auto store = [&](int sl, int buf, Stage& st) __attribute__((always_inline)) {
      turn++;
      const bool nodes_in = (sl + 1) * SL > sq.len;  // (uniform)
      if (PAGED && st.dead) holes[buf] = turn;
      // what is not held, and what some row may not see, must be finite: 0 * inf in
      // the products would reach every row
      if (!Q8 && (nodes_in || (PAGED && __any(st.dead)))) {
        bool bad = false;
#pragma unroll
        for (int j = 0; j < PER; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t f = finite_halves(st.vw[j][e]);
            bad |= f != st.vw[j][e];
            st.vw[j][e] = f;
          }
        if (bad) spoilt[run & 1] = run;
      }
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const int i = tid + 256 * j, key = i / WPK, pc = i % WPK;
        if constexpr (Q8) {
          *(th8*)(ks[buf] + key * KR + 16 * pc) = int8_halves(st.kw[j].x, st.kw[j].y);
          *(th8*)(ks[buf] + key * KR + 16 * pc + 8) = int8_halves(st.kw[j].z, st.kw[j].w);
          *(th8*)(vs[buf] + key * VR + 16 * pc) = int8_halves(st.vw[j].x, st.vw[j].y);
          *(th8*)(vs[buf] + key * VR + 16 * pc + 8) = int8_halves(st.vw[j].z, st.vw[j].w);
        } else {
          *(tu4*)(ks[buf] + key * KR + 8 * pc) = st.kw[j];
          *(tu4*)(vs[buf] + key * VR + 8 * pc) = st.vw[j];
        }
      }
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < FPER; j++) {
          const int i = tid + 256 * j, u = fblock(j);
          float f = half_bits_to_float(st.f[j]);
          if (i >= SL * KS) {  // (uniform: the second half of the threads, or of a thread's factors)
            const float af = fabsf(f);
            const float fm = lanes::reduce<SL>(sl * SL + fkey(j) < sq.len && af < INFINITY ? af : 0.0f, lanes::Max{});
            if (fm > 0.0f) xrun[j] = max(xrun[j], __builtin_amdgcn_frexp_expf(fm));
            f = ldexpf(f, kFactor - xrun[j]);
            if (i % SL == 0) xs[buf][u] = xrun[j];
          }
          fac[buf][i / (SL * KS)][u][fkey(j)] = f;
        }
      }
    };

    // the first two slices and the queries at once
    find(s0, st);
    Stage ahead;
    if (s0 + 1 < s1) find(s0 + 1, ahead);
    tf4 raw[NC][KS][2];
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const float* qr = a.q + (int64_t)(sq.t0 + min(node[c], sq.nodes - 1)) * a.q_stride +
                        (int64_t)(kvh * group + ((first_row + 16 * c + lm) & (group - 1))) * D + 8 * lk;
#pragma unroll
      for (int u = 0; u < KS; u++)
#pragma unroll
        for (int w = 0; w < 2; w++) raw[c][u][w] = *(const tf4*)(qr + 32 * u + 4 * w);
    }
    __builtin_amdgcn_sched_barrier(0);
    load(s0, st);
    if (s0 + 1 < s1) {
      load(s0 + 1, ahead);
      if (s0 + 2 < s1) find(s0 + 2, ahead);
    }
    __builtin_amdgcn_sched_barrier(0);

    // the queries as B fragments, each scaled by a power of two that c2 takes back
    th8 qf[2][NC][KS];
    float c2[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
      float mx = 0.0f;
#pragma unroll
      for (int u = 0; u < KS; u++)
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
          for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(raw[c][u][w][e]));
      mx = across(mx, lanes::Max{});
      const int e2 = mx > 0.0f ? max(__builtin_amdgcn_frexp_expf(mx) - 15, -126) : 0;
      c2[c] = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, e2), 1e-38f);  // (never zero: a key that is not seen scores -inf)
      const float sc = ldexpf(a.scale < 0.0f ? -1.0f : 1.0f, -e2);
#pragma unroll
      for (int u = 0; u < KS; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float f = raw[c][u][e >> 2][e & 3] * sc;
          const _Float16 h = (_Float16)f;
          qf[0][c][u][e] = h;
          qf[1][c][u][e] = (_Float16)fmaf((float)h, -1.0f, f);
        }
    }

    tf4 o[NC][NT];
    // running maximum (of the scores, before c2), the same times c2, and this lane's part of the sum
    float mc[NC], mk[NC], l[NC];
    int xo[Q8 ? KS : 1];  // q8_0: (uniform) the X that a 32-dim block of o is held at
#pragma unroll
    for (int c = 0; c < NC; c++) {
      mc[c] = -1e30f;
      mk[c] = -3e38f;
      l[c] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < NT; dt++) o[c][dt] = tf4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int u = 0; u < (Q8 ? KS : 1); u++) xo[u] = kNoFactor;
    // a row's mk is too large for a weight's exponent; (uniform) some row's is
    auto large = [&](int c) __attribute__((always_inline)) { return mc[c] > -1e30f && !(fabsf(mk[c]) <= 4e6f); };
    bool huge = false;
    constexpr float lift = Q8 ? 0.0f : kLift;
    float one = 1.0f;
    asm("" : "+s"(one));

    // the scores of keys 32 kt .. of a slice, and whether all its cells are held
    // and (q8_0) the X that its values' factors are at
    auto scores = [&](int sl, int kt, int buf, tf4 (&s)[NC][2], int& hole, int (&xv)[Q8 ? KS : 1]) __attribute__((always_inline)) {
      const _Float16* kp = &ks[buf][32 * kt * KR + kat];
      if (PAGED) hole = holes[buf];
      if constexpr (Q8) {
#pragma unroll
        for (int u = 0; u < KS; u++) xv[u] = xs[buf][u];
      }
      // key fragments of as many products as there are registers for on their way
      // before the first (one at a time, the compiler's order, left each product
      // waiting for LDS)
      if constexpr (Q8) {
        // a group: the products of 16 keys over up to four 32-dim blocks, each with
        // its keys' factors; the next group's fragments on their way (at D = 256 there
        // are no registers for them)
        constexpr int UG = KS < 4 ? KS : 4, G = 2 * KS / UG, AH = KS <= 4 ? 2 : 1;
        th8 k8[AH][UG];
        tf4 f[AH][UG];  // the factors of lane group lk's four keys
        auto read = [&](int g) __attribute__((always_inline)) {
          const int h = g * UG / KS, u0 = g * UG % KS;
#pragma unroll
          for (int u = 0; u < UG; u++) k8[g % AH][u] = *(const th8*)(kp + 16 * h * KR + 32 * (u0 + u));
#pragma unroll
          for (int u = 0; u < UG; u++) f[g % AH][u] = *(const tf4*)&fac[buf][0][u0 + u][32 * kt + 16 * h + 4 * lk];
        };
        if (AH == 2) read(0);
#pragma unroll
        for (int g = 0; g < G; g++) {
          const int h = g * UG / KS, u0 = g * UG % KS;
          if (g + AH - 1 < G) read(g + AH - 1);
          __builtin_amdgcn_sched_barrier(0);
          tf4 d[NC][UG];
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int u = 0; u < UG; u++)
#pragma unroll
              for (int c = 0; c < NC; c++)
                d[c][u] = mfma16(k8[g % AH][u], qf[k][c][u0 + u], k ? d[c][u] : tf4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
          for (int c = 0; c < NC; c++)
#pragma unroll
            for (int u = 0; u < UG; u++)
#pragma unroll
              for (int i = 0; i < 4; i++)
                s[c][h][i] = u0 + u ? fmaf(f[g % AH][u][i], d[c][u][i], s[c][h][i]) : f[g % AH][u][i] * d[c][u][i];
        }
      } else {
        constexpr bool both = KS <= 4;
        th8 k8[2][KS];
        auto kread = [&](int h) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < KS; u++) k8[h][u] = *(const th8*)(kp + 16 * h * KR + 32 * u);
        };
        kread(0);
        if (both) kread(1);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int HG = both ? 2 : 1;
#pragma unroll
        for (int h0 = 0; h0 < 2; h0 += HG) {
          if (!both && h0) {
            kread(1);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int h = h0; h < h0 + HG; h++)
#pragma unroll
            for (int c = 0; c < NC; c++) s[c][h] = tf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int u = 0; u < KS; u++)
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
              for (int h = h0; h < h0 + HG; h++)
#pragma unroll
                for (int c = 0; c < NC; c++) s[c][h] = mfma16(k8[h][u], qf[k][c][u], s[c][h]);
        }
      }
      if (PAGED) hole = __builtin_amdgcn_readfirstlane(hole) - (first_turn + sl - s0);
    };
    // their softmax and weighted values
    auto values = [&](int sl, int kt, int buf, tf4 (&s)[NC][2], int hole, int (&xv)[Q8 ? KS : 1]) __attribute__((always_inline)) {
      const int base = sl * SL + 32 * kt;
      const _Float16* vp = &vs[buf][32 * kt * VR + vat];
      ts4 v4[2][VG][2];
      auto vread = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < VG; d++)
#pragma unroll
          for (int w = 0; w < 2; w++)
            v4[g & 1][d][w] =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ts4*)(vp + 16 * w * VR + 16 * (g * VG + d)));
      };
      vread(0);
      const bool all = base + 32 <= sq.len && !(PAGED && hole == 0);  // (uniform)
      uint32_t mine[NC];  // bit (i & 3) + 16 (i >> 2): key 4 lk + that is seen
      if (!all) {
        const int key = base + (lane & 31);
        uint32_t there = 0xffffffffu;
        if constexpr (PAGED) there = (uint32_t)__ballot(cell_at(key) >= 0);
#pragma unroll
        for (int c = 0; c < NC; c++) {
          mine[c] = (seen_bits(mask_row(c), words, base - sq.len, sq.count - sq.len) & there) >> (4 * lk);
#pragma unroll
          for (int i = 0; i < 8; i++)
            s[c][i >> 2][i & 3] = (mine[c] >> ((i & 3) + 16 * (i >> 2))) & 1 ? s[c][i >> 2][i & 3] : -INFINITY;
        }
      }
      th8 ph[NC], pl[NC];
      float p[NC][8];
#pragma unroll
      for (int c = 0; c < NC; c++) {
        float m = s[c][0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) m = fmaxf(m, s[c][i >> 2][i & 3]);
        m = across(m, lanes::Max{});
        const bool rose = huge && large(c) ? m > mc[c] : fmaf(m, c2[c], -mk[c]) > lift + kSlack;
        if (__any(rose)) {
          const float mn = rose ? m : mc[c];
          const float mkn = rose ? fmaf(mn, c2[c], -lift) : mk[c];
          const float f = __builtin_amdgcn_exp2f(large(c) ? (mc[c] - mn) * c2[c] : mk[c] - mkn);
          l[c] *= f;
#pragma unroll
          for (int dt = 0; dt < NT; dt++) o[c][dt] *= f;
          mc[c] = mn;
          mk[c] = mkn;
          huge = huge || __any(large(c));
        }
        if (__builtin_expect(huge, 0)) {
#pragma unroll
          for (int i = 0; i < 8; i++)
            p[c][i] = __builtin_amdgcn_exp2f(large(c) ? fmaf(s[c][i >> 2][i & 3] - mc[c], c2[c], lift) : fmaf(s[c][i >> 2][i & 3], c2[c], -mk[c]));
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) p[c][i] = __builtin_amdgcn_exp2f(fmaf(s[c][i >> 2][i & 3], c2[c], -mk[c]));
        }
        l[c] += ((p[c][0] + p[c][1]) + (p[c][2] + p[c][3])) + ((p[c][4] + p[c][5]) + (p[c][6] + p[c][7]));
        if constexpr (!Q8) split<true>(p[c], [&](int) __attribute__((always_inline)) { return one; }, ph[c], pl[c]);
      }
      if constexpr (Q8) {  // (uniform) X has risen with this slice's factors
        int rise = 0;
#pragma unroll
        for (int u = 0; u < KS; u++) rise |= __builtin_amdgcn_readfirstlane(xv[u]) ^ xo[u];
        if (rise) {
#pragma unroll
          for (int u = 0; u < KS; u++) {
            const int x = __builtin_amdgcn_readfirstlane(xv[u]);
            const float f = ldexpf(1.0f, xo[u] - x);
#pragma unroll
            for (int c = 0; c < NC; c++) o[c][2 * u] *= f, o[c][2 * u + 1] *= f;
            xo[u] = x;
          }
        }
      }
      // value fragments of group dt / VG, the next group's on their way
      auto vtile = [&](int dt) __attribute__((always_inline)) {
        ts8 v;
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
          for (int e = 0; e < 4; e++) v[4 * w + e] = v4[(dt / VG) & 1][dt % VG][w][e];
        return __builtin_bit_cast(th8, v);
      };
      if constexpr (Q8) {
        static_assert(VG == 2, "a group is a 32-dim block");
        tf4 f[2][2];  // a block's factors, the next one's on their way
        auto fread = [&](int u) __attribute__((always_inline)) {
#pragma unroll
          for (int w = 0; w < 2; w++) f[u & 1][w] = *(const tf4*)&fac[buf][1][u][32 * kt + 16 * w + 4 * lk];
        };
        fread(0);
        if (all) {
#pragma unroll
          for (int u = 0; u < KS; u++) {
            if (u + 1 < KS) {
              vread(u + 1);
              fread(u + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < NC; c++) {
              split<false>(p[c], [&](int i) __attribute__((always_inline)) { return f[u & 1][i >> 2][i & 3]; }, ph[c], pl[c]);
#pragma unroll
              for (int dt = 2 * u; dt < 2 * u + 2; dt++) o[c][dt] = mfma16(vtile(dt), ph[c], o[c][dt]);
#pragma unroll
              for (int dt = 2 * u; dt < 2 * u + 2; dt++) o[c][dt] = mfma16(vtile(dt), pl[c], o[c][dt]);
            }
          }
        } else {
#pragma unroll
          for (int u = 0; u < KS; u++) {
            if (u) {
              vread(u);
              fread(u);
            }
#pragma unroll
            for (int c = 0; c < NC; c++) {
              // (whatever the factor of a key that is not seen)
              float w[8], wm = 0.0f;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                w[i] = (mine[c] >> ((i & 3) + 16 * (i >> 2))) & 1 ? p[c][i] * f[u & 1][i >> 2][i & 3] : 0.0f;
                wm = fmaxf(wm, fabsf(w[i]));
              }
              wm = across(wm, lanes::Max{});
              const int xc = wm > 0.0f && wm < INFINITY ? __builtin_amdgcn_frexp_expf(wm) : 0;
              const float unit = ldexpf(1.0f, 15 - xc), back = ldexpf(1.0f, xc - 15);
#pragma unroll
              for (int i = 0; i < 8; i++) {
                ph[c][i] = (_Float16)fmaf(w[i], unit, 0.0f);
                pl[c][i] = (_Float16)fmaf(w[i], unit, -(float)ph[c][i]);
              }
#pragma unroll
              for (int dt = 2 * u; dt < 2 * u + 2; dt++) {
                const tf4 t = mfma16(vtile(dt), pl[c], mfma16(vtile(dt), ph[c], tf4{0.0f, 0.0f, 0.0f, 0.0f}));
#pragma unroll
                for (int e = 0; e < 4; e++) o[c][dt][e] = fmaf(t[e], back, o[c][dt][e]);
              }
            }
          }
        }
      } else {
#pragma unroll
        for (int dt = 0; dt < NT; dt++) {
          if (dt % VG == 0) {
            if (dt + VG < NT) vread(dt / VG + 1);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int c = 0; c < NC; c++) o[c][dt] = mfma16(vtile(dt), ph[c], o[c][dt]);
#pragma unroll
          for (int c = 0; c < NC; c++) o[c][dt] = mfma16(vtile(dt), pl[c], o[c][dt]);
        }
      }
    };

    store(s0, 0, st);
    if (s0 + 1 < s1) st = ahead;
    __syncthreads();
    for (int sl = s0, buf = 0; sl < s1; sl++, buf ^= 1) {
      tf4 s[SL / 32][NC][2];
      int hole = 1, xv[Q8 ? KS : 1];
      if constexpr (KW == 2) {
        if (busy && sl * SL + 32 * half < sq.count) scores(sl, half, buf, s[0], hole, xv);
      } else if (busy) {
        scores(sl, 0, buf, s[0], hole, xv);
        if constexpr (SL > 32) scores(sl, 1, buf, s[1], hole, xv);
      }
      // the next slice from registers to the other buffer, and the one behind it on
      // its way (written once for busy and idle waves: with a copy for each the
      // registers differ, and the busy ones wait for loads at every step)
      __builtin_amdgcn_sched_barrier(0);
      if (sl + 1 < s1) {
        store(sl + 1, buf ^ 1, st);
        if (sl + 2 < s1) {
          load(sl + 2, st);
          if (sl + 3 < s1) find(sl + 3, st);
        }
      }
      if constexpr (KW == 2) {
        if (busy && sl * SL + 32 * half < sq.count) values(sl, half, buf, s[0], hole, xv);
      } else if (busy) {
        values(sl, 0, buf, s[0], hole, xv);
        if constexpr (SL > 32) {
          if (sl * SL + 32 < sq.count) values(sl, 1, buf, s[1], hole, xv);
        }
      }
      __syncthreads();
    }

    if constexpr (KW == 2) {
      // the two waves of a row to one, by way of the keys' buffers (no more in use; the
      // next run's first slice waits behind the second barrier)
      static_assert(Q8 && NC == 1 && sizeof(ks) >= 2 * 64 * (NT + 1) * sizeof(tf4), "room for two waves' sums");
      tf4* put = (tf4*)ks + (wave * 64 + lane) * (NT + 1);
      if (half && busy) {
#pragma unroll
        for (int dt = 0; dt < NT; dt++) put[dt] = o[0][dt] * ldexpf(1.0f, xo[dt / 2] - kFactor);
        put[NT] = tf4{mk[0], l[0], 0.0f, 0.0f};
      }
      __syncthreads();
      if (!half && busy) {
        const float om = put[NT][0], m = fmaxf(mk[0], om);
        const float f0 = mk[0] == m ? 1.0f : __builtin_amdgcn_exp2f(mk[0] - m), f1 = om == m ? 1.0f : __builtin_amdgcn_exp2f(om - m);
#pragma unroll
        for (int dt = 0; dt < NT; dt++) o[0][dt] = o[0][dt] * (ldexpf(f0, xo[dt / 2] - kFactor)) + put[dt] * f1;
        l[0] = l[0] * f0 + put[NT][1] * f1;
        mk[0] = m;
      }
      __syncthreads();
    }
    if (!busy || half) return;
    float sum[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) sum[c] = across(l[c], lanes::Add{});
    auto write = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < NC; c++) {
        if (node[c] >= sq.nodes) continue;
        const int64_t slot = (int64_t)part * ROWS + wave * 16 * NC + 16 * c + lm;
        float* dst = part < 0 ? a.out + ((int64_t)(sq.t0 + node[c]) * a.heads + kvh * group + ((first_row + 16 * c + lm) & (group - 1))) * D
                              : parts.acc + slot * D;
        const float w = part >= 0 ? 1.0f : sum[c] != 0.0f ? 1.0f / sum[c] : 0.0f;
#pragma unroll
        for (int dt = 0; dt < NT; dt++) {
          const float f = Q8 && KW == 1 ? w * ldexpf(1.0f, xo[dt / 2] - kFactor) : w;
          *(tf4*)(dst + 16 * dt + 4 * lk) = o[c][dt] * f;
        }
        if (part >= 0 && lk == 0) *(float2*)(parts.ml + 2 * slot) = make_float2(mk[c], sum[c]);
      }
    };
    write();
    // Values that are not finite.  Of slices that were staged without them they are
    // missing in o; of the others the halves' products have made NaN (inf times a lower
    // half of zero): each such sum starts anew from the values that the row sees.  Where
    // the weights are NaN so is their sum, and the result with it, whatever o is.  (Behind
    // the stores, which need not wait for the look: 1 x 8 over 2048 15.2 us ahead of them.)
    if constexpr (!Q8) {
      bool lost = spoilt[run & 1] == run;
#pragma unroll
      for (int c = 0; c < NC; c++) {
        tf4 none = {0.0f, 0.0f, 0.0f, 0.0f};  // (zero, or NaN)
#pragma unroll
        for (int dt = 0; dt < NT; dt++)
#pragma unroll
          for (int e = 0; e < 4; e++) none[e] = fmaf(o[c][dt][e], 0.0f, none[e]);
        lost |= (none[0] + none[1]) + (none[2] + none[3]) != 0.0f && sum[c] == sum[c];
      }
      if (__builtin_expect(!__any(lost), 1)) return;
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int dt = 0; dt < NT; dt++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[c][dt][e] = fabsf(o[c][dt][e]) < INFINITY ? o[c][dt][e] : 0.0f;
      for (int j = s0 * SL; j < min(s1 * SL, sq.count); j++) {
        const int cell = PAGED ? index[j] : j;
        if (cell < 0) continue;
        const __half* vr = vc + (int64_t)cell * crow + 4 * lk;
        const int i = j - sq.len;
#pragma unroll
        for (int c = 0; c < NC; c++) {
          const bool sees = i < 0 || ((mask_row(c)[max(i, 0) >> 5] >> (i & 31)) & 1);
#pragma unroll
          for (int dt = 0; dt < NT; dt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float v = __half2float(vr[16 * dt + e]);
              if (sees && !(fabsf(v) < INFINITY)) o[c][dt][e] += v;
            }
        }
      }
      write();
    }
  });
}

// Folds the parts of each row whose tile several blocks share: W waves a row, up
// to eight parts' sums of each on their way at once.  A part that no key of the
// row fell in has sum 0 and weight 0; a row without any other is zero.
template <int V, int W>
__global__ __launch_bounds__(256) void attend_tree_fold_kernel(TreeAttend a, TreeParts parts,
                                                               const int32_t* __restrict__ plan, int rows, int slice) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ vec sums[W > 1 ? W : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int D = a.head_dim, shift = a.group_shift;
  const uint32_t i = grid_block() * (4 / W) + wave / W, step = (uint32_t)a.tree.max_nodes * a.heads;  // (both below 2^31)
  const int b = (int)(i / step);
  if (b >= a.tree.batch) return;  // (W > 1: every wave of the block)
  const int at = (int)(i - b * step), node = at / a.heads, h = at - node * a.heads;
  const int per = plan[0], b_first = plan[1 + b];
  const TreeSeq sq = tree_seq(a.tree, b);
  if (node >= sq.nodes) return;
  const int kvh = h >> shift, r = (node << shift) + (h & ((1 << shift) - 1)), tile = r / rows, slices = tree_slices(sq, slice);
  const int u0 = b_first + (kvh * tree_tiles(sq, shift, rows) + tile) * tree_units(sq, slice) + kStart;
  const int g0 = u0 / per, n = (u0 + slices - 1) / per - g0 + 1;
  if (n == 1) return;  // one block's: finished
  // part k is block g0 + k's: its last one (1) for the block that the tile starts in, else its first (0)
  auto slot = [&](int k) { return (int64_t)(2 * (g0 + k) + (k == 0 ? 1 : 0)) * rows + r % rows; };
  const int per_wave = (n + W - 1) / W, k0 = (wave % W) * per_wave, k1 = min(k0 + per_wave, n);
  float2 ml[2];
#pragma unroll
  for (int k = 0; k < 2; k++) ml[k] = ((const float2*)parts.ml)[slot(min(64 * k + lane, n - 1))];
  // eight parts' sums from k on (past the end the last one again, weight 0)
  vec x[8];
  auto send = [&](int k, int d) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = *(const vec*)(parts.acc + slot(min(k + j, n - 1)) * D + d);
  };
  send(k0, min(lane * V, D - V));  // (behind the maxima, and waited for with them)
  float w[2], m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (64 * k + lane >= n) ml[k].y = 0.0f;
    if (ml[k].y != 0.0f) m = fmaxf(m, ml[k].x);
  }
  m = lanes::reduce<64>(m, lanes::Max{});
#pragma unroll
  for (int k = 0; k < 2; k++) {
    w[k] = ml[k].y == 0.0f ? 0.0f : ml[k].x == m ? 1.0f : __builtin_amdgcn_exp2f(ml[k].x - m);
    sum += ml[k].y == 0.0f ? 0.0f : ml[k].y * w[k];
  }
  sum = lanes::reduce<64>(sum, lanes::Add{});
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  float* dst = a.out + ((int64_t)(sq.t0 + node) * a.heads + h) * D;
  for (int d0 = 0; d0 < D; d0 += 64 * V) {
    const int d = min(d0 + lane * V, D - V);
    vec o = {};
    for (int k = k0; k < k1; k += 8) {
      if (d0 || k != k0) send(k, d);
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (k + j < k1)  // (uniform)
          o += x[j] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(k + j < 64 ? w[0] : w[1]), (k + j) & 63));
    }
    if constexpr (W > 1) {
      if (d0) __syncthreads();
      sums[wave][lane] = o;
      __syncthreads();
      if (wave) continue;
#pragma unroll
      for (int v = 1; v < W; v++) o += sums[v][lane];
    }
    if (d0 + lane * V < D) *(vec*)(dst + d) = o * inv;
  }
}

// The same for rows of 64 and 128 values where there are many: 64 / L rows a wave,
// L lanes of four values each.  They are consecutive rows of a tile, so that their
// parts lie in the same blocks (12288 rows of 64 in 5 parts 9.3 us with a wave each,
// 5.1; 16384 of 128 13 and 8.6).
template <int L>
__global__ __launch_bounds__(256) void attend_tree_fold_rows_kernel(TreeAttend a, TreeParts parts,
                                                                    const int32_t* __restrict__ plan, int rows,
                                                                    int slice) {
  constexpr int R = 64 / L, D = 4 * L, J = kMaxParts / L;
  const int lane = threadIdx.x & 63, l = lane % L, shift = a.group_shift;
  const uint32_t job = grid_block() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t runs = ((a.tree.max_nodes << shift) + R - 1) / R, pair = job / runs;
  const int b = (int)(pair / a.kv_heads), kvh = (int)(pair - b * a.kv_heads), r0 = (int)(job - pair * runs) * R;
  if (b >= a.tree.batch) return;
  const int per = plan[0], b_first = plan[1 + b];
  const TreeSeq sq = tree_seq(a.tree, b);
  if (r0 >= sq.nodes << shift) return;
  const int slices = tree_slices(sq, slice);
  const int u0 = b_first + (kvh * tree_tiles(sq, shift, rows) + r0 / rows) * tree_units(sq, slice) + kStart;
  const int g0 = u0 / per, n = (u0 + slices - 1) / per - g0 + 1;
  if (n == 1) return;
  const int r = r0 + lane / L;
  auto slot = [&](int k) { return (int64_t)(2 * (g0 + k) + (k == 0 ? 1 : 0)) * rows + r % rows; };
  tf4 x[8];
  auto send = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = *(const tf4*)(parts.acc + slot(min(k + j, n - 1)) * D + 4 * l);
  };
  // part L j + l of the row: its maximum and sum, then its weight
  float2 ml[J];
#pragma unroll
  for (int j = 0; j < J; j++)
    if (j == 0 || L * j < n) ml[j] = ((const float2*)parts.ml)[slot(min(L * j + l, n - 1))];
  send(0);
  float w[J], m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int j = 0; j < J; j++) {
    if (L * j + l >= n) ml[j].y = 0.0f;
    if (ml[j].y != 0.0f) m = fmaxf(m, ml[j].x);
  }
  m = lanes::reduce<L>(m, lanes::Max{});
#pragma unroll
  for (int j = 0; j < J; j++) {
    w[j] = ml[j].y == 0.0f ? 0.0f : ml[j].x == m ? 1.0f : __builtin_amdgcn_exp2f(ml[j].x - m);
    sum += ml[j].y == 0.0f ? 0.0f : ml[j].y * w[j];
  }
  sum = lanes::reduce<L>(sum, lanes::Add{});
  tf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < J; j++)
    for (int k = L * j; k < min(L * (j + 1), n); k += 8) {
      if (k) send(k);
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (k + i < n) o += x[i] * __shfl(w[j], (lane & ~(L - 1)) + k + i - L * j);  // (uniform)
    }
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  const int node = r >> shift;
  if (node < sq.nodes)
    *(tf4*)(a.out + ((int64_t)(sq.t0 + node) * a.heads + (kvh << shift) + (r & ((1 << shift) - 1))) * D + 4 * l) = o * inv;
}

struct TreeGrid {
  bool mfma;
  int columns, split;  // NC and KW of attend_tree_kernel
  int rows, slice;
  int64_t units;  // of the largest step
  int blocks;
};

TreeGrid tree_grid(int heads, int kv_heads, int head_dim, int form, const mi_tree& t) {
  TreeGrid g;
  const int group = heads / kv_heads;
  g.mfma = head_dim == 64 || head_dim == 128 || head_dim == 256;
  // two columns a lane read each key fragment once for twice the rows, but only
  // where a sequence has more rows than one column's 64: 8 x 32 nodes at D = 128 74
  // us with two and 89 with one, 8 x 16 62 and 50, 1 x 13 47 and 37 (at D = 64 the
  // registers cost the third block: 8 x 48 over 3000 31 us for 29, over 12000 80 for
  // 83; with q8_0 they spill)
  g.columns = head_dim == 128 && form != MI_CACHE_Q8 && t.max_nodes * group > 64 ? 2 : 1;
  // up to 32 rows are two waves' work, at q8_0 long enough for the other two to take
  // half of each slice's keys: 64 x 1 nodes over 4096 212 us, so 173; 8 x 8 over 16384
  // 122 and 101 (f16 waits for its loads, 150 us and 5.4 TB/s)
  g.split = form == MI_CACHE_Q8 && (head_dim == 64 || head_dim == 128) && t.max_nodes * group <= 32 ? 2 : 1;
  g.rows = g.mfma ? 64 * g.columns / g.split : kRowsTile;
  g.slice = g.split == 2 ? 64 : g.mfma ? mfma_slice(head_dim) : rows_slice(head_dim);
  g.units = (int64_t)t.batch * ((t.max_nodes * group + g.rows - 1) / g.rows) * kv_heads *
            (((int64_t)t.max_count + g.slice - 1) / g.slice + kStart);
  g.blocks = (int)std::min<int64_t>(g.units, (int64_t)cu_count() * (g.mfma ? mfma_blocks(head_dim) : 3));
  return g;
}

// The workspace: each block's two parts of a tile (sums, then maxima and sums),
// then the plan of the walk.
struct TreeCarve {
  size_t ml, plan, total;
};
TreeCarve tree_carve(const TreeGrid& g, int head_dim, int batch) {
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  TreeCarve c;
  c.ml = up((size_t)2 * g.blocks * g.rows * head_dim * sizeof(float));
  c.plan = c.ml + up((size_t)2 * g.blocks * g.rows * 2 * sizeof(float));
  c.total = c.plan + up(((size_t)batch + 1) * sizeof(int32_t));
  return c;
}

}  // namespace

size_t tree_attend_workspace(int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t form, const mi_tree& t) {
  return tree_carve(tree_grid(heads, kv_heads, head_dim, form, t), head_dim, t.batch).total;
}

// Whether units and rows, whose sums the device takes in 32 bits, are few enough.
bool tree_attend_fits(int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t form, const mi_tree& t) {
  return tree_grid(heads, kv_heads, head_dim, form, t).units <= 1 << 30 &&
         (int64_t)t.batch * t.max_nodes * heads <= 1 << 30;
}

int launch_tree_attend(hipStream_t s, const TreeAttend& step, void* work) {
  TreeAttend a = step;
  a.group_shift = __builtin_ctz(a.heads / a.kv_heads);  // (1, 2, 4 or 8 query heads a key head)
  const TreeGrid g = tree_grid(a.heads, a.kv_heads, a.head_dim, a.form, a.tree);
  // few rows: four waves each (416 rows of 62 parts 8.5 us with one, 5.6 with four;
  // 3200 of 10 5.8 and 12.2), else several rows a wave where a row is 64 or 128 values
  const int64_t rows = (int64_t)a.tree.batch * a.tree.max_nodes * a.heads;
  const int waves = rows <= 1024 ? 4 : 1;
  const dim3 fold = grid_of((rows * waves + 3) / 4);
  const TreeCarve c = tree_carve(g, a.head_dim, a.tree.batch);
  const TreeParts parts{(float*)work, (float*)((char*)work + c.ml)};
  int32_t* plan = (int32_t*)((char*)work + c.plan);
  const dim3 grid(g.blocks);
#define MI_TREE(D, NC, Q, P) \
  hipLaunchKernelGGL((attend_tree_kernel<D, NC, Q, P>), grid, dim3(256), 0, s, a, parts, plan)
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
                       a, parts, plan);                                                                              \
  else                                                                                                               \
    hipLaunchKernelGGL((attend_tree_rows_kernel<false, ND>), grid, dim3(kRowsThreads), rows_lds_bytes(a.head_dim), s, \
                       a, parts, plan)
#define MI_TREE_SPLIT(D)                                                                                         \
  if (a.kv_index)                                                                                                \
    hipLaunchKernelGGL((attend_tree_kernel<D, 1, true, true, 2>), grid, dim3(256), 0, s, a, parts, plan);        \
  else                                                                                                           \
    hipLaunchKernelGGL((attend_tree_kernel<D, 1, true, false, 2>), grid, dim3(256), 0, s, a, parts, plan)
  if (g.split == 2) {
    if (a.head_dim == 64) MI_TREE_SPLIT(64);
    else MI_TREE_SPLIT(128);
  } else if (a.head_dim == 64) {
    MI_TREE_F(64, 1)
  } else if (a.head_dim == 128) {
    if (g.columns == 1) { MI_TREE_F(128, 1) }
    else if (a.kv_index) MI_TREE(128, 2, false, true);
    else MI_TREE(128, 2, false, false);
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
#undef MI_TREE_SPLIT
#undef MI_TREE_ROWS
  if (int rc = hip_check(hipGetLastError(), "attend_tree launch")) return rc;
#define MI_TREE_FOLD(V)                                                                                            \
  if (waves == 4)                                                                                                  \
    hipLaunchKernelGGL((attend_tree_fold_kernel<V, 4>), fold, dim3(256), 0, s, a, parts, plan, g.rows, \
                       g.slice);                                                                                   \
  else                                                                                                             \
    hipLaunchKernelGGL((attend_tree_fold_kernel<V, 1>), fold, dim3(256), 0, s, a, parts, plan, g.rows, \
                       g.slice)
  if (waves == 1 && (a.head_dim == 64 || a.head_dim == 128)) {
    const int per_wave = a.head_dim == 64 ? 4 : 2;
    const int64_t runs = ((int64_t)a.tree.max_nodes * a.heads / a.kv_heads + per_wave - 1) / per_wave;
    const dim3 folds = grid_of(((int64_t)a.tree.batch * a.kv_heads * runs + 3) / 4);
    if (a.head_dim == 64)
      hipLaunchKernelGGL(attend_tree_fold_rows_kernel<16>, folds, dim3(256), 0, s, a, parts, plan, g.rows, g.slice);
    else
      hipLaunchKernelGGL(attend_tree_fold_rows_kernel<32>, folds, dim3(256), 0, s, a, parts, plan, g.rows, g.slice);
  } else if (a.head_dim % 256 == 0) MI_TREE_FOLD(4);
  else if (a.head_dim % 128 == 0) MI_TREE_FOLD(2);
  else MI_TREE_FOLD(1);
#undef MI_TREE_FOLD
  return hip_check(hipGetLastError(), "attend_tree fold launch");
}

}  // namespace mi
