// prefill.hip -- the many-token matmul of one matrix, or of up to three laid end
// to end: the launchers of prefill_kernel.h's kernel, the sum of its parts, and
// how a block is cut by size.
#include "prefill_kernel.h"

namespace mi {
namespace {

// A token's activations, one block a token (256 threads, 8 consecutive values
// a thread and round): its scale, the power of two 2^e with the largest
// |x| * 2^-e in [2^13, 2^14) (e clamped so that the scale stays a normal
// float; 1 for a zero or padding token), xs[t] = 2^e; its halves; and the
// means of its 32-value groups.  A row of up to 16384 values stays in
// registers between the maximum and the split (one launch and one reading of
// x, where two launches were 9.8 us at 256 x 4096).
constexpr int kPrepRounds = 8;
__global__ __launch_bounds__(256) void prefill_prep_kernel(const float* __restrict__ x, int cols, int tokens,
                                                           uint8_t* __restrict__ work) {
  const Prep P = prep_layout(cols, tokens);
  const int t = blockIdx.x, tile = t >> 5, m = t & 31;
  const int n8 = cols >> 3;  // runs of 8 values
  const float* row = x + (int64_t)t * cols;
  typedef float v4f __attribute__((ext_vector_type(4)));
  __shared__ float red[4];
  v4f v[kPrepRounds][2];
  float mx = 0.0f;
  if (t < tokens) {
#pragma unroll
    for (int k = 0; k < kPrepRounds; k++) {
      const int i = min((int)threadIdx.x + 256 * k, n8 - 1);  // (a repeated run changes no maximum)
      if (256 * k < n8) {
        v[k][0] = *(const v4f*)(row + 8 * i);
        v[k][1] = *(const v4f*)(row + 8 * i + 4);
      }
    }
#pragma unroll
    for (int k = 0; k < kPrepRounds; k++)
      if (256 * k < n8) {
#pragma unroll
        for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(v[k][i >> 2][i & 3]));
      }
    for (int i = threadIdx.x + 256 * kPrepRounds; i < n8; i += 256) {
      const v4f a = *(const v4f*)(row + 8 * i), b = *(const v4f*)(row + 8 * i + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) mx = fmaxf(mx, fmaxf(fabsf(a[e]), fabsf(b[e])));
    }
    mx = lanes::reduce<64>(mx, lanes::Max{});
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  }
  const int e = scale_exp(mx);
  if (threadIdx.x == 0) ((float*)(work + P.xs))[t] = ldexpf(1.0f, e);
  uint8_t* xp = work + P.xp + (size_t)tile * P.ks * 2048 + 16 * m;
  _Float16* xm = (_Float16*)(work + P.xm) + (size_t)tile * P.nch * 512 + 8 * m;
  auto put = [&](int i, v4f a, v4f b) __attribute__((always_inline)) {
    // run i: values 8 i .. +8, half wave (i >> 1) & 1 of step 2 (i >> 2) + (i & 1)
    v8h hi, lo;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      constexpr int order[4] = {0, 2, 1, 3};  // the order of K (above)
      const int c = order[k & 3];
      const float f = ldexpf(k < 4 ? a[c] : b[c], -e);
      _Float16 h, l;
      split_half(f, h, l);
      hi[k] = h;
      lo[k] = l;
      sum += f;
    }
    uint8_t* dst = xp + (size_t)(2 * (i >> 2) + (i & 1)) * 2048 + 512 * ((i >> 1) & 1);
    *(v8h*)dst = hi;
    *(v8h*)(dst + 1024) = lo;
    // the mean of the group's 32 values (a mean, since 32 values of up to
    // 2^14 overflow a half): four neighbouring lanes
    sum = lanes::reduce<4>(sum, lanes::Add{}) * (1.0f / 32.0f);
    _Float16 h, l;
    split_half(sum, h, l);
    const int g = i >> 2;
    if ((i & 3) == 0) {
      xm[(size_t)(g >> 3) * 512 + (g & 7)] = h;
      xm[(size_t)(g >> 3) * 512 + 256 + (g & 7)] = l;
    }
  };
  // (n8 is a multiple of 8: a group's four lanes go together)
#pragma unroll
  for (int k = 0; k < kPrepRounds; k++) {
    const int i = threadIdx.x + 256 * k;
    if (i < n8) put(i, t < tokens ? v[k][0] : v4f{}, t < tokens ? v[k][1] : v4f{});
  }
  for (int i = threadIdx.x + 256 * kPrepRounds; i < n8; i += 256)
    put(i, t < tokens ? *(const v4f*)(row + 8 * i) : v4f{}, t < tokens ? *(const v4f*)(row + 8 * i + 4) : v4f{});
  // groups past cols in the last chunk
  for (int g = (cols >> 5) + threadIdx.x; g < 8 * P.nch; g += 256) {
    xm[(size_t)(g >> 3) * 512 + (g & 7)] = (_Float16)0.0f;
    xm[(size_t)(g >> 3) * 512 + 256 + (g & 7)] = (_Float16)0.0f;
  }
}

// Adds the splits' partial sums in split order and applies the epilogue.
__global__ __launch_bounds__(256) void prefill_reduce_kernel(const float* __restrict__ part, int splits, int rows,
                                                             int tokens, float* __restrict__ y, int64_t ldy, int epi,
                                                             const float* __restrict__ aux) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t n = (int64_t)rows * tokens;
  if (i >= n) return;
  float v = part[i];
  for (int z = 1; z < splits; z++) v += part[z * n + i];
  const int t = (int)(i / rows), r = (int)(i - (int64_t)t * rows);
  mv::epilogue(y, aux, epi, (int64_t)t * ldy + r, r, v);
}

// How a block is cut: (row tiles, token tiles) of 32 a wave, waves over rows,
// groups over K.
struct Shape {
  int rt, tt, wr, ks;
  int block_rows() const { return wr * rt * 32; }
};
// Each measured against the others (us a call).  Up to 32 tokens (1, 1, 4, 2) /
// (1, 2, 4, 2) / (1, 1, 4, 4): Q4_K 4096x4096 12.7 / 13.8 / 13.5, Q6_K 17.2 / - /
// 22.9, Q8_0 17.7 / 19.1 / 24.6.
// Small matrices want more, smaller blocks.  (1, 2, 4, 2) / (2, 2, 4, 2) by `work`,
// the 256-value chunks of 256 x 64 outputs:
//   896   14336x4096, 64 tokens   Q4_K 35.6 / 37.9  Q8_0 44.5 / 47.9  Q4_0 39.0 / 39.3
//   1232  5632x2048, 400          Q4_K 54.2 / 44.8  Q8_0 59.7 / 61.9  Q4_0 48.8 / 51.2
//   1536  6144x4096, 256          Q4_K 47.3 / 49.5  Q8_0 65.5 / 66.8  Q4_0 60.5 / 56.0
//   1792  14336x4096, 128         Q4_K 47.6 / 51.7  Q8_0 68.5 / 72.3  Q4_0 58.1 / 55.8
//   2064  11008x4096, 192         Q4_K 87.3 / 65.5  Q8_0 107.9 / 105.9  Q4_0 80.5 / 83.2
//   2688  4096x14336, 192         Q4_K 82.1 / 76.9  Q8_0 122.7 / 116.1  Q4_0 103.2 / 88.8
//   3584  14336x4096, 256         Q4_K 89.8 / 77.8  Q8_0 111.5 / 113.9  Q4_0 87.7 / 86.4
// The line is a rough one: the smaller blocks lose where they need a second round
// of the chip (up to 25 %) and for Q4_K and Q8_0 win up to there, to 2048 (11 %).
// Q6_K, three products a step, pays for the larger token tile also where half of
// it is empty: (1, 2, 4, 2) / (2, 2, 4, 2) / (1, 4, 8, 1) 14336x4096 at 96 tokens
// 68 / 73 / 62, at 128 69 / 74 / 68, at 150 124 / 117 / 98, 4096x14336 at 192 121 /
// 120 / 107, at 256 127 / 127 / 114; at 64 48 / 54 / 62.
// (The (2, 2, 4, 2) block of Q5_1 spills 10 registers in its stage and is still the
// faster one at 14336x4096, 256 tokens: 118 / 106.)
Shape shape_for(int kind, int rows, int cols, int tokens) {
  if (tokens <= 32) return Shape{1, 1, 4, 2};
  const int64_t work = (int64_t)((rows + 255) / 256) * ((tokens + 63) / 64) * ((cols + kChunk - 1) / kChunk);
  if (work <= 1536) return Shape{1, 2, 4, 2};
  if (kind == MI_Q6_K && tokens > 64) return Shape{1, 4, 8, 1};
  return Shape{2, 2, 4, 2};
}

template <int KIND>
int launch_kind(hipStream_t s, const RowSegs& sg, int cols, int tokens, const void* work, int splits, int cps,
                float* y, int64_t ldy, int epi, const float* aux, float* part) {
  const int rows = sg.end[sg.nseg - 1];
  const Shape sh = shape_for(KIND, rows, cols, tokens);
  const int tiles = (tokens + kTileTok - 1) / kTileTok;
  const dim3 grid((rows + sh.block_rows() - 1) / sh.block_rows(), (tiles + sh.tt - 1) / sh.tt, splits);
  const dim3 block(sh.wr * sh.ks * 64);
#define MI_PF(R, T, W, G)                                                                                  \
  hipLaunchKernelGGL((prefill_kernel<KIND, R, T, W, G>), grid, block, 0, s, sg, cols, tokens,               \
                     (const uint8_t*)work, cps, y, ldy, epi, aux, splits > 1 ? part : nullptr)
  if (sh.tt == 1) MI_PF(1, 1, 4, 2);
  else if (sh.rt == 1 && sh.tt == 2) MI_PF(1, 2, 4, 2);
  else if constexpr (KIND == MI_Q6_K) {
    if (sh.tt == 4) MI_PF(1, 4, 8, 1);
    else MI_PF(2, 2, 4, 2);
  } else {
    MI_PF(2, 2, 4, 2);
  }
#undef MI_PF
  return hip_check(hipGetLastError(), "prefill launch");
}

// Splits of K over blocks (in whole 256-value chunks): the largest power of
// two whose blocks still fit one round of the chip, one block a compute unit,
// each K group of a block at least one chunk.
int choose_splits(int kind, int rows, int cols, int tokens) {
  const Shape sh = shape_for(kind, rows, cols, tokens);
  const int tiles = (tokens + kTileTok - 1) / kTileTok;
  const int64_t blocks = (int64_t)((rows + sh.block_rows() - 1) / sh.block_rows()) * ((tiles + sh.tt - 1) / sh.tt);
  const int chunks = (cols + kChunk - 1) / kChunk;
  int s = 1;
  const int places = cu_count();
  while (blocks * 2 * s <= places && chunks >= 2 * s * sh.ks) s *= 2;
  return s;
}

}  // namespace

bool prefill_fits(int kind, int32_t cols, int64_t row_bytes, const void* w) {
  if (cols % kStage) return false;
  switch (kind) {
    case MI_Q4_K:
    case MI_Q5_K:
      return cols % 256 == 0 && ((uintptr_t)w & 15) == 0 && row_bytes % 16 == 0;
    case MI_Q6_K:
      return cols % 256 == 0 && ((uintptr_t)w & 1) == 0 && row_bytes % 2 == 0;
    case MI_Q4_1:
      return ((uintptr_t)w & 3) == 0 && row_bytes % 4 == 0;
    case MI_Q5_1:
      return ((uintptr_t)w & 7) == 0 && row_bytes % 8 == 0;
    case MI_Q8_0:
    case MI_Q4_0:
    case MI_Q5_0:
      return ((uintptr_t)w & 1) == 0 && row_bytes % 2 == 0;
  }
  return false;
}

size_t prefill_workspace(int32_t rows, int32_t cols, int32_t tokens) {
  const Prep P = prep_layout(cols, tokens);
  int splits = 1;  // the most any kind takes (shape_for tells two apart)
  for (int k : {MI_Q4_K, MI_Q6_K}) splits = std::max(splits, rows > 0 ? choose_splits(k, rows, cols, tokens) : 1);
  size_t part = splits > 1 ? (size_t)splits * tokens * rows * 4 : 0;
  return P.total + ((part + 255) & ~(size_t)255);
}

size_t prefill_prep_bytes(int32_t cols, int32_t tokens) { return prep_layout(cols, tokens).total; }

int prefill_prepare(hipStream_t s, const float* x, int32_t cols, int32_t tokens, void* work) {
  const Prep P = prep_layout(cols, tokens);
  hipLaunchKernelGGL(prefill_prep_kernel, dim3(P.ttp * kTileTok), dim3(256), 0, s, x, cols, tokens, (uint8_t*)work);
  return hip_check(hipGetLastError(), "prefill activation launch");
}

int launch_prefill_segs(hipStream_t s, int kind, const RowSegs& sg, int32_t cols, int32_t tokens, float* y,
                        int64_t ldy, int32_t epi, const float* aux, void* work, size_t work_bytes) {
  const Prep P = prep_layout(cols, tokens);
  const int rows = sg.end[sg.nseg - 1];
  int splits = choose_splits(kind, rows, cols, tokens);
  const size_t need = (size_t)splits * tokens * rows * 4;
  if (splits > 1 && work_bytes < P.total + need) splits = 1;  // no room for partial sums
  const int cps = (P.nch + splits - 1) / splits;
  splits = (P.nch + cps - 1) / cps;
  float* part = (float*)((uint8_t*)work + P.total);
  int rc;
  switch (kind) {
    case MI_Q4_K: rc = launch_kind<MI_Q4_K>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q5_K: rc = launch_kind<MI_Q5_K>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q6_K: rc = launch_kind<MI_Q6_K>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q8_0: rc = launch_kind<MI_Q8_0>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q4_0: rc = launch_kind<MI_Q4_0>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q4_1: rc = launch_kind<MI_Q4_1>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q5_0: rc = launch_kind<MI_Q5_0>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    case MI_Q5_1: rc = launch_kind<MI_Q5_1>(s, sg, cols, tokens, work, splits, cps, y, ldy, epi, aux, part); break;
    default: return fail(MI_ERR_KIND, "prefill: ggml type %d has no tile", kind);
  }
  if (rc || splits == 1) return rc;
  const int64_t n = (int64_t)rows * tokens;
  hipLaunchKernelGGL(prefill_reduce_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, part, splits, rows,
                     tokens, y, ldy, epi, aux);
  return hip_check(hipGetLastError(), "prefill reduce launch");
}

int launch_prefill(hipStream_t s, int kind, const void* w, int64_t row_bytes, int32_t rows, int32_t cols,
                   const float* x, int32_t tokens, float* y, int64_t ldy, int32_t epi, const float* aux, void* work,
                   size_t work_bytes) {
  int rc = prefill_prepare(s, x, cols, tokens, work);
  if (rc) return rc;
  return launch_prefill_segs(s, kind, rows::one_matrix(w, row_bytes, rows), cols, tokens, y, ldy, epi, aux, work,
                             work_bytes);
}

}  // namespace mi
