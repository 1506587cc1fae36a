// experts_tile.hip -- products of many rows with stacked experts' matrices on the
// matrix cores: prefill_kernel.h's kernel over rows grouped by expert, and the
// activations in its layout.
#include "experts.h"
#include "prefill_kernel.h"

namespace mi {
namespace {

// A block's activation layout has room for the widest block past the last slot.
int prep_slots(const GroupPlan& g) { return g.slots + (kPadTiles - 1) * kTileTok; }

// The activations of 8 slots x 1024 columns a block, in prefill_prep_kernel's layout
// (and its arithmetic), the rows' largest sizes known: a wave takes 8 slots x 8 runs of
// 8 values, so that the 16-byte pieces of a step's 8 neighbouring slots leave as whole
// 128-byte lines.  (A row a block left them to blocks on different chiplets, an eighth
// of a line each: 1018 rows of 14336 columns in 64 us, of 4096 in 16; now 37 together.)
constexpr int kPrepCols = 1024;
__global__ __launch_bounds__(256) void group_prep_kernel(const float* __restrict__ x, int cols, int slots, int share,
                                                         const int32_t* __restrict__ order,
                                                         const int32_t* __restrict__ count,
                                                         const float* __restrict__ top, int tops, int64_t top_stride,
                                                         uint8_t* __restrict__ work) {
  typedef float v4f __attribute__((ext_vector_type(4)));
  const Prep P = prep_layout(cols, slots);
  const int s0 = blockIdx.x * 8;
  if (s0 >= count[1]) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slot = s0 + (lane & 7), tile = slot >> 5, m = slot & 31;
  const int pair = order[slot];
  const int64_t from = (pair < 0 ? 0 : pair) / share;
  const float* row = x + from * cols;
  // the row's largest size: the wave's lanes of a slot, then the waves
  __shared__ float most[4][8];
  float mx = 0.0f;
  for (int j = 8 * wave + (lane >> 3); j < tops; j += 32) mx = fmaxf(mx, top[j * top_stride + from]);
  mx = fmaxf(mx, __uint_as_float(lanes::dpp<0x128>(__float_as_uint(mx))));  // row_ror:8
  auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
  mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
  mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  if (lane < 8) most[wave][lane] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(most[0][lane & 7], most[1][lane & 7]), fmaxf(most[2][lane & 7], most[3][lane & 7]));
  const int e = pair < 0 ? 0 : scale_exp(mx);
  if (blockIdx.y == 0 && threadIdx.x < 8) ((float*)(work + P.xs))[slot] = ldexpf(1.0f, e);
  uint8_t* xp = work + P.xp + (size_t)tile * P.ks * 2048 + 16 * m;
  _Float16* xm = (_Float16*)(work + P.xm) + (size_t)tile * P.nch * 512 + 8 * m;
  const int n8 = cols >> 3;
  constexpr int kRounds = kPrepCols / 8 / 32;
  v4f v[kRounds][2];
#pragma unroll
  for (int k = 0; k < kRounds; k++) {
    const int i = min((int)blockIdx.y * (kPrepCols / 8) + 32 * k + 8 * wave + (lane >> 3), n8 - 1);
    v[k][0] = *(const v4f*)(row + 8 * i);
    v[k][1] = *(const v4f*)(row + 8 * i + 4);
  }
#pragma unroll
  for (int k = 0; k < kRounds; k++) {
    // run i: values 8 i .. +8, half wave (i >> 1) & 1 of step 2 (i >> 2) + (i & 1)
    const int i = blockIdx.y * (kPrepCols / 8) + 32 * k + 8 * wave + (lane >> 3);
    v8h hi, lo;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      constexpr int kOrder[4] = {0, 2, 1, 3};  // the order of K
      const float f = ldexpf(v[k][j >> 2][kOrder[j & 3]], -e);
      _Float16 h, l;
      split_half(f, h, l);
      hi[j] = h;
      lo[j] = l;
      sum += f;
    }
    // the mean of a group's 32 values: its four runs are 8 lanes apart
    sum += __uint_as_float(lanes::dpp<0x128>(__float_as_uint(sum)));  // row_ror:8
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = (__uint_as_float(p[0]) + __uint_as_float(p[1])) * (1.0f / 32.0f);
    if (i >= n8) continue;  // (n8 is a multiple of 8: whole waves)
    uint8_t* dst = xp + (size_t)(2 * (i >> 2) + (i & 1)) * 2048 + 512 * ((i >> 1) & 1);
    *(v8h*)dst = hi;
    *(v8h*)(dst + 1024) = lo;
    if ((i & 3) == 0) {
      const int g = i >> 2;
      _Float16 h, l;
      split_half(sum, h, l);
      xm[(size_t)(g >> 3) * 512 + (g & 7)] = h;
      xm[(size_t)(g >> 3) * 512 + 256 + (g & 7)] = l;
    }
  }
  // groups past cols in the last chunk
  if (blockIdx.y == gridDim.y - 1 && wave == 0)
    for (int g = (cols >> 5) + (lane >> 3); g < 8 * P.nch; g += 8) {
      xm[(size_t)(g >> 3) * 512 + (g & 7)] = (_Float16)0.0f;
      xm[(size_t)(g >> 3) * 512 + 256 + (g & 7)] = (_Float16)0.0f;
    }
}

// How a block is cut, by the tiles it takes (prefill.hip's Shape): (1, 1, 4, 2),
// (1, 2, 4, 2) or, for the kinds with one scale a superblock and one limb, (2, 2, 4,
// 2), and (1, 4, 8, 1).
constexpr bool long_scales(int kind) { return kind == MI_Q4_K || kind == MI_Q5_K; }
int block_rows(int kind, int tiles) { return tiles == 1 ? 128 : tiles == 2 && !long_scales(kind) ? 128 : 256; }

template <int KIND, bool GLU>
int launch_kind(hipStream_t s, const RowSegs& sg, int cols, int act, const GroupPlan& g, int tiles, int64_t expert_bytes,
                int pairs, int splits, const void* prep, float* y, float* top) {
  const int rows = sg.end[0], nch = (cols + kChunk - 1) / kChunk;
  const Groups gr{(const GroupTile*)g.tiles, g.count, g.order, expert_bytes, (int64_t)pairs * rows, pairs, top};
  const int epi = GLU ? MI_EPI_GLU | act : MI_EPI_NONE, mine = block_rows(KIND, tiles) / (GLU ? 2 : 1);
  const dim3 grid((rows + mine - 1) / mine, g.blocks, splits);
#define MI_GT(R, T, W, G)                                                                                              \
  hipLaunchKernelGGL((group_kernel<KIND, R, T, W, G, GLU>), grid, dim3(W * G * 64), 0, s, sg, cols, prep_slots(g), \
                     (const uint8_t*)prep, (nch + splits - 1) / splits, y, (int64_t)rows, epi, gr)
  if (tiles == 1) MI_GT(1, 1, 4, 2);
  else if constexpr (long_scales(KIND)) MI_GT(2, 2, 4, 2);
  else if (tiles == 2) MI_GT(1, 2, 4, 2);
  else MI_GT(1, 4, 8, 1);
#undef MI_GT
  return hip_check(hipGetLastError(), "experts tile launch");
}

}  // namespace

// By the rows of an expert, on average.  us a product by tiles a block 1 / 2 / 4 (Q4_K's
// 2: (2, 2, 4, 2)), 64 experts of 2048x1024 and 8 of 14336x4096:
//   rows           16              38              64              100             160
//   Q4_K 64   49 / 53         63 / 76         85 / 87         125 / 125       180 / 174
//   Q4_K 8    119 / 114       158 / 149       245 / 209       332 / 286       477 / 400
//   Q6_K 64   88 / 92 / 83    114 / 101 / 100 153 / 128 / 124 216 / 177 / 152 330 / 259 / 213
//   Q6_K 8    255 / 264 / 270 354 / 280 / 306 503 / 381 / 313 697 / 475 / 421 1045 / 706 / 589
//   Q8_0 64   68 / 69 / 67    88 / 78 / 84    119 / 98 / 98   170 / 132 / 127 270 / 203 / 192
//   Q8_0 8    221 / 220 / 238 299 / 249 / 255 426 / 332 / 279 588 / 436 / 381 833 / 585 / 502
// (24 rows: Q6_K 102 / 92, 307 / 266, Q8_0 77 / 73, 261 / 240.)
int group_tiles(int kind, int32_t pairs, int32_t experts) {
  const int each = pairs / experts;
  if (long_scales(kind)) return each < 56 ? 1 : 2;
  return each < 24 ? 1 : each < 56 ? 2 : 4;
}

// Parts of K (in whole 256-value chunks): while the blocks that the experts take on
// average are few for the chip and a part stays eight chunks long.
int group_splits(int kind, int32_t rows, int32_t cols, int32_t pairs, int32_t experts, int32_t tiles_a_block) {
  const int64_t lists = pairs / (32 * tiles_a_block) + (std::min(pairs, experts) + 1) / 2;
  const int br = block_rows(kind, tiles_a_block), nch = (cols + kChunk - 1) / kChunk;
  const int64_t blocks = lists * ((rows + br - 1) / br);
  int z = 1;
  while (z < 8 && blocks * 2 * z <= 4 * cu_count() && nch >= 16 * z) z *= 2;
  return z;
}

int group_most_splits(int32_t cols) {
  const int nch = (cols + kChunk - 1) / kChunk;
  int z = 1;
  while (z < 8 && nch >= 16 * z) z *= 2;
  return z;
}

GroupPlan group_plan(void* work, int32_t pairs, int32_t experts, int32_t tiles_a_block) {
  GroupPlan g{};
  const int64_t some = std::min(pairs, experts);  // experts that have a pair
  g.slots = (int32_t)(32 * (pairs / 32 + some));
  g.blocks = (int32_t)(pairs / (32 * tiles_a_block) + some);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    void* p = work ? (char*)work + at : nullptr;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  g.count = (int32_t*)take(8);
  g.xtop = (float*)take(4 * (size_t)pairs);
  g.order = (int32_t*)take(4 * (size_t)g.slots);
  g.tiles = take(sizeof(GroupTile) * (size_t)(pairs / 32 + some));
  g.bytes = at;
  return g;
}

size_t group_prep_bytes(int32_t cols, const GroupPlan& g) { return prep_layout(cols, prep_slots(g)).total; }

int group_tops(int kind, int32_t rows, int32_t tiles_a_block) {
  const int mine = block_rows(kind, tiles_a_block) / 2;
  return (rows + mine - 1) / mine;
}

int launch_group_prep(hipStream_t s, const float* x, int32_t cols, int32_t pairs, int32_t share, const float* top,
                      int32_t tops, const GroupPlan& g, void* prep) {
  hipLaunchKernelGGL(group_prep_kernel, dim3(g.slots / 8, (cols + kPrepCols - 1) / kPrepCols), dim3(256), 0, s, x, cols,
                     prep_slots(g), share, g.order, g.count, top, tops, (int64_t)pairs, (uint8_t*)prep);
  return hip_check(hipGetLastError(), "experts activation launch");
}

int launch_group_tile(hipStream_t s, int kind, const void* w0, const void* w1, int64_t row_bytes, int32_t rows,
                      int32_t cols, int32_t act, const GroupPlan& g, int32_t tiles_a_block, int32_t pairs, int32_t splits,
                      const void* prep, float* y, float* top) {
  RowSegs sg = rows::one_matrix(w0, row_bytes, rows);
  if (w1) sg.w[1] = (const uint8_t*)w1;
  const int64_t eb = rows * row_bytes;
#define MI_GK(K)                                                                                               \
  case K:                                                                                                      \
    return w1 ? launch_kind<K, true>(s, sg, cols, act, g, tiles_a_block, eb, pairs, splits, prep, y, top)      \
              : launch_kind<K, false>(s, sg, cols, act, g, tiles_a_block, eb, pairs, splits, prep, y, nullptr)
  switch (kind) {
    MI_GK(MI_Q4_K);
    MI_GK(MI_Q5_K);
    MI_GK(MI_Q6_K);
    MI_GK(MI_Q8_0);
    MI_GK(MI_Q4_0);
    MI_GK(MI_Q4_1);
    MI_GK(MI_Q5_0);
    MI_GK(MI_Q5_1);
  }
#undef MI_GK
  return fail(MI_ERR_KIND, "experts: ggml type %d has no tile", kind);
}

}  // namespace mi
