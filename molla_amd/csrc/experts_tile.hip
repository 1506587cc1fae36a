// experts_tile.hip -- products of many rows with stacked experts' matrices on the
// matrix cores: prefill_kernel.h's kernel over rows grouped by expert.
#include "experts.h"
#include "prefill_kernel.h"

namespace mi {
namespace {

// A block's activation layout has room for the widest block past the last slot.
int prep_slots(const GroupPlan& g) { return g.slots + (kPadTiles - 1) * kTileTok; }

template <int KIND, bool GLU>
int launch_kind(hipStream_t s, const RowSegs& sg, int cols, int act, const GroupPlan& g, int tiles, int64_t expert_bytes,
                const void* prep, float* y) {
  const int rows = sg.end[0], nch = (cols + kChunk - 1) / kChunk;
  const Groups gr{(const GroupTile*)g.tiles, g.count, g.order, expert_bytes};
  const int epi = GLU ? MI_EPI_GLU | act : MI_EPI_NONE;
#define MI_GT(R, T, W, G)                                                                                              \
  do {                                                                                                                 \
    const int mine = W * R * 32 / (GLU ? 2 : 1);                                                                       \
    hipLaunchKernelGGL((prefill_kernel<KIND, R, T, W, G, Groups, GLU>), dim3((rows + mine - 1) / mine, g.blocks),      \
                       dim3(W * G * 64), 0, s, sg, cols, prep_slots(g), (const uint8_t*)prep, nch, y, (int64_t)rows, epi, \
                       nullptr, nullptr, gr);                                                                          \
  } while (0)
  if (tiles == 1) MI_GT(1, 1, 4, 2);
  else if constexpr (KIND == MI_Q6_K) MI_GT(1, 4, 8, 1);
  else MI_GT(2, 2, 4, 2);
#undef MI_GT
  return hip_check(hipGetLastError(), "experts tile launch");
}

}  // namespace

int group_tiles(int kind, int32_t pairs, int32_t experts) {
  if (pairs <= 32 * (int64_t)experts) return 1;
  return kind == MI_Q6_K ? 4 : 2;
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
  g.count = (int32_t*)take(4);
  g.tiles = take(sizeof(GroupTile) * (size_t)g.blocks);
  g.slot = (int32_t*)take(4 * (size_t)pairs);
  g.order = (int32_t*)take(4 * (size_t)g.slots);
  g.bytes = at;
  return g;
}

size_t group_prep_bytes(int32_t cols, const GroupPlan& g) { return prep_layout(cols, prep_slots(g)).total; }

int launch_group_prep(hipStream_t s, const float* x, int32_t cols, int32_t pairs, int32_t share, const GroupPlan& g,
                      void* prep) {
  hipLaunchKernelGGL(prefill_prep_kernel<Slots>, dim3(pairs), dim3(256), 0, s, x, cols, prep_slots(g), (uint8_t*)prep,
                     Slots{g.slot, share});
  return hip_check(hipGetLastError(), "experts activation launch");
}

int launch_group_tile(hipStream_t s, int kind, const void* w0, const void* w1, int64_t row_bytes, int32_t rows,
                      int32_t cols, int32_t act, const GroupPlan& g, int32_t tiles_a_block, const void* prep, float* y) {
  RowSegs sg = rows::one_matrix(w0, row_bytes, rows);
  if (w1) sg.w[1] = (const uint8_t*)w1;
  const int64_t eb = rows * row_bytes;
#define MI_GK(K)                                                                                          \
  case K:                                                                                                 \
    return w1 ? launch_kind<K, true>(s, sg, cols, act, g, tiles_a_block, eb, prep, y)                     \
              : launch_kind<K, false>(s, sg, cols, act, g, tiles_a_block, eb, prep, y)
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
