// experts_api.cpp -- the C ABI of the sparse-expert entry points
// (include/molla_mi.h): argument checks, workspaces, the launches of a call.
#include <algorithm>
#include <cmath>

#include "experts.h"

namespace mi {
int check_weight(const char* name, int kind, const void* w, int64_t row_bytes, int32_t rows, int32_t cols);

namespace {

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

// Whether two buffers share a byte.
bool meet(const void* a, size_t an, const void* b, size_t bn) {
  return a && b && (const char*)a < (const char*)b + bn && (const char*)b < (const char*)a + an;
}

// Stacked experts' matrices: one GGUF tensor of experts * rows rows.
int check_stack(const char* name, const mi_weight& w, int32_t experts, int32_t rows, int32_t cols) {
  if ((int64_t)experts * rows > INT32_MAX)
    return fail(MI_ERR_SHAPE, "%s: %d experts of %d rows are too many rows", name, experts, rows);
  if (w.rows != experts * rows || w.cols != cols)
    return fail(MI_ERR_SHAPE, "%s is %d x %d where %d experts of %d x %d are wanted", name, w.rows, w.cols, experts, rows,
                cols);
  const int rc = check_weight(name, w.kind, w.data, w.row_bytes, w.rows, w.cols);
  if (rc) return rc;
  // (every kind's tile takes an expert at its offset from there: rows are whole
  // multiples of the alignment that their kind's loads need)
  if ((uintptr_t)w.data & 15) return fail(MI_ERR_ALIGN, "%s: experts' matrices must be 16-byte aligned", name);
  return MI_OK;
}

int check_counts(const char* name, int32_t experts, int64_t pairs) {
  if (experts < 1 || experts > kMaxExperts) return fail(MI_ERR_SHAPE, "%s: %d experts, outside 1..%d", name, experts, kMaxExperts);
  if (pairs < 1 || pairs > kMaxPairs) return fail(MI_ERR_SHAPE, "%s: %lld rows, outside 1..%d", name, (long long)pairs, kMaxPairs);
  return MI_OK;
}

// Whether a call's pairs take the row kernel: up to three an expert, on average, or
// where the products are small beside the tile's chain of launches.  us of an MLP, rows
// / tile: 8 experts of 4096 x 14336, 16 pairs Q4_K 246 / 279, with Q6_K down 305 / 440,
// Q8_0 328 / 575, 24 pairs 345 / 316, 420 / 442, 434 / 580, 32 pairs 444 / 318, 536 /
// 439, 537 / 582; 16 of 2048 x 4096, 48 pairs Q4_K 124 / 108, Q8_0 132 / 186; 64 of 2048
// x 1024, 64 pairs 52 / 89, 69 / 151; 4 of 1024 x 2048, 24 pairs 41 / 43, 32 pairs 55 /
// 41.
bool few_pairs(int64_t pairs, int32_t experts, int64_t weights) {
  return pairs <= kFewPairs && (pairs <= 3 * (int64_t)experts || pairs * weights <= 48 << 20);
}

// Whether they take the matrix cores instead, eight rows an operand (experts_pack.hip):
// from where an expert's weights, unpacked once for all its pairs there, cost the row
// kernel more.  us of an MLP, rows (or the tile, the last) / packed, by pairs: 8 experts
// of 4096 x 14336 Q4_K 12 pairs 221 / 193, 16 244 / 213, 32 345 / 228, 64 330 / 289; with
// Q6_K down 12 272 / 269, 16 303 / 288, 32 448 / 377, 48 444 / 452; all Q6_K 16 405 /
// 435, 24 565 / 436, 48 698 / 691; 16 of 2048 x 4096 Q4_K 16 48 / 53, 24 69 / 67, 64 102 /
// 76; 64 of 2048 x 1024 48 43 / 53, 64 50 / 64.  A product of 8 of 14336 x 4096: Q4_K 12
// 61 / 63, 16 72 / 63, 64 108 / 88; Q6_K 16 152 / 165, 24 196 / 166, 64 262 / 258.
bool pack_pairs(int kind, int64_t pairs, int32_t experts) {
  if (!pack_fits(kind) || pairs > kFewPairs) return false;
  return kind == MI_Q4_K ? 2 * pairs >= 3 * (int64_t)experts && pairs <= 8 * (int64_t)experts
                         : pairs >= 3 * (int64_t)experts && pairs <= 6 * (int64_t)experts;
}
bool pack_mlp(const mi_experts& d, int64_t pairs) {
  if (!pack_pairs(d.gate.kind, pairs, d.experts)) return false;
  return d.down.kind == MI_Q4_K ||
         (d.down.kind == MI_Q6_K && pairs >= 2 * (int64_t)d.experts && pairs <= 5 * (int64_t)d.experts);
}

struct MatmulCarve {
  size_t x, plan, total;
};
// Few rows: their activations in matvec form.  Many: by slot, and the plan.  (The
// larger of the two where it hangs on the rows.)
MatmulCarve matmul_carve(int32_t experts, int32_t cols, int32_t share, int32_t pairs, bool few) {
  MatmulCarve c{};
  const size_t rows = up256((size_t)xq_token_bytes(cols) * (pairs / share));
  const GroupPlan g = group_plan(nullptr, pairs, experts, 1);  // (the most lists)
  const size_t tile = g.bytes + up256(group_prep_bytes(cols, g));
  c.x = few ? 0 : g.bytes;
  c.total = pairs > kFewPairs ? tile : few_pairs(pairs, experts, INT32_MAX) ? rows : std::max(rows, tile);
  return c;
}

struct MlpCarve {
  bool few, pack;
  size_t x, h, hx, part, plan, top, total;
  int gate_tiles, down_tiles, splits;  // many rows: tiles a block; parts of down's K
};
// Packed: h and part alone.  x: the input in the form its product reads; h: act(gate) *
// up in f32, top: the largest sizes in its rows; hx: the same as the down projection
// reads it; part: what that gives.
MlpCarve mlp_carve(const mi_experts& d, int32_t tokens, int32_t used) {
  const int32_t experts = d.experts, width = d.width, hidden = d.hidden;
  MlpCarve c{};
  const size_t pairs = (size_t)tokens * used;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += up256(bytes);
    return p;
  };
  c.few = few_pairs(pairs, experts, (int64_t)width * hidden);
  c.pack = pack_mlp(d, pairs);
  if (c.pack) {
    c.splits = pack_splits(width, hidden, pairs, experts);
    c.h = take(4 * (size_t)hidden * pairs);
    c.part = take(4 * (size_t)width * pairs * c.splits);
  } else if (c.few) {
    c.x = take((size_t)xq_token_bytes(width) * tokens);
    c.hx = take((size_t)xq_token_bytes(hidden) * pairs);
  } else {
    c.gate_tiles = group_tiles(d.gate.kind, (int32_t)pairs, experts);
    c.down_tiles = group_tiles(d.down.kind, (int32_t)pairs, experts);
    c.splits = group_splits(d.down.kind, width, hidden, (int32_t)pairs, experts, c.down_tiles);
    const GroupPlan g = group_plan(nullptr, (int32_t)pairs, experts, 1);
    c.plan = take(g.bytes);
    c.top = take(4 * pairs * group_tops(d.gate.kind, hidden, c.gate_tiles));
    // (the input is dead where h's form is made, h where the down projection writes)
    c.x = c.hx = take(std::max(group_prep_bytes(width, g), group_prep_bytes(hidden, g)));
    c.h = c.part = take(4 * (size_t)std::max<int64_t>((int64_t)width * c.splits, hidden) * pairs);
  }
  c.total = at;
  return c;
}

}  // namespace

// Of calls of up to as many tokens: a workspace of the largest holds a smaller call's,
// which may take another way or be cut into more parts.
size_t experts_workspace(const mi_experts& d, int32_t tokens, int32_t used) {
  const int64_t pairs = (int64_t)tokens * used, some = std::min<int64_t>(pairs, kFewPairs);
  const int32_t width = d.width, hidden = d.hidden;
  size_t most = up256((size_t)xq_token_bytes(width) * std::min<int64_t>(tokens, kFewPairs)) +
                up256((size_t)xq_token_bytes(hidden) * some);
  if (pack_fits(d.gate.kind) && pack_fits(d.down.kind))
    most = std::max(most, up256(4 * (size_t)hidden * some) + up256(4 * (size_t)width * some * pack_most_splits(hidden)));
  if (!few_pairs(pairs, d.experts, (int64_t)width * hidden)) {
    const GroupPlan g = group_plan(nullptr, (int32_t)pairs, d.experts, 1);
    const size_t top = 4 * (size_t)pairs * group_tops(d.gate.kind, hidden, 1);
    const int64_t row = std::max<int64_t>((int64_t)width * group_most_splits(hidden), hidden);
    most = std::max(most, up256(g.bytes) + up256(top) +
                              up256(std::max(group_prep_bytes(width, g), group_prep_bytes(hidden, g))) +
                              up256(4 * (size_t)row * pairs));
  }
  return most;
}

int launch_experts_mlp(hipStream_t s, const mi_experts& d, const float* x, int32_t tokens, int32_t used,
                       const int32_t* ids, const float* weights, float* out, bool add, void* work) {
  const int32_t pairs = tokens * used;
  const MlpCarve c = mlp_carve(d, tokens, used);
  char* base = (char*)work;
  int rc;
  if (c.pack) {
    float *h = (float*)(base + c.h), *part = (float*)(base + c.part);
    if ((rc = launch_expert_pack(s, d.gate.kind, d.gate.data, d.up.data, d.gate.row_bytes, d.hidden, d.width, d.experts, x,
                                 used, ids, pairs, d.act, 1, h)))
      return rc;
    if ((rc = launch_expert_pack(s, d.down.kind, d.down.data, nullptr, d.down.row_bytes, d.width, d.hidden, d.experts, h, 1,
                                 ids, pairs, 0, c.splits, part)))
      return rc;
    return launch_expert_sum(s, part, ids, weights, d.width, tokens, used, d.experts, add, c.splits, out);
  }
  if (c.few) {
    const bool one = one_row_fits(d.width, used, pairs);
    if (!one && (rc = launch_quantize(s, x, d.width, tokens, base + c.x))) return rc;
    ExpertRows a{};
    a.w0 = d.gate.data;
    a.w1 = d.up.data;
    a.row_bytes = d.gate.row_bytes;
    a.rows = d.hidden;
    a.cols = d.width;
    a.experts = d.experts;
    a.xq = base + c.x;
    a.x = one ? x : nullptr;
    a.share = used;
    a.pairs = pairs;
    a.ids = ids;
    a.act = d.act;
    a.xq_out = base + c.hx;
    if ((rc = launch_expert_rows(s, d.gate.kind, a))) return rc;
    ExpertRows b{};
    b.w0 = d.down.data;
    b.row_bytes = d.down.row_bytes;
    b.rows = d.width;
    b.cols = d.hidden;
    b.experts = d.experts;
    b.xq = base + c.hx;
    b.pairs = pairs;
    b.ids = ids;
    b.y = out;
    b.weights = weights;
    b.used = used;
    b.add = add;
    return launch_expert_rows(s, d.down.kind, b);
  }
  float *h = (float*)(base + c.h), *part = (float*)(base + c.part), *top = (float*)(base + c.top);
  void *xp = base + c.x, *hp = base + c.hx;
  const int ta = c.gate_tiles, tb = c.down_tiles;
  GroupPlan g = group_plan(base + c.plan, pairs, d.experts, ta);
  if ((rc = launch_group_plan(s, ids, pairs, d.experts, ta, g, x, tokens, d.width))) return rc;
  if ((rc = launch_group_prep(s, x, d.width, pairs, used, g.xtop, 1, g, xp))) return rc;
  if ((rc = launch_group_tile(s, d.gate.kind, d.gate.data, d.up.data, d.gate.row_bytes, d.hidden, d.width, d.act, g, ta,
                              pairs, 1, xp, h, top)))
    return rc;
  if (tb != ta) {
    // (other block lists; the slots may be others too, each pair's row is the same)
    g = group_plan(base + c.plan, pairs, d.experts, tb);
    if ((rc = launch_group_plan(s, ids, pairs, d.experts, tb, g, nullptr, 0, 0))) return rc;
  }
  if ((rc = launch_group_prep(s, h, d.hidden, pairs, 1, top, group_tops(d.gate.kind, d.hidden, ta), g, hp))) return rc;
  if ((rc = launch_group_tile(s, d.down.kind, d.down.data, nullptr, d.down.row_bytes, d.width, d.hidden, 0, g, tb, pairs,
                              c.splits, hp, part)))
    return rc;
  return launch_expert_sum(s, part, ids, weights, d.width, tokens, used, d.experts, add, c.splits, out);
}

// The descriptor of a gated MLP of experts.
int check_experts(const char* name, const mi_experts* d) {
  if (!d) return fail(MI_ERR_ARG, "%s: null descriptor", name);
  int rc = check_counts(name, d->experts, 1);
  if (rc) return rc;
  if (d->width <= 0 || d->hidden <= 0 || d->width % 64 || d->hidden % 64)
    return fail(MI_ERR_SHAPE, "%s: width %d / hidden %d must be positive multiples of 64", name, d->width, d->hidden);
  if (d->act != 0 && d->act != MI_ACT_GELU) return fail(MI_ERR_ARG, "%s: act %d is neither silu (0) nor gelu", name, d->act);
  if ((rc = check_stack("experts' gate", d->gate, d->experts, d->hidden, d->width))) return rc;
  if ((rc = check_stack("experts' up", d->up, d->experts, d->hidden, d->width))) return rc;
  if ((rc = check_stack("experts' down", d->down, d->experts, d->width, d->hidden))) return rc;
  if (d->gate.kind != d->up.kind)
    return fail(MI_ERR_KIND, "%s: gate of type %d and up of type %d: they are of one", name, d->gate.kind, d->up.kind);
  return MI_OK;
}

int check_router(const char* name, const float* router, int32_t width, int32_t experts, int32_t used, int32_t tokens,
                 int32_t flags, float scale) {
  if (!router) return fail(MI_ERR_ARG, "%s: null router", name);
  if (width <= 0 || width % 4) return fail(MI_ERR_SHAPE, "%s: a router of %d values a row, not a multiple of 4", name, width);
  if (tokens < 1 || tokens > kMaxPrefill) return fail(MI_ERR_ARG, "%s: tokens %d outside 1..%d", name, tokens, kMaxPrefill);
  const int rc = check_counts(name, experts, 1);
  if (rc) return rc;
  if (used < 1 || used > std::min(experts, kMaxUsed))
    return fail(MI_ERR_SHAPE, "%s: %d of %d experts a token, at most %d", name, used, experts, kMaxUsed);
  if (flags & ~(MI_ROUTER_SIGMOID | MI_ROUTER_NORM)) return fail(MI_ERR_ARG, "%s: unknown router bits 0x%x", name, flags);
  if (!std::isfinite(scale)) return fail(MI_ERR_ARG, "%s: the weights' scale has to be finite", name);
  if ((uintptr_t)router & 15) return fail(MI_ERR_ALIGN, "%s: the router must be 16-byte aligned", name);
  return MI_OK;
}

size_t router_workspace(int32_t experts, int32_t tokens) { return up256(sizeof(double) * (size_t)experts * tokens); }

}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_router_workspace(int32_t experts, int32_t tokens) {
  if (experts < 1 || experts > kMaxExperts || tokens < 1 || tokens > kMaxPrefill) return 0;
  return router_workspace(experts, tokens);
}

int mi_router(mi_stream stream, const float* x, const float* router, const float* bias, int32_t width, int32_t experts,
              int32_t used, int32_t tokens, int32_t flags, float scale, int32_t* ids, float* weights, void* work,
              size_t work_bytes) {
  if (!x || !ids || !weights) return fail(MI_ERR_ARG, "router: null pointer");
  int rc = check_router("router", router, width, experts, used, tokens, flags, scale);
  if (rc) return rc;
  if ((uintptr_t)x & 15) return fail(MI_ERR_ALIGN, "router: the input must be 16-byte aligned");
  const size_t picks = 4 * (size_t)tokens * used, xb = 4 * (size_t)tokens * width, rb = 4 * (size_t)experts * width;
  if (meet(ids, picks, weights, picks) || meet(ids, picks, bias, 4 * (size_t)experts) ||
      meet(weights, picks, bias, 4 * (size_t)experts))
    return fail(MI_ERR_ARG, "router: an output lies in another buffer");
  const size_t need = router_workspace(experts, tokens);
  if (!work || ((uintptr_t)work & 255) || work_bytes < need)
    return fail(MI_ERR_WORKSPACE, "router: workspace of %zu bytes (256-aligned), %zu needed", work_bytes, need);
  if (meet(work, need, x, xb) || meet(work, need, router, rb) || meet(work, need, bias, 4 * (size_t)experts) ||
      meet(work, need, ids, picks) || meet(work, need, weights, picks))
    return fail(MI_ERR_ARG, "router: the workspace lies in another buffer");
  return launch_router((hipStream_t)stream, x, router, bias, width, experts, used, tokens, flags, scale, ids, weights,
                       work);
}

size_t mi_experts_matmul_workspace(int32_t experts, int32_t cols, int32_t share, int32_t pairs) {
  if (experts < 1 || experts > kMaxExperts || cols <= 0 || cols % 64 || pairs < 1 || pairs > kMaxPairs || share < 1 ||
      pairs % share)
    return 0;
  return matmul_carve(experts, cols, share, pairs, true).total;
}

int mi_experts_matmul(mi_stream stream, int kind, const void* w, int64_t row_bytes, int32_t experts, int32_t rows,
                      int32_t cols, const float* x, int32_t share, const int32_t* ids, int32_t pairs, float* y,
                      void* work, size_t work_bytes) {
  int rc = check_counts("experts_matmul", experts, pairs);
  if (rc) return rc;
  if (rows < 1) return fail(MI_ERR_SHAPE, "experts_matmul: experts of %d rows", rows);
  if ((int64_t)experts * rows > INT32_MAX)
    return fail(MI_ERR_SHAPE, "experts_matmul: %d experts of %d rows are too many rows", experts, rows);
  if ((rc = check_stack("experts_matmul", mi_weight{w, kind, experts * rows, cols, row_bytes}, experts, rows, cols))) return rc;
  if (!x || !ids || !y) return fail(MI_ERR_ARG, "experts_matmul: null pointer");
  if (share < 1 || pairs % share)
    return fail(MI_ERR_SHAPE, "experts_matmul: %d rows, %d for each row of the input", pairs, share);
  if (((uintptr_t)x | (uintptr_t)y) & 15)
    return fail(MI_ERR_ALIGN, "experts_matmul: the input and the output must be 16-byte aligned");
  const size_t xb = 4 * (size_t)(pairs / share) * cols, yb = 4 * (size_t)pairs * rows;
  if (meet(y, yb, x, xb) || meet(y, yb, ids, 4 * (size_t)pairs) || meet(y, yb, w, (size_t)experts * rows * row_bytes))
    return fail(MI_ERR_ARG, "experts_matmul: the output lies in an input");
  const bool few = few_pairs(pairs, experts, (int64_t)rows * cols);
  const MatmulCarve c = matmul_carve(experts, cols, share, pairs, few);
  if (!work || ((uintptr_t)work & 255) || work_bytes < c.total)
    return fail(MI_ERR_WORKSPACE, "experts_matmul: workspace of %zu bytes (256-aligned), %zu needed", work_bytes, c.total);
  if (meet(work, c.total, x, xb) || meet(work, c.total, y, yb) || meet(work, c.total, ids, 4 * (size_t)pairs) ||
      meet(work, c.total, w, (size_t)experts * rows * row_bytes))
    return fail(MI_ERR_ARG, "experts_matmul: the workspace lies in another buffer");
  hipStream_t s = (hipStream_t)stream;
  char* base = (char*)work;
  if (pack_pairs(kind, pairs, experts))
    return launch_expert_pack(s, kind, w, nullptr, row_bytes, rows, cols, experts, x, share, ids, pairs, 0, 1, y);
  if (few) {
    const bool one = one_row_fits(cols, share, pairs);
    if (!one && (rc = launch_quantize(s, x, cols, pairs / share, base + c.x))) return rc;
    ExpertRows a{};
    a.w0 = w;
    a.row_bytes = row_bytes;
    a.rows = rows;
    a.cols = cols;
    a.experts = experts;
    a.xq = base + c.x;
    a.x = one ? x : nullptr;
    a.share = share;
    a.pairs = pairs;
    a.ids = ids;
    a.y = y;
    return launch_expert_rows(s, kind, a);
  }
  const int tiles = group_tiles(kind, pairs, experts);
  const GroupPlan g = group_plan(base + c.plan, pairs, experts, tiles);
  if ((rc = launch_group_plan(s, ids, pairs, experts, tiles, g, x, pairs / share, cols))) return rc;
  if ((rc = launch_group_prep(s, x, cols, pairs, share, g.xtop, 1, g, base + c.x))) return rc;
  return launch_group_tile(s, kind, w, nullptr, row_bytes, rows, cols, 0, g, tiles, pairs, 1, base + c.x, y);
}

size_t mi_experts_workspace(const mi_experts* d, int32_t tokens, int32_t used) {
  if (!d || d->experts < 1 || d->experts > kMaxExperts || d->width <= 0 || d->hidden <= 0 || d->width % 64 ||
      d->hidden % 64 || tokens < 1 || tokens > kMaxPrefill || used < 1 || used > kMaxUsed ||
      (int64_t)tokens * used > kMaxPairs)
    return 0;
  return experts_workspace(*d, tokens, used);
}

int mi_experts_mlp(mi_stream stream, const mi_experts* d, const float* x, int32_t tokens, int32_t used,
                   const int32_t* ids, const float* weights, float* out, int32_t epi, void* work, size_t work_bytes) {
  int rc = check_experts("experts_mlp", d);
  if (rc) return rc;
  if (!x || !ids || !weights || !out) return fail(MI_ERR_ARG, "experts_mlp: null pointer");
  if (tokens < 1 || tokens > kMaxPrefill)
    return fail(MI_ERR_ARG, "experts_mlp: tokens %d outside 1..%d", tokens, kMaxPrefill);
  if (used < 1 || used > kMaxUsed) return fail(MI_ERR_SHAPE, "experts_mlp: %d experts a token, outside 1..%d", used, kMaxUsed);
  if ((rc = check_counts("experts_mlp", d->experts, (int64_t)tokens * used))) return rc;
  if (epi != MI_EPI_NONE && epi != MI_EPI_ADD) return fail(MI_ERR_ARG, "experts_mlp: epilogue 0x%x is neither none nor add", epi);
  if (((uintptr_t)x | (uintptr_t)out) & 15)
    return fail(MI_ERR_ALIGN, "experts_mlp: the input and the output must be 16-byte aligned");
  const size_t xb = 4 * (size_t)tokens * d->width, pb = 4 * (size_t)tokens * used;
  // (of the experts' matrices)
  auto in_stacks = [d](const void* p, size_t n) {
    for (const mi_weight* w : {&d->gate, &d->up, &d->down})
      if (meet(p, n, w->data, (size_t)w->rows * w->row_bytes)) return true;
    return false;
  };
  if (meet(out, xb, ids, pb) || meet(out, xb, weights, pb) || in_stacks(out, xb))
    return fail(MI_ERR_ARG, "experts_mlp: the output lies in an input");
  const size_t need = experts_workspace(*d, tokens, used);
  if (!work || ((uintptr_t)work & 255) || work_bytes < need)
    return fail(MI_ERR_WORKSPACE, "experts_mlp: workspace of %zu bytes (256-aligned), %zu needed", work_bytes, need);
  if (meet(work, need, x, xb) || meet(work, need, out, xb) || meet(work, need, ids, pb) || meet(work, need, weights, pb) ||
      in_stacks(work, need))
    return fail(MI_ERR_ARG, "experts_mlp: the workspace lies in another buffer");
  return launch_experts_mlp((hipStream_t)stream, *d, x, tokens, used, ids, weights, out, epi == MI_EPI_ADD, work);
}

}  // extern "C"
