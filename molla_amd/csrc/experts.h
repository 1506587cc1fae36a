// experts.h -- what the sparse-expert kernels and their callers share.
#pragma once

#include "mi_internal.h"

namespace mi {

constexpr int kMaxExperts = 512;       // a plan's thread each
constexpr int kMaxUsed = 64;           // of a token: a lane each
constexpr int kMaxPairs = 1 << 20;     // of a call
constexpr int kFewPairs = 64;          // up to here the row kernel: a lane each

int launch_router(hipStream_t s, const float* x, const float* router, const float* bias, int32_t width, int32_t experts,
                  int32_t used, int32_t tokens, int32_t flags, float scale, int32_t* ids, float* weights, void* work);

// A few pairs' products (experts_rows.h), x in matvec form (xq), or one row of floats
// for every pair (x; one_row_fits): y[p] = W[ids[p]] .
// x[p / share]; with w1, act(w0) * w1 in matvec form to xq_out instead; with
// weights, y[t] (+)= sum over k < used of weights[t * used + k] * W[ids[t * used +
// k]] . x[t * used + k].
struct ExpertRows {
  const void *w0, *w1;
  int64_t row_bytes;
  int32_t rows, cols, experts;
  const void* xq;
  const float* x;
  int32_t share, pairs;
  const int32_t* ids;
  float* y;
  // GLU
  int32_t act;
  void* xq_out;
  // the weighted sum
  const float* weights;
  int32_t used, add;
};
bool one_row_fits(int32_t cols, int32_t share, int32_t pairs);
int launch_expert_rows(hipStream_t s, int kind, const ExpertRows& a);
int launch_expert_sum(hipStream_t s, const float* part, const int32_t* ids, const float* weights, int32_t width,
                      int32_t tokens, int32_t used, int32_t experts, bool add, int32_t splits, float* out);

// A few pairs' products on the matrix cores (experts_pack.hip): y[z][p] = W[ids[p]] .
// x[p / share] over part z of the columns; with w1, act(w0) * w1.
int launch_expert_pack(hipStream_t s, int kind, const void* w0, const void* w1, int64_t row_bytes, int32_t rows,
                       int32_t cols, int32_t experts, const float* x, int32_t share, const int32_t* ids, int32_t pairs,
                       int32_t act, int32_t splits, float* y);
bool pack_fits(int kind);
int pack_most_splits(int32_t cols);
int pack_splits(int32_t rows, int32_t cols, int32_t pairs, int32_t experts);

// The lists of many pairs by expert: order[slot] (the pair, -1 behind an expert's
// last), the blocks' tiles (experts_tile.hip), count (of lists, of slots), and the
// largest size in each row of x.
struct GroupPlan {
  int32_t *order, *count;
  float* xtop;
  void* tiles;
  int32_t slots;   // the most that are numbered, whole tiles of 32
  int32_t blocks;  // the most lists
  size_t bytes;
};
// x: rows x cols; null: they stay as an earlier plan left them.
int launch_group_plan(hipStream_t s, const int32_t* ids, int32_t pairs, int32_t experts, int32_t tiles_a_block,
                      const GroupPlan& g, const float* x, int32_t rows, int32_t cols);

// Products of many pairs on the matrix cores: a plan, the activations by slot,
// then the products.  group_plan lays a plan out in `work` (null: sizes only).
GroupPlan group_plan(void* work, int32_t pairs, int32_t experts, int32_t tiles_a_block);
int group_tiles(int kind, int32_t pairs, int32_t experts);  // 32-slot tiles a block
// Parts of K of a product whose sum a later launch takes.
int group_splits(int kind, int32_t rows, int32_t cols, int32_t pairs, int32_t experts, int32_t tiles_a_block);
int group_most_splits(int32_t cols);
size_t group_prep_bytes(int32_t cols, const GroupPlan& g);
// Row p / share of x for pair p, whose largest size is that among top[j * pairs + p /
// share], j < tops.
int launch_group_prep(hipStream_t s, const float* x, int32_t cols, int32_t pairs, int32_t share, const float* top,
                      int32_t tops, const GroupPlan& g, void* prep);
// y[z][p] = W[expert of p] . x over part z of K; with w1, act(w0) * w1, and group_tops
// of its rows' largest sizes to top[j * pairs + p].  tiles_a_block as the plan's.
int group_tops(int kind, int32_t rows, int32_t tiles_a_block);
int launch_group_tile(hipStream_t s, int kind, const void* w0, const void* w1, int64_t row_bytes, int32_t rows,
                      int32_t cols, int32_t act, const GroupPlan& g, int32_t tiles_a_block, int32_t pairs, int32_t splits,
                      const void* prep, float* y, float* top = nullptr);

// experts_api.cpp: the MLP, checked, and its checks for the layer.
size_t experts_workspace(const mi_experts& d, int32_t tokens, int32_t used);
int launch_experts_mlp(hipStream_t s, const mi_experts& d, const float* x, int32_t tokens, int32_t used,
                       const int32_t* ids, const float* weights, float* out, bool add, void* work);
int check_experts(const char* name, const mi_experts* d);
int check_router(const char* name, const float* router, int32_t width, int32_t experts, int32_t used, int32_t tokens,
                 int32_t flags, float scale);
size_t router_workspace(int32_t experts, int32_t tokens);

}  // namespace mi
