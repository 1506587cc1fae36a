// plan.hip -- the plans of a step over drafted tokens, gfx950: which cell each
// new position gets (mi_page_plan) and what each node of a tree sees
// (mi_tree_plan).  No counterpart in the reference, whose host fills the paging
// vectors (gpu.mojo:571 DevicePaging).  Both are small integer work, bound by
// the launch and a chain of a few memory latencies.
#include "mi_internal.h"

namespace mi {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = kMaxPlanBatch / kPlanThreads;  // requests a thread scans

// Inclusive sum over a block of 1024, each partial sum at most `most` (with
// values at least 0 the capped sum is associative); wsum: 16 ints of LDS.
__device__ __forceinline__ int scan_block(int v, int most, int* wsum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v = min(v + u, most);
  }
  __syncthreads();  // (wsum of an earlier scan has been read)
  if (lane == 63) wsum[wave] = v;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; w++) before = min(before + wsum[w], most);
  return min(before + v, most);
}

// Every block scans all requests (at most 4096, four a thread, from the cache)
// and then fills its share of the token rows: no second launch, and nothing
// between blocks.  A position that is a multiple of the page opens a new page:
// pages a request holds are full up to its length, but for the last one.
__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(PagePlan p) {
  __shared__ int start[kMaxPlanBatch + 1];   // of each request's new tokens
  __shared__ int before[kMaxPlanBatch + 1];  // new pages of the requests ahead
  __shared__ int wsum[kPlanThreads / 64];
  const int tid = threadIdx.x, b0 = tid * kPlanPer;
  int len[kPlanPer], n[kPlanPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPlanPer; i++) {
    const bool live = b0 + i < p.batch;
    len[i] = live ? max(p.lengths[b0 + i], 0) : 0;
    n[i] = live ? min(max(p.news[b0 + i], 0), p.max_tokens) : 0;
    sum = min(sum + n[i], p.max_tokens);
  }
  const int free0 = min(max(p.free_count[0], 0), p.free_size);
  // token rows: what does not fit into max_tokens is not planned
  int at = scan_block(sum, p.max_tokens, wsum);
  {
    // (the capped total cannot be taken back: the exclusive sum again from the left)
    const int up = __shfl_up(at, 1);
    __shared__ int last[kPlanThreads / 64];
    if ((tid & 63) == 63) last[tid >> 6] = at;
    __syncthreads();
    at = (tid & 63) ? up : (tid ? last[(tid >> 6) - 1] : 0);
  }
  int grow[kPlanPer], pages = 0;
#pragma unroll
  for (int i = 0; i < kPlanPer; i++) {
    const int end = min(at + n[i], p.max_tokens);
    const int64_t cap = p.max_pos;  // positions the table and the list have room for
    const int64_t have = (min<int64_t>(len[i], cap) + p.page - 1) / p.page;
    const int64_t need = (min<int64_t>((int64_t)len[i] + (end - at), cap) + p.page - 1) / p.page;
    start[b0 + i] = at;
    grow[i] = (int)(need - have);
    pages += grow[i];
    at = end;
  }
  if (tid == kPlanThreads - 1) start[kMaxPlanBatch] = at;
  // (a new page holds at least one new token, so their sum is below 2^31 too)
  const int upto = scan_block(pages, 0x7fffffff, wsum);
  int ahead = upto - pages;
#pragma unroll
  for (int i = 0; i < kPlanPer; i++) {
    before[b0 + i] = ahead;
    ahead += grow[i];
  }
  if (tid == kPlanThreads - 1) before[kMaxPlanBatch] = ahead;
  __syncthreads();
  const int total = start[kMaxPlanBatch];
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.batch; b += kPlanThreads) p.starts[b] = b < p.batch ? start[b] : total;
    if (tid == 0) {
      const int want = before[kMaxPlanBatch];
      p.free_left[0] = max(free0 - want, 0);
      p.free_left[1] = max(want - free0, 0);
    }
  }
  for (int64_t t64 = (int64_t)blockIdx.x * kPlanThreads + tid; t64 < total; t64 += (int64_t)gridDim.x * kPlanThreads) {
    const int t = (int)t64;
    int lo = 0, hi = p.batch;  // the last request that starts at or ahead of t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int64_t held = max(p.lengths[lo], 0);
    const int64_t pos = held + (t - start[lo]);
    int cell = -1;
    if (pos < p.max_pos) {
      const int64_t col = pos / p.page, off = pos - col * p.page, have = (held + p.page - 1) / p.page;
      int32_t* entry = p.table + lo * p.table_stride + col;
      int page;
      if (col < have) {
        page = *entry;
      } else {
        const int take = free0 - 1 - (before[lo] + (int)(col - have));
        page = take >= 0 ? p.free_pages[take] : -1;
        if (off == 0) *entry = page;
      }
      const int64_t c = (int64_t)page * p.page + off;
      if (page >= 0 && c <= 0x7fffffff) cell = (int)c;
      if (p.kv_index) p.kv_index[lo * p.index_stride + pos] = cell;
    }
    if (p.seq) p.seq[t] = lo;
    if (p.pos) p.pos[t] = (int)min<int64_t>(pos, 0x7fffffff);
    p.cells[t] = cell;
  }
}

// A block is one sequence, a thread one node: each round joins a node's set
// with that of the node its chain has reached and doubles the reach, so a tree
// of depth d takes log2(d) rounds.  A parent that is not an earlier node of the
// sequence makes the node a root.
__global__ __launch_bounds__(kMaxTreeNodes) void tree_plan_kernel(const int32_t* __restrict__ starts,
                                                                  const int32_t* __restrict__ lengths,
                                                                  const int32_t* __restrict__ parents, int max_nodes,
                                                                  int words, int tokens, int32_t* __restrict__ pos,
                                                                  uint32_t* __restrict__ mask) {
  __shared__ uint32_t set[kMaxTreeNodes / 32][kMaxTreeNodes];
  __shared__ int jump[kMaxTreeNodes], depth[kMaxTreeNodes];
  const int b = blockIdx.x, i = threadIdx.x;
  const int s0 = min(max(starts[b], 0), tokens), s1 = min(max(starts[b + 1], s0), tokens);
  const int n = s1 - s0;
  const bool node = i < min(n, max_nodes);
  int up = node ? parents[s0 + i] : -1;
  if (up < 0 || up >= i) up = -1;
  int far = up >= 0 ? 1 : 0;
  uint32_t own[kMaxTreeNodes / 32];
#pragma unroll
  for (int w = 0; w < kMaxTreeNodes / 32; w++) {
    own[w] = node && w == (i >> 5) ? 1u << (i & 31) : 0u;
    if (w < words) set[w][i] = own[w];
  }
  jump[i] = up;
  depth[i] = far;
  while (__syncthreads_or(up >= 0)) {
    int next = -1, more = 0;
    if (up >= 0) {
      next = jump[up];
      more = depth[up];
#pragma unroll
      for (int w = 0; w < kMaxTreeNodes / 32; w++)
        if (w < words) own[w] |= set[w][up];
    }
    __syncthreads();
    up = next;
    far += more;
    jump[i] = up;
    depth[i] = far;
#pragma unroll
    for (int w = 0; w < kMaxTreeNodes / 32; w++)
      if (w < words) set[w][i] = own[w];
  }
  if (node) {
#pragma unroll
    for (int w = 0; w < kMaxTreeNodes / 32; w++)
      if (w < words) mask[(int64_t)(s0 + i) * words + w] = own[w];
    if (pos) pos[s0 + i] = (int)min<int64_t>((int64_t)max(lengths[b], 0) + far, 0x7fffffff);
  }
  // rows past the largest tree see nothing of it
  for (int t = s0 + max_nodes + i; t < s1; t += blockDim.x) {
    for (int w = 0; w < words; w++) mask[(int64_t)t * words + w] = 0;
    if (pos) pos[t] = max(lengths[b], 0);
  }
}

}  // namespace

int launch_page_plan(hipStream_t s, const PagePlan& p) {
  // a block for each 4096 token rows, at most one a compute unit
  const int64_t want = ((int64_t)p.max_tokens + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  const int blocks = (int)(want < cu_count() ? want : cu_count());
  hipLaunchKernelGGL(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, s, p);
  return hip_check(hipGetLastError(), "page_plan launch");
}

int launch_tree_plan(hipStream_t s, int32_t batch, const int32_t* starts, const int32_t* lengths,
                     const int32_t* parents, int32_t max_nodes, int32_t tokens, int32_t* pos, uint32_t* mask) {
  hipLaunchKernelGGL(tree_plan_kernel, dim3(batch), dim3((max_nodes + 63) / 64 * 64), 0, s, starts, lengths, parents,
                     max_nodes, (max_nodes + 31) / 32, tokens, pos, mask);
  return hip_check(hipGetLastError(), "tree_plan launch");
}

}  // namespace mi
