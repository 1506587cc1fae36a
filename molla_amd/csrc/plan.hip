// plan.hip -- the plans of a step over drafted tokens, gfx950: which cell each
// new position gets (mi_page_plan) and what each node of a tree sees
// (mi_tree_plan).  No counterpart in the reference, whose host fills the paging
// vectors (gpu.mojo:571 DevicePaging).  Both are small integer work, bound by
// the launch and a chain of a few memory latencies.
#include "mi_internal.h"

namespace mi {
namespace {

// a + b of values from 0 to `most`, at most that (their sum may pass 31 bits)
__device__ __forceinline__ int capped(int a, int b, int most) {
  return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)most);
}

// Inclusive sum over a block of T threads, each partial sum at most `most` (with
// values at least 0 the capped sum is associative); wsum: an int a wave, of LDS.
template <int T>
__device__ __forceinline__ int scan_block(int v, int most, int* wsum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v = capped(v, u, most);
  }
  __syncthreads();  // (wsum of an earlier scan has been read)
  if (lane == 63) wsum[wave] = v;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < T / 64 - 1; w++) before = capped(before, w < wave ? wsum[w] : 0, most);
  return capped(before, v, most);
}

// Every block of T threads scans all requests (at most T * PER, from the cache)
// and then fills its share of the token rows: no second launch, and nothing
// between blocks.  A position that is a multiple of the page opens a new page:
// pages a request holds are full up to its length, but for the last one.  (All
// positions are below 2^32: a length and a row of tokens are below 2^31.)
template <int T, int PER>
__global__ __launch_bounds__(T) void page_plan_kernel(PagePlan p) {
  __shared__ int start[T * PER + 1];   // of each request's new tokens
  __shared__ int before[T * PER + 1];  // new pages of the requests ahead
  __shared__ int wsum[T / 64];
  const int tid = threadIdx.x, b0 = tid * PER;
  const uint32_t page = p.page, cap = (uint32_t)min<int64_t>(p.max_pos, 0xffffffff);  // positions there is room for
  auto pages_of = [&](uint32_t n) { return min(n, cap) / page + (min(n, cap) % page != 0); };
  int len[PER], n[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const bool live = b0 + i < p.batch;
    len[i] = live ? max(p.lengths[b0 + i], 0) : 0;
    n[i] = live ? min(max(p.news[b0 + i], 0), p.max_tokens) : 0;
    sum = capped(sum, n[i], p.max_tokens);
  }
  const int free0 = min(max(p.free_count[0], 0), p.free_size);
  // token rows: what does not fit into max_tokens is not planned
  int at = scan_block<T>(sum, p.max_tokens, wsum);
  {
    // (the capped total cannot be taken back: the exclusive sum again from the left)
    const int up = __shfl_up(at, 1);
    __shared__ int last[T / 64];
    if ((tid & 63) == 63) last[tid >> 6] = at;
    __syncthreads();
    at = (tid & 63) ? up : (tid ? last[(tid >> 6) - 1] : 0);
  }
  int grow[PER], pages = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int end = (int)min((uint32_t)at + n[i], (uint32_t)p.max_tokens);
    start[b0 + i] = at;
    grow[i] = (int)(pages_of((uint32_t)len[i] + (end - at)) - pages_of(len[i]));
    pages += grow[i];
    at = end;
  }
  if (tid == T - 1) start[T * PER] = at;
  // (a new page holds at least one new token, so their sum is below 2^31 too)
  const int upto = scan_block<T>(pages, 0x7fffffff, wsum);
  int ahead = upto - pages;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    before[b0 + i] = ahead;
    ahead += grow[i];
  }
  if (tid == T - 1) before[T * PER] = ahead;
  __syncthreads();
  const int total = start[T * PER];
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.batch; b += T) p.starts[b] = b < p.batch ? start[b] : total;
    if (tid == 0) {
      const int want = before[T * PER];
      p.free_left[0] = max(free0 - want, 0);
      p.free_left[1] = max(want - free0, 0);
    }
  }
  for (int64_t t64 = (int64_t)blockIdx.x * T + tid; t64 < total; t64 += (int64_t)gridDim.x * T) {
    const int t = (int)t64;
    int lo = 0, hi = p.batch;  // the last request that starts at or ahead of t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= t) lo = mid;
      else hi = mid;
    }
    const uint32_t held = max(p.lengths[lo], 0), pos = held + (t - start[lo]);
    int cell = -1;
    if (pos < cap) {
      const uint32_t col = pos / page, off = pos - col * page, have = held / page + (held % page != 0);
      int32_t* entry = p.table + (int64_t)lo * p.table_stride + col;
      int got;
      if (col < have) {
        got = *entry;
      } else {
        const int take = free0 - 1 - (before[lo] + (int)(col - have));
        got = take >= 0 ? p.free_pages[take] : -1;
        if (off == 0) *entry = got;
      }
      const int64_t c = (int64_t)got * page + off;
      if (got >= 0 && c <= 0x7fffffff) cell = (int)c;
      if (p.kv_index) p.kv_index[lo * p.index_stride + pos] = cell;
    }
    if (p.seq) p.seq[t] = lo;
    if (p.pos) p.pos[t] = (int)min(pos, 0x7fffffffu);
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
                                                                  int words, int batch, int tokens,
                                                                  int32_t* __restrict__ pos, uint32_t* __restrict__ mask) {
  __shared__ uint32_t set[kMaxTreeNodes / 32][kMaxTreeNodes];
  __shared__ int jump[kMaxTreeNodes], depth[kMaxTreeNodes];
  const int i = threadIdx.x;
  const uint32_t b = grid_block();
  if (b >= (uint32_t)batch) return;  // (the whole block)
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
  // up to 256 requests: one a thread of four waves, whose scan is short (64 requests
  // of a token 3.6 us, 5.7 with the larger block; 200 prompts of 274000 tokens 6.2 and
  // 8.8); a block for each T token rows, at most four (or one) a compute unit (for
  // each 4 T of them the 200 prompts take 7.4)
  const bool few = p.batch <= 256;
  const int T = few ? 256 : 1024;
  const int64_t want = ((int64_t)p.max_tokens + T - 1) / T, most = (int64_t)cu_count() * (few ? 4 : 1);
  const int blocks = (int)(want < most ? want : most);
  if (few) hipLaunchKernelGGL((page_plan_kernel<256, 1>), dim3(blocks), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((page_plan_kernel<1024, kMaxPlanBatch / 1024>), dim3(blocks), dim3(1024), 0, s, p);
  return hip_check(hipGetLastError(), "page_plan launch");
}

int launch_tree_plan(hipStream_t s, int32_t batch, const int32_t* starts, const int32_t* lengths,
                     const int32_t* parents, int32_t max_nodes, int32_t tokens, int32_t* pos, uint32_t* mask) {
  hipLaunchKernelGGL(tree_plan_kernel, grid_of(batch), dim3((max_nodes + 63) / 64 * 64), 0, s, starts, lengths, parents,
                     max_nodes, (max_nodes + 31) / 32, batch, tokens, pos, mask);
  return hip_check(hipGetLastError(), "tree_plan launch");
}

}  // namespace mi
