// experts_pack.hip -- products of a few rows an expert (up to kFewPairs rows in all)
// with stacked experts' Q4_K or Q6_K matrices on the matrix cores: v_mfma_f32_16x16x32_f16,
// gfx950.
//
// The arithmetic of prefill_kernel.h: a weight's code sc * q is an exact half, an
// activation two halves of its value over a power of two, the scales of a superblock
// multiply its sum, and the mins meet the means of 32 values in one more product.  Eight
// rows of activations fill the 16 rows of one operand, their high halves in rows 0..7 and
// their low halves in 8..15.
//
// What bounds it is the experts' weights, so nothing waits for anything else: a block
// takes its expert's rows of x as floats, kPackCols columns at a time, makes their halves
// itself (no launch ahead, no list of rows: a block finds its eight among the ids) and
// keeps them in LDS, the next columns on their
// way, while each wave streams its own 32 rows of weights, one or two superblocks
// ahead.  A chunk has a power of two a row, of the largest size in it.
//
// Fragments: lane l holds row l % 16 and the 8 values of a step's 32 that belong to
// kq = l / 16; result j of lane l is activation row 4 (l / 16) + j, weight row l % 16.
// A lane's two 16-byte loads of a superblock's nibbles are bytes 64 L + 16 kq on: the half
// kq % 2 of two groups of 32 values, one in the low and one in the high nibbles.  Step
// (L, nibble, half) takes 8 of the bytes; the activations lie in the same order.
#include "experts.h"
#include "prefill_kernel.h"

namespace mi {
namespace {

constexpr int kPackRows = 8;    // of activations an operand takes
constexpr int kPackCols = 512;  // columns of them in LDS at a time, in two buffers
constexpr int kPackWaves = 4;

typedef float v4f __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4f mfma16(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// A superblock of 16 rows: what a lane holds of it; step (L, up, half) of its codes (b1
// where codes have two limbs); what ends it.  SLOTS: superblocks in registers.
template <int KIND>
struct PackUnit;
template <>
struct PackUnit<MI_Q4_K> {
  static constexpr int SLOTS = 3, LIMBS = 1;
  static constexpr bool MINS = true;
  v4u h, q[2];
  // group g is nibble `up` of the lanes whose kq / 2 is `which`
  static __device__ __forceinline__ int up_of(int g) { return g & 1; }
  static __device__ __forceinline__ int which_of(int g) { return (g >> 1) & 1; }
  __device__ __forceinline__ void load(const uint8_t* row, int sb, int kq) {
    const uint8_t* p = row + (int64_t)sb * 144;
    h = *(const v4u*)p;
    q[0] = *(const v4u*)(p + 16 + 16 * kq);
    q[1] = *(const v4u*)(p + 80 + 16 * kq);
  }
  __device__ __forceinline__ void codes(int L, int up, int half, int kq, v8h& b0, v8h&) const {
    uint32_t lo, hi;
    kscales(h.y, h.w, lo, hi);
    const uint32_t word = L ? hi : lo, sel = 0x04000400u + 0x00020002u * (kq >> 1), mk = up ? kHigh : kLow;
    // (a high nibble is left in place: its scale a sixteenth)
    const v2h sc = up ? as_v2h(__builtin_amdgcn_perm(0x54545454u, word, sel + 0x00010001u)) + splat2(-64.0f)
                      : as_v2h(__builtin_amdgcn_perm(0x64646464u, word, sel)) + splat2(-1024.0f);
    const uint32_t x = q[L][2 * half], y = q[L][2 * half + 1];
    b0 = scaled(v4u{pair(x, mk), pair(x >> 8, mk), pair(y, mk), pair(y >> 8, mk)}, sc, sc * splat2(-1024.0f));
  }
  __device__ __forceinline__ float d() const { return f16f(h.x); }
  __device__ __forceinline__ float dmin() const { return f16f(h.x >> 16); }
  __device__ __forceinline__ v8h mins() const { return kmins(h.z, h.w); }
};
template <>
struct PackUnit<MI_Q6_K> {
  static constexpr int SLOTS = 2, LIMBS = 2;
  static constexpr bool MINS = false;
  v4u ql[2], qh[2], sc;
  uint32_t dbits;
  static __device__ __forceinline__ int up_of(int g) { return (g >> 1) & 1; }
  static __device__ __forceinline__ int which_of(int g) { return g & 1; }
  __device__ __forceinline__ void load(const uint8_t* row, int sb, int kq) {
    const uint8_t* p = row + (int64_t)sb * 210;
#pragma unroll
    for (int L = 0; L < 2; L++) {
      ql[L] = ld16(p + 64 * L + 16 * kq);
      qh[L] = ld16(p + 128 + 32 * L + 16 * (kq & 1));
    }
    sc = ld16(p + 192);
    dbits = ld2(p + 208);
  }
  // sc * (q - 32) reaches 4096: b0 its nearest half, b1 the rest (-1, 0 or 1)
  __device__ __forceinline__ void codes(int L, int up, int half, int kq, v8h& b0, v8h& b1) const {
    const _Float16 f = (_Float16)(float)(int)__builtin_amdgcn_sbfe((int)sc[2 * L + up], 8 * kq, 8);
    const v2h s = {f, f};
    v4u c0, c1;
#pragma unroll
    for (int w = 0; w < 2; w++) {
      // bits 2 (kq / 2) + 4 up and one more of the byte to bits 4, 5
      const uint32_t hi = ((qh[L][2 * half + w] >> (2 * (kq >> 1) + 4 * up)) & 0x03030303u) << 4;
      const uint32_t u = ((ql[L][2 * half + w] >> (4 * up)) & 0x0F0F0F0Fu) | hi;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const v2h v = as_v2h(__builtin_amdgcn_perm(0x64646464u, u, k ? 0x04030401u : 0x04020400u)) + splat2(-1056.0f);
        const v2h r = v * s;
        c0[2 * w + k] = as_u32(r);
        c1[2 * w + k] = as_u32(__builtin_elementwise_fma(v, s, -r));
      }
    }
    b0 = __builtin_bit_cast(v8h, c0);
    b1 = __builtin_bit_cast(v8h, c1);
  }
  __device__ __forceinline__ float d() const { return f16f(dbits); }
  __device__ __forceinline__ float dmin() const { return 0.0f; }
  __device__ __forceinline__ v8h mins() const { return v8h{}; }
};

template <int KIND, bool GLU>
__global__ __launch_bounds__(64 * kPackWaves, 2) void experts_pack_kernel(
    const uint8_t* __restrict__ w0, const uint8_t* __restrict__ w1, int64_t expert_bytes, int64_t rb, int rows, int cols,
    const float* __restrict__ x, int share, const int32_t* __restrict__ ids, int pairs, int experts, int act,
    int chunks_per_split, float* __restrict__ y, int64_t split_stride) {
  using Unit = PackUnit<KIND>;
  constexpr int RT = 2, S = Unit::SLOTS, kSb = kPackCols / kChunk, kRuns = 2;
  static_assert(kPackCols * kPackRows == 64 * kPackWaves * 8 * kRuns, "a thread's runs of 8 values");
  __shared__ __align__(16) uint8_t xl[2][kSb][8][1024];               // [step][lane][8 halves]
  __shared__ __align__(16) _Float16 xm[2][kSb][2 * kPackRows][8];     // means of 32 values
  __shared__ float scale[2][kPackRows];
  __shared__ int pair_of[kPackRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kq = lane >> 4;
  const int first = blockIdx.y, id = lane < pairs ? ids[lane] : -1;
  const int e = __builtin_amdgcn_readlane(id, first);
  // (uniform over the block) every eighth pair's block takes it and the seven behind it
  uint64_t mine = __ballot(id == e);
  const uint64_t before = mine & ((1ull << first) - 1);
  if ((uint32_t)e >= (uint32_t)experts || __builtin_popcountll(before) % kPackRows) return;
  mine ^= before;

  // this wave's rows: two tiles of 16 of one matrix, or the same 16 of both
  const int row0 = (blockIdx.x * kPackWaves + wave) * (GLU ? 16 : 32);
  const uint8_t* wrow[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++)
    wrow[rt] = (GLU && rt ? w1 : w0) + e * expert_bytes + (int64_t)min(row0 + (GLU ? 0 : 16 * rt) + n, rows - 1) * rb;
  const int nsb = cols / kChunk, chunks = (cols + kPackCols - 1) / kPackCols;
  const int c0 = blockIdx.z * chunks_per_split, c1 = min(c0 + chunks_per_split, chunks);
  const int sb0 = c0 * kSb, sb1 = min(c1 * kSb, nsb);

  int count = 0;
  for (; mine && count < kPackRows; mine &= mine - 1, count++)
    if ((int)threadIdx.x == count) pair_of[count] = __builtin_ctzll(mine);
  // rows that are not there
  if (count < kPackRows) {
    for (int i = threadIdx.x; i < (int)(sizeof(xl) / 16); i += 64 * kPackWaves) ((v4u*)xl)[i] = v4u{0, 0, 0, 0};
    for (int i = threadIdx.x; i < (int)(sizeof(xm) / 16); i += 64 * kPackWaves) ((v4u*)xm)[i] = v4u{0, 0, 0, 0};
  }
  __syncthreads();

  Unit un[S][RT];
  auto load = [&](Unit(&u)[RT], int sb) __attribute__((always_inline)) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++) u[rt].load(wrow[rt], min(sb, sb1 - 1), kq);
  };
#pragma unroll
  for (int k = 0; k < S - 1; k++) load(un[k], sb0 + k);

  // A chunk's activations: a row has 32 lanes, lane c takes its runs 32 k + c of 8 values
  const int m = 2 * wave + (lane >> 5), c = lane & 31;
  const bool there = m < count;
  const float* xrow = x + (int64_t)(pair_of[min(m, count - 1)] / share) * cols;
  v4f v[kRuns][2];
  auto load_x = [&](int ch) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kRuns; k++) {
      const float* p = xrow + min(ch * kPackCols + 8 * (32 * k + c), cols - 8);
      v[k][0] = *(const v4f*)p;
      v[k][1] = *(const v4f*)(p + 4);
    }
  };
  auto store_x = [&](int ch, int buf) __attribute__((always_inline)) {
    float mx = 0.0f;
#pragma unroll
    for (int k = 0; k < kRuns; k++) {
      if (ch * kPackCols + 8 * (32 * k + c) >= cols) v[k][0] = v[k][1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(v[k][j >> 2][j & 3]));
    }
    const int ex = scale_exp(lanes::reduce<32>(mx, lanes::Max{}));
    if (c == 0) scale[buf][m] = there ? ldexpf(1.0f, ex) : 0.0f;
#pragma unroll
    for (int k = 0; k < kRuns; k++) {
      v8h hi, lo;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        constexpr int kOrder[4] = {0, 2, 1, 3};  // the order of K
        const float f = ldexpf(v[k][j >> 2][kOrder[j & 3]], -ex);
        _Float16 h, l;
        split_half(f, h, l);
        hi[j] = h;
        lo[j] = l;
        sum += f;
      }
      sum = lanes::reduce<4>(sum, lanes::Add{}) * (1.0f / 32.0f);
      if (!there) continue;
      const int i = 32 * k + c, sb = i >> 5, g = (i >> 2) & 7, r = i & 3;  // superblock, group, run of it
      uint8_t* dst = &xl[buf][sb][4 * (g >> 2) + 2 * Unit::up_of(g) + (r & 1)][256 * (2 * Unit::which_of(g) + (r >> 1)) + 16 * m];
      *(v8h*)dst = hi;
      *(v8h*)(dst + 16 * kPackRows) = lo;
      if (Unit::MINS && r == 0) {
        _Float16 h, l;
        split_half(sum, h, l);
        xm[buf][sb][m][g] = h;
        xm[buf][sb][kPackRows + m][g] = l;
      }
    }
  };

  const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
  v4f tot[RT], out[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) out[rt] = zero;
  auto use = [&](const Unit(&u)[RT], int local, int buf) __attribute__((always_inline)) {
    v4f acc[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) acc[rt] = zero;
    const uint8_t* at = &xl[buf][local][0][16 * lane];
#pragma unroll
    for (int st = 0; st < 8; st++) {
      const v8h a = *(const v8h*)(at + 1024 * st);
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        v8h b0, b1;
        u[rt].codes(st >> 2, (st >> 1) & 1, st & 1, kq, b0, b1);
        acc[rt] = mfma16(a, b0, acc[rt]);
        if constexpr (Unit::LIMBS == 2) acc[rt] = mfma16(a, b1, acc[rt]);
      }
    }
    if constexpr (Unit::MINS) {
      // (lanes past the first 16 hold values 8..31 of the mins' step: zeros)
      const v8h am = kq == 0 ? *(const v8h*)xm[buf][local][n] : v8h{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        const v4f cm = mfma16(am, u[rt].mins(), zero);
        const float dm = -32.0f * u[rt].dmin();
#pragma unroll
        for (int j = 0; j < 4; j++) tot[rt][j] = fmaf(dm, cm[j], tot[rt][j]);
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int j = 0; j < 4; j++) tot[rt][j] = fmaf(u[rt].d(), acc[rt][j], tot[rt][j]);
  };

  load_x(c0);
  store_x(c0, 0);
  __syncthreads();
  int ch = c0, local = 0;
#pragma unroll
  for (int rt = 0; rt < RT; rt++) tot[rt] = zero;
  load_x(min(c0 + 1, chunks - 1));
  // superblock sb, after sending for sb + S - 1; at a chunk's end the next one's halves
  auto step = [&](int sb, Unit(&now)[RT], Unit(&refill)[RT]) __attribute__((always_inline)) {
    if (sb >= sb1) return;
    load(refill, sb + S - 1);
    __builtin_amdgcn_sched_barrier(0);
    const int buf = (ch - c0) & 1;
    use(now, local, buf);
    if (++local < kSb && sb + 1 < sb1) return;
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        out[rt][j] = fmaf(scale[buf][(4 * kq + j) & 7], tot[rt][j], out[rt][j]);
        tot[rt][j] = 0.0f;
      }
    local = 0;
    if (++ch >= c1) return;
    store_x(ch, 1 - buf);  // (read before the last barrier)
    __syncthreads();
    load_x(min(ch + 1, chunks - 1));
  };
  for (int sb = sb0; sb < sb1; sb += S) {
#pragma unroll
    for (int k = 0; k < S; k++) step(sb + k, un[k], un[(k + S - 1) % S]);
  }

  // high and low halves' sums: 32 lanes apart
#pragma unroll
  for (int rt = 0; rt < RT; rt++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(out[rt][j]), __float_as_uint(out[rt][j]), false, false);
      out[rt][j] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
  if (lane < 32) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int k = 4 * kq + j;
      if (k >= count) continue;
      float* to = y + blockIdx.z * split_stride + (int64_t)pair_of[k] * rows + row0 + n;
      if constexpr (GLU) {
        if (row0 + n < rows) *to = ((act & MI_ACT_GELU) ? mv::gelu(out[0][j]) : mv::silu(out[0][j])) * out[1][j];
      } else {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
          if (row0 + 16 * rt + n < rows) to[16 * rt] = out[rt][j];
      }
    }
  }
}

}  // namespace

bool pack_fits(int kind) { return kind == MI_Q4_K || kind == MI_Q6_K; }

int pack_most_splits(int32_t cols) { return std::min((cols + kPackCols - 1) / kPackCols, 8); }

// Parts of the columns: three blocks a CU, where the chunks allow it.
int pack_splits(int32_t rows, int32_t cols, int32_t pairs, int32_t experts) {
  const int chunks = (cols + kPackCols - 1) / kPackCols, blocks = (rows + 127) / 128 * std::min(pairs, experts);
  const int most = std::min(std::max(3 * cu_count() / blocks, 1), pack_most_splits(cols)), each = (chunks + most - 1) / most;
  return (chunks + each - 1) / each;
}

int launch_expert_pack(hipStream_t s, int kind, const void* w0, const void* w1, int64_t row_bytes, int32_t rows,
                       int32_t cols, int32_t experts, const float* x, int32_t share, const int32_t* ids, int32_t pairs,
                       int32_t act, int32_t splits, float* y) {
  if (!pack_fits(kind)) return fail(MI_ERR_KIND, "experts: ggml type %d is not packed", kind);
  const int chunks = (cols + kPackCols - 1) / kPackCols, mine = (w1 ? 16 : 32) * kPackWaves;
  const dim3 grid((rows + mine - 1) / mine, pairs, splits);
#define MI_PK(K, GLU)                                                                                                   \
  hipLaunchKernelGGL((experts_pack_kernel<K, GLU>), grid, dim3(64 * kPackWaves), 0, s, (const uint8_t*)w0,             \
                     (const uint8_t*)w1, rows * row_bytes, row_bytes, rows, cols, x, share, ids, pairs, experts, act,  \
                     (chunks + splits - 1) / splits, y, (int64_t)pairs * rows)
  if (kind == MI_Q4_K && w1) MI_PK(MI_Q4_K, true);
  else if (kind == MI_Q4_K) MI_PK(MI_Q4_K, false);
  else if (w1) MI_PK(MI_Q6_K, true);
  else MI_PK(MI_Q6_K, false);
#undef MI_PK
  return hip_check(hipGetLastError(), "experts pack launch");
}

}  // namespace mi
