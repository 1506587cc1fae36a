// matvec_q6k_unit.h -- one lane's 64-value unit of a Q6_K row (half n, part a of a
// superblock; matvec_q6k_rows.hip has the format): its activation, its bytes, its
// dot.
#pragma once

#include "matvec_units.h"

namespace mi {
namespace mv {

// The activation of one lane's unit: groups g0 = 4n + a and g1 = g0 + 2 of
// its superblock.
struct XQ6Regs {
  uint4 l[2][3][2];  // [group][limb][16-value half]
  float scale[2];
  int lsum1[2][2], lsum23[2][2];
};

// The 22 dwords of one row's unit, 4-byte aligned; `sh` realigns them.
struct Q6Piece {
  uint32_t ql[9], qh[9], sc[3], d;
};

__device__ __forceinline__ void load_piece(Q6Piece& p, const uint8_t* blk4, uint32_t sh, int n, int a) {
  const uint8_t* q = blk4 + 64 * n + 32 * a;
  const uint4 q0 = ld16a4(q), q1 = ld16a4(q + 16);
  p.ql[0] = q0.x; p.ql[1] = q0.y; p.ql[2] = q0.z; p.ql[3] = q0.w;
  p.ql[4] = q1.x; p.ql[5] = q1.y; p.ql[6] = q1.z; p.ql[7] = q1.w;
  p.ql[8] = ld4(q + 32);
  const uint8_t* h = blk4 + 128 + 32 * n;
  const uint4 h0 = ld16a4(h), h1 = ld16a4(h + 16);
  p.qh[0] = h0.x; p.qh[1] = h0.y; p.qh[2] = h0.z; p.qh[3] = h0.w;
  p.qh[4] = h1.x; p.qh[5] = h1.y; p.qh[6] = h1.z; p.qh[7] = h1.w;
  p.qh[8] = ld4(h + 32);
  // sc[8n .. 8n+7] spans three dwords only when the block is 2 bytes off
  // alignment; aligned, the third would read past the superblock (past the
  // tensor, for its last one), so it re-reads the second instead.
  const uint8_t* s = blk4 + 192 + 8 * n;
  p.sc[0] = ld4(s);
  p.sc[1] = ld4(s + 4);
  p.sc[2] = ld4(s + (sh ? 8 : 4));
  // d as a 16-bit load at its own (even) address, for the same reason
  p.d = *(const uint16_t*)(blk4 + sh + 208);
}

__device__ __forceinline__ float piece_dot(const Q6Piece& p, uint32_t sh, int a, const XQ6Regs& x) {
  const uint32_t s_lo = 2u * a, s_hi = 4u + 2u * a;
  uint32_t scw[2];
  scw[0] = align(p.sc[1], p.sc[0], sh);  // sc[8n .. 8n+3]
  scw[1] = align(p.sc[2], p.sc[1], sh);  // sc[8n+4 .. 8n+7]
  const float d = half_bits_to_float(p.d);
  float part = 0.0f;
#pragma unroll
  for (int hh = 0; hh < 2; hh++) {
    int s0[3] = {0, 0, 0}, s1[3] = {0, 0, 0};
#pragma unroll
    for (int ii = 0; ii < 4; ii++) {
      const int i = 4 * hh + ii;
      const uint32_t A = align(p.ql[i + 1], p.ql[i], sh);
      const uint32_t H = align(p.qh[i + 1], p.qh[i], sh);
      const uint32_t q0 = (A & 0x0F0F0F0Fu) | (((H >> s_lo) & 0x03030303u) << 4);
      const uint32_t q1 = ((A >> 4) & 0x0F0F0F0Fu) | (((H >> s_hi) & 0x03030303u) << 4);
#pragma unroll
      for (int j = 0; j < 3; j++) {
        s0[j] = dot4(q0, comp(x.l[0][j][hh], ii), s0[j]);
        s1[j] = dot4(q1, comp(x.l[1][j][hh], ii), s1[j]);
      }
    }
    // sc[8n + hh + 2a] for group g0, sc[8n + hh + 4 + 2a] for g1
    const uint32_t b0 = hh + 2u * a, b1 = hh + 4u + 2u * a;
    const float sc0 = (float)(int8_t)((scw[b0 >> 2] >> (8 * (b0 & 3))) & 0xFF);
    const float sc1 = (float)(int8_t)((scw[b1 >> 2] >> (8 * (b1 & 3))) & 0xFF);
    const float f0 = limbs_to_float(s0[0] - 32 * x.lsum1[0][hh], s0[1] * 256 + s0[2] - 32 * x.lsum23[0][hh]);
    const float f1 = limbs_to_float(s1[0] - 32 * x.lsum1[1][hh], s1[1] * 256 + s1[2] - 32 * x.lsum23[1][hh]);
    part = fmaf(sc0 * x.scale[0], f0, part);
    part = fmaf(sc1 * x.scale[1], f1, part);
  }
  return d * part;
}

template <class XA>
__device__ __forceinline__ void load_x6(XQ6Regs& x, const XA& xa, int g0) {
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int g = g0 + 2 * e;
#pragma unroll
    for (int j = 0; j < 3; j++)
#pragma unroll
      for (int hh = 0; hh < 2; hh++) x.l[e][j][hh] = xa.limb(0, j, hh, g);
    const XMeta m = xa.meta(0, g);
    const int2 l23 = xa.lsum23(0, g);
    x.scale[e] = m.scale;
    x.lsum1[e][0] = m.lsum1[0];
    x.lsum1[e][1] = m.lsum1[1];
    x.lsum23[e][0] = l23.x;
    x.lsum23[e][1] = l23.y;
  }
}

}  // namespace mv
}  // namespace mi
