// kv_device.h -- device side of the KV cache rows that the stores share.
#pragma once

#include "mi_internal.h"

namespace mi {

// One q8_0 block of a cache row: the 32 lanes of a half-wave each bring one
// value x of block b; rowp is the position's row (quants, then factors).
__device__ __forceinline__ void q8_store_block(float x, __half* __restrict__ rowp, int b, int kv_width,
                                               int lane32) {
#pragma clang fp contract(off)
  float amax = fabsf(x);
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 32));
  const float inv = amax == 0.0f ? 0.0f : 127.0f / amax;
  const float y = x * inv;
  const float r = y >= 0.0f ? y + 0.5f : y - 0.5f;
  const int qi = max(-127, min(127, (int)r));
  ((int8_t*)rowp)[b * 32 + lane32] = (int8_t)qi;
  if (lane32 == 0) rowp[(kv_width >> 1) + b] = __float2half_rn(amax / 127.0f);
}

}  // namespace mi
