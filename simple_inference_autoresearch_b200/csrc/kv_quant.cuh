// How a row of a quantised cache is formed (formats: top of kv_quant.cu), shared by the kernel that stores
// prompts' rows and the attention kernel that stores the row of its new token.
#pragma once

#include "common.cuh"

#include <math.h>

namespace siar {

constexpr int kQuantGroup = 64;      // dims that share a scale in the 4-bit format

__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One pair of a rotation: rounded products, a rounded sum (no fused multiply-add), so that the codes
// are a function of the row and the position alone, whatever kernel forms them.
__device__ __forceinline__ float rotate_lo(float a, float c, float cosv, float sinv) {
  return __fsub_rn(__fmul_rn(a, cosv), __fmul_rn(c, sinv));
}
__device__ __forceinline__ float rotate_hi(float a, float c, float cosv, float sinv) {
  return __fadd_rn(__fmul_rn(c, cosv), __fmul_rn(a, sinv));
}
// Cosine and sine of position x frequency, each rounded once: the product of two 24-bit numbers is exact
// in 64 bits (as a float32 it is off by up to 2^-8 at 131,072 positions).
__device__ __forceinline__ void rotation(int pos, float freq, float* cosv, float* sinv) {
  double sn, cn;
  sincos((double)pos * (double)freq, &sn, &cn);
  *cosv = (float)cn;
  *sinv = (float)sn;
}

// One warp quantises a row x[0 .. D) (shared memory): lane l holds dims 64 i + 2l, + 2l + 1 of run i.
// codes(d, c): the codes of dims d, d + 1 (8 bits: two bytes; 4 bits: one byte); scales: 8 bits (0, s),
// 4 bits (run, s, m), from lane 0.
template <int BITS, typename Codes, typename Scales>
__device__ __forceinline__ void quantize_row(const float* row, int D, int lane, Codes codes, Scales scales) {
  const float nan = __int_as_float(0x7fc00000);
  if (BITS == 8) {
    float amax = 0.f;
    bool bad = false;
    for (int d = lane; d < D; d += 32) {
      amax = fmaxf(amax, fabsf(row[d]));
      bad |= !isfinite(row[d]);
    }
    amax = warp_max(amax);
    bad = __any_sync(0xffffffffu, bad);
    const float s = __fdiv_rn(amax, 127.f);
    for (int d = 2 * lane; d < D; d += 64) {
      int c[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        c[e] = bad || !(s > 0.f) ? 0 : max(-127, min(127, __float2int_rn(__fdiv_rn(row[d + e], s))));
      codes(d, (uint32_t)((c[0] & 0xff) | ((c[1] & 0xff) << 8)));
    }
    if (lane == 0) scales(0, bad ? nan : s, __floats2bfloat162_rn(0.f, 0.f));
  } else {
    for (int g = 0; g * kQuantGroup < D; ++g) {
      const int d = g * kQuantGroup + 2 * lane;
      const bool in = d < D;
      const float x0 = in ? row[d] : 0.f, x1 = in ? row[d + 1] : 0.f;
      const bool bad = __any_sync(0xffffffffu, !isfinite(x0) || !isfinite(x1));
      const float lo = warp_min(in ? fminf(x0, x1) : INFINITY), hi = warp_max(in ? fmaxf(x0, x1) : -INFINITY);
      const __nv_bfloat16 sb = __float2bfloat16_rn(__fsub_rn(__fdiv_rn(hi, 15.f), __fdiv_rn(lo, 15.f)));
      const float s = __bfloat162float(sb);
      const __nv_bfloat16 mb = __float2bfloat16_rn(__fadd_rn(lo, 8.f * s));
      const float m = __bfloat162float(mb);
      if (in) {
        int c[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          c[e] = bad || !(s > 0.f) ? 8 : max(0, min(15, __float2int_rn(__fdiv_rn(__fsub_rn(e ? x1 : x0, m), s)) + 8));
        codes(d, (uint32_t)(c[0] | (c[1] << 4)));
      }
      if (lane == 0) scales(g, 0.f, bad ? __floats2bfloat162_rn(nan, nan) : __halves2bfloat162(sb, mb));
    }
  }
}

}  // namespace siar
