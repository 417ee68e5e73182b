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
// Cosine and sine of position x frequency, each rounded to 32 bits once: the product of two 24-bit numbers is
// exact in 64 bits (as a float32 it is off by up to 2^-8 at 131,072 positions).  The angle is brought to
// |r| <= pi/4 by Cody and Waite's two-part reduction, x - n (pi/2 as a sum of two doubles), each step one fused
// multiply-add (n is below 2^31, so what the two parts leave of n pi/2 is below 2^-75), and the two Taylor
// series are taken as far as r^15 and r^16, whose next terms are below 2^-54: about twenty 64-bit operations for
// both functions where a call of sincos takes several times that.
__device__ __forceinline__ void rotation(int pos, float freq, float* cosv, float* sinv) {
  const double x = (double)pos * (double)freq;
  const double n = rint(x * 0.63661977236758134308);                // 2 / pi
  double r = fma(-n, 1.57079632679489661923, x);
  r = fma(-n, 6.12323399573676603587e-17, r);
  const double r2 = r * r;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;    // 1/15!, 1/16!
  s = fma(s, r2, 1.0 / 6227020800.0);
  c = fma(c, r2, -1.0 / 87178291200.0);
  s = fma(s, r2, -1.0 / 39916800.0);
  c = fma(c, r2, 1.0 / 479001600.0);
  s = fma(s, r2, 1.0 / 362880.0);
  c = fma(c, r2, -1.0 / 3628800.0);
  s = fma(s, r2, -1.0 / 5040.0);
  c = fma(c, r2, 1.0 / 40320.0);
  s = fma(s, r2, 1.0 / 120.0);
  c = fma(c, r2, -1.0 / 720.0);
  s = fma(s, r2, -1.0 / 6.0);
  c = fma(c, r2, 1.0 / 24.0);
  c = fma(c, r2, -0.5);
  s = fma(s * r2, r, r);
  c = fma(c, r2, 1.0);
  const int q = (int)((long long)n & 3);
  const float sf = (float)((q & 1) ? c : s), cf = (float)((q & 1) ? s : c);
  *sinv = (q & 2) ? -sf : sf;
  *cosv = (q == 1 || q == 2) ? -cf : cf;
}

// The scale of a row in 8 bits, and a code against it (0 without a scale).
__device__ __forceinline__ float scale8(float amax) { return __fdiv_rn(amax, 127.f); }
__device__ __forceinline__ int code8(float x, float s, bool bad) {
  return bad || !(s > 0.f) ? 0 : max(-127, min(127, __float2int_rn(__fdiv_rn(x, s))));
}
// Scale and mid of a run in 4 bits, and a code against them.
__device__ __forceinline__ __nv_bfloat162 scale4(float lo, float hi, bool bad) {
  const __nv_bfloat16 s = __float2bfloat16_rn(__fsub_rn(__fdiv_rn(hi, 15.f), __fdiv_rn(lo, 15.f)));
  const __nv_bfloat16 m = __float2bfloat16_rn(__fadd_rn(lo, 8.f * __bfloat162float(s)));
  const float nan = __int_as_float(0x7fc00000);
  return bad ? __floats2bfloat162_rn(nan, nan) : __halves2bfloat162(s, m);
}
__device__ __forceinline__ int code4(float x, float s, float m) {        // s, m: NaN for a bad run
  return !(s > 0.f) ? 8 : max(0, min(15, __float2int_rn(__fdiv_rn(__fsub_rn(x, m), s)) + 8));
}

// One warp quantises a row x[0 .. D) (shared memory): lane l holds dims 64 i + 2l, + 2l + 1 of run i.
// codes(d, c): the codes of dims d, d + 1 (8 bits: two bytes; 4 bits: one byte); scales: 8 bits (0, s),
// 4 bits (run, s, m), from lane 0.
template <int BITS, typename Codes, typename Scales>
__device__ __forceinline__ void quantize_row(const float* row, int D, int lane, Codes codes, Scales scales) {
  if (BITS == 8) {
    float amax = 0.f;
    bool bad = false;
    for (int d = lane; d < D; d += 32) {
      amax = fmaxf(amax, fabsf(row[d]));
      bad |= !isfinite(row[d]);
    }
    amax = warp_max(amax);
    bad = __any_sync(0xffffffffu, bad);
    const float s = scale8(amax);
    for (int d = 2 * lane; d < D; d += 64)
      codes(d, (uint32_t)((code8(row[d], s, bad) & 0xff) | ((code8(row[d + 1], s, bad) & 0xff) << 8)));
    if (lane == 0) scales(0, bad ? __int_as_float(0x7fc00000) : s, __floats2bfloat162_rn(0.f, 0.f));
  } else {
    for (int g = 0; g * kQuantGroup < D; ++g) {
      const int d = g * kQuantGroup + 2 * lane;
      const bool in = d < D;
      const float x0 = in ? row[d] : 0.f, x1 = in ? row[d + 1] : 0.f;
      const bool bad = __any_sync(0xffffffffu, !isfinite(x0) || !isfinite(x1));
      const float lo = warp_min(in ? fminf(x0, x1) : INFINITY), hi = warp_max(in ? fmaxf(x0, x1) : -INFINITY);
      const __nv_bfloat162 sm = scale4(lo, hi, bad);
      const float s = __low2float(sm), m = __high2float(sm);
      if (in) codes(d, (uint32_t)(code4(x0, s, m) | (code4(x1, s, m) << 4)));
      if (lane == 0) scales(g, 0.f, sm);
    }
  }
}

}  // namespace siar
