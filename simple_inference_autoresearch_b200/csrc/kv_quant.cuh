// How a row of a quantised cache is formed (formats: top of kv_quant.cu), shared by the kernel that stores
// prompts' rows and the attention kernel that stores the row of its new token.
#pragma once

#include "common.cuh"

#include <math.h>
#include <string.h>

#include <type_traits>
#include <utility>

namespace siar {

// A launcher's arguments as 64-bit words, one each (whole numbers and pointers as they are, floats as doubles): a call from
// Python with one buffer of words takes 1 us where one with 33 arguments takes 4.
template <typename T>
T from_word(long long w) {
  if constexpr (std::is_pointer<T>::value) {
    return reinterpret_cast<T>(w);
  } else if constexpr (std::is_floating_point<T>::value) {
    double d;
    memcpy(&d, &w, sizeof(d));
    return (T)d;
  } else {
    return (T)w;
  }
}
template <typename... A, size_t... I>
int call_with(int (*f)(A...), const long long* w, std::index_sequence<I...>) {
  return f(from_word<A>(w[I])...);
}
template <typename... A>
int call_with_words(int (*f)(A...), const void* words) {
  long long w[sizeof...(A)];
  memcpy(w, words, sizeof(w));
  return call_with(f, w, std::index_sequence_for<A...>{});
}
#define SIAR_TAKES_WORDS(name) \
  extern "C" int name(const void* words) { return siar::call_with_words(name##_of, words); }

constexpr int kQuantGroup = 64;      // dims that share a scale in the 4-bit format

__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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

// x / s rounded to nearest for all the values of a row, which share s: with r the rounded reciprocal of s, the
// quotient x r is off by little more than its last bit, and Markstein's correction (q + (x - q s) r, both fused)
// rounds it as a division does, while nothing under- or overflows on the way.  A scale outside 2^-90 .. 2^90 is
// brought inside by a power of two (k), the values with it.  Without a scale (zero, infinite, NaN) quotients of
// finite values are 0.
struct Divisor {
  float s, r, k;
};
__device__ __forceinline__ Divisor divisor(float s) {
  if (!(s > 0.f && s < INFINITY)) return Divisor{0.f, 0.f, 1.f};
  const float k = s < 0x1p-90f ? 0x1p60f : s > 0x1p90f ? 0x1p-60f : 1.f;
  return Divisor{s * k, __frcp_rn(s * k), k};
}
__device__ __forceinline__ float corrected(float x, const Divisor& by) {       // x already times k
  const float q = __fmul_rn(x, by.r);
  return fmaf(fmaf(-q, by.s, x), by.r, q);
}
__device__ __forceinline__ float quotient(float x, const Divisor& by) { return corrected(x * by.k, by); }
// rint(y) for |y| < 2^22, in the low bits (two's complement): adding 1.5 x 2^23 rounds to a whole number.
__device__ __forceinline__ uint32_t whole_bits(float y) { return __float_as_uint(__fadd_rn(y, 12582912.f)); }

// The scale of a row in 8 bits, and a code against it in the low byte (0 without a scale).  127 and 15 divide by a product
// with the float32 reciprocal, as torch divides a tensor on the GPU by a number: where a scale is rounded to 16 bits, the
// last bit of the quotient decides about one run in 500,000.
__device__ __forceinline__ float scale8(float amax) { return __fmul_rn(amax, 1.f / 127.f); }
__device__ __forceinline__ uint32_t code8(float x, const Divisor& by, bool bad) {
  return bad ? 0u : whole_bits(fmaxf(-127.f, fminf(127.f, quotient(x, by))));
}
// Scale and mid of a run in 4 bits, and a code against them in the low four bits.
__device__ __forceinline__ __nv_bfloat162 scale4(float lo, float hi, bool bad) {
  const __nv_bfloat16 s = __float2bfloat16_rn(__fsub_rn(__fmul_rn(hi, 1.f / 15.f), __fmul_rn(lo, 1.f / 15.f)));
  const __nv_bfloat16 m = __float2bfloat16_rn(__fadd_rn(lo, 8.f * __bfloat162float(s)));
  const float nan = __int_as_float(0x7fc00000);
  return bad ? __floats2bfloat162_rn(nan, nan) : __halves2bfloat162(s, m);
}
__device__ __forceinline__ uint32_t code4(float x, const Divisor& by, float m, bool bad) {
  return bad ? 8u : (whole_bits(fmaxf(-8.f, fminf(7.f, quotient(__fsub_rn(x, m), by)))) + 8u) & 15u;
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
    const Divisor by = divisor(s);
    for (int d = 2 * lane; d < D; d += 64) codes(d, __byte_perm(code8(row[d], by, bad), code8(row[d + 1], by, bad), 0x7740) & 0xffffu);
    if (lane == 0) scales(0, bad ? __int_as_float(0x7fc00000) : s, __floats2bfloat162_rn(0.f, 0.f));
  } else {
    for (int g = 0; g * kQuantGroup < D; ++g) {
      const int d = g * kQuantGroup + 2 * lane;
      const bool in = d < D;
      const float x0 = in ? row[d] : 0.f, x1 = in ? row[d + 1] : 0.f;
      const bool bad = __any_sync(0xffffffffu, !isfinite(x0) || !isfinite(x1));
      const float lo = warp_min(in ? fminf(x0, x1) : INFINITY), hi = warp_max(in ? fmaxf(x0, x1) : -INFINITY);
      const __nv_bfloat162 sm = scale4(lo, hi, bad);
      const Divisor by = divisor(__low2float(sm));
      const float m = __high2float(sm);
      if (in) codes(d, code4(x0, by, m, bad) | (code4(x1, by, m, bad) << 4));
      if (lane == 0) scales(g, 0.f, sm);
    }
  }
}

}  // namespace siar
