// codes8.cuh — 8-bit codes of a quantised key/value cache: whole numbers -127 .. 127, or e4m3 floats
// up to 448.  A block of kScaleBlock tokens of one page and head has one fp32 scale; a code stands
// for code * scale.  The scales that the cache's own writes make are powers of two, so dividing by
// one is exact, a code is the correctly rounded quotient whatever the arithmetic around it, and a
// block rounded again and again to growing scales is off by less than one step in all (half a step
// of the last scale, a quarter for the one before, ...).  That costs int8 up to one of its seven
// bits, e4m3 nothing but the ends of its range.
#pragma once
#include "common.cuh"

namespace enigma_codes8 {

constexpr int kScaleBlock = ENIGMA_SCALE_BLOCK;

// Four codes (low byte first) as two pairs of halves; both kinds are exact in fp16.
template <bool E4M3>
__device__ __forceinline__ void halves_of4(uint32_t four, uint32_t* lo, uint32_t* hi) {
  if (E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(*lo), "=r"(*hi) : "r"(four));
  } else {
    // 0x6400 + u is the half 1024 + u: the code's byte with its sign bit turned is code + 128.
    const uint32_t u = four ^ 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(*lo) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(*hi) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(0x64806480u));
  }
}

__device__ __forceinline__ float2 floats_of(uint32_t halves) {
  float2 f;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(f.x), "=f"(f.y) : "r"(halves));
  return f;
}

// Four values times `unit` (one over their scale) rounded to codes: to nearest, ties to even.  No value of a
// block passes the codes' range but one that is not a number, whose block reads as NaN.
template <bool E4M3>
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d, float unit) {
  if (E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * unit), "f"(a * unit));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * unit), "f"(c * unit));
    return uint32_t(lo) | uint32_t(hi) << 16;
  }
  // 1.5 * 2^23 + x is x rounded to a whole number, in the low bits (conversions to integers run at a
  // quarter of the rate of additions).
  constexpr float kWhole = 0x1.8p23f;
  const uint32_t x = __float_as_uint(fmaf(a, unit, kWhole)), y = __float_as_uint(fmaf(b, unit, kWhole));
  const uint32_t z = __float_as_uint(fmaf(c, unit, kWhole)), w = __float_as_uint(fmaf(d, unit, kWhole));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// The scale of values whose largest magnitude has these bits (finite): the least power of two 2^e
// with top <= 127 * 2^e, or 448 * 2^e; tops below 2^-110 count as that.
template <bool E4M3>
__device__ __forceinline__ float scale_of(uint32_t top) {
  top = max(top, uint32_t(127 - 110) << 23);
  const int e = int(top >> 23) - (E4M3 ? 8 : 6);                 // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const bool over = (top & 0x7fffffu) > (E4M3 ? 0x600000u : 0x7e0000u);
  return __uint_as_float(uint32_t(e + (over ? 1 : 0)) << 23);
}

}  // namespace enigma_codes8
