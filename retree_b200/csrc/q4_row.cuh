// The 4-bit cache row: one head's 128 values of one token in 72 bytes.
//
//   bytes 0-63   codes: 32-bit word i holds values 8i..8i+7, nibbles 0-3 the
//                even ones (8i, 8i+2, 8i+4, 8i+6), nibbles 4-7 the odd ones,
//                so (word >> 4j) & 0x000F000F is the pair (8i+2j, 8i+2j+1)
//   bytes 64-71  four 16-bit words, one per 32 values: bits 4-14 are bits 4-14
//                of the bf16 scale s (exponent and three mantissa bits), bits
//                0-3 the zero point z
//
// A value is (u - z) * s: |u - z| <= 15 has four significant bits and s four,
// so the product is a bf16 number and nothing is rounded when a row is read.
// Writing a row (x its bf16 values, per group of 32):
//   lo = min(0, min x), hi = max(0, max x)
//   s  = (hi - lo) / 15 rounded up to four significant bits (0 below 2^-126)
//   z  = rne(-lo / s),  u = clamp(rne(x / s) + z, 0, 15)
// Both quotients are correctly rounded in fp32, and x (8 significant bits)
// either equals a half-integer times s (9 bits) or is off it by 2^-9 or more,
// so every rounding decision is the exact one.  A row holding a value that is
// not finite gets NaN scales: all of its 128 values read as NaN.
#pragma once

#include "common.cuh"

namespace rt {

constexpr int kQ4Row = 72;
constexpr int kQ4Codes = 64;
constexpr uint32_t kQ4NanWord = 0x7FF0;

// The 16-bit word's scale as bf16 in both halves, and 128 + z likewise.
__device__ __forceinline__ uint32_t q4_scale2(uint32_t w) {
  const uint32_t s = w & 0x7FF0u;
  return s | (s << 16);
}
__device__ __forceinline__ uint32_t q4_zero2(uint32_t w) { return 0x43004300u | ((w & 15u) * 0x00010001u); }

// Values 2j, 2j+1 of a code word as a bf16 pair: 0x4300 | u is 128 + u, the
// difference to 128 + z and the product are exact.
__device__ __forceinline__ uint32_t q4_pair(uint32_t shifted, uint32_t zero2, uint32_t scale2) {
  uint32_t t;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;" : "=r"(t) : "r"(shifted));  // (a & b) | c
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t),
                                   *reinterpret_cast<const __nv_bfloat162*>(&zero2));
  const __nv_bfloat162 v = __hmul2(d, *reinterpret_cast<const __nv_bfloat162*>(&scale2));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight values of a code word as four bf16 pairs (16 bytes, in order).
__device__ __forceinline__ uint4 q4_decode8(uint32_t word, uint32_t zero2, uint32_t scale2) {
  uint4 r;
  r.x = q4_pair(word, zero2, scale2);
  r.y = q4_pair(word >> 4, zero2, scale2);
  r.z = q4_pair(word >> 8, zero2, scale2);
  r.w = q4_pair(word >> 12, zero2, scale2);
  return r;
}

}  // namespace rt
