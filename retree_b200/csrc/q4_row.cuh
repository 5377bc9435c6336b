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
// hi - lo is rounded up in fp32 and its quotient correctly, which gives the exact s.
// The other two quotients are correctly rounded in fp32, and x (8 significant bits)
// either equals a half-integer times s (9 bits) or is off it by 2^-9 or more,
// so every rounding decision is the exact one.  A row holding a value that is
// not finite gets NaN scales: all of its 128 values read as NaN.
#pragma once

#include "common.cuh"

namespace rt {

constexpr int kQ4Row = 72;
constexpr int kQ4Codes = 64;
constexpr uint32_t kQ4NanWord = 0x7FF0;

// The 16-bit word's scale as bf16 in both halves.
__device__ __forceinline__ uint32_t q4_scale2(uint32_t w) {
  const uint32_t s = w & 0x7FF0u;
  return s | (s << 16);
}

// Eight values of a code word as four bf16 pairs (16 bytes, in order), three and
// a quarter instructions a pair: the nibbles as bytes, 64 - z added to each,
// then 0x43 above a byte b makes the bf16 number 128 + b = 192 + (u - z),
// and (192 + (u - z)) * s - 192 * s is one fused multiply-add whose result
// (u - z) * s is representable, so it is exact.  192 * s has as few bits as s, but
// must not overflow: s < 2^120.
struct Q4Group {
  uint32_t add4, scale2, shift2;  // 64 - z in four bytes, s and -192 s in two halves
};
__device__ __forceinline__ uint32_t q4_shift(uint32_t scale2) {
  const __nv_bfloat162 c = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&scale2),
                                   __floats2bfloat162_rn(-192.f, -192.f));
  return *reinterpret_cast<const uint32_t*>(&c);
}
__device__ __forceinline__ Q4Group q4_group(uint32_t w) {
  const uint32_t s2 = q4_scale2(w);
  return {0x40404040u - (w & 15u) * 0x01010101u, s2, q4_shift(s2)};
}
// The same for a word whose low half comes from one row and high half from another.
__device__ __forceinline__ Q4Group q4_group2(uint32_t wlo, uint32_t whi) {
  const uint32_t s2 = (wlo & 0x7FF0u) | ((whi & 0x7FF0u) << 16);
  return {0x40404040u - ((wlo & 15u) | ((whi & 15u) << 16)) * 0x0101u, s2, q4_shift(s2)};
}
// x43: 0x43434343, which the callers read from shared memory: one token over 131071
// rows then runs 735 instructions a 32-key tile and warp (897 with the constant written
// here; counted by a profiler together with explicit shared loads), 43.0 us and not 47.2.
__device__ __forceinline__ uint4 q4_decode8(uint32_t word, const Q4Group& g, uint32_t x43) {
  const uint32_t lo = (word & 0x0F0F0F0Fu) + g.add4, hi = ((word >> 4) & 0x0F0F0F0Fu) + g.add4;
  auto value = [&](uint32_t bytes, uint32_t sel) {
    const uint32_t x = __byte_perm(bytes, x43, sel);
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                     *reinterpret_cast<const __nv_bfloat162*>(&g.scale2),
                                     *reinterpret_cast<const __nv_bfloat162*>(&g.shift2));
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  return make_uint4(value(lo, 0x4240), value(hi, 0x4240), value(lo, 0x4341), value(hi, 0x4341));
}

}  // namespace rt
