// 4-bit KV cache rows: append (quantise) and read (decode).
//
// Both are data movement with a few operations a value: 256 bytes in and 72
// out for a row of one head (append), 72 in and 256 out (read).  Sixteen lanes
// hold a row, eight values (16 bytes of bf16, one code word) each; the four
// lanes of a 32-value group reduce its range with two shuffles.  A lane takes
// kRowsEach rows, whose loads are all in flight at once.
// Measured, 8191 rows of 8 heads, K and V (43 MB), in a graph: append 13.8 us (3.1
// TB/s; bound by the quantisation: ALU pipe 67 % and issue slots 74 % busy), read
// 6.4 us (6.7 TB/s).  With one row a lane and fp32 divisions both took 36.9 us.
#include "common.cuh"
#include "host_util.h"
#include "q4_row.cuh"

namespace rt {

constexpr int kRowsEach = 4;
constexpr int kRowsBlock = 16 * kRowsEach;  // 256 threads

// x / s correctly rounded, from an approximate reciprocal of s and the exact
// remainder of the first quotient (Markstein's correction; s with few bits, nothing
// near the ends of the range: s in [2^-60, 2^100], |x| <= 16 s).
__device__ __forceinline__ float quotient(float x, float s, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, s, x), inv, q);
}
__device__ __forceinline__ __nv_bfloat162 as_bf16x2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }

// Code word and group word of a lane's eight values.  No lower clamp: rne is odd
// and increasing, so rne(x / s) + rne(-lo / s) >= rne(lo / s) + rne(-lo / s) = 0.
__device__ __forceinline__ void quantise8(const uint4& raw, uint32_t& code, uint32_t& word) {
  // range of the group; NaN stays NaN, so that one look at the ends finds every
  // value that is not finite
  const __nv_bfloat162 top = __hmax2_nan(__hmax2_nan(as_bf16x2(raw.x), as_bf16x2(raw.y)),
                                         __hmax2_nan(as_bf16x2(raw.z), as_bf16x2(raw.w)));
  const __nv_bfloat162 low = __hmin2_nan(__hmin2_nan(as_bf16x2(raw.x), as_bf16x2(raw.y)),
                                         __hmin2_nan(as_bf16x2(raw.z), as_bf16x2(raw.w)));
  const float2 t = __bfloat1622float2(top), b = __bfloat1622float2(low);
  float hi, lo;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(hi) : "f"(t.x), "f"(t.y));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(lo) : "f"(b.x), "f"(b.y));
  const uint32_t bad = !(hi < INFINITY) || !(lo > -INFINITY);
  hi = fmaxf(hi, 0.f);
  lo = fminf(lo, 0.f);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
  }
  // one such value spoils the row: its sixteen lanes
  const bool spoilt = ((__ballot_sync(0xFFFFFFFFu, bad != 0) >> (threadIdx.x & 16)) & 0xFFFFu) != 0;
  code = 0;
  word = kQ4NanWord;
  if (spoilt) return;
  // (hi - lo) / 15, halved first so that the difference cannot overflow, and up to
  // four significant bits.  The difference is rounded up: 7.5 times a scale has 8
  // bits, so one that the exact difference passes, by however little, d passes by a
  // step of fp32, and the quotient by more than half a step, which its rounding keeps.
  const float d = __fsub_ru(0.5f * hi, 0.5f * lo);
  const bool plain = d >= 1.7347235e-17f && d <= 1.2676506e30f;  // 2^-56, 2^100
  float s = plain ? quotient(d, 7.5f, 1.f / 7.5f) : __fdiv_rn(d, 7.5f);
  // (asked before: below 2^-126 a step of this rounding is 2^-129, not four bits; the
  // largest four-bit number there is 15/16 of 2^-126)
  const bool flat = s <= 1.10202596e-38f;
  s = __uint_as_float((__float_as_uint(s) + 0xFFFFFu) & ~0xFFFFFu);
  word = 0;
  if (flat) return;
  float x[8];
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  float z = -lo, top_x = hi;
  if (plain) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = quotient(x[i], s, inv);
    z = quotient(z, s, inv);
    top_x = quotient(top_x, s, inv);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(x[i], s);
    z = __fdiv_rn(z, s);
    top_x = __fdiv_rn(top_x, s);
  }
  // adding 1.5 * 2^23 rounds to the nearest integer (ties to even) in the low
  // bits; the codes are summed with that offset and it is taken off at the end
  constexpr float kRound = 12582912.f;
  const uint32_t zi = __float_as_uint(z + kRound) - __float_as_uint(kRound), base = __float_as_uint(kRound) - zi;
  word = ((__float_as_uint(s) >> 16) & 0x7FF0u) | zi;
  // (the upper clamp matters only where the group's largest code would be 16)
  if (__float_as_uint(top_x + kRound) > base + 15u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(x[i], __uint_as_float(base + 15u) - kRound);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) code += __float_as_uint(x[i] + kRound) << (4 * ((i >> 1) + 4 * (i & 1)));
  code -= base * 0x11111111u;
}

__global__ void __launch_bounds__(256) kv_append_q4_kernel(char* k_cache, char* v_cache, int64_t c_head_stride,
                                                           const char* k_new, const char* v_new,
                                                           int64_t n_head_stride, int64_t n_row_stride, int n_new,
                                                           int64_t capacity, int64_t offset,
                                                           const int64_t* offset_dev, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t off = offset_dev != nullptr ? *offset_dev : offset;
  char* dst = (blockIdx.z == 0 ? k_cache : v_cache) + blockIdx.y * c_head_stride;
  const char* src = (blockIdx.z == 0 ? k_new : v_new) + blockIdx.y * n_head_stride;
  const int lane = threadIdx.x & 15, r0 = blockIdx.x * kRowsBlock + (threadIdx.x >> 4);
  uint4 raw[kRowsEach];
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i) {
    const int r = r0 + 16 * i;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (r < n_new) raw[i] = *(reinterpret_cast<const uint4*>(src + r * n_row_stride) + lane);
  }
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i) {
    const int r = r0 + 16 * i;
    uint32_t code, word;
    quantise8(raw[i], code, word);
    if (r >= n_new) continue;
    const int64_t row = off + r;
    if (row < 0 || row >= capacity) {
      if (lane == 0) set_status(status, RT_DEV_OVERFLOW);
      continue;
    }
    char* p = dst + row * kQ4Row;
    *reinterpret_cast<uint32_t*>(p + lane * 4) = code;
    if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(p + kQ4Codes + (lane >> 2) * 2) = static_cast<uint16_t>(word);
  }
}

// Every scale the format holds, the largest too: 0x4300 | u is 128 + u, and the
// difference to 128 + z and its product with s are exact.
__device__ __forceinline__ uint4 q4_decode8_any(uint32_t word, uint32_t w) {
  const uint32_t z2 = 0x43004300u | ((w & 15u) * 0x00010001u), s2 = q4_scale2(w);
  auto value = [&](uint32_t x) {
    x = (x & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                     *reinterpret_cast<const __nv_bfloat162*>(&z2));
    const __nv_bfloat162 v = __hmul2(d, *reinterpret_cast<const __nv_bfloat162*>(&s2));
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  return make_uint4(value(word), value(word >> 4), value(word >> 8), value(word >> 12));
}

__global__ void __launch_bounds__(256) kv_read_q4_kernel(const char* cache, int64_t c_head_stride, char* out,
                                                         int64_t o_head_stride, int64_t o_row_stride, int n,
                                                         int64_t start) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 15, r0 = blockIdx.x * kRowsBlock + (threadIdx.x >> 4);
  const char* src = cache + blockIdx.y * c_head_stride + start * kQ4Row;
  char* dst = out + blockIdx.y * o_head_stride;
  uint32_t code[kRowsEach], word[kRowsEach];
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i) {
    const int r = r0 + 16 * i;
    code[i] = word[i] = 0;
    if (r < n) {
      code[i] = *reinterpret_cast<const uint32_t*>(src + static_cast<int64_t>(r) * kQ4Row + lane * 4);
      word[i] = *reinterpret_cast<const uint16_t*>(src + static_cast<int64_t>(r) * kQ4Row + kQ4Codes + (lane >> 2) * 2);
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i) {
    const int r = r0 + 16 * i;
    if (r < n) *(reinterpret_cast<uint4*>(dst + r * o_row_stride) + lane) = q4_decode8_any(code[i], word[i]);
  }
}

}  // namespace rt

using namespace rt;

extern "C" int rt_kv_append_q4(void* k_cache, void* v_cache, int64_t cache_head_stride, const void* k_new,
                               const void* v_new, int64_t new_head_stride, int64_t new_row_stride, int n_heads,
                               int n_new, int head_dim, int64_t capacity, int64_t offset, const int64_t* offset_dev,
                               int* status, rt_stream_t stream) {
  if (n_heads < 0 || n_new < 0 || capacity < 0) return RT_ERR_INVALID_ARGUMENT;
  if (head_dim != 128) return RT_ERR_UNSUPPORTED;
  if (n_heads == 0 || n_new == 0) return RT_OK;
  if (!k_cache || !v_cache || !k_new || !v_new) return RT_ERR_INVALID_ARGUMENT;
  if (offset_dev == nullptr && (offset < 0 || offset > capacity - n_new)) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t a16 = reinterpret_cast<uint64_t>(k_new) | reinterpret_cast<uint64_t>(v_new) |
                       static_cast<uint64_t>(new_head_stride) | static_cast<uint64_t>(new_row_stride);
  const uint64_t a8 = reinterpret_cast<uint64_t>(k_cache) | reinterpret_cast<uint64_t>(v_cache) |
                      static_cast<uint64_t>(cache_head_stride);
  if ((a16 & 15) || (a8 & 7)) return RT_ERR_INVALID_ARGUMENT;
  if (n_heads > 65535) return RT_ERR_UNSUPPORTED;
  const dim3 grid((n_new + kRowsBlock - 1) / kRowsBlock, n_heads, 2);
  return record_cuda(launch_ex(kv_append_q4_kernel, grid, dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), 1,
                               static_cast<char*>(k_cache), static_cast<char*>(v_cache), cache_head_stride,
                               static_cast<const char*>(k_new), static_cast<const char*>(v_new), new_head_stride,
                               new_row_stride, n_new, capacity, offset, offset_dev, status));
}

extern "C" int rt_kv_read_q4(const void* cache, int64_t cache_head_stride, void* out, int64_t out_head_stride,
                             int64_t out_row_stride, int n_heads, int n, int head_dim, int64_t capacity,
                             int64_t start, rt_stream_t stream) {
  if (n_heads < 0 || n < 0 || capacity < 0 || start < 0 || start > capacity - n) return RT_ERR_INVALID_ARGUMENT;
  if (head_dim != 128) return RT_ERR_UNSUPPORTED;
  if (n_heads == 0 || n == 0) return RT_OK;
  if (!cache || !out) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t a16 = reinterpret_cast<uint64_t>(out) | static_cast<uint64_t>(out_head_stride) |
                       static_cast<uint64_t>(out_row_stride);
  const uint64_t a8 = reinterpret_cast<uint64_t>(cache) | static_cast<uint64_t>(cache_head_stride);
  if ((a16 & 15) || (a8 & 7)) return RT_ERR_INVALID_ARGUMENT;
  if (n_heads > 65535) return RT_ERR_UNSUPPORTED;
  const dim3 grid((n + kRowsBlock - 1) / kRowsBlock, n_heads);
  return record_cuda(launch_ex(kv_read_q4_kernel, grid, dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), 1,
                               static_cast<const char*>(cache), cache_head_stride, static_cast<char*>(out),
                               out_head_stride, out_row_stride, n, start));
}
