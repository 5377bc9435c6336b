// 4-bit KV cache rows: append (quantise) and read (decode).
//
// Both are data movement with a few operations a value: 256 bytes in and 72
// out for a row of one head (append), 72 in and 256 out (read).  Sixteen lanes
// hold a row, eight values (16 bytes of bf16, one code word) each; the four
// lanes of a 32-value group reduce its range with two shuffles.
#include "common.cuh"
#include "host_util.h"
#include "q4_row.cuh"

namespace rt {

__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

__global__ void __launch_bounds__(256) kv_append_q4_kernel(char* k_cache, char* v_cache, int64_t c_head_stride,
                                                           const char* k_new, const char* v_new,
                                                           int64_t n_head_stride, int64_t n_row_stride, int n_heads,
                                                           int n_new, int64_t capacity, int64_t offset,
                                                           const int64_t* offset_dev, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t off = offset_dev != nullptr ? *offset_dev : offset;
  char* dst_base = blockIdx.y == 0 ? k_cache : v_cache;
  const char* src_base = blockIdx.y == 0 ? k_new : v_new;
  const int lane = threadIdx.x & 15;
  const int64_t rows = static_cast<int64_t>(n_heads) * n_new;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  // all 32 lanes of a warp stay in the loop together (two rows a warp)
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 5) * 2; base < rows; base += step) {
    const int64_t hr = base + ((threadIdx.x >> 4) & 1);
    const bool live = hr < rows;
    const int h = live ? static_cast<int>(hr / n_new) : 0;
    const int r = live ? static_cast<int>(hr - static_cast<int64_t>(h) * n_new) : 0;
    const int64_t row = off + r;
    float x[8];
    unpack8(*(reinterpret_cast<const uint4*>(src_base + h * n_head_stride + r * n_row_stride) + lane), x);
    float lo = 0.f, hi = 0.f;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      bad |= (__float_as_uint(x[i]) & 0x7F800000u) == 0x7F800000u;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) bad |= __shfl_xor_sync(0xFFFFFFFFu, bad, o);
    // (hi - lo) / 15, halved first so that the difference cannot overflow
    float s = __fdiv_rn(__fsub_rn(0.5f * hi, 0.5f * lo), 7.5f);
    s = __uint_as_float((__float_as_uint(s) + 0xFFFFFu) & ~0xFFFFFu);
    uint32_t word = kQ4NanWord, code = 0;
    if (!bad) {
      word = 0;
      if (s >= 1.17549435e-38f) {
        const float z = rintf(__fdiv_rn(-lo, s));
        word = ((__float_as_uint(s) >> 16) & 0x7FF0u) | static_cast<uint32_t>(z);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)) + z, 0.f), 15.f);
          code |= static_cast<uint32_t>(u) << (4 * ((i >> 1) + 4 * (i & 1)));
        }
      }
    }
    if (!live) continue;
    if (row < 0 || row >= capacity) {
      if (lane == 0) set_status(status, RT_DEV_OVERFLOW);
      continue;
    }
    char* dst = dst_base + h * c_head_stride + row * kQ4Row;
    *reinterpret_cast<uint32_t*>(dst + lane * 4) = code;
    if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(dst + kQ4Codes + (lane >> 2) * 2) = static_cast<uint16_t>(word);
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
                                                         int64_t o_head_stride, int64_t o_row_stride, int n_heads,
                                                         int n, int64_t start) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 15;
  const int64_t rows = static_cast<int64_t>(n_heads) * n;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  for (int64_t hr = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); hr < rows; hr += step) {
    const int h = static_cast<int>(hr / n);
    const int r = static_cast<int>(hr - static_cast<int64_t>(h) * n);
    const char* src = cache + h * c_head_stride + (start + r) * kQ4Row;
    const uint32_t code = *reinterpret_cast<const uint32_t*>(src + lane * 4);
    const uint32_t word = *reinterpret_cast<const uint16_t*>(src + kQ4Codes + (lane >> 2) * 2);
    *(reinterpret_cast<uint4*>(out + h * o_head_stride + r * o_row_stride) + lane) =
        q4_decode8_any(code, word);
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
  if (offset_dev == nullptr && (offset < 0 || offset + n_new > capacity)) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t a16 = reinterpret_cast<uint64_t>(k_new) | reinterpret_cast<uint64_t>(v_new) |
                       static_cast<uint64_t>(new_head_stride) | static_cast<uint64_t>(new_row_stride);
  const uint64_t a8 = reinterpret_cast<uint64_t>(k_cache) | reinterpret_cast<uint64_t>(v_cache) |
                      static_cast<uint64_t>(cache_head_stride);
  if ((a16 & 15) || (a8 & 7)) return RT_ERR_INVALID_ARGUMENT;
  const int64_t rows = static_cast<int64_t>(n_heads) * n_new;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + 15) / 16, 148 * 8)), 2);
  return record_cuda(launch_ex(kv_append_q4_kernel, grid, dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), 1,
                               static_cast<char*>(k_cache), static_cast<char*>(v_cache), cache_head_stride,
                               static_cast<const char*>(k_new), static_cast<const char*>(v_new), new_head_stride,
                               new_row_stride, n_heads, n_new, capacity, offset, offset_dev, status));
}

extern "C" int rt_kv_read_q4(const void* cache, int64_t cache_head_stride, void* out, int64_t out_head_stride,
                             int64_t out_row_stride, int n_heads, int n, int head_dim, int64_t capacity,
                             int64_t start, rt_stream_t stream) {
  if (n_heads < 0 || n < 0 || capacity < 0 || start < 0 || start + n > capacity) return RT_ERR_INVALID_ARGUMENT;
  if (head_dim != 128) return RT_ERR_UNSUPPORTED;
  if (n_heads == 0 || n == 0) return RT_OK;
  if (!cache || !out) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t a16 = reinterpret_cast<uint64_t>(out) | static_cast<uint64_t>(out_head_stride) |
                       static_cast<uint64_t>(out_row_stride);
  const uint64_t a8 = reinterpret_cast<uint64_t>(cache) | static_cast<uint64_t>(cache_head_stride);
  if ((a16 & 15) || (a8 & 7)) return RT_ERR_INVALID_ARGUMENT;
  const int64_t rows = static_cast<int64_t>(n_heads) * n;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + 15) / 16, 148 * 16)));
  return record_cuda(launch_ex(kv_read_q4_kernel, grid, dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), 1,
                               static_cast<const char*>(cache), cache_head_stride, static_cast<char*>(out),
                               out_head_stride, out_row_stride, n_heads, n, start));
}
