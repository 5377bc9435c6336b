// One 128-key block of the online softmax for one query row held by one thread
// (S, P and O of the row live in the thread's TMEM lane).
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace rt {

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}

constexpr float kLazyRescale = 8.0f;  // log2 units

// sr: the row's 128 raw scores (-inf where hidden), read from the S tile whose
// first 64 columns (ts) take the weights P = 2^(s * sl2 - m) as 16-bit pairs.
// The running maximum m moves only when a score passes it by 2^8, so weights stay
// below that and O (128 columns at `to`) is rescaled rarely; O must hold every
// earlier block (`rescale` is false for a row's first block).  l sums the
// weights in fp32, before they are rounded.  fp16 weights sit 2^6 above the
// maximum's 1 (2^14 at most), which keeps weights down to 2^-20 of it out of the
// subnormal range.
// part1() runs once the weights of the first kPart1 keys are in TMEM, so that
// their product can start under the last quarter's exponentials; the caller
// announces the rest.
constexpr int kPart1 = 96;
template <typename T, typename Part1>
__device__ __forceinline__ void softmax_block(const uint32_t (&sr)[4][32], uint32_t ts, uint32_t to, bool rescale,
                                              float sl2, float& m, float& l, Part1 part1) {
  constexpr float kLift = std::is_same_v<T, __half> ? 6.f : 0.f;
  float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 32; ++i) a[i & 3] = fmaxf(a[i & 3], __uint_as_float(sr[c][i]));
  const float m_new = fmaxf(m, fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * sl2);
  const bool need = m_new > m + kLazyRescale;  // false while m_new is -inf
  if (__any_sync(0xFFFFFFFFu, need)) {
    if (rescale) {
      const float f = need ? ex2(m - m_new) : 1.f;
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        uint32_t o[16];
        tmem_ld16(to + c * 16, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st16(to + c * 16, o);
      }
      l *= f;
    }
    if (need) m = m_new;
  }
  const float mu = (m == -INFINITY ? 0.f : m) - kLift;
  const float2 sc2 = make_float2(sl2, sl2), sh2 = make_float2(-mu, -mu);
  float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 x =
          ffma2(make_float2(__uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1])), sc2, sh2);
      const float p0 = ex2(x.x), p1 = ex2(x.y);
      acc[i & 1] = fadd2(acc[i & 1], make_float2(p0, p1));
      pk[i] = pack2<T>(p0, p1);
    }
    tmem_st16(ts + c * 16, pk);
    if (c == kPart1 / 32 - 1) {
      tmem_wait_st();
      tc_fence_before();
      part1();
    }
  }
  tmem_wait_st();
  tc_fence_before();
  l += (acc[0].x + acc[1].x) + (acc[0].y + acc[1].y);
}

// A warp's 32 output rows, a lane a row, written through 2 KB of shared memory four
// lanes a row, so that a store touches 8 rows and not 32.
struct RowsOut {
  uint32_t stage;
  uint64_t to[4];  // rows lane / 4 + 0, 8, 16, 24 (0: no row)
  __device__ __forceinline__ RowsOut(uint32_t stage, uint64_t row) : stage(stage) {
#pragma unroll
    for (int q = 0; q < 4; ++q) to[q] = __shfl_sync(0xFFFFFFFFu, row, q * 8 + ((threadIdx.x & 31) >> 2));
  }
  // 64 bytes of each row, `at` bytes into it
  __device__ __forceinline__ void put(const uint4 (&v)[4], int at) const {
    const int lane = threadIdx.x & 31, piece = lane & 3;
#pragma unroll
    for (int q = 0; q < 4; ++q) sts128(stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4), v[q]);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int from = q * 8 + (lane >> 2);
      const uint4 x = lds128(stage + from * 64 + ((piece ^ ((from >> 1) & 3)) << 4));
      if (to[q] != 0) *reinterpret_cast<uint4*>(to[q] + at + piece * 16) = x;
    }
    __syncwarp();
  }
  // values 32c .. 32c + 31 of each row, in T or in fp32
  template <typename T>
  __device__ __forceinline__ void put32(const float (&x)[32], int c) const {
    uint4 v[4];
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float* f = x + h * 16 + q * 4;
          v[q] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        }
        put(v, c * 128 + h * 64);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float* f = x + q * 8;
        v[q] = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
      }
      put(v, c * 64);
    }
  }
};

}  // namespace rt
