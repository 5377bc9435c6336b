// Tree-verify attention over the 4-bit cache: one warp per (node, query head).
#include "common.cuh"
#include "host_util.h"
#include "q4_row.cuh"

namespace rt {

struct Q4AttnParams {
  const char* q;
  int64_t q_tok_stride, q_head_stride;
  const char* k;
  const char* v;
  int64_t kv_head_stride;
  char* out;
  int64_t out_tok_stride, out_head_stride;
  const uint32_t* mask;
  int mask_words, n, hq, group;
  int64_t prefix_len;
  const int64_t* prefix_len_dev;
  float scale_log2;
  int64_t capacity;
  int* status;
};

__global__ void __launch_bounds__(128) tree_attn_q4_simple(const Q4AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int gw = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (gw >= p.n * p.hq) return;
  const int node = gw / p.hq, h = gw - node * p.hq, g = h / p.group;
  const int64_t L = p.prefix_len_dev ? *p.prefix_len_dev : p.prefix_len;
  if (L < 0 || L + p.n > p.capacity) {
    if (lane == 0) set_status(p.status, RT_DEV_BAD_INDEX);
    return;
  }
  const char* kb = p.k + g * p.kv_head_stride;
  const char* vb = p.v + g * p.kv_head_stride;
  const uint2 qr = *reinterpret_cast<const uint2*>(p.q + node * p.q_tok_stride + h * p.q_head_stride + lane * 8);
  const float q0 = __uint_as_float(qr.x << 16), q1 = __uint_as_float(qr.x & 0xFFFF0000u);
  const float q2 = __uint_as_float(qr.y << 16), q3 = __uint_as_float(qr.y & 0xFFFF0000u);
  auto decode4 = [&](const char* row, float (&x)[4]) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + (lane >> 1) * 4) >> ((lane & 1) * 8);
    const uint32_t m = *reinterpret_cast<const uint16_t*>(row + kQ4Codes + (lane >> 3) * 2);
    const uint32_t a = q4_pair(w, q4_zero2(m), q4_scale2(m)), b = q4_pair(w >> 4, q4_zero2(m), q4_scale2(m));
    x[0] = __uint_as_float(a << 16);
    x[1] = __uint_as_float(a & 0xFFFF0000u);
    x[2] = __uint_as_float(b << 16);
    x[3] = __uint_as_float(b & 0xFFFF0000u);
  };
  float m = -INFINITY, l = 0.f, acc[4] = {};
  for (int64_t key = 0; key < L + p.n; ++key) {
    const int64_t t = key - L;
    if (t >= 0 && !((p.mask[static_cast<int64_t>(node) * p.mask_words + (t >> 5)] >> (t & 31)) & 1u)) continue;
    float x[4];
    decode4(kb + key * kQ4Row, x);
    float s = q0 * x[0] + q1 * x[1] + q2 * x[2] + q3 * x[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s);
    const float f = ex2(m - mn), e = ex2(s - mn);
    decode4(vb + key * kQ4Row, x);
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * f + e * x[i];
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint2 pk;
  pk.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  pk.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<uint2*>(p.out + node * p.out_tok_stride + h * p.out_head_stride + lane * 8) = pk;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_tree_attn_q4_workspace_size(int, int, int, int, int64_t, int) { return 0; }

extern "C" int rt_tree_attn_q4(const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* k,
                               const void* v, int64_t kv_head_stride, int64_t kv_capacity, void* out,
                               int64_t out_tok_stride, int64_t out_head_stride, const uint32_t* mask, int mask_words,
                               int n, int64_t prefix_len, const int64_t* prefix_len_dev, int num_q_heads,
                               int num_kv_heads, int head_dim, float scale, int num_splits, void* workspace,
                               size_t workspace_bytes, int* status, rt_stream_t stream) {
  if (!q || !k || !v || !out || !mask) return RT_ERR_INVALID_ARGUMENT;
  if (n <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || prefix_len < 0)
    return RT_ERR_INVALID_ARGUMENT;
  if (!(scale >= 0.f) || scale > 3e38f) return RT_ERR_INVALID_ARGUMENT;
  if (head_dim != 128) return RT_ERR_UNSUPPORTED;
  if (mask_words < (n + 31) / 32) return RT_ERR_INVALID_ARGUMENT;
  if (prefix_len_dev == nullptr && prefix_len + n > kv_capacity) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t align_bits = reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(k) |
                              reinterpret_cast<uint64_t>(v) | reinterpret_cast<uint64_t>(out) |
                              static_cast<uint64_t>(q_tok_stride) | static_cast<uint64_t>(q_head_stride) |
                              static_cast<uint64_t>(kv_head_stride) | static_cast<uint64_t>(out_tok_stride) |
                              static_cast<uint64_t>(out_head_stride);
  if ((align_bits & 15) || (kv_capacity & 1)) return RT_ERR_INVALID_ARGUMENT;
  Q4AttnParams p{static_cast<const char*>(q), q_tok_stride, q_head_stride, static_cast<const char*>(k),
                 static_cast<const char*>(v), kv_head_stride, static_cast<char*>(out), out_tok_stride,
                 out_head_stride, mask, mask_words, n, num_q_heads, num_q_heads / num_kv_heads, prefix_len,
                 prefix_len_dev, scale * 1.4426950408889634f, kv_capacity, status};
  return record_cuda(launch_ex(tree_attn_q4_simple, dim3((n * num_q_heads + 3) / 4), dim3(128), 0,
                               reinterpret_cast<cudaStream_t>(stream), 1, p));
}
