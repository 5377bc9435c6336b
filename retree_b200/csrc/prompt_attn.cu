// Causal attention over whole prompts (packed sequences): one warp per (token, query head).
#include <cuda_fp16.h>

#include "common.cuh"
#include "host_util.h"

namespace rt {

struct PromptParams {
  const char* q;
  int64_t q_tok_stride, q_head_stride;
  const char* k;
  const char* v;
  int64_t kv_head_stride, kv_row_stride;
  char* out;
  int64_t out_tok_stride, out_head_stride;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int num_seqs, total_q, total_k, hq, group;
  float scale_log2;
  int* status;
};

template <typename T>
__device__ __forceinline__ float2 up2(uint32_t w) {
  if constexpr (sizeof(T) == 2 && std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<__half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t down2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  return pack_bf16x2(a, b);
}

template <typename T>
__global__ void __launch_bounds__(128) prompt_attn_simple(const PromptParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t gw = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (gw >= static_cast<int64_t>(p.total_q) * p.hq) return;
  const int tok = static_cast<int>(gw / p.hq), h = static_cast<int>(gw - static_cast<int64_t>(tok) * p.hq);
  int q0 = 0, q1 = p.total_q, k0 = 0, k1 = p.total_k;
  if (p.cu_q != nullptr) {
    int b = 0;
    for (; b < p.num_seqs; ++b) {
      q0 = p.cu_q[b];
      q1 = p.cu_q[b + 1];
      k0 = p.cu_k[b];
      k1 = p.cu_k[b + 1];
      if (q0 < 0 || q1 < q0 || q1 > p.total_q || k0 < 0 || k1 < k0 || k1 > p.total_k) {
        set_status(p.status, RT_DEV_BAD_INDEX);
        continue;
      }
      if (tok >= q0 && tok < q1) break;
    }
    if (b == p.num_seqs) return;
  }
  const int last = k0 + (tok - q0) + (k1 - k0) - (q1 - q0);
  const char* kb = p.k + (h / p.group) * p.kv_head_stride;
  const char* vb = p.v + (h / p.group) * p.kv_head_stride;
  const uint2 qr = *reinterpret_cast<const uint2*>(p.q + tok * p.q_tok_stride + h * p.q_head_stride + lane * 8);
  const float2 qa = up2<T>(qr.x), qb = up2<T>(qr.y);
  float m = -INFINITY, l = 0.f, acc[4] = {};
  for (int key = k0; key <= last; ++key) {
    const uint2 kr = *reinterpret_cast<const uint2*>(kb + key * p.kv_row_stride + lane * 8);
    const uint2 vr = *reinterpret_cast<const uint2*>(vb + key * p.kv_row_stride + lane * 8);
    const float2 ka = up2<T>(kr.x), kc = up2<T>(kr.y), va = up2<T>(vr.x), vc = up2<T>(vr.y);
    float s = qa.x * ka.x + qa.y * ka.y + qb.x * kc.x + qb.y * kc.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float f = ex2(m - mu), e = ex2(s - mu);
    l = l * f + e;
    acc[0] = acc[0] * f + e * va.x;
    acc[1] = acc[1] * f + e * va.y;
    acc[2] = acc[2] * f + e * vc.x;
    acc[3] = acc[3] * f + e * vc.y;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(p.out + tok * p.out_tok_stride + h * p.out_head_stride + lane * 8) =
      make_uint2(down2<T>(acc[0] * inv, acc[1] * inv), down2<T>(acc[2] * inv, acc[3] * inv));
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_prompt_attn_workspace_size(int64_t, int64_t, int, int, int) { return 0; }

extern "C" int rt_prompt_attn(const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* k,
                              const void* v, int64_t kv_head_stride, int64_t kv_row_stride, void* out,
                              int64_t out_tok_stride, int64_t out_head_stride, int dtype, const int32_t* cu_q,
                              const int32_t* cu_k, int num_seqs, int64_t total_q, int64_t total_k, int num_q_heads,
                              int num_kv_heads, int head_dim, float scale, void* workspace, size_t workspace_bytes,
                              int* status, rt_stream_t stream) {
  if (num_seqs < 0 || total_q < 0 || total_k < 0 || num_kv_heads <= 0 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads)
    return RT_ERR_INVALID_ARGUMENT;
  if (!(scale >= 0.f) || scale > 3e38f) return RT_ERR_INVALID_ARGUMENT;
  if (cu_q == nullptr && (cu_k != nullptr || num_seqs != 1)) return RT_ERR_INVALID_ARGUMENT;
  if (head_dim != 128 || (dtype != 1 && dtype != 2)) return RT_ERR_UNSUPPORTED;
  const int G = num_q_heads / num_kv_heads;
  if (G > 128 || total_q > INT32_MAX || total_k > INT32_MAX) return RT_ERR_UNSUPPORTED;
  if (total_q == 0 || num_seqs == 0) return RT_OK;
  if (!q || !out || (total_k > 0 && (!k || !v))) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t align_bits = reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(k) |
                              reinterpret_cast<uint64_t>(v) | reinterpret_cast<uint64_t>(out) |
                              static_cast<uint64_t>(q_tok_stride) | static_cast<uint64_t>(q_head_stride) |
                              static_cast<uint64_t>(kv_head_stride) | static_cast<uint64_t>(kv_row_stride) |
                              static_cast<uint64_t>(out_tok_stride) | static_cast<uint64_t>(out_head_stride);
  if (align_bits & 15) return RT_ERR_INVALID_ARGUMENT;
  PromptParams p{static_cast<const char*>(q), q_tok_stride, q_head_stride, static_cast<const char*>(k),
                 static_cast<const char*>(v), kv_head_stride, kv_row_stride, static_cast<char*>(out), out_tok_stride,
                 out_head_stride, cu_q, cu_k ? cu_k : cu_q, num_seqs, static_cast<int>(total_q),
                 static_cast<int>(total_k), num_q_heads, G, scale * 1.4426950408889634f, status};
  const int64_t warps = total_q * num_q_heads;
  const dim3 grid(static_cast<unsigned>((warps + 3) / 4));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return record_cuda(dtype == 1 ? launch_ex(prompt_attn_simple<__nv_bfloat16>, grid, dim3(128), 0, s, 1, p)
                                : launch_ex(prompt_attn_simple<__half>, grid, dim3(128), 0, s, 1, p));
}
