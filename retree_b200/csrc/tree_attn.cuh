// What the tree-attention kernels share: the launch's parameters, key ranges and
// visibility, and the merge of key splits (inside a cluster, or from the
// workspace by a second kernel).
#pragma once

#include "common.cuh"

namespace rt {

constexpr int kHD = 128;
constexpr int kBM = 128;       // query rows of a tile (and of a workspace slot)
constexpr int kMaxMerge = 16;  // cluster size limit (16 needs the non-portable cluster attribute)

struct AttnParams {
  const char* q;
  int64_t q_tok_stride, q_head_stride;
  char* out;
  int64_t out_tok_stride, out_head_stride;
  const uint32_t* mask;
  int mask_words;
  int n;
  int64_t prefix_len;
  const int64_t* prefix_len_dev;
  int group, num_kv_heads, tiles, num_splits;
  int merge;       // 1: the splits of a (kv head, tile) form one cluster and are merged in the kernel
  float scale_log2;
  float* ws_o;     // [split][kv_head][tiles*128][128]
  float2* ws_ml;   // [split][kv_head][tiles*128]  (m in log2 units, l)
  int* status;
  // warp-level path only
  const char* k;
  const char* v;
  int64_t kv_head_stride, kv_row_stride;
  // 4-bit cache: rows of a head; a prefix length that does not fit writes nothing (0: not checked)
  int64_t capacity;
  // with tail_splits > 0 the rows from tail_row on have so many splits and those before
  // them row_splits; num_splits is the larger count
  int row_splits, tail_splits, tail_row;
};

__device__ __forceinline__ int64_t prefix_rows(const AttnParams& p) {
  return p.prefix_len_dev != nullptr ? *p.prefix_len_dev : p.prefix_len;
}
__device__ __forceinline__ int64_t key_count(const AttnParams& p) { return prefix_rows(p) + p.n; }
// Whether the keys are rows of the cache (asked before a sum that a wild length could overflow).
__device__ __forceinline__ bool prefix_fits(const AttnParams& p, int64_t L) { return L >= 0 && L <= p.capacity - p.n; }

// Block range [b0, b1) of this split: the blocks spread evenly (range sizes
// differ by at most one, so no split runs two blocks while another idles).
__device__ __forceinline__ void split_range(int64_t total_keys, int split, int splits, int64_t blk, int64_t& b0,
                                            int64_t& b1) {
  const int64_t nblk = (total_keys + blk - 1) / blk;
  b0 = nblk * split / splits;
  b1 = nblk * (split + 1) / splits;
}

// Visibility of the 32 keys [k0, k0+32) for one node: prefix keys (< L) are
// visible, tree key t = key - L uses bit t of the node's mask row, keys at or
// past L + n are hidden.
__device__ __forceinline__ uint32_t visible_word(int64_t k0, int64_t L, int n, const uint32_t* mrow, int words) {
  const int64_t pre = L - k0;  // prefix columns at the start of the window
  if (pre >= 32) return 0xFFFFFFFFu;
  uint32_t bits = pre > 0 ? ((1u << pre) - 1u) : 0u;
  const int64_t t0 = k0 - L;  // tree index of column 0 (negative: starts in the prefix)
  uint32_t tb;
  if (t0 >= 0) {
    const int w = static_cast<int>(t0 >> 5), sh = static_cast<int>(t0 & 31);
    const uint32_t lo = w < words ? mrow[w] : 0u;
    const uint32_t hi = (sh != 0 && w + 1 < words) ? mrow[w + 1] : 0u;
    tb = sh ? ((lo >> sh) | (hi << (32 - sh))) : lo;
  } else {
    tb = mrow[0] << static_cast<int>(-t0);
  }
  // tree columns past the last node are hidden
  const int64_t lim = static_cast<int64_t>(n) - t0;  // columns c < lim have t < n
  if (lim < 32) tb &= lim <= 0 ? 0u : ((1u << lim) - 1u);
  return bits | tb;
}

__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float4 merge_chunk(const float4 (&o)[kMaxMerge], int S, const float* wrow) {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int u = 0; u < kMaxMerge; ++u) {
    const float wu = wrow[u];
    if (u < S && wu != 0.f) {
      acc.x = fmaf(wu, o[u].x, acc.x);
      acc.y = fmaf(wu, o[u].y, acc.y);
      acc.z = fmaf(wu, o[u].z, acc.z);
      acc.w = fmaf(wu, o[u].w, acc.w);
    }
  }
  return acc;
}

// The rank weights of one row from every rank's (m, l).
__device__ __forceinline__ void merge_weights(const float2 (&ml)[kMaxMerge], float (&w)[kMaxMerge]) {
  float M = -INFINITY;
#pragma unroll
  for (int u = 0; u < kMaxMerge; ++u) M = fmaxf(M, ml[u].x);
  float lsum = 0.f;
#pragma unroll
  for (int u = 0; u < kMaxMerge; ++u) {
    w[u] = (M == -INFINITY || ml[u].x == -INFINITY) ? 0.f : ex2(ml[u].x - M);
    lsum = fmaf(w[u], ml[u].y, lsum);
  }
  const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
#pragma unroll
  for (int u = 0; u < kMaxMerge; ++u) w[u] = w[u] * inv;
}

// In-kernel split merge: once a CTA's last PV product is final, the Q / K / V
// ring is idle and holds the CTA's unnormalised fp32 O tile (rows of 512 B,
// 16-byte chunks XOR-swizzled by row) and its rows' (m, l).
constexpr uint32_t kOffStage = 0;
constexpr uint32_t kOffMl = 65536;
constexpr uint32_t kOffWeights = 98304;  // [owned rows][kMaxMerge] fp32 merge weights

// Byte offset of 16-byte chunk `c` (0..31) of row `r` in the merge's O stage.
__device__ __forceinline__ uint32_t stage_off(int r, int c) {
  return kOffStage + static_cast<uint32_t>(r) * 512u + static_cast<uint32_t>((c ^ (r & 31)) << 4);
}

// The split merge inside the cluster (every thread of every CTA calls it, or the
// first kThreads of each while the others pass its two cluster barriers; the
// cluster is the S = num_splits CTAs of one (kv head, tile), rank = split).
// Each CTA has staged its unnormalised O rows and (m, l) in its own shared
// memory.  Rank c merges the tile rows r = c, c + S, ...: the rank weights of
// a row are 2^(m_s - M) / L (L = sum_s 2^(m_s - M) l_s, in rank order), and the
// chunks are summed in rank order (a rank of weight 0 -- no key of the row, or
// a row it did not stage -- is skipped, never multiplied) into the bf16
// output.  When every thread has at most one (row, 4-dim chunk) item, each
// item's thread loads every rank's (m, l) and chunk at once and forms the
// weights itself: one distributed-shared-memory round trip.  Otherwise one
// thread per row forms the weights into a shared table first and the item
// threads then load only the chunks.  The last barrier keeps every CTA's
// shared memory until all ranks have read it.
template <int kThreads, bool kWholeBlock = true>
__device__ __forceinline__ void merge_splits(const AttnParams& p, unsigned char* smem, int rank, int kvh, int row0,
                                             int rows_total) {
  __syncwarp();
  cluster_sync_all();
  const int tid = threadIdx.x;
  const int S = p.num_splits, G = p.group;
  const int rows_here = min(kBM, rows_total - row0);
  const int owned = rows_here > rank ? (rows_here - rank + S - 1) / S : 0;
  const uint32_t base = smem_u32(smem);
  float* wtab = reinterpret_cast<float*>(smem + kOffWeights);
  auto store = [&](int rr, int c, const float4& acc) {
    const int R = row0 + rr;
    const int node = R / G, h = kvh * G + (R - node * G);
    uint2 pk;
    pk.x = pack_bf16x2(acc.x, acc.y);
    pk.y = pack_bf16x2(acc.z, acc.w);
    *reinterpret_cast<uint2*>(p.out + node * p.out_tok_stride + h * p.out_head_stride + c * 8) = pk;
  };
  if (owned * 32 <= kThreads) {  // the same in every thread of the CTA
    const int it = tid;
    if (it < owned * 32) {
      const int i = it >> 5, c = it & 31;
      const int rr = rank + S * i;
      const uint32_t off = base + stage_off(rr, c);
      float2 ml[kMaxMerge];
      float4 o[kMaxMerge];
#pragma unroll
      for (int u = 0; u < kMaxMerge; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u < S) {
          ml[u] = ld_cluster_f32x2(cluster_map(base + kOffMl + rr * 8, u));
          o[u] = ld_cluster_f32x4(cluster_map(off, u));
        }
      }
      float w[kMaxMerge];
      merge_weights(ml, w);
      store(rr, c, merge_chunk(o, S, w));
    }
  } else {
    for (int i = tid; i < owned; i += kThreads) {
      const int rr = rank + S * i;
      float2 ml[kMaxMerge];
#pragma unroll
      for (int u = 0; u < kMaxMerge; ++u)
        ml[u] = u < S ? ld_cluster_f32x2(cluster_map(base + kOffMl + rr * 8, u)) : make_float2(-INFINITY, 0.f);
      float w[kMaxMerge];
      merge_weights(ml, w);
#pragma unroll
      for (int u = 0; u < kMaxMerge; ++u) wtab[i * kMaxMerge + u] = w[u];
    }
    if constexpr (kWholeBlock) __syncthreads();
    else asm volatile("bar.sync 2, %0;" ::"n"(kThreads) : "memory");
    for (int it = tid; it < owned * 32; it += kThreads) {
      const int i = it >> 5, c = it & 31;
      const int rr = rank + S * i;
      const uint32_t off = base + stage_off(rr, c);
      float4 o[kMaxMerge];
#pragma unroll
      for (int u = 0; u < kMaxMerge; ++u) {
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u < S && wtab[i * kMaxMerge + u] != 0.f) o[u] = ld_cluster_f32x4(cluster_map(off, u));
      }
      store(rr, c, merge_chunk(o, S, wtab + i * kMaxMerge));
    }
  }
  __syncwarp();
  cluster_sync_all();
}

// ---------------------------------------------------------------------------
// Split merge: one warp per (kv head, tile row); lane owns 4 dims.
// ---------------------------------------------------------------------------
constexpr int kFastSplits = 24;  // up to this many splits: every load of a row issued at once

static __global__ void __launch_bounds__(128) attn_combine_kernel(const AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rows = p.n * p.group;
  if (p.capacity > 0 && !prefix_fits(p, prefix_rows(p))) return;
  const int64_t rows_ws = static_cast<int64_t>(p.tiles) * kBM;
  auto splits_of = [&](int R) {
    return p.tail_splits == 0 ? p.num_splits : R >= p.tail_row ? p.tail_splits : p.row_splits;
  };
  const float2 none = make_float2(-INFINITY, 0.f);
  if (p.num_splits <= kFastSplits) {
    // Two warps per (kv head, row), one per 64-dim half, lane owns 2 dims.
    // Every load of the row is independent of the others, so all of them --
    // the splits' partial rows and (max, sum) pairs -- go out at once: one
    // L2 round trip instead of one for the maxima and one per batch of rows.
    // A split whose weight is zero (max -inf) is skipped, never multiplied;
    // the per-element sum runs over the splits in order, as below.
    const int gw = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (gw >= 2 * p.num_kv_heads * rows) return;
    const int half = gw & 1, pair = gw >> 1;
    const int kvh = pair / rows, R = pair - kvh * rows, S = splits_of(R);
    auto slot = [&](int s) { return (static_cast<int64_t>(s) * p.num_kv_heads + kvh) * rows_ws + R; };
    const int d0 = half * 64 + lane * 2;
    float2 o[kFastSplits];
#pragma unroll
    for (int u = 0; u < kFastSplits; ++u)
      o[u] = u < S ? *reinterpret_cast<const float2*>(p.ws_o + slot(u) * kHD + d0) : make_float2(0.f, 0.f);
    const float2 ml = lane < S ? p.ws_ml[slot(lane)] : none;
    float M = ml.x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, off));
    float2 acc = make_float2(0.f, 0.f);
    float lsum = 0.f;
    if (M > -INFINITY) {
      const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      lsum = w * ml.y;
#pragma unroll
      for (int u = 0; u < kFastSplits; ++u) {
        const float wu = __shfl_sync(0xFFFFFFFFu, w, u);
        if (u < S && wu != 0.f) {
          acc.x = fmaf(wu, o[u].x, acc.x);
          acc.y = fmaf(wu, o[u].y, acc.y);
        }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) lsum += __shfl_xor_sync(0xFFFFFFFFu, lsum, off);
    }
    const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
    const int node = R / p.group, h = kvh * p.group + (R - node * p.group);
    *reinterpret_cast<uint32_t*>(p.out + node * p.out_tok_stride + h * p.out_head_stride + d0 * 2) =
        pack_bf16x2(acc.x * inv, acc.y * inv);
    return;
  }
  const int gw = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (gw >= p.num_kv_heads * rows) return;
  const int kvh = gw / rows, R = gw - kvh * rows, S = splits_of(R);
  auto slot = [&](int s) { return (static_cast<int64_t>(s) * p.num_kv_heads + kvh) * rows_ws + R; };
  // lane s holds split s's (max, sum); one load per lane instead of a serial walk
  const float2 first = lane < S ? p.ws_ml[slot(lane)] : none;
  float M = first.x;
  for (int base = 32; base < S; base += 32) M = fmaxf(M, base + lane < S ? p.ws_ml[slot(base + lane)].x : -INFINITY);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float lsum = 0.f;
  if (M > -INFINITY) {
    for (int base = 0; base < S; base += 32) {
      const float2 ml = base == 0 ? first : (base + lane < S ? p.ws_ml[slot(base + lane)] : none);
      const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      lsum += w * ml.y;
      const int cnt = min(32, S - base);
      for (int j = 0; j < cnt; j += 8) {
        float4 o[8];
        float ww[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          ww[u] = __shfl_sync(0xFFFFFFFFu, w, (j + u) & 31);
          o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (j + u < cnt && ww[u] != 0.f)
            o[u] = *reinterpret_cast<const float4*>(p.ws_o + slot(base + j + u) * kHD + lane * 4);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          acc.x = fmaf(ww[u], o[u].x, acc.x);
          acc.y = fmaf(ww[u], o[u].y, acc.y);
          acc.z = fmaf(ww[u], o[u].z, acc.z);
          acc.w = fmaf(ww[u], o[u].w, acc.w);
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xFFFFFFFFu, lsum, o);
  }
  const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
  const int node = R / p.group, h = kvh * p.group + (R - node * p.group);
  uint2 pk;
  pk.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  pk.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(p.out + node * p.out_tok_stride + h * p.out_head_stride + lane * 8) = pk;
}

static inline int tiles_for(int n, int G) { return (n * G + kBM - 1) / kBM; }


}  // namespace rt
