// Tree-verify attention over the 4-bit cache (q4_row.cuh): bf16 queries, GQA,
// head_dim 128, packed ancestor bits over the tree block.
//
// Few query rows (n * group <= 16: single tokens, small trees)
// ---------------------------------------------------------------------------
// One CTA per (key split, kv head), sixteen warps that work alone: each streams
// 32-key tiles (2304 bytes of K, 2304 of V, contiguous) through its own 3-stage
// ring of bulk copies and keeps its rows' running maximum, sum and output in
// registers.  The codes go from shared memory to mma.sync fragments in
// registers, so nothing decoded is stored:
//   S^T = K Q^T      m16n8k16, m = keys, n = query rows: lane (g, t) = (lane / 4,
//                    lane % 4) decodes group t of keys g and g + 8, and the
//                    contraction runs over values in the order the code words
//                    hold them -- Q's fragments are laid out once in that order;
//   O^T += V^T P^T   m = values, k = keys: lane (g, t) decodes code words 2g,
//                    2g+1 of keys 2t, 2t+1, 2t+8, 2t+9, pairing two keys' nibbles
//                    with one byte permute; P^T comes from S^T by 8 x 8
//                    transposes between the lanes.
// With the queries on the n side a single token of a group of four to eight
// heads costs one 8-wide tile, not a 16-wide one.
// The warps' results are merged in shared memory, the splits' in the cluster
// (distributed shared memory) or through the workspace (attn_combine_kernel).
// Measured (32 / 8 heads, in a graph): one token over 2048 rows 7.0 us (launch and
// merges), over 131071 rows 42.7 us (3.5 TB/s).  735 instructions a tile and warp fill 64 % of
// the issue slots, the ALU pipe is 54 % busy; of a warp's cycles an instruction it
// spends 1.1 on a busy pipe, 1.0 on the latency of the instruction before, 0.6 at the
// barriers and 0.4 each on memory and dispatch, and four warps a scheduler do not cover them.
//
// Up to 16 rows come here: over a short cache the other kernel is ahead at 9-16 rows
// (32 / 8 heads, four nodes: 500 rows 10.5 us, 8.0 there; 2048 rows 11.5, 9.6), over a long
// one this (32768 rows 24.4, 28.4; 131071 rows 59.1, 86.0), and so few rows are
// single tokens of wide groups, or the smallest trees, for which the long cache counts.
//
// More query rows
// ---------------------------------------------------------------------------
// One CTA per (key split, kv head, 256 query rows): two 128-row tiles (row r of
// a tile is (node r / group, query head r % group)) in ping-pong on tcgen05 as in
// the prompt attention.  Sixteen warps:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one thread per row;
//   warps 8-14      decode: a lane turns the 72 bytes of a key's K (or V) into its
//                   row of a bf16 SW128 tile, 32 keys a task, the next task's
//                   bytes already on their way from global memory;
//   warp 15         Q by TMA, MMA issuer.
// When only one tile has queries (n * group <= 128, or the last rows) the two
// softmax groups take turns at its key blocks instead: two chains of S, P and O
// for the same queries, merged at the end, so that one chain's softmax still runs
// under the other's products.
// Measured (32 / 8 heads, 32768 rows, in a graph): 17 nodes 28.7 us, of which 12.6 do
// not depend on the length; decode (2140 cycles a block) and the two chains (2050)
// bound the rest alike.  257 nodes 157 us (880 TFLOP/s): a tile's chain (softmax 2250 cycles,
// P to the next S 1500) bounds the block, whose products take 2048.
//
// What hides: the rows behind the tree are stale bytes, so the last tile reads
// their scales as zero; a tree row that reads as NaN turns the scores of the
// nodes that see it into NaN and counts as zero otherwise.
#include <cuda.h>

#include <mutex>

#include "attn_softmax.cuh"
#include "common.cuh"
#include "host_util.h"
#include "q4_row.cuh"
#include "tmap.h"
#include "tree_attn.cuh"

namespace rt {

constexpr int kQsWarps = 16;
constexpr int kQsThreads = kQsWarps * 32;
constexpr int kQsKeys = 32;                               // keys per tile
constexpr uint32_t kQsHalf = kQsKeys * kQ4Row;            // one tile of K (or V)
constexpr int kQsStages = 3;
constexpr uint32_t kQsRing = kQsStages * 2 * kQsHalf;     // of one warp
constexpr uint32_t kQsOffQ = kQsWarps * kQsRing;          // Q fragments [8-row tile][code word][32 lanes] x 16 bytes
constexpr uint32_t kQsOffBar = kQsOffQ + 2 * 4 * 32 * 16;
constexpr uint32_t kQsOffX43 = kQsOffBar + kQsWarps * kQsStages * 8 + 8;
constexpr uint32_t kQsSmem = kQsOffX43 + 8 + 128;
// after the key loop the rings hold the warps' results, then the CTA's
constexpr int kQsRows = 16;
constexpr uint32_t kQsOffPart = 0;                                        // [warp][fragment][lane] x 16 bytes
constexpr uint32_t kQsOffPartMl = kQsOffPart + kQsWarps * kQsRows * 512;  // [warp][row] (m, l)
constexpr uint32_t kQsOffW = kQsOffPartMl + kQsWarps * kQsRows * 8;       // [warp][row] merge weights
constexpr uint32_t kQsStageRow = 132 * 4;                                 // (padded against bank conflicts)
constexpr uint32_t kQsOffStage = kQsOffW + kQsWarps * kQsRows * 4;        // [row][128] fp32
constexpr uint32_t kQsOffStageMl = kQsOffStage + kQsRows * kQsStageRow;   // [row] (m, l)
static_assert(kQsOffStageMl + kQsRows * 8 <= kQsOffQ, "results fit in the rings");

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 tile of 16-bit values, two of a row in each lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ bool q4_is_nan(uint32_t w) { return (w & 0x7F80u) == 0x7F80u; }

__device__ __forceinline__ void store_bf16x4(char* dst, const float4& v) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

// NT: 8-row tiles of queries (rows <= 8 * NT).
template <int NT>
__global__ void __launch_bounds__(kQsThreads, 1) tree_attn_q4_small_kernel(const AttnParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kQsOffBar) + (threadIdx.x >> 5) * kQsStages;
  int* abort_word = reinterpret_cast<int*>(smem + kQsOffBar + kQsWarps * kQsStages * 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y, G = p.group, rows = p.n * G;
  if (lane == 0) {
    for (int i = 0; i < kQsStages; ++i) mbar_init(&full[i], 1);
    if (warp == 0) {
      *abort_word = 0;
      *reinterpret_cast<uint2*>(smem + kQsOffX43) = make_uint2(0x43434343u, 0);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  pdl_launch_dependents();
  pdl_wait();
  const int64_t L = prefix_rows(p);
  if (!prefix_fits(p, L)) {  // the same in every CTA of the launch
    if (tid == 0) set_status(p.status, RT_DEV_BAD_INDEX);
    return;
  }
  const int64_t total = L + p.n;
  int64_t b0, b1;
  split_range(total, split, p.num_splits, kQsKeys, b0, b1);
  const char* kb = p.k + kvh * p.kv_head_stride;
  const char* vb = p.v + kvh * p.kv_head_stride;
  unsigned char* ring = smem + warp * kQsRing;
  const int tiles = static_cast<int>(b1 - b0) > warp ? (static_cast<int>(b1 - b0) - warp + kQsWarps - 1) / kQsWarps : 0;
  auto issue = [&](int i) {  // tile i of this warp (lane 0)
    const int s = i % kQsStages;
    const int64_t key0 = (b0 + warp + static_cast<int64_t>(i) * kQsWarps) * kQsKeys;
    // an even number of rows: 16-byte pieces that end inside the (even) capacity
    const uint32_t bytes = static_cast<uint32_t>((min(static_cast<int64_t>(kQsKeys), total - key0) + 1) & ~int64_t(1)) * kQ4Row;
    mbar_arrive_expect_tx(&full[s], 2 * bytes);
    bulk_load(ring + s * 2 * kQsHalf, kb + key0 * kQ4Row, bytes, &full[s]);
    bulk_load(ring + s * 2 * kQsHalf + kQsHalf, vb + key0 * kQ4Row, bytes, &full[s]);
  };
  if (lane == 0)
    for (int i = 0; i < min(tiles, kQsStages); ++i) issue(i);
  // Q fragments in the code words' order: word wd of lane (g, t) is values 32t + 8wd .. + 7 of row g
  uint4* qs = reinterpret_cast<uint4*>(smem + kQsOffQ);
  if (warp < 4 * NT) {
    const int R = g + 8 * (warp >> 2);
    uint4 x = make_uint4(0, 0, 0, 0);
    if (R < rows) {
      const int node = R / G, h = kvh * G + (R - node * G);
      x = *reinterpret_cast<const uint4*>(p.q + node * p.q_tok_stride + h * p.q_head_stride +
                                          (32 * t + 8 * (warp & 3)) * 2);
    }
    qs[tid] = x;
  }
  __syncthreads();

  const uint32_t sbase = smem_u32(smem);
  const uint32_t x43 = lds64(sbase + kQsOffX43).x;
  const float sl2 = p.scale_log2;
  uint4 qr[NT == 1 ? 4 : 1];  // one tile of queries stays in registers
  if constexpr (NT == 1) {
#pragma unroll
    for (int wd = 0; wd < 4; ++wd) qr[wd] = lds128(sbase + kQsOffQ + (wd * 32 + lane) * 16);
  }
  float O[8][NT][4];
  float m[NT][2], l[NT][2];  // rows 8nt + 2t, + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) O[i][nt][c] = 0.f;
  }
  bool ok = true;
  int i = 0;
#pragma unroll 1
  for (; i < tiles; ++i) {
    const int s = i % kQsStages;
    ok = mbar_wait(&full[s], (i / kQsStages) & 1, abort_word, p.status, RT_DEV_WAIT_TIMEOUT);
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (!ok) break;
    const int64_t key0 = (b0 + warp + static_cast<int64_t>(i) * kQsWarps) * kQsKeys;
    const uint32_t kt = sbase + warp * kQsRing + s * 2 * kQsHalf, vt = kt + kQsHalf;
    // ---- S^T = K Q^T: 16 keys (rows g, g + 8) a step
    float S[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t kw[2][4];
      Q4Group kg[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t row = kt + (mt * 16 + e * 8 + g) * kQ4Row;
        const uint2 a = lds64(row + t * 16), b = lds64(row + t * 16 + 8);
        const uint32_t w = lds16(row + kQ4Codes + t * 2);
        kw[e][0] = a.x;
        kw[e][1] = a.y;
        kw[e][2] = b.x;
        kw[e][3] = b.y;
        kg[e] = q4_group(w);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) S[mt][nt][c] = 0.f;
#pragma unroll
      for (int wd = 0; wd < 4; ++wd) {
        const uint4 a = q4_decode8(kw[0][wd], kg[0], x43), b = q4_decode8(kw[1][wd], kg[1], x43);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 q = NT == 1 ? qr[wd] : lds128(sbase + kQsOffQ + ((nt * 4 + wd) * 32 + lane) * 16);
          mma_bf16(S[mt][nt], a.x, b.x, a.y, b.y, q.x, q.y);
          mma_bf16(S[mt][nt], a.z, b.z, a.w, b.w, q.z, q.w);
        }
      }
    }
    // ---- this lane's V codes: keys 16ks + {2t, 2t+1, 2t+8, 2t+9}, code words 2g, 2g+1
    uint2 vw[2][4];
    uint32_t vm[2][4];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t row = vt + (ks * 16 + 2 * t + (c & 1) + 8 * (c >> 1)) * kQ4Row;
        vw[ks][c] = lds64(row + g * 8);
        vm[ks][c] = lds16(row + kQ4Codes + (g >> 1) * 2);
      }
    // ---- hide, online softmax
    if (key0 + kQsKeys > L) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // (a tree row of NaN shows up in its key's scores instead)
          const int64_t key = key0 + ks * 16 + 2 * t + (c & 1) + 8 * (c >> 1);
          if (key >= total || (key >= L && q4_is_nan(vm[ks][c]))) vm[ks][c] = 0;
        }
      uint32_t bad = 0;  // bit 2 mt + e: this lane's key 16mt + 8e + g is such a row
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = e * 8 + g;
        if (key0 + key >= L && key0 + key < total &&
            q4_is_nan(lds16(vt + key * kQ4Row + kQ4Codes)))
          bad |= 1u << e;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int R = nt * 8 + 2 * t + c;
          const uint32_t vis =
              R < rows ? visible_word(key0, L, p.n, p.mask + static_cast<int64_t>(R / G) * p.mask_words, p.mask_words)
                       : 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float& x = S[e >> 1][nt][2 * (e & 1) + c];
            if ((bad >> e) & 1u) x = __int_as_float(0x7FC00000);
            if (!((vis >> (e * 8 + g)) & 1u)) x = -INFINITY;
          }
        }
    }
    // lazy: the maximum moves when a score passes it by 8 in log2, so weights stay below 2^8
    bool need = false;
    float mx[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[nt][c] = sl2 * fmaxf(fmaxf(S[0][nt][c], S[0][nt][2 + c]), fmaxf(S[1][nt][c], S[1][nt][2 + c]));
        need |= mx[nt][c] > m[nt][c] + 8.f;
      }
    if (__any_sync(0xFFFFFFFFu, need)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = mx[nt][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, o));
          const float mn = fmaxf(m[nt][c], x);
          const float f = mn == -INFINITY ? 1.f : ex2(m[nt][c] - mn);
          m[nt][c] = mn;
          l[nt][c] *= f;
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            O[n][nt][c] *= f;
            O[n][nt][2 + c] *= f;
          }
        }
    }
    // weights, transposed into the B fragments of P V: pf[ks][nt] = keys 2t, 2t+1 | + 8 of row g
    uint2 pf[2][NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mu0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], mu1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float p0 = ex2(fmaf(S[mt][nt][0], sl2, -mu0)), p1 = ex2(fmaf(S[mt][nt][1], sl2, -mu1));
        const float p2 = ex2(fmaf(S[mt][nt][2], sl2, -mu0)), p3 = ex2(fmaf(S[mt][nt][3], sl2, -mu1));
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        pf[mt][nt] = make_uint2(transpose8x8(pack_bf16x2(p0, p1)), transpose8x8(pack_bf16x2(p2, p3)));
      }
    }
    // refill the stage once every lane has read it
    __syncwarp();
    if (lane == 0 && i + kQsStages < tiles) issue(i + kQsStages);
    // ---- O^T += V^T P^T: a step is 16 keys; an m-tile two values of every lane g's sixteen
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const Q4Group ga = q4_group2(vm[ks][0], vm[ks][1]), gb = q4_group2(vm[ks][2], vm[ks][3]);
#pragma unroll
      for (int wd = 0; wd < 2; ++wd) {
        const uint32_t w0 = wd ? vw[ks][0].y : vw[ks][0].x, w1 = wd ? vw[ks][1].y : vw[ks][1].x;
        const uint32_t w2 = wd ? vw[ks][2].y : vw[ks][2].x, w3 = wd ? vw[ks][3].y : vw[ks][3].x;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          // nibbles of two keys: the words' low (or high) halves side by side
          const uint4 x = q4_decode8(__byte_perm(w0, w1, hf ? 0x7632 : 0x5410), ga, x43);
          const uint4 y = q4_decode8(__byte_perm(w2, w3, hf ? 0x7632 : 0x5410), gb, x43);
          const int o = wd * 4 + hf * 2;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16(O[o][nt], x.x, x.y, y.x, y.y, pf[ks][nt].x, pf[ks][nt].y);
            mma_bf16(O[o + 1][nt], x.z, x.w, y.z, y.w, pf[ks][nt].x, pf[ks][nt].y);
          }
        }
      }
    }
  }
  if (!ok && lane == 0)  // copies in flight land before the block leaves
    for (int j = i; j < min(tiles, i + kQsStages); ++j) mbar_wait_drain(&full[j % kQsStages], (j / kQsStages) & 1);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], o);
      if (l[nt][c] != l[nt][c]) m[nt][c] = INFINITY;  // a NaN weight wins every merge
    }
  __syncthreads();  // every warp is done with its ring
  float4* part = reinterpret_cast<float4*>(smem + kQsOffPart);
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      part[((warp * 8 + n) * NT + nt) * 32 + lane] = make_float4(O[n][nt][0], O[n][nt][1], O[n][nt][2], O[n][nt][3]);
  if (g == 0) {
    float2* ml = reinterpret_cast<float2*>(smem + kQsOffPartMl) + warp * kQsRows;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) ml[nt * 8 + 2 * t + c] = make_float2(m[nt][c], l[nt][c]);
  }
  __syncthreads();
  // ---- the warps' merge weights 2^(m_u - M), and the rows' (M, sum)
  float* wtab = reinterpret_cast<float*>(smem + kQsOffW);
  if (tid < kQsWarps * 8 * NT) {
    const float2* ml = reinterpret_cast<const float2*>(smem + kQsOffPartMl);
    const int R = tid % (8 * NT), u = tid / (8 * NT);
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kQsWarps; ++x) M = fmaxf(M, ml[x * kQsRows + R].x);
    auto weight = [&](int x) { return ml[x * kQsRows + R].x == -INFINITY ? 0.f : ex2(ml[x * kQsRows + R].x - M); };
    wtab[u * kQsRows + R] = weight(u);
    if (u == 0) {
      float lsum = 0.f;
#pragma unroll
      for (int x = 0; x < kQsWarps; ++x) lsum = fmaf(weight(x), ml[x * kQsRows + R].y, lsum);
      reinterpret_cast<float2*>(smem + kQsOffStageMl)[R] = make_float2(M, lsum);
    }
  }
  __syncthreads();
  // ---- their sum, into rows: lane (g, t) of fragment n = 4wd + 2hf + q holds values 16g + 8wd + (nibble order)
  for (int it = tid; it < 8 * NT * 32; it += kQsThreads) {
    const int nt = (it >> 5) % NT, n = (it >> 5) / NT, it_g = (it & 31) >> 2, R = nt * 8 + 2 * (it & 3);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < kQsWarps; ++u) {
      const float2 w = *reinterpret_cast<const float2*>(wtab + u * kQsRows + R);
      const float4 o = part[((u * 8 + n) * NT + nt) * 32 + (it & 31)];
      acc.x = fmaf(w.x, o.x, acc.x);
      acc.y = fmaf(w.y, o.y, acc.y);
      acc.z = fmaf(w.x, o.z, acc.z);
      acc.w = fmaf(w.y, o.w, acc.w);
    }
    const int d = 16 * it_g + 8 * (n >> 2) + ((n >> 1) & 1) + 4 * (n & 1);
    float* row = reinterpret_cast<float*>(smem + kQsOffStage + R * kQsStageRow) + d;
    float* next = reinterpret_cast<float*>(smem + kQsOffStage + (R + 1) * kQsStageRow) + d;
    row[0] = acc.x;
    next[0] = acc.y;
    row[2] = acc.z;
    next[2] = acc.w;
  }
  __syncthreads();
  const int S = p.num_splits;
  auto out_at = [&](int R, int c) {
    const int node = R / G, h = kvh * G + (R - node * G);
    return p.out + node * p.out_tok_stride + h * p.out_head_stride + c * 8;
  };
  if (p.merge > 1) {
    cluster_sync_all();
    const uint32_t base = smem_u32(smem);
    for (int it = tid * S + split; it < rows * 32; it += kQsThreads * S) {
      const int R = it >> 5, c = it & 31;
      float2 ml[kMaxMerge];
      float4 o[kMaxMerge];
#pragma unroll
      for (int u = 0; u < kMaxMerge; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u < S) {
          ml[u] = ld_cluster_f32x2(cluster_map(base + kQsOffStageMl + R * 8, u));
          o[u] = ld_cluster_f32x4(cluster_map(base + kQsOffStage + R * kQsStageRow + c * 16, u));
        }
      }
      float w[kMaxMerge];
      merge_weights(ml, w);
      store_bf16x4(out_at(R, c), merge_chunk(o, S, w));
    }
    __syncwarp();
    cluster_sync_all();
    return;
  }
  for (int it = tid; it < rows * 32; it += kQsThreads) {
    const int R = it >> 5, c = it & 31;
    float4 acc = *reinterpret_cast<const float4*>(smem + kQsOffStage + R * kQsStageRow + c * 16);
    const float2 ml = reinterpret_cast<const float2*>(smem + kQsOffStageMl)[R];
    if (S > 1) {
      const int64_t slot = (static_cast<int64_t>(split) * p.num_kv_heads + kvh) * kBM + R;
      *reinterpret_cast<float4*>(p.ws_o + slot * kHD + c * 4) = acc;
      if (c == 0) p.ws_ml[slot] = ml;
    } else {
      const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
      store_bf16x4(out_at(R, c), make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
  }
}

// ---------------------------------------------------------------------------
// More query rows: decoded tiles on tcgen05
// ---------------------------------------------------------------------------
constexpr int kQtThreads = 512;
constexpr int kQtDecodeWarps = 7, kQtMmaWarp = 15;    // warps 8-14, 15
// registers a thread; the block is launched with 128 x 512 (2 x 176 + 2 x 80 = 4 x 128).
// (Spilling on either side shows: 257 nodes over 32768 rows, three splits, 204 us, 222 with 168 / 88,
// 216 with 184 / 72.  With 4 / 5 / 6 / 7 decode warps 17 nodes take 33.8 / 33.8 / 30.5 / 28.7.)
constexpr int kQtRegsSoftmax = 176, kQtRegsOther = 80;
constexpr int kQtAhead = 4;                           // blocks between L2 prefetch and products
constexpr int kQtKeys = 128;
constexpr uint32_t kQtTile = 128 * 128 * 2, kQtHalf = kQtTile / 2;
constexpr int kQtStages = 4;                          // decoded tiles
constexpr uint32_t kQtOffQ = 0;
constexpr uint32_t kQtOffKV = 2 * kQtTile;
constexpr uint32_t kQtOffBar = kQtOffKV + kQtStages * kQtTile;
constexpr uint32_t kQtOffMl = kQtOffBar + 512;        // [chain][row] (m, l)
constexpr uint32_t kQtSmem = kQtOffMl + 2 * 128 * 8 + 1024;
constexpr uint32_t kQtTmemO = 256;                    // S0 | S1 | O0 | O1, P_t in S_t's first 64 columns

struct Q4Bars {
  uint64_t q_full[2], kv_full[kQtStages], kv_empty[kQtStages], s_full[2],
      p_part[2], p_full[2], o_full[2], fin;
  uint32_t tmem_base;
  int abort_flag;
  uint2 x43;  // (.x)
};

// Order in which the blocks are decoded and consumed: K of the
// first `ahead` blocks (1, or 2 with two chains), then V_b and K_{b + ahead} in turn.
__device__ __forceinline__ int q4_entry(int n, int nb, int ahead, bool& is_v) {
  const int a = min(ahead, nb), m = n - a, pairs = nb - a;
  is_v = m >= 2 * pairs || (m >= 0 && !(m & 1));
  if (m < 0) return n;
  return m >= 2 * pairs ? m - pairs : (m >> 1) + ((m & 1) ? a : 0);
}

// A key's row as its thread holds it.
struct Q4Packed {
  uint2 w[8];  // code words
  uint2 meta;  // group words
};

__device__ __forceinline__ void q4_load_row(const char* src, bool have, Q4Packed& x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x.w[i] = have ? *reinterpret_cast<const uint2*>(src + i * 8) : make_uint2(0, 0);
  x.meta = have ? *reinterpret_cast<const uint2*>(src + kQ4Codes) : make_uint2(0, 0);  // (scale 0: reads as zero)
}

// Its 128 bf16 values into row r of a decoded tile (two SW128 halves).
__device__ __forceinline__ void q4_decode_row(const Q4Packed& x, uint32_t tile, int r, uint32_t x43) {
  const uint32_t meta[4] = {x.meta.x & 0xFFFFu, x.meta.x >> 16, x.meta.y & 0xFFFFu, x.meta.y >> 16};
  const uint32_t dst = tile + r * 128;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const Q4Group q = q4_group(meta[g]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ch = g * 4 + i * 2;
      const uint32_t half = dst + (ch >> 3) * kQtHalf;
      sts128(half + (((ch & 7) ^ (r & 7)) << 4), q4_decode8(x.w[g * 2 + i].x, q, x43));
      sts128(half + ((((ch + 1) & 7) ^ (r & 7)) << 4), q4_decode8(x.w[g * 2 + i].y, q, x43));
    }
  }
}

__global__ void __launch_bounds__(kQtThreads, 1)
    tree_attn_q4_tile_kernel(const __grid_constant__ CUtensorMap tmap_q, const AttnParams p, const int tok, const int pairs,
                             const int heavy) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Q4Bars& bar = *reinterpret_cast<Q4Bars*>(smem + kQtOffBar);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // CTAs of two tiles (`pairs` a kv head and split), then those of a last single one
  const int two = pairs * heavy * p.num_kv_heads, G = p.group;
  const bool dual = static_cast<int>(blockIdx.x) >= two;  // two chains over one tile's keys
  const int tiles = dual ? 1 : 2, mine = dual ? p.tail_splits : heavy;
  const int rank = blockIdx.x - (dual ? two : 0), split = rank % mine;
  const int kvh = rank / mine % p.num_kv_heads;
  const int node0 = (dual ? pairs : rank / (mine * p.num_kv_heads)) * 2 * tok;  // first node of tile 0
  const int ahead = dual ? 2 : 1;
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tmap_q);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.q_full[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_part[i], 4);
      mbar_init(&bar.p_full[i], 4);
      mbar_init(&bar.o_full[i], 1);
    }
    for (int i = 0; i < kQtStages; ++i) {
      mbar_init(&bar.kv_full[i], 4);
      mbar_init(&bar.kv_empty[i], 1);
    }
    mbar_init(&bar.fin, 1);
    bar.abort_flag = 0;
    bar.x43 = make_uint2(0x43434343u, 0);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == kQtMmaWarp) {
    tmem_alloc(&bar.tmem_base, 512);
    tmem_relinquish();
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = bar.tmem_base;
  volatile int* abort_flag = &bar.abort_flag;
  const int64_t L = prefix_rows(p);
  const bool inside = prefix_fits(p, L);                // the same in every thread of the launch
  const int64_t total = inside ? L + p.n : 0;
  if (!inside && tid == 0) set_status(p.status, RT_DEV_BAD_INDEX);
  __syncwarp();  // (whole warps for setmaxnreg)
  int64_t b0 = 0, b1 = 0;
  if (inside) split_range(total, split, mine, kQtKeys, b0, b1);
  const int nb = static_cast<int>(b1 - b0);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kQtRegsOther));
    if (warp == kQtMmaWarp) {
      // ---------------- MMA issuer (and Q by TMA) ----------------
      if (lane == 0 && nb > 0) {
        const uint32_t qbytes = static_cast<uint32_t>(tok * G) * 256u;
        for (int t = 0; t < tiles; ++t) {
          unsigned char* dst = smem + kQtOffQ + t * kQtTile;
          mbar_arrive_expect_tx(&bar.q_full[t], qbytes);
          tma_load_3d(dst, &tmap_q, &bar.q_full[t], 0, kvh * G, node0 + t * tok);
          tma_load_3d(dst + kQtHalf, &tmap_q, &bar.q_full[t], 64, kvh * G, node0 + t * tok);
        }
      }
      __syncwarp();
      constexpr uint32_t idesc_qk = idesc_bf16_f32(kBM, kQtKeys, false, false);
      constexpr uint32_t idesc_pv = idesc_bf16_f32(kBM, kHD, false, true);
      const bool me = elect_one();
      const uint32_t tm = warp_uniform(tmem);
      // (descriptors: the low words; Q and K differ from V in the high one)
      const uint64_t desc_q = smem_desc_sw128(smem_u32(smem + kQtOffQ), 16, 1024);
      const uint64_t desc_v = smem_desc_sw128(smem_u32(smem + kQtOffKV), kQtHalf, 1024);
      const uint32_t dq = warp_uniform(static_cast<uint32_t>(desc_q)), dk = dq + ((kQtOffKV - kQtOffQ) >> 4);
      const uint32_t dv = warp_uniform(static_cast<uint32_t>(desc_v));
      const uint32_t hi_qk = warp_uniform(static_cast<uint32_t>(desc_q >> 32));
      const uint32_t hi_v = warp_uniform(static_cast<uint32_t>(desc_v >> 32));
      auto wait = [&](uint64_t* b, uint32_t ph) { mbar_wait_fast(b, ph & 1, abort_flag, p.status); };
      auto qk = [&](int t, int qt, int stage) {
        const uint32_t a = dq + qt * (kQtTile >> 4), b = dk + stage * (kQtTile >> 4);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kHD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kQtHalf + (kk & 3) * 32) >> 4;
          umma_f16_if(me, tm + t * 128, a + off, b + off, hi_qk, idesc_qk, kk > 0);
        }
        umma_commit_if(me, &bar.s_full[t]);
      };
      auto pv = [&](int t, int stage, int j, bool last) {
        const uint32_t b = dv + stage * (kQtTile >> 4);
        auto mma = [&](int kk) {
          umma_f16_ts_if(me, tm + kQtTmemO + t * kHD, tm + t * 128 + kk * 8, b + kk * (2048 >> 4), hi_v, idesc_pv,
                         j > 0 || kk > 0);
        };
        wait(&bar.p_part[t], j);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kPart1 / 16; ++kk) mma(kk);
        wait(&bar.p_full[t], j);
        tc_fence_after();
#pragma unroll
        for (int kk = kPart1 / 16; kk < kQtKeys / 16; ++kk) mma(kk);
        umma_commit_if(me && last, &bar.o_full[t]);
      };
      auto release = [&](int stage) { umma_commit_if(me, &bar.kv_empty[stage]); };
      // The blocks some way ahead into L2: the decode warps' registers hold too little
      // to cover the memory's latency (a cache that is not in L2, 32768 rows: 17 nodes
      // 33.8 -> 31.5 us, 257 nodes 167 -> 158; 3, 6 and 8 blocks ahead alike; asked
      // for by the decode warps themselves 34.1 and 174).
      const char* kb = p.k + kvh * p.kv_head_stride + b0 * kQtKeys * kQ4Row;
      const char* vb = p.v + kvh * p.kv_head_stride + b0 * kQtKeys * kQ4Row;
      const int whole = static_cast<int>(min(static_cast<int64_t>(nb), total / kQtKeys - b0));  // blocks of 128 rows
      auto prefetch = [&](int b) {
        if (me && b < whole) {
          prefetch_l2(kb + static_cast<int64_t>(b) * kQtKeys * kQ4Row, kQtKeys * kQ4Row);
          prefetch_l2(vb + static_cast<int64_t>(b) * kQtKeys * kQ4Row, kQtKeys * kQ4Row);
        }
      };
      for (int b = 0; b < kQtAhead; ++b) prefetch(b);
      if (dual && nb > 0) {
        wait(&bar.q_full[0], 0);
        int n = 0;
        for (; n < min(2, nb); ++n) {
          wait(&bar.kv_full[n], 0);
          qk(n, 0, n);
          release(n);
        }
        for (int b = 0; b < nb; ++b) {
          const int t = warp_uniform2(b & 1), sv = warp_uniform2(n % kQtStages), sk = (sv + 1) % kQtStages;
          const bool more = b + 2 < nb;
          prefetch(b + kQtAhead);
          wait(&bar.kv_full[sv], n / kQtStages);
          if (more) wait(&bar.kv_full[sk], (n + 1) / kQtStages);
          pv(t, sv, b >> 1, !more);
          release(sv);
          if (more) qk(t, 0, sk);
          if (more) release(sk);
          n += more ? 2 : 1;
        }
      }
      for (int j = -1; j < nb && nb > 0 && !dual; ++j) {
        // entries 2j+1 = V_j and 2j+2 = K_{j+1}
        const int nv = 2 * j + 1, nk = 2 * j + 2;
        const int sk = warp_uniform2(nk % kQtStages), sv = (sk + kQtStages - 1) % kQtStages;
        const bool more = j + 1 < nb;
        prefetch(j + kQtAhead);
        if (j >= 0) wait(&bar.kv_full[sv], nv / kQtStages);
        if (more) wait(&bar.kv_full[sk], nk / kQtStages);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j >= 0) pv(t, sv, j, !more);
          else wait(&bar.q_full[t], 0);
          if (more) qk(t, t, sk);
        }
        if (j >= 0) release(sv);
        if (more) release(sk);
      }
      // all issued MMAs complete before TMEM is released
      umma_commit_if(me, &bar.fin);
      if (me) mbar_wait_drain(&bar.fin, 0);
      __syncwarp();
      if (nb > 0)
        for (int t = 0; t < tiles; ++t) mbar_wait_drain(&bar.q_full[t], 0);  // (long done, but for an abort)
    } else if (warp < 8 + kQtDecodeWarps) {
      // ---------------- decode ----------------
      // A task is 32 keys of K or V of a block, a lane a key; the warps take turns.
      // The next task's rows are on their way from global memory meanwhile.
      const uint32_t sbase = smem_u32(smem), x43 = lds64(smem_u32(&bar.x43)).x;
      const char* kb = p.k + kvh * p.kv_head_stride;
      const char* vb = p.v + kvh * p.kv_head_stride;
      const int tasks = 8 * nb;
      Q4Packed next;
      auto load = [&](int task) {
        bool is_v;
        const int64_t key = (b0 + q4_entry(task >> 2, nb, ahead, is_v)) * kQtKeys + (task & 3) * 32 + lane;
        // (behind the tree: zeros)
        q4_load_row((is_v ? vb : kb) + key * kQ4Row, task < tasks && key < total, next);
        // A tree row of V that reads as NaN: zero in V, and NaN in K, so that only
        // the nodes that see the key get it.
        if (task < tasks && key >= L && key < total &&
            q4_is_nan(*reinterpret_cast<const uint16_t*>(vb + key * kQ4Row + kQ4Codes)))
          next.meta = is_v ? make_uint2(0, 0) : make_uint2(0x7FF07FF0u, 0x7FF07FF0u);
      };
      load(warp - 8);
      for (int task = warp - 8; task < tasks; task += kQtDecodeWarps) {
        const Q4Packed x = next;
        load(task + kQtDecodeWarps);
        const int n = task >> 2, so = n % kQtStages;
        mbar_wait_fast(&bar.kv_empty[so], ((n / kQtStages) & 1) ^ 1, abort_flag, p.status);
        q4_decode_row(x, sbase + kQtOffKV + so * kQtTile, (task & 3) * 32 + lane, x43);
        fence_proxy_async_smem();
        mbar_arrive_warp(&bar.kv_full[so]);
      }
    }
  } else {
    // ---------------- softmax and result of tile (or chain) t ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kQtRegsSoftmax));
    const int t = warp >> 2, r = tid & 127;
    const int rt = r / G;
    const int first = node0 + (dual ? 0 : t * tok);     // first node of the tile
    const int node = first + rt;
    const bool valid = rt < tok && node < p.n;
    const int h = kvh * G + (r - rt * G);
    const int64_t R = static_cast<int64_t>(node) * G + (r - rt * G);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + t * 128, tmo = tmem + lane_base + kQtTmemO, to = tmo + t * kHD;
    const uint32_t* mrow = p.mask + static_cast<int64_t>(valid ? node : 0) * p.mask_words;
    // a warp without a query only keeps the barriers' count
    const bool warp_live = ((warp & 3) * 32) / G < tok && first + ((warp & 3) * 32) / G < p.n;
    const float sl2 = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    const int step = dual ? 2 : 1;
    int j = 0;
    for (int b = dual ? t : 0; b < nb; b += step, ++j) {
      mbar_wait_fast(&bar.s_full[t], j & 1, abort_flag, p.status);
      if (warp_live) {
        tc_fence_after();
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, sr[c]);
        tmem_wait_ld();
        const int64_t key0 = (b0 + b) * kQtKeys;
        if (key0 + kQtKeys > L) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t vm = valid ? visible_word(key0 + c * 32, L, p.n, mrow, p.mask_words) : 0u;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((vm >> i) & 1u)) sr[c][i] = __float_as_uint(-INFINITY);
          }
        }
        softmax_block<__nv_bfloat16>(sr, ts, to, j > 0, sl2, m, l, [&] { mbar_arrive_warp(&bar.p_part[t]); });
      } else {
        mbar_arrive_warp(&bar.p_part[t]);
      }
      mbar_arrive_warp(&bar.p_full[t]);
    }
    if (l != l) m = INFINITY;  // a NaN weight wins the merges
    float w0 = 1.f, w1 = 0.f;  // of the two O tiles; with one chain t's own is the first
    if (j > 0) mbar_wait_fast(&bar.o_full[t], 0, abort_flag, p.status);
    if (dual) {
      float2* ml = reinterpret_cast<float2*>(smem + kQtOffMl);
      ml[t * 128 + r] = make_float2(m, l);
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // both chains' products are done, too
      const float2 x0 = ml[r], x1 = ml[128 + r];
      m = fmaxf(x0.x, x1.x);
      w0 = x0.x == -INFINITY ? 0.f : ex2(x0.x - m);
      w1 = x1.x == -INFINITY ? 0.f : ex2(x1.x - m);
      l = fmaf(w0, x0.y, w1 * x1.y);
    }
    const int64_t rows_ws = static_cast<int64_t>(p.tiles) * kBM;
    const int64_t slot = (static_cast<int64_t>(split) * p.num_kv_heads + kvh) * rows_ws + R;
    if (p.merge > 1) {
      // park the unnormalised O rows and (m, l) for the merge in the cluster: the
      // rings are idle, every load was consumed and the last products are done
      const bool have = inside && warp_live && nb > 0 && !__any_sync(0xFFFFFFFFu, *abort_flag);
      if (have) {
        tc_fence_after();
#pragma unroll 1
        for (int c = 2 * t; c < 2 * t + 2; ++c) {
          uint32_t o[32], o1[32];
          tmem_ld32(tmo + c * 32, o);
          tmem_ld32(tmo + kHD + c * 32, o1);
          tmem_wait_ld();
          float x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            x[i] = w0 == 0.f ? 0.f : __uint_as_float(o[i]) * w0;
            if (w1 != 0.f) x[i] = fmaf(w1, __uint_as_float(o1[i]), x[i]);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(smem + stage_off(r, c * 8 + q)) =
                make_float4(x[q * 4], x[q * 4 + 1], x[q * 4 + 2], x[q * 4 + 3]);
        }
      }
      if (t == 0)
        reinterpret_cast<float2*>(smem + kOffMl)[r] = have ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
      // (one tile, so the launch's rows are the tile's)
      if (inside) merge_splits<256, false>(p, smem, split, kvh, 0, p.n * G);
    } else if (inside && nb == 0) {
      if (valid && p.num_splits > 1 && (t == 0 || !dual)) p.ws_ml[slot] = make_float2(-INFINITY, 0.f);
    } else if (inside && warp_live && !__any_sync(0xFFFFFFFFu, *abort_flag)) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const uint32_t stage = smem_u32(smem) + kQtOffQ + (dual ? warp : t * 8 + (warp & 3)) * 4096;  // (Q is done with)
      char* row = p.num_splits > 1 ? reinterpret_cast<char*>(p.ws_o + slot * kHD)
                                   : p.out + node * p.out_tok_stride + h * p.out_head_stride;
      const RowsOut rows(stage, valid ? reinterpret_cast<uint64_t>(row) : 0);
      // one chain: all four column groups of the tile's O; two: half of them, of both O
#pragma unroll 1
      for (int c = dual ? 2 * t : 0; c < (dual ? 2 * t + 2 : 4); ++c) {
        float x[32];
        uint32_t o[32];
        tmem_ld32((dual ? tmo : to) + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = w0 == 0.f ? 0.f : __uint_as_float(o[i]) * w0;
        if (dual) {
          tmem_ld32(tmo + kHD + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = w1 == 0.f ? x[i] : fmaf(w1, __uint_as_float(o[i]), x[i]);
        }
        if (p.num_splits == 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = l == 0.f ? 0.f : x[i] * inv;
          rows.put32<__nv_bfloat16>(x, c);
        } else {
          rows.put32<float>(x, c);
        }
      }
      if (valid && p.num_splits > 1 && (t == 0 || !dual)) p.ws_ml[slot] = make_float2(m, l);
    }
    tc_fence_before();
  }
  if (p.merge > 1 && inside && warp >= 8) {  // the merge's two cluster barriers
    __syncwarp();
    cluster_sync_all();
    cluster_sync_all();
  }
  __syncthreads();
  if (warp == kQtMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Q viewed as [n nodes][Hq heads][128]: one box is `tok` nodes x G heads x 64 values.
static int make_q4_query_tmap(CUtensorMap* m, const void* q, int64_t tok_stride, int64_t head_stride, int n, int hq,
                              int G, int tok) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return RT_ERR_CUDA;
  const cuuint64_t dims[3] = {kHD, static_cast<cuuint64_t>(hq), static_cast<cuuint64_t>(n)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride), static_cast<cuuint64_t>(tok_stride)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(tok)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? RT_OK : RT_ERR_INVALID_ARGUMENT;
}

struct Q4Plan {
  bool small;  // the mma.sync path
  int splits;  // of the keys, the most any tile has
  bool merge;
  int heavy, tail;  // of the tiles of two-tile CTAs, of a last single one
};

// Clusters of `c` CTAs of `kernel` that fit on the GPU at once (-1 when the query
// fails, e.g. without a device).
template <typename Kernel>
static int clusters_fit(Kernel kernel, int threads, uint32_t smem, int c) {
  int n = -1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) ==
          cudaSuccess &&
      (c <= 8 || cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess)) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c, 1, 1);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(c);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = -1;
  }
  cudaGetLastError();
  return n;
}

// ... of the few-rows kernel, or of the tile kernel: an answer is kept per device and
// size, a failed query counts as none and is asked again.
static int q4_clusters_fit(bool small, int c) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static int cache[kDevices][2][kMaxMerge + 1] = {};  // answer + 1, 0: not asked yet
  if (c < 2 || c > kMaxMerge) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) {
    cudaGetLastError();
    return 0;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (cache[dev][small][c] > 0) return cache[dev][small][c] - 1;
  const int n = small ? clusters_fit(tree_attn_q4_small_kernel<2>, kQsThreads, kQsSmem, c)
                      : clusters_fit(tree_attn_q4_tile_kernel, kQtThreads, kQtSmem, c);
  if (n < 0) return 0;
  cache[dev][small][c] = n + 1;
  return n;
}

template <int NT>
static int launch_q4_small(dim3 grid, dim3 cluster, cudaStream_t s, const AttnParams& p) {
  set_smem_limit(tree_attn_q4_small_kernel<NT>, kQsSmem);
  if (cluster.x > 8) cudaFuncSetAttribute(tree_attn_q4_small_kernel<NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return record_cuda(
      launch_ex_cluster(tree_attn_q4_small_kernel<NT>, grid, dim3(kQsThreads), kQsSmem, s, cluster, p));
}

// A launch of two-tile CTAs ("heavy") may end in a single-tile one a kv head
// ("light", started last): a root and a power of two of others leave just that.
// A block costs them 2.3 and 1.24 us (measured at 32768 rows), a CTA 6 us besides.
struct Q4Load {
  int heavy, light;  // CTAs for each split
};
constexpr double kQtHeavyBlock = 2.3, kQtLightBlock = 1.24, kQtCta = 6;

// Time on 148 SMs of heavy CTAs of `h` and light ones of `l`, which take the SMs as they come free.
static double q4_time(int heavy, double h, int light, double l) {
  const int rounds = (heavy + 147) / 148, idle = rounds * 148 - heavy;
  double t_idle = (rounds - 1) * h, t_busy = rounds * h;
  while (light > 0) {
    const bool on_idle = idle > 0 && t_idle <= t_busy;
    light -= on_idle ? idle : 148 - idle;
    (on_idle ? t_idle : t_busy) += l;
  }
  return std::max(t_idle, t_busy);
}

// Splits of the light CTAs beside heavy ones of `s` splits: the fewest that come within 2 % of
// the shortest time over many blocks (no use of the prefix length: launches that are given
// one count split alike).  257 nodes over 32768 rows: 172 us with 4 splits of both, 161 with
// 4 of the heavy and 5 of the light ones.
static int tail_splits(const Q4Load& w, int s) {
  if (w.light == 0 || w.heavy == 0 || s == 1) return s;
  double t[33], best = 1e30;
  for (int i = 1; i <= 32; ++i) {
    t[i] = q4_time(w.heavy * s, kQtHeavyBlock / s, w.light * i, kQtLightBlock / i);
    best = std::min(best, t[i]);
  }
  int tail = 1;
  while (t[tail] > 1.02 * best) ++tail;
  return tail;
}

// The split count with the shortest estimated time.  257 nodes over 32768 rows: 4 (161 us);
// 205 with 3, 179 with 8 (of both kinds).
static int tile_splits(const Q4Load& w, int64_t blocks) {
  int best_s = 1;
  double best = 1e30;
  auto cost = [&](double block, int s) { return block * static_cast<double>((blocks + s - 1) / s) + kQtCta; };
  for (int s = 1; s <= 32 && s <= blocks; ++s) {
    const double h = cost(kQtHeavyBlock, s);
    if ((w.heavy * s + 147) / 148 * h >= best) continue;
    const int tail = tail_splits(w, s);
    const double t = q4_time(w.heavy * s, h, w.light * tail, cost(kQtLightBlock, tail));
    if (t < best) best = t, best_s = s;
  }
  return best_s;
}

static Q4Plan q4_plan(int n, int G, int hkv, int64_t prefix_len, int num_splits) {
  const bool small = n * G <= kQsRows;
  if (small) {
    const int64_t tiles = (prefix_len + n + kQsKeys - 1) / kQsKeys;
    int64_t want = num_splits;
    if (want <= 0) want = std::max<int64_t>(1, std::min<int64_t>(148 / hkv, (tiles + 7) / 8));
    want = std::min<int64_t>(want, 256);
    const int s = static_cast<int>(want);
    return {true, s, s >= 2 && s <= kMaxMerge && hkv <= q4_clusters_fit(true, s), s, s};
  }
  const int64_t blocks = (prefix_len + n + kQtKeys - 1) / kQtKeys;
  const int tok = kBM / G;
  int64_t want = num_splits;
  if (n > tok) {
    const int rest = n % (2 * tok);
    const Q4Load w = {hkv * (n / (2 * tok) + (rest > tok)), hkv * (rest > 0 && rest <= tok)};
    const int heavy = want > 0 ? static_cast<int>(std::min<int64_t>(want, 256)) : tile_splits(w, blocks);
    const int tail = tail_splits(w, heavy);
    return {false, std::max(heavy, tail), false, heavy, tail};
  }
  if (want <= 0) want = std::min<int64_t>(std::max<int64_t>(1, 148 / hkv), blocks);
  want = std::min<int64_t>(want, 256);
  if (want > 1) {
    // one tile: its splits merge in a cluster when it takes all of them, or (where
    // the count is ours to choose) leaves each CTA three blocks at most
    int c = static_cast<int>(std::min<int64_t>(want, kMaxMerge));
    if (num_splits <= 0)
      while (c >= 2 && hkv > q4_clusters_fit(false, c)) --c;
    if (c >= 2 && hkv <= q4_clusters_fit(false, c) && (c == want || (num_splits <= 0 && blocks <= 3 * c)))
      return {false, c, true, c, c};
  }
  const int s = static_cast<int>(want);
  return {false, s, false, s, s};
}

}  // namespace rt

using namespace rt;

extern "C" int rt_tree_attn_q4_default_splits(int n, int num_q_heads, int num_kv_heads, int64_t prefix_len) {
  if (n <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || prefix_len < 0) return 1;
  return q4_plan(n, num_q_heads / num_kv_heads, num_kv_heads, prefix_len, 0).heavy;
}

extern "C" size_t rt_tree_attn_q4_workspace_size(int n, int num_q_heads, int num_kv_heads, int head_dim,
                                                 int64_t prefix_len, int num_splits) {
  if (n <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || head_dim != kHD ||
      prefix_len < 0)
    return 0;
  const Q4Plan pl = q4_plan(n, num_q_heads / num_kv_heads, num_kv_heads, prefix_len, num_splits);
  if (pl.splits <= 1 || pl.merge) return 0;
  const size_t slots = static_cast<size_t>(pl.splits) * num_kv_heads * tiles_for(n, num_q_heads / num_kv_heads) * kBM;
  return align_up(slots * kHD * 4, 256) + align_up(slots * 8, 256);
}

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
  if (head_dim != kHD) return RT_ERR_UNSUPPORTED;
  if (mask_words < (n + 31) / 32) return RT_ERR_INVALID_ARGUMENT;
  if (kv_capacity < n || (prefix_len_dev == nullptr && prefix_len > kv_capacity - n)) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t align_bits = reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(k) |
                              reinterpret_cast<uint64_t>(v) | reinterpret_cast<uint64_t>(out) |
                              static_cast<uint64_t>(q_tok_stride) | static_cast<uint64_t>(q_head_stride) |
                              static_cast<uint64_t>(kv_head_stride) | static_cast<uint64_t>(out_tok_stride) |
                              static_cast<uint64_t>(out_head_stride);
  if ((align_bits & 15) || (kv_capacity & 1)) return RT_ERR_INVALID_ARGUMENT;
  const int G = num_q_heads / num_kv_heads;
  if (n * G > kQsRows && G > kBM) return RT_ERR_UNSUPPORTED;
  const Q4Plan pl = q4_plan(n, G, num_kv_heads, prefix_len, num_splits);
  AttnParams p{};
  p.q = static_cast<const char*>(q);
  p.q_tok_stride = q_tok_stride;
  p.q_head_stride = q_head_stride;
  p.out = static_cast<char*>(out);
  p.out_tok_stride = out_tok_stride;
  p.out_head_stride = out_head_stride;
  p.mask = mask;
  p.mask_words = mask_words;
  p.n = n;
  p.prefix_len = prefix_len;
  p.prefix_len_dev = prefix_len_dev;
  p.group = G;
  p.num_kv_heads = num_kv_heads;
  p.tiles = tiles_for(n, G);
  p.num_splits = pl.splits;
  p.row_splits = pl.heavy;
  p.merge = pl.merge ? pl.splits : 1;
  // (never 0: a hidden score is -inf and stays so; scores times 2^-126 are 0 in the sum)
  p.scale_log2 = std::max(scale * 1.4426950408889634f, 1.17549435e-38f);
  p.status = status;
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.kv_head_stride = kv_head_stride;
  p.capacity = kv_capacity;
  if (pl.splits > 1 && !pl.merge) {
    const size_t need = rt_tree_attn_q4_workspace_size(n, num_q_heads, num_kv_heads, head_dim, prefix_len, num_splits);
    if (workspace == nullptr || workspace_bytes < need) return RT_ERR_WORKSPACE;
    const size_t slots = static_cast<size_t>(pl.splits) * num_kv_heads * p.tiles * kBM;
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + align_up(slots * kHD * 4, 256));
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int rc;
  if (pl.small) {
    const dim3 grid(pl.splits, num_kv_heads), cluster(pl.merge ? pl.splits : 1, 1, 1);
    rc = n * G <= 8 ? launch_q4_small<1>(grid, cluster, s, p) : launch_q4_small<2>(grid, cluster, s, p);
  } else {
    if (q_tok_stride <= 0 || q_head_stride <= 0) return RT_ERR_UNSUPPORTED;
    const int tok = kBM / G;
    CUtensorMap tq;
    rc = make_q4_query_tmap(&tq, q, q_tok_stride, q_head_stride, n, num_q_heads, G, tok);
    if (rc != RT_OK) return rc;
    const int pairs = n / (2 * tok) + (n % (2 * tok) > tok);
    const bool last = n > pairs * 2 * tok;
    p.tail_splits = last ? pl.tail : 0;
    p.tail_row = pairs * 2 * tok * G;
    const dim3 grid(num_kv_heads * (pairs * pl.heavy + p.tail_splits));
    set_smem_limit(tree_attn_q4_tile_kernel, kQtSmem);
    if (pl.merge && pl.splits > 8)
      cudaFuncSetAttribute(tree_attn_q4_tile_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    rc = record_cuda(launch_ex_cluster(tree_attn_q4_tile_kernel, grid, dim3(kQtThreads), kQtSmem, s,
                                       dim3(pl.merge ? pl.splits : 1, 1, 1), tq, p, tok, pairs, pl.heavy));
  }
  if (rc != RT_OK || pl.merge || pl.splits == 1) return rc;
  const int warps = num_kv_heads * n * G * (pl.splits <= kFastSplits ? 2 : 1);
  return record_cuda(launch_ex(attn_combine_kernel, dim3((warps + 3) / 4), dim3(128), 0, s, 1, p));
}
