// Causal attention over whole prompts for B200 (sm_100a): packed sequences, GQA,
// head_dim 128, bf16 or fp16 in and out.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(scale*log2(e) q_i.k_j - m_i),
//   j <= i + lk - lq within the sequence, m_i a running maximum.
//
// A work item is 256 query rows of one kv head -- two 128-row tiles, row r of a
// tile being (token r / G, query head r % G) of G = Hq / Hkv, so the heads of a
// group share every K/V tile -- and all the 128-key blocks they see.  CTAs are
// persistent (one per SM) and take items longest first.  Twelve warps:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one thread per row: S from TMEM, the
//                   online softmax in the exp2 domain with a lazy (> 8 in log2)
//                   rescale of O in TMEM, P back into S's own columns, and the
//                   tile's output rows;
//   warp 8          TMA producer: Q tiles, and K / V blocks into a 4-stage ring;
//   warp 9          MMA issuer: per block PV of tile 0, next QK of
//                   tile 0, PV of tile 1, next QK of tile 1 -- while one tile's
//                   softmax runs the tensor core has the other tile's products;
//   warp 10         checks the V blocks that some row must not see in full
//                   (the causal diagonal, the sequence's end) for values that
//                   are not finite: 0 * NaN would reach rows that hide the key.
//                   It zeroes them; rows that do see the key add the value back
//                   at the end.
// Every mbarrier wait is bounded (common.cuh): on time-out the CTA records
// RT_DEV_WAIT_TIMEOUT, drains what it issued, frees TMEM and exits.
#include <cuda.h>
#include <cuda_fp16.h>

#include "attn_softmax.cuh"
#include "common.cuh"
#include "host_util.h"
#include "tmap.h"

namespace rt {

constexpr int kPD = 128;                       // head_dim
constexpr int kPB = 128;                       // keys per block, rows per tile
constexpr int kPThreads = 384;
// Registers a thread: the block is launched with 168 x 384; the two softmax
// warpgroups hold a 128-key row of S each and take what the third gives up
// (2 x 208 + 88 = 3 x 168).
constexpr int kPRegsSoftmax = 208, kPRegsOther = 88;
constexpr uint32_t kPTile = 128 * 128 * 2;
constexpr uint32_t kPHalf = kPTile / 2;        // 128 rows x 64 columns, one SW128 box
constexpr int kPStages = 4;
constexpr uint32_t kPOffQ = 0;
constexpr uint32_t kPOffKV = 2 * kPTile;
constexpr uint32_t kPOffTab = kPOffKV + kPStages * kPTile;  // prefix sums of the sequences' pair counts
constexpr int kPMaxSeqs = 4096;
constexpr uint32_t kPOffBar = kPOffTab + (kPMaxSeqs + 1) * 4 + 12;
constexpr uint32_t kPSmem = kPOffBar + 512 + 1024;
constexpr uint32_t kPTmemO = 256;              // S0 | S1 | O0 | O1, P_t in S_t's first 64 columns
constexpr int kPSms = 148;

struct PromptParams {
  char* out;
  int64_t out_tok_stride, out_head_stride;
  const char* v;
  int64_t kv_head_stride, kv_row_stride;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int num_seqs, total_q, total_k, hkv, group, tok;  // tok: tokens per 128-row tile
  int tiles;                                        // tiles per item: 2, or 1 when the call is small
  float scale_log2;
  int* status;
};

struct PromptBars {
  uint64_t q_full[2], q_empty[2], kv_full[kPStages], kv_empty[kPStages], s_full[2], p_part[2], p_full[2], o_full[2],
      v_look, v_ok, fin;
  uint32_t tmem_base;
  int abort_flag;
  int poison;  // set once a checked V block held a value that is not finite
};

struct PromptItem {
  int q0, lq, k0, lk, tok0, g;
  int nb[2];  // key blocks of each tile
  int jm;     // first block that some row of the item hides in part
};

__device__ __forceinline__ bool prompt_seq(const PromptParams& p, int b, int& q0, int& lq, int& k0, int& lk) {
  int q1 = p.total_q, k1 = p.total_k;
  q0 = k0 = 0;
  if (p.cu_q != nullptr) {
    q0 = p.cu_q[b];
    q1 = p.cu_q[b + 1];
    k0 = p.cu_k[b];
    k1 = p.cu_k[b + 1];
  }
  lq = q1 - q0;
  lk = k1 - k0;
  return q0 >= 0 && q1 >= q0 && q1 <= p.total_q && k0 >= 0 && k1 >= k0 && k1 <= p.total_k;
}

// Item `it` of this CTA: round r runs through the list forwards or backwards
// (the list is sorted by length within a sequence, so a CTA's items average out).
__device__ __forceinline__ bool prompt_item(const PromptParams& p, const int* tab, int it, PromptItem& w) {
  const int grid = gridDim.x;
  const int64_t idx = static_cast<int64_t>(it) * grid + ((it & 1) ? grid - 1 - blockIdx.x : blockIdx.x);
  const int64_t pos64 = idx / p.hkv;
  const int total = tab[p.num_seqs];
  if (static_cast<int64_t>(it) * grid >= static_cast<int64_t>(total) * p.hkv) return false;
  w.nb[0] = w.nb[1] = 0;
  w.jm = 0;
  w.lq = w.tok0 = 0;
  if (pos64 >= total) return true;  // an empty place of the last round
  const int pos = static_cast<int>(pos64);
  w.g = static_cast<int>(idx - pos64 * p.hkv);
  int lo = 0, hi = p.num_seqs;  // tab[lo] <= pos < tab[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab[mid] <= pos) lo = mid; else hi = mid;
  }
  prompt_seq(p, lo, w.q0, w.lq, w.k0, w.lk);
  const int tile = tab[lo + 1] - 1 - pos;  // the longest (last) tiles first
  w.tok0 = tile * p.tiles * p.tok;
  const int shift = w.lk - w.lq;
  for (int t = 0; t < p.tiles; ++t) {
    const int first = w.tok0 + t * p.tok;
    const int lim = min(first + p.tok, w.lq) + shift;  // keys the tile's last token sees
    w.nb[t] = (first < w.lq && lim > 0) ? (lim + kPB - 1) / kPB : 0;
  }
  w.jm = max(w.tok0 + 1 + shift, 0) / kPB;
  return true;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
}
// Sign bits of the halves of a 16-bit pair whose exponent is all ones.
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  constexpr uint32_t kExp = std::is_same_v<T, __half> ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t kOne = std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
  return ((w & kExp) + kOne) & 0x80008000u;
}

// The values of v rows [key0, key1) that are not finite, added to 32 columns of
// one output row (the rare path: those values were zero in the product).
template <typename T>
__device__ __forceinline__ void add_not_finite(const char* v, int64_t row_stride, int key0, int key1,
                                               float (&o)[32]) {
#pragma unroll 1
  for (int key = key0; key < key1; ++key) {
    const uint4* row = reinterpret_cast<const uint4*>(v + key * row_stride);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 x = row[c];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bad = not_finite2<T>(w[i]);
        const float2 f = unpack2<T>(w[i]);
        if (bad & 0x8000u) o[c * 8 + 2 * i] += f.x;
        if (bad & 0x80000000u) o[c * 8 + 2 * i + 1] += f.y;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kPThreads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const PromptParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PromptBars& bar = *reinterpret_cast<PromptBars*>(smem + kPOffBar);
  int* tab = reinterpret_cast<int*>(smem + kPOffTab);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bar.q_full[t], 1);
      mbar_init(&bar.q_empty[t], 1);
      mbar_init(&bar.s_full[t], 1);
      mbar_init(&bar.p_part[t], 4);
      mbar_init(&bar.p_full[t], 4);
      mbar_init(&bar.o_full[t], 1);
    }
    for (int s = 0; s < kPStages; ++s) {
      mbar_init(&bar.kv_full[s], 1);
      mbar_init(&bar.kv_empty[s], 1);
    }
    mbar_init(&bar.v_look, 1);
    mbar_init(&bar.v_ok, 1);
    mbar_init(&bar.fin, 1);
    bar.abort_flag = 0;
    bar.poison = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc(&bar.tmem_base, 512);
    tmem_relinquish();
  }
  pdl_wait();
  // prefix sums of the sequences' item counts, by warp 10
  if (warp == 10) {
    const int span = p.tiles * p.tok;
    int carry = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
      int n = 0;
      if (b0 + lane < p.num_seqs) {
        int q0, lq, k0, lk;
        if (prompt_seq(p, b0 + lane, q0, lq, k0, lk)) n = (lq + span - 1) / span;
        else set_status(p.status, RT_DEV_BAD_INDEX);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, n, o);
        if (lane >= o) n += up;
      }
      if (b0 + lane < p.num_seqs) tab[b0 + lane + 1] = carry + n;
      carry += __shfl_sync(0xFFFFFFFFu, n, 31);
    }
    if (lane == 0) tab[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = bar.tmem_base;
  volatile int* abort_flag = &bar.abort_flag;
  PromptItem w{};
  // (inside the roles' own branches: ptxas budgets the code after a merge for the smaller count)
  auto fewer_registers = [] { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsOther)); };
  if (warp == 8) {
    // ---------------- TMA producer ----------------
    fewer_registers();
    if (lane == 0) {
      int n = 0;          // ring loads issued
      int nq[2] = {0, 0};  // Q loads issued per tile
      bool ok = true;
      const uint32_t qbytes = static_cast<uint32_t>(p.tok * p.group) * 256u;
      auto load = [&](const CUtensorMap* map, int row) {
        const int s = n % kPStages;
        ok = mbar_wait(&bar.kv_empty[s], ((n / kPStages) & 1) ^ 1, abort_flag, p.status, RT_DEV_WAIT_TIMEOUT);
        if (!ok) return;
        unsigned char* dst = smem + kPOffKV + s * kPTile;
        mbar_arrive_expect_tx(&bar.kv_full[s], kPTile);
        tma_load_3d(dst, map, &bar.kv_full[s], 0, row, w.g);
        tma_load_3d(dst + kPHalf, map, &bar.kv_full[s], 64, row, w.g);
        ++n;
      };
      for (int it = 0; ok && prompt_item(p, tab, it, w); ++it) {
        const int nb = max(w.nb[0], w.nb[1]);
        for (int j = 0; j < nb && ok; ++j) {
          load(&tmap_k, w.k0 + j * kPB);
          if (j == 0) {
            for (int t = 0; t < 2 && ok; ++t) {
              if (w.nb[t] == 0) continue;
              ok = mbar_wait(&bar.q_empty[t], (nq[t] & 1) ^ 1, abort_flag, p.status, RT_DEV_WAIT_TIMEOUT);
              if (!ok) break;
              unsigned char* dst = smem + kPOffQ + t * kPTile;
              mbar_arrive_expect_tx(&bar.q_full[t], qbytes);
              tma_load_3d(dst, &tmap_q, &bar.q_full[t], 0, w.g * p.group, w.q0 + w.tok0 + t * p.tok);
              tma_load_3d(dst + kPHalf, &tmap_q, &bar.q_full[t], 64, w.g * p.group, w.q0 + w.tok0 + t * p.tok);
              ++nq[t];
            }
          }
          if (ok) load(&tmap_v, w.k0 + j * kPB);
        }
      }
      if (*abort_flag) {
        for (int i = max(0, n - kPStages); i < n; ++i)
          mbar_wait_drain(&bar.kv_full[i % kPStages], (i / kPStages) & 1);
        for (int t = 0; t < 2; ++t)
          if (nq[t] > 0) mbar_wait_drain(&bar.q_full[t], (nq[t] - 1) & 1);
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer ----------------
    fewer_registers();
    constexpr uint32_t kFmt = std::is_same_v<T, __half> ? (1u << 7 | 1u << 10) : 0u;  // clears the bf16 format bits
    constexpr uint32_t idesc_qk = idesc_bf16_f32(kPB, kPB, false, false) & ~kFmt;
    constexpr uint32_t idesc_pv = idesc_bf16_f32(kPB, kPD, false, true) & ~kFmt;
    const uint32_t tm = warp_uniform(tmem);
    const uint64_t dq = warp_uniform(smem_desc_sw128(smem_u32(smem + kPOffQ), 16, 1024));
    const uint64_t dk = warp_uniform(smem_desc_sw128(smem_u32(smem + kPOffKV), 16, 1024));
    const uint64_t dv = warp_uniform(smem_desc_sw128(smem_u32(smem + kPOffKV), kPHalf, 1024));
    int n = 0;  // ring loads consumed
    int nq[2] = {0, 0}, np[2] = {0, 0};
    uint32_t looks = 0;  // V blocks handed to warp 10
    auto wait = [&](uint64_t* b, uint32_t ph) { mbar_wait_fast(b, ph & 1, abort_flag, p.status); };
    // S_t = Q_t K^T of the block in `stage`; the last one of an item frees Q_t
    auto qk = [&](int t, int stage, bool last) {
      const uint64_t b = dk + static_cast<uint64_t>(warp_uniform(stage) * (kPTile >> 4));
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kPD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kPHalf + (kk & 3) * 32) >> 4;
          umma_f16(tm + t * kPB, dq + t * (kPTile >> 4) + off, b + off, idesc_qk, kk > 0);
        }
        umma_commit(&bar.s_full[t]);
        if (last) umma_commit(&bar.q_empty[t]);
      }
    };
    auto commit = [&](uint64_t* b) {
      if (elect_one()) umma_commit(b);
    };
    for (int it = 0; prompt_item(p, tab, it, w); ++it) {
      if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
      const int nb = max(w.nb[0], w.nb[1]);
      if (nb == 0) continue;
      const int s = n % kPStages;
      wait(&bar.kv_full[s], n / kPStages);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (w.nb[t] == 0) continue;
        wait(&bar.q_full[t], nq[t]++);
        tc_fence_after();
        qk(t, s, w.nb[t] == 1);
      }
      commit(&bar.kv_empty[s]);
      ++n;
      for (int j = 0; j < nb; ++j) {
        const int sv = n % kPStages, sk = (n + 1) % kPStages;
        const bool more = j + 1 < nb;
        wait(&bar.kv_full[sv], n / kPStages);
        bool look = j >= w.jm;
        if (look && elect_one()) mbar_arrive(&bar.v_look);
        if (more) wait(&bar.kv_full[sk], (n + 1) / kPStages);
        const uint64_t b = dv + static_cast<uint64_t>(warp_uniform(sv) * (kPTile >> 4));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j < w.nb[t]) {
            auto pv = [&](int kk) {
              umma_f16_ts(tm + kPTmemO + t * kPD, tm + t * kPB + kk * 8, b + kk * (2048 >> 4), idesc_pv,
                          (j > 0 || kk > 0) ? 1u : 0u);
            };
            if (kPart1 < kPB) {
              wait(&bar.p_part[t], np[t]);
              if (look) wait(&bar.v_ok, looks++);
              look = false;
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kPart1 / 16; ++kk) pv(kk);
              }
            }
            wait(&bar.p_full[t], np[t]++);
            if (look) wait(&bar.v_ok, looks++);
            look = false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = (kPart1 < kPB ? kPart1 / 16 : 0); kk < kPB / 16; ++kk) pv(kk);
              if (j + 1 == w.nb[t]) umma_commit(&bar.o_full[t]);
            }
          }
          if (j + 1 < w.nb[t]) qk(t, sk, j + 2 == w.nb[t]);
          if (t == 1) commit(&bar.kv_empty[sv]);
        }
        if (more) commit(&bar.kv_empty[sk]);
        n += more ? 2 : 1;
      }
    }
    // all issued MMAs complete before TMEM is released
    if (elect_one()) {
      umma_commit(&bar.fin);
      mbar_wait_drain(&bar.fin, 0);
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---------------- V blocks that are partly hidden: values that are not finite ----------------
    fewer_registers();
    // (the MMA warp hands them over in order, right after the block's QK, so
    // the check runs beside the block's softmax)
    int n = 0;
    uint32_t looks = 0;
    for (int it = 0; prompt_item(p, tab, it, w); ++it) {
      if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
      const int nb = max(w.nb[0], w.nb[1]);
      for (int j = min(w.jm, nb); j < nb; ++j) {
        const int m = n + 2 * j + 1, s = m % kPStages;
        mbar_wait_fast(&bar.v_look, looks++ & 1, abort_flag, p.status);
        mbar_wait_fast(&bar.kv_full[s], (m / kPStages) & 1, abort_flag, p.status);
        uint4* v = reinterpret_cast<uint4*>(smem + kPOffKV + s * kPTile) + lane;
        uint32_t bad = 0;
#pragma unroll 8
        for (int i = 0; i < static_cast<int>(kPTile / 512); ++i) {
          const uint4 x = v[i * 32];
          bad |= not_finite2<T>(x.x) | not_finite2<T>(x.y) | not_finite2<T>(x.z) | not_finite2<T>(x.w);
        }
        if (__any_sync(0xFFFFFFFFu, bad != 0)) {
          auto fix = [](uint32_t x) {
            const uint32_t b = not_finite2<T>(x);
            return x & ~(((b >> 15) & 0x00010001u) * 0xFFFFu);
          };
#pragma unroll 1
          for (int i = 0; i < static_cast<int>(kPTile / 512); ++i) {
            uint4 x = v[i * 32];
            x.x = fix(x.x);
            x.y = fix(x.y);
            x.z = fix(x.z);
            x.w = fix(x.w);
            v[i * 32] = x;
          }
          fence_proxy_async_smem();
          if (lane == 0) *const_cast<volatile int*>(&bar.poison) = 1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.v_ok);
      }
      n += 2 * nb;
    }
  } else if (warp < 8) {
    // ---------------- softmax and output of tile t ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsSoftmax));
    const int t = warp >> 2;
    const int r = tid & (kPB - 1);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + t * kPB, to = tmem + lane_base + kPTmemO + t * kPD;
    const int rt = r / p.group, rh = r - rt * p.group;
    const float sl2 = p.scale_log2;
    int ns = 0, no = 0;
    for (int it = 0; prompt_item(p, tab, it, w); ++it) {
      if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
      const int tok = w.tok0 + t * p.tok + rt;
      const bool valid = t < p.tiles && rt < p.tok && tok < w.lq;
      const int lim = valid ? min(max(tok + 1 + w.lk - w.lq, 0), w.lk) : 0;  // keys this row sees
      const int jmask = max(w.tok0 + t * p.tok + 1 + w.lk - w.lq, 0) / kPB;
      const int nb = t == 0 ? w.nb[0] : w.nb[1];
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nb; ++j) {
        mbar_wait_fast(&bar.s_full[t], ns++ & 1, abort_flag, p.status);
        tc_fence_after();
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, sr[c]);
        tmem_wait_ld();
        if (j >= jmask) {
          const int left = lim - j * kPB;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= left) sr[c][i] = __float_as_uint(-INFINITY);
        }
        softmax_block<T>(sr, ts, to, j > 0, sl2, m, l, [&] { mbar_arrive_warp(&bar.p_part[t]); });
        mbar_arrive_warp(&bar.p_full[t]);
      }
      char* dst = p.out + static_cast<int64_t>(w.q0 + tok) * p.out_tok_stride +
                  static_cast<int64_t>(w.g * p.group + rh) * p.out_head_stride;
      if (nb == 0) {
        if (valid)
          for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(dst + c * 16) = make_uint4(0, 0, 0, 0);
        continue;
      }
      mbar_wait_fast(&bar.o_full[t], no++ & 1, abort_flag, p.status);
      if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
      tc_fence_after();
      const float inv = lim > 0 ? 1.f / l : 0.f;
      const bool poison = *const_cast<volatile int*>(&bar.poison) != 0;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(to + c * 32, o);
        tmem_wait_ld();
        if (!valid) continue;
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = lim > 0 ? __uint_as_float(o[i]) * inv : 0.f;
        if (poison)
          add_not_finite<T>(p.v + w.g * p.kv_head_stride + w.k0 * p.kv_row_stride + c * 64, p.kv_row_stride,
                            w.jm * kPB, lim, x);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(dst + c * 64 + q * 16) =
              make_uint4(pack2<T>(x[q * 8], x[q * 8 + 1]), pack2<T>(x[q * 8 + 2], x[q * 8 + 3]),
                         pack2<T>(x[q * 8 + 4], x[q * 8 + 5]), pack2<T>(x[q * 8 + 6], x[q * 8 + 7]));
      }
      tc_fence_before();
    }
  } else {
    fewer_registers();
  }
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// [rows of 128][mid][outer] of 16-bit values read in boxes of 64 columns x
// box_mid x box_outer with the 128-byte swizzle; out-of-range rows read as zero.
static int make_prompt_tmap(CUtensorMap* m, const void* base, bool half, int64_t mid, int64_t mid_stride,
                            int64_t outer, int64_t outer_stride, int box_mid, int box_outer) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return RT_ERR_CUDA;
  const cuuint64_t dims[3] = {kPD, static_cast<cuuint64_t>(mid), static_cast<cuuint64_t>(outer)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(mid_stride), static_cast<cuuint64_t>(outer_stride)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_mid), static_cast<cuuint32_t>(box_outer)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? RT_OK : RT_ERR_INVALID_ARGUMENT;
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
  if (head_dim != kPD || (dtype != 1 && dtype != 2)) return RT_ERR_UNSUPPORTED;
  const int G = num_q_heads / num_kv_heads;
  if (G > kPB || total_q > INT32_MAX || total_k > INT32_MAX) return RT_ERR_UNSUPPORTED;
  if (total_q == 0 || num_seqs == 0) return RT_OK;
  if (!q || !out || (total_k > 0 && (!k || !v))) return RT_ERR_INVALID_ARGUMENT;
  const uint64_t align_bits = reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(k) |
                              reinterpret_cast<uint64_t>(v) | reinterpret_cast<uint64_t>(out) |
                              static_cast<uint64_t>(q_tok_stride) | static_cast<uint64_t>(q_head_stride) |
                              static_cast<uint64_t>(kv_head_stride) | static_cast<uint64_t>(kv_row_stride) |
                              static_cast<uint64_t>(out_tok_stride) | static_cast<uint64_t>(out_head_stride);
  if (align_bits & 15) return RT_ERR_INVALID_ARGUMENT;
  if (q_tok_stride <= 0 || q_head_stride <= 0 || kv_head_stride <= 0 || kv_row_stride <= 0) return RT_ERR_UNSUPPORTED;
  const bool half = dtype == 2;
  const int tok = kPB / G;
  // without keys there is nothing to load: every row is zero, and the maps describe Q
  const bool keys = total_k > 0;
  CUtensorMap tq, tk, tv;
  int rc = make_prompt_tmap(&tq, q, half, num_q_heads, q_head_stride, total_q, q_tok_stride, G, tok);
  if (rc == RT_OK && keys)
    rc = make_prompt_tmap(&tk, k, half, total_k, kv_row_stride, num_kv_heads, kv_head_stride, kPB, 1);
  if (rc == RT_OK && keys)
    rc = make_prompt_tmap(&tv, v, half, total_k, kv_row_stride, num_kv_heads, kv_head_stride, kPB, 1);
  if (rc != RT_OK) return rc;
  if (!keys) tk = tv = tq;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  for (int b0 = 0; b0 < num_seqs; b0 += kPMaxSeqs) {
    const int nb = std::min(kPMaxSeqs, num_seqs - b0);
    PromptParams p{};
    p.out = static_cast<char*>(out);
    p.out_tok_stride = out_tok_stride;
    p.out_head_stride = out_head_stride;
    p.v = static_cast<const char*>(v);
    p.kv_head_stride = kv_head_stride;
    p.kv_row_stride = kv_row_stride;
    p.cu_q = cu_q == nullptr ? nullptr : cu_q + b0;
    p.cu_k = cu_q == nullptr ? nullptr : (cu_k != nullptr ? cu_k : cu_q) + b0;
    p.num_seqs = nb;
    p.total_q = static_cast<int>(total_q);
    p.total_k = static_cast<int>(total_k);
    p.hkv = num_kv_heads;
    p.group = G;
    p.tok = tok;
    // items, at most: full ones and one partial a sequence
    const int64_t pairs = (total_q / (2 * tok) + nb) * num_kv_heads;
    p.tiles = pairs >= kPSms ? 2 : 1;
    // (never 0: a hidden score is -inf and stays so; scores times 2^-126 are 0 in the sum)
    p.scale_log2 = std::max(scale * 1.4426950408889634f, 1.17549435e-38f);
    p.status = status;
    const int64_t items = (total_q / (p.tiles * tok) + nb) * num_kv_heads;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(items, kPSms)));
    if (half) {
      set_smem_limit(prompt_attn_kernel<__half>, kPSmem);
      rc = record_cuda(launch_ex(prompt_attn_kernel<__half>, grid, dim3(kPThreads), kPSmem, s, 1, tq, tk, tv, p));
    } else {
      set_smem_limit(prompt_attn_kernel<__nv_bfloat16>, kPSmem);
      rc = record_cuda(
          launch_ex(prompt_attn_kernel<__nv_bfloat16>, grid, dim3(kPThreads), kPSmem, s, 1, tq, tk, tv, p));
    }
    if (rc != RT_OK) return rc;
  }
  return RT_OK;
}
