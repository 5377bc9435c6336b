// Causal attention over whole prompts for B200 (sm_100a): packed sequences, GQA,
// head_dim 128, bf16 or fp16 in and out.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(scale*log2(e) q_i.k_j - m_i),
//   j <= i + lk - lq within the sequence, m_i a running maximum.
//
// A work item is 256 query rows of one kv head -- two 128-row tiles, row r of a
// tile being (token r / G, query head r % G) of G = Hq / Hkv, so the heads of a
// group share every K/V tile -- and all the 128-key blocks they see (or one of
// `splits` shares of them, when the items alone would leave SMs without work; the
// shares are merged through the workspace by prompt_combine_kernel).  The items
// are ordered longest first and handed out by the hardware: a CTA runs the item
// of its own block index, then takes over the next block that has not started.
// Twelve warps:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one thread per row: S from TMEM, the
//                   online softmax in the exp2 domain with a lazy (> 8 in log2)
//                   rescale of O in TMEM, P back into S's own columns, and the
//                   tile's output rows;
//   warp 8          producer: Q tiles and K / V blocks (a 4-stage ring) by TMA, and
//                   the requests for further items (cluster launch control);
//   warp 9          MMA issuer: per block PV of tile 0, next QK of
//                   tile 0, PV of tile 1, next QK of tile 1 -- while one tile's
//                   softmax runs the tensor core has the other tile's products;
//   warps 10, 11    check the V blocks that some row must not see in full
//                   (the causal diagonal, the sequence's end) for values that
//                   are not finite: 0 * NaN would reach rows that hide the key.
//                   They zero them; rows that do see the key add the value back
//                   at the end.  (Half a block each: one warp took longer than the
//                   block's softmax.)
// Every mbarrier wait is bounded (common.cuh): on time-out the CTA records
// RT_DEV_WAIT_TIMEOUT, drains what it issued, frees TMEM and exits.
//
// Measured (32 / 8 heads, bf16, in a graph): 2048 tokens 39.0-40.3 us, 7122
// tokens 334 us in a short burst (1250 TFLOP/s; 244 us at the burst rate of a plain matrix
// product), 394 us in a loop of seconds, where the GPU is at its power limit (990 W, SM
// clock 1.63 GHz).  A block of two tiles takes the MMA warp 3200 cycles, of which its products fill
// 2048 (tensor pipe 60 % active); with the exponentials, maxima and sums left out, and that warp's
// waits kept, 7122 tokens took 340 us where the whole took 362.
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
constexpr uint32_t kPOffOrd = kPOffTab + (kPMaxSeqs + 1) * 4 + 12;  // up to 32 sequences, longest first
constexpr uint32_t kPOffOut = kPOffOrd + 32 * 4;                       // a warp's 32 rows x 64 bytes of output
constexpr uint32_t kPOffBar = kPOffOut + 8 * 2048;
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
  int splits;                                       // shares of an item's keys
  int hq;
  float* ws_o;                                      // [split][token][head][128]
  float2* ws_ml;                                    // [split][token][head] (m in log2 units, l)
  float scale_log2;
  int* status;
};

struct PromptBars {
  uint64_t q_full[2], q_empty[2], kv_full[kPStages], kv_empty[kPStages], s_full[2], p_part[2], p_full[2], o_full[2],
      v_look, v_ok, clc_full[2], clc_empty[2], fin;
  uint4 clc[2];
  uint32_t tmem_base;
  int abort_flag;
  int poison;  // set once a checked V block held a value that is not finite
};

struct PromptItem {
  int q0, lq, k0, lk, tok0, g, split;
  int jb;     // first key block of this share
  int nb[2];  // its blocks in each tile
  int jm;     // the first of them that some row of the item hides in part
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

// The item of block index `idx`: kv head fastest, then share, then tile (the
// last, longest one of a sequence first), then sequence.
__device__ __forceinline__ void prompt_item(const PromptParams& p, const int* tab, const int* ord, int idx,
                                            PromptItem& w) {
  w.nb[0] = w.nb[1] = 0;
  w.jm = w.jb = w.lq = w.tok0 = 0;
  int pos = idx / p.hkv;
  w.g = idx - pos * p.hkv;
  w.split = pos % p.splits;
  pos /= p.splits;
  if (pos >= tab[p.num_seqs]) return;  // (the grid is sized for the most items there can be)
  int lo = 0, hi = p.num_seqs;         // tab[lo] <= pos < tab[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab[mid] <= pos) lo = mid; else hi = mid;
  }
  prompt_seq(p, p.num_seqs <= 32 ? ord[lo] : lo, w.q0, w.lq, w.k0, w.lk);
  const int tile = tab[lo + 1] - 1 - pos;
  w.tok0 = tile * p.tiles * p.tok;
  const int shift = w.lk - w.lq;
  int nb[2] = {0, 0};
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = w.tok0 + t * p.tok;
    const int lim = min(first + p.tok, w.lq) + shift;  // keys the tile's last token sees
    if (t < p.tiles && first < w.lq && lim > 0) nb[t] = (lim + kPB - 1) / kPB;
  }
  const int all = max(nb[0], nb[1]);
  w.jb = all * w.split / p.splits;
  const int je = all * (w.split + 1) / p.splits;
  w.nb[0] = max(min(nb[0], je) - w.jb, 0);
  w.nb[1] = max(min(nb[1], je) - w.jb, 0);
  w.jm = max(max(w.tok0 + 1 + shift, 0) / kPB - w.jb, 0);
}

// The `it`-th item of this CTA for one converged warp (or one lane that acts for
// it): its own block's, then those taken over.  False when there is none.
template <bool kWarp>
__device__ __forceinline__ bool prompt_next(const PromptParams& p, PromptBars& bar, const int* tab, const int* ord,
                                            int it, PromptItem& w) {
  int idx = blockIdx.x;
  if (it > 0) {
    const int s = (it - 1) & 1;
    if constexpr (kWarp) mbar_wait_fast(&bar.clc_full[s], ((it - 1) >> 1) & 1, &bar.abort_flag, p.status);
    else mbar_wait(&bar.clc_full[s], ((it - 1) >> 1) & 1, &bar.abort_flag, p.status, RT_DEV_WAIT_TIMEOUT);
    idx = *const_cast<volatile int*>(&bar.abort_flag) ? -1 : clc_taken(smem_u32(&bar.clc[s]));
    fence_proxy_async_smem();  // the slot's next answer is an async-proxy write: this read comes first
    if constexpr (kWarp) {
      idx = __reduce_min_sync(0xFFFFFFFFu, idx);  // (the same in every lane but for an abort in between)
      mbar_arrive_warp(&bar.clc_empty[s]);
    } else {
      mbar_arrive(&bar.clc_empty[s]);
    }
  }
  if (idx < 0) return false;
  prompt_item(p, tab, ord, idx, w);
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

// Larger magnitude of the halves of two 16-bit pairs (NaN stays).
template <typename T>
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                         __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
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

// kSplit: the items' keys are shared out (splits > 1), and results go to the workspace.
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kPThreads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const PromptParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PromptBars& bar = *reinterpret_cast<PromptBars*>(smem + kPOffBar);
  int* tab = reinterpret_cast<int*>(smem + kPOffTab);
  int* ord = reinterpret_cast<int*>(smem + kPOffOrd);
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
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.clc_full[i], 1);
      mbar_init(&bar.clc_empty[i], 12);  // every warp
    }
    mbar_init(&bar.v_look, 1);
    mbar_init(&bar.v_ok, 2);
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
    int q0, lq, k0, lk;
    if (p.num_seqs <= 32) {  // longest keys first (stable)
      const int key = lane < p.num_seqs ? (prompt_seq(p, lane, q0, lq, k0, lk) ? lk : -1) : -2;
      int rank = 0;
      for (int i = 0; i < p.num_seqs; ++i) {
        const int other = __shfl_sync(0xFFFFFFFFu, key, i);
        rank += other > key || (other == key && i < lane);
      }
      if (lane < p.num_seqs) ord[rank] = lane;
      __syncwarp();
    }
    int carry = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
      int n = 0;
      if (b0 + lane < p.num_seqs) {
        if (prompt_seq(p, p.num_seqs <= 32 ? ord[lane] : b0 + lane, q0, lq, k0, lk)) n = (lq + span - 1) / span;
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
  if (warp >= 8) {
    // (one instruction for the whole warpgroup; what follows stays inside the branch, as the
    // compiler budgets code after a merge for the smaller count)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsOther));
    if (warp == 8) {
      // ---------------- TMA producer ----------------
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
        // The next item is asked for when five blocks of this one are left to load:
        // late, so that whoever is done first gets it, and early enough that the
        // answer is there in time.  (Asked for at once, 256 items on 148 CTAs were
        // all handed out in the first microsecond: 2048 tokens took 52 us, not 43.)
        int asked = 0;
        auto take_over = [&](int it) {
          const int s = it & 1;
          if (!mbar_wait(&bar.clc_empty[s], ((it >> 1) & 1) ^ 1, abort_flag, p.status, RT_DEV_WAIT_TIMEOUT))
            return false;
          mbar_arrive_expect_tx(&bar.clc_full[s], 16);
          clc_try_cancel(smem_u32(&bar.clc[s]), &bar.clc_full[s]);
          asked = it + 1;
          return true;
        };
        for (int it = 0; ok && prompt_next<false>(p, bar, tab, ord, it, w); ++it) {
          const int nb = max(w.nb[0], w.nb[1]);
          if (nb == 0) ok = take_over(it);
          for (int j = 0; j < nb && ok; ++j) {
            if (j == max(nb - 5, 0)) {
              ok = take_over(it);
              if (!ok) break;
            }
            load(&tmap_k, w.k0 + (w.jb + j) * kPB);
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
            if (ok) load(&tmap_v, w.k0 + (w.jb + j) * kPB);
          }
        }
        if (*abort_flag) {
          for (int i = max(0, n - kPStages); i < n; ++i)
            mbar_wait_drain(&bar.kv_full[i % kPStages], (i / kPStages) & 1);
          for (int t = 0; t < 2; ++t)
            if (nq[t] > 0) mbar_wait_drain(&bar.q_full[t], (nq[t] - 1) & 1);
          if (asked > 0) mbar_wait_drain(&bar.clc_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1);
        }
      }
    } else if (warp == 9) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t kFmt = std::is_same_v<T, __half> ? (1u << 7 | 1u << 10) : 0u;  // clears the bf16 format bits
      constexpr uint32_t idesc_qk = idesc_bf16_f32(kPB, kPB, false, false) & ~kFmt;
      constexpr uint32_t idesc_pv = idesc_bf16_f32(kPB, kPD, false, true) & ~kFmt;
      const bool me = elect_one();
      const uint32_t tm = warp_uniform(tmem);
      // (descriptors: the low words; Q, K and V differ in the high one)
      const uint64_t desc_q = smem_desc_sw128(smem_u32(smem + kPOffQ), 16, 1024);
      const uint64_t desc_v = smem_desc_sw128(smem_u32(smem + kPOffKV), kPHalf, 1024);
      const uint32_t dq = warp_uniform(static_cast<uint32_t>(desc_q));
      const uint32_t hi_qk = warp_uniform(static_cast<uint32_t>(desc_q >> 32));
      const uint32_t dk = dq + ((kPOffKV - kPOffQ) >> 4);
      const uint32_t dv = warp_uniform(static_cast<uint32_t>(desc_v));
      const uint32_t hi_v = warp_uniform(static_cast<uint32_t>(desc_v >> 32));
      int n = 0;  // ring loads consumed
      int nq[2] = {0, 0}, np[2] = {0, 0};
      uint32_t looks = 0;  // V blocks handed to warps 10 and 11
      auto wait = [&](uint64_t* b, uint32_t ph, uint32_t known = 0) {
        mbar_wait_fast(b, ph & 1, abort_flag, p.status, known);
      };
      auto test = [](uint64_t* b, uint32_t ph) { return mbar_test(b, ph & 1); };
      // S_t = Q_t K^T of the block in `stage`; the last one of an item frees Q_t
      auto qk = [&](int t, int stage, bool last) {
        const uint32_t a = dq + t * (kPTile >> 4), b = dk + stage * (kPTile >> 4);
  #pragma unroll
        for (int kk = 0; kk < kPD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kPHalf + (kk & 3) * 32) >> 4;
          umma_f16_if(me, tm + t * kPB, a + off, b + off, hi_qk, idesc_qk, kk > 0);
        }
        umma_commit_if(me, &bar.s_full[t]);
        umma_commit_if(me && last, &bar.q_empty[t]);
      };
      for (int it = 0; prompt_next<true>(p, bar, tab, ord, it, w); ++it) {
        const int nb = max(w.nb[0], w.nb[1]);
        if (nb == 0) continue;
        const int s = warp_uniform2(n % kPStages);
        wait(&bar.kv_full[s], n / kPStages);
  #pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (w.nb[t] == 0) continue;
          wait(&bar.q_full[t], nq[t]++);
          tc_fence_after();
          qk(t, s, w.nb[t] == 1);
        }
        umma_commit_if(me, &bar.kv_empty[s]);
        ++n;
        // Each wait's barrier is asked some products ahead (`known`), so that the answer
        // of one that is there does not hold up the tensor core.
        uint32_t known_v = 0, known_p = 0;
        for (int j = 0; j < nb; ++j) {
          const int sv = warp_uniform2(n % kPStages), sk = (sv + 1) % kPStages;
          const bool more = j + 1 < nb;
          bool look = j >= w.jm;
          wait(&bar.kv_full[sv], n / kPStages, known_v);
          if (look && me) mbar_arrive(&bar.v_look);
          uint32_t known_k = more ? test(&bar.kv_full[sk], (n + 1) / kPStages) : 0;
          const uint32_t b = dv + sv * (kPTile >> 4);
  #pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j < w.nb[t]) {
              auto pv = [&](int kk) {
                umma_f16_ts_if(me, tm + kPTmemO + t * kPD, tm + t * kPB + kk * 8, b + kk * (2048 >> 4), hi_v, idesc_pv,
                               j > 0 || kk > 0);
              };
              wait(&bar.p_part[t], np[t], known_p);
              if (look) wait(&bar.v_ok, looks++);
              look = false;
              tc_fence_after();
              const uint32_t known = test(&bar.p_full[t], np[t]);
  #pragma unroll
              for (int kk = 0; kk < kPart1 / 16; ++kk) pv(kk);
              wait(&bar.p_full[t], np[t]++, known);
              tc_fence_after();
  #pragma unroll
              for (int kk = kPart1 / 16; kk < kPB / 16; ++kk) pv(kk);
              umma_commit_if(me && j + 1 == w.nb[t], &bar.o_full[t]);
            }
            if (more && t == 0) wait(&bar.kv_full[sk], (n + 1) / kPStages, known_k);
            known_p = test(&bar.p_part[t ^ 1], np[t ^ 1]);
            if (t == 1 && more) known_v = test(&bar.kv_full[(sv + 2) % kPStages], (n + 2) / kPStages);
            if (j + 1 < w.nb[t]) qk(t, sk, j + 2 == w.nb[t]);
            if (t == 1) umma_commit_if(me, &bar.kv_empty[sv]);
          }
          umma_commit_if(me && more, &bar.kv_empty[sk]);
          n += more ? 2 : 1;
        }
      }
      // all issued MMAs complete before TMEM is released
      umma_commit_if(me, &bar.fin);
      if (me) mbar_wait_drain(&bar.fin, 0);
      __syncwarp();
    } else {
      // ---------------- V blocks that are partly hidden: values that are not finite ----------------
      // (the MMA warp hands them over in order, right after the block's QK, so
      // the check runs beside the block's softmax)
      int n = 0;
      uint32_t looks = 0;
      for (int it = 0; prompt_next<true>(p, bar, tab, ord, it, w); ++it) {
        const int nb = max(w.nb[0], w.nb[1]);
        for (int j = min(w.jm, nb); j < nb; ++j) {
          const int m = n + 2 * j + 1, s = m % kPStages;
          mbar_wait_fast(&bar.v_look, looks++ & 1, abort_flag, p.status);
          mbar_wait_fast(&bar.kv_full[s], (m / kPStages) & 1, abort_flag, p.status);
          // this warp's half, 512 bytes a step
          constexpr int kSteps = static_cast<int>(kPTile / 1024);
          const uint32_t v = smem_u32(smem + kPOffKV + s * kPTile) + (warp - 10) * (kPTile / 2) + lane * 16;
          uint32_t top = 0;  // largest magnitudes, NaN above all
  #pragma unroll 8
          for (int i = 0; i < kSteps; ++i) {
            const uint4 x = lds128(v + i * 512);
            top = abs_max2<T>(abs_max2<T>(abs_max2<T>(abs_max2<T>(top, x.x), x.y), x.z), x.w);
          }
          if (__any_sync(0xFFFFFFFFu, not_finite2<T>(top) != 0)) {
            auto fix = [](uint32_t x) {
              const uint32_t b = not_finite2<T>(x);
              return x & ~(((b >> 15) & 0x00010001u) * 0xFFFFu);
            };
  #pragma unroll 1
            for (int i = 0; i < kSteps; ++i) {
              uint4 x = lds128(v + i * 512);
              x.x = fix(x.x);
              x.y = fix(x.y);
              x.z = fix(x.z);
              x.w = fix(x.w);
              sts128(v + i * 512, x);
            }
            fence_proxy_async_smem();
            if (lane == 0) *const_cast<volatile int*>(&bar.poison) = 1;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.v_ok);
        }
        n += 2 * nb;
      }
    }
  } else {
    // ---------------- softmax and output of tile t ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsSoftmax));
    const int t = warp >> 2;
    const int r = tid & (kPB - 1);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + t * kPB, to = tmem + lane_base + kPTmemO + t * kPD;
    const int rt = r / p.group, rh = r - rt * p.group;
    const float sl2 = p.scale_log2;
    int ns = 0, no = 0;
    const uint32_t stage = smem_u32(smem + kPOffOut + warp * 2048);
    bool more = prompt_next<true>(p, bar, tab, ord, 0, w);
    PromptItem next{};
    for (int it = 0; more; ++it, w = next) {
      const int tok = w.tok0 + t * p.tok + rt;
      const bool valid = t < p.tiles && rt < p.tok && tok < w.lq;
      const int lim = valid ? min(max(tok + 1 + w.lk - w.lq, 0), w.lk) : 0;  // keys this row sees
      const int jmask = max(w.tok0 + t * p.tok + 1 + w.lk - w.lq, 0) / kPB - w.jb;
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
          const int left = lim - (w.jb + j) * kPB;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= left) sr[c][i] = __float_as_uint(-INFINITY);
        }
        softmax_block<T>(sr, ts, to, j > 0, sl2, m, l, [&] { mbar_arrive_warp(&bar.p_part[t]); });
        mbar_arrive_warp(&bar.p_full[t]);
      }
      const int64_t row = static_cast<int64_t>(w.q0 + tok), head = w.g * p.group + rh;
      char* dst = p.out + row * p.out_tok_stride + head * p.out_head_stride;
      const int64_t slot = (static_cast<int64_t>(w.split) * p.total_q + row) * p.hq + head;
      // (found out while the last products run)
      more = prompt_next<true>(p, bar, tab, ord, it + 1, next);
      if (nb == 0) {
        if (kSplit && valid) p.ws_ml[slot] = make_float2(-INFINITY, 0.f);
        if (!kSplit && valid)
          for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(dst + c * 16) = make_uint4(0, 0, 0, 0);
        continue;
      }
      mbar_wait_fast(&bar.o_full[t], no++ & 1, abort_flag, p.status);
      if (__any_sync(0xFFFFFFFFu, *abort_flag)) break;
      tc_fence_after();
      // (a row that sees no key of this share has l == 0, and its O is 0 or not a number)
      const float inv = kSplit ? 1.f : 1.f / l;
      const bool none = lim <= w.jb * kPB;
      const bool poison = *const_cast<volatile int*>(&bar.poison) != 0;
      const RowsOut rows(stage, !valid   ? 0
                                : kSplit ? reinterpret_cast<uint64_t>(p.ws_o + slot * kPD)
                                         : reinterpret_cast<uint64_t>(dst));
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(to + c * 32, o);
        tmem_wait_ld();
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = none ? 0.f : __uint_as_float(o[i]) * inv;
        if (poison && valid)
          add_not_finite<T>(p.v + w.g * p.kv_head_stride + w.k0 * p.kv_row_stride + c * 64, p.kv_row_stride,
                            (w.jb + w.jm) * kPB, min(lim, (w.jb + nb) * kPB), x);
        rows.put32<std::conditional_t<kSplit, float, T>>(x, c);
      }
      // (a NaN weight wins the merge)
      if (kSplit && valid) p.ws_ml[slot] = none ? make_float2(-INFINITY, 0.f) : make_float2(l == l ? m : INFINITY, l);
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One warp per (token, query head): the sum of the row's shares.  Tokens outside
// every (valid) sequence have none and are left alone.
template <typename T>
__global__ void __launch_bounds__(128) prompt_combine_kernel(const PromptParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t gw = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (gw >= static_cast<int64_t>(p.total_q) * p.hq) return;
  const int row = static_cast<int>(gw / p.hq), head = static_cast<int>(gw - static_cast<int64_t>(row) * p.hq);
  bool mine = false;
  for (int b = lane; b < p.num_seqs; b += 32) {
    int q0, lq, k0, lk;
    mine |= prompt_seq(p, b, q0, lq, k0, lk) && row >= q0 && row < q0 + lq;
  }
  if (!__any_sync(0xFFFFFFFFu, mine)) return;
  const int64_t step = static_cast<int64_t>(p.total_q) * p.hq, slot = static_cast<int64_t>(row) * p.hq + head;
  const float2 ml = lane < p.splits ? p.ws_ml[slot + lane * step] : make_float2(-INFINITY, 0.f);
  float M = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
  const float wt = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
  float lsum = wt * ml.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xFFFFFFFFu, lsum, o);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < p.splits; s0 += 4) {
    float4 o[4];
    float w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      w[u] = __shfl_sync(0xFFFFFFFFu, wt, (s0 + u) & 31);
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + u < p.splits && w[u] != 0.f)
        o[u] = *reinterpret_cast<const float4*>(p.ws_o + (slot + (s0 + u) * step) * kPD + lane * 4);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (s0 + u >= p.splits || w[u] == 0.f) continue;
      acc.x = fmaf(w[u], o[u].x, acc.x);
      acc.y = fmaf(w[u], o[u].y, acc.y);
      acc.z = fmaf(w[u], o[u].z, acc.z);
      acc.w = fmaf(w[u], o[u].w, acc.w);
    }
  }
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
  *reinterpret_cast<uint2*>(p.out + row * p.out_tok_stride + head * p.out_head_stride + lane * 8) =
      make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
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

struct PromptPlan {
  int tiles, splits;
  int64_t items;
};

// Two tiles an item when that fills the GPU.  When it does not, an item's keys
// are split if there are enough of them (at least eight blocks a share; twice the
// SMs' number of shares), and short prompts go one tile an item.  The sequences'
// lengths are on the device, so their mean stands for them.
static PromptPlan prompt_plan(int64_t total_q, int64_t total_k, int seqs, int hkv, int tok) {
  PromptPlan pl{2, 1, (total_q / (2 * tok) + seqs) * hkv};
  if (pl.items >= kPSms) return pl;
  const int64_t blocks = total_k / seqs / kPB;
  if (blocks < 16 || total_q / seqs <= tok) {
    pl.tiles = 1;
    pl.items = (total_q / tok + seqs) * hkv;
  }
  if (blocks >= 16)
    pl.splits = static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(32, blocks / 8), (2 * kPSms + pl.items - 1) / pl.items)));
  return pl;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_prompt_attn_workspace_size(int64_t total_q, int64_t total_k, int num_seqs, int num_q_heads,
                                                int num_kv_heads) {
  if (total_q <= 0 || total_k < 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads || num_q_heads / num_kv_heads > kPB)
    return 0;
  const PromptPlan pl = prompt_plan(total_q, total_k, num_seqs, num_kv_heads, kPB / (num_q_heads / num_kv_heads));
  if (pl.splits == 1) return 0;
  const size_t rows = static_cast<size_t>(pl.splits) * total_q * num_q_heads;
  return align_up(rows * kPD * 4, 256) + align_up(rows * 8, 256);
}

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
  const PromptPlan plan = prompt_plan(total_q, total_k, num_seqs, num_kv_heads, tok);
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
    p.hq = num_q_heads;
    p.group = G;
    p.tok = tok;
    p.tiles = plan.tiles;
    p.splits = plan.splits;
    // (never 0: a hidden score is -inf and stays so; scores times 2^-126 are 0 in the sum)
    p.scale_log2 = std::max(scale * 1.4426950408889634f, 1.17549435e-38f);
    p.status = status;
    if (plan.splits > 1) {  // (fewer than kPMaxSeqs sequences: one launch)
      const size_t rows = static_cast<size_t>(plan.splits) * total_q * num_q_heads;
      if (workspace == nullptr ||
          workspace_bytes < rt_prompt_attn_workspace_size(total_q, total_k, num_seqs, num_q_heads, num_kv_heads))
        return RT_ERR_WORKSPACE;
      p.ws_o = static_cast<float*>(workspace);
      p.ws_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + align_up(rows * kPD * 4, 256));
    }
    // items, at most: full ones and one partial a sequence
    const int64_t items = (total_q / (plan.tiles * tok) + nb) * num_kv_heads * plan.splits;
    if (items > INT32_MAX) return RT_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(items));
    const dim3 rows_grid(static_cast<unsigned>((total_q * num_q_heads + 3) / 4));
    auto launch = [&](auto kernel, auto combine) {
      set_smem_limit(kernel, kPSmem);
      int status = record_cuda(launch_ex(kernel, grid, dim3(kPThreads), kPSmem, s, 1, tq, tk, tv, p));
      if (status == RT_OK && plan.splits > 1) status = record_cuda(launch_ex(combine, rows_grid, dim3(128), 0, s, 1, p));
      return status;
    };
    if (half)
      rc = plan.splits > 1 ? launch(prompt_attn_kernel<__half, true>, prompt_combine_kernel<__half>)
                           : launch(prompt_attn_kernel<__half, false>, prompt_combine_kernel<__half>);
    else
      rc = plan.splits > 1 ? launch(prompt_attn_kernel<__nv_bfloat16, true>, prompt_combine_kernel<__nv_bfloat16>)
                           : launch(prompt_attn_kernel<__nv_bfloat16, false>, prompt_combine_kernel<__nv_bfloat16>);
    if (rc != RT_OK) return rc;
  }
  return RT_OK;
}
