// tcgen05 / TMEM / TMA form of the ragged attention (gqa_ragged.cuh has the masks, the
// scores and the work of a tile): requests of more than kRaggedStreamRows packed rows, i.e.
// prompts, chunks of them and long drafts. The pipeline is the dense prefill kernel's (gqa_prefill.cuh): one CTA
// owns two 128-row query tiles of one (request, kv head), a TMA warp streams 128-key
// tiles of K and V from the paged cache, one thread issues the UMMAs
//   S_i = Q_i K_j^T (f32 in TMEM),   O_i += P_i V_j (P from TMEM)
// and a warpgroup per tile turns S into P with the online softmax, the two tiles taking
// turns on the tensor core. What differs:
//  - Rows are packed token-major (row = token x group + head), so a tile's tokens are
//    consecutive rows of the packed queries and any group up to 64 fits:
//    bm = 128 / group tokens per tile, 128 - bm x group rows idle.
//  - The key range is the union of the two tiles' intervals, and every row has its own
//    [lo, hi) in it. A row's running maximum starts at a finite -3e38, so that tiles
//    where it sees nothing add exp2(-inf) = 0; rows that saw nothing end with l = 0.
//  - Scores may be capped or biased (MOD), see below.
//  - A tile whose tokens fit the first query tile runs solo: the two warpgroups take the
//    even and the odd key tiles of the same 128 rows (own S, O, maximum and sum) and merge
//    at the end, so that a request of few rows keeps both warpgroups busy.
//  - O leaves through shared memory with ordinary 16-byte stores, since a tile may end
//    where the next request's rows begin.
//
// Work is found on the device: every CTA scans the requests' lengths (one load and one
// block scan per 384 requests) and takes its tile from the end, so that of one prompt the
// tiles with the most keys start first. The host's grid covers the most tiles that the
// step can have; CTAs past the real number return before they touch TMEM.
//
// Bound by the tensor core and the softmax's exponentials together (gqa_prefill.cuh has
// the accounting). The cap would cost two more MUFU operations per score (exp2 and a
// reciprocal), three times the exponential's alone. So while every score of a warp's rows
// in the tile has |y| <= 0.6, y = s scale / cap,
//   cap log2 e tanh(y) = s (a0 + a1 s^2 + a2 s^4 + a3 s^6),
// an odd polynomial fitted to tanh (tests/tanh_fit.py, absolute error 6.5e-7 of the cap)
// whose last product merges with the subtraction of the maximum: four more operations per
// pair of scores (packed; 5 % faster than with a scalar square) on the FMA pipe. Neither that
// pipe nor the MUFU is full: a step waits for the magnitude of all its columns and the vote
// before P. Tiles with larger scores, rare in models that cap them,
// take the MUFU form.
//
// Measured, 32 query and 8 kv heads of 128, bf16, two prompts' chunks of up to 4096 tokens
// on up to 12288 cached keys: causal 985 us, 1080 TFLOP/s; capped 1.24 to 1.33 ms on different
// boxes (2.3 ms with every tile in the MUFU form); capped and with a distance bias 1.8 ms (3.8 ms). A pair's step
// of 128 keys takes 2.0 us (the softmax chain, then the wait for its S), a solo step
// 1.05 us per 128 keys, and a CTA about 10 us besides: the scan 2, the first S 2.5, a
// masked tile 1.3, the epilogue 3 to 4. Slower, and not kept: P beside S in TMEM, which at
// head size 128 leaves room for 64- or 80-key tiles only (677 and 836 TFLOP/s).
#pragma once

#include "gqa_prefill.cuh"
#include "gqa_ragged.cuh"

namespace gqa {

constexpr int kMaxRaggedChunks = 16;  // key chunks of a tile

// Score transforms of an instantiation: kRaggedPlain none; kRaggedCap the cap alone
// (monotone, so the row maximum is taken before it); kRaggedBias a distance bias alone,
// kRaggedCapBias both. An instantiation each: code that a call does not use costs the
// softmax warps registers (one for bias with and without a cap: 7 % slower without).
enum : int { kRaggedPlain = 0, kRaggedCap = 1, kRaggedBias = 2, kRaggedCapBias = 3 };

// tanh(y) ~ y (c0 + c1 y^2 + c2 y^4 + c3 y^6), |y| <= kTanhRange.
constexpr float kTanhRange = 0.6f;
constexpr float kTanhC0 = 0.9999909996986389f, kTanhC1 = -0.33298975229263306f;
constexpr float kTanhC2 = 0.12974554300308228f, kTanhC3 = -0.039611268788576126f;

// The polynomial's coefficients for raw scores s (host side).
inline void set_cap_polynomial(RaggedParams& p, double scale_over_cap, double cap_log2e) {
  const double c[4] = {kTanhC0, kTanhC1, kTanhC2, kTanhC3};
  double k = scale_over_cap;
  for (int i = 0; i < 4; ++i) {
    p.cap_a[i] = (float)(cap_log2e * c[i] * k);
    k *= scale_over_cap * scale_over_cap;
  }
  p.cap_most = (float)(kTanhRange / scale_over_cap);
}

// With bf16, a bound of the row's scores may stand for their maximum: P has fp32's range.
// At most this large (log2 units), so that the smallest P, 2^-2 kBoundMost, is far from it.
constexpr float kBoundMost = 44.f;

// Three-input maximum of magnitudes.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int HD>
struct RaggedTileCfg : PrefillCfg<HD> {
  using Base = PrefillCfg<HD>;
  static constexpr int kTileBytes = Base::kTileBytes;
  // K and V have a ring each (K_j's slot is free once QK_j is done, V_j's only after the
  // softmax and PV_j), filled by a warp each. A pair's rings start after its two Q tiles;
  // a solo tile has one, and less work per key to hide the loads behind, so its rings are
  // longer: they fill the shared memory that an SM has.
  static constexpr int kPairSlots = HD == 128 ? 2 : 4;  // of each of K and V
  static constexpr int kSoloSlots = HD == 128 ? 3 : 6;
  static constexpr int kRingTiles = 2 * kPairSlots + 1 > 2 * kSoloSlots ? 2 * kPairSlots + 1 : 2 * kSoloSlots;
  static constexpr int kBarOff = (1 + kRingTiles) * kTileBytes;
  // q_full[2] k_full[S] k_empty[S] v_full[S] v_empty[S] s_full[2] p_full[2][kPParts] o_final[2] mma_done
  static constexpr int kNumBars = 2 + 4 * kSoloSlots + 2 + 2 * Base::kPParts + 2 + 1;
  // tmem base, abort flag, last-CTA flag, then the work item and the scan's warp sums
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kWorkOff = kMiscOff + 16;
  static constexpr int kTileSmem = kWorkOff + 64 + 64 + 1024;
  static constexpr int kSmemBytes = kTileSmem > StreamCfg<HD>::kSmemBytes ? kTileSmem : StreamCfg<HD>::kSmemBytes;
  static_assert(kSmemBytes <= 227 * 1024, "one CTA's shared memory");
};

template <int HD, bool BF16, int MOD>
__global__ void __launch_bounds__(384, 1)
    gqa_ragged_tile_kernel(const __grid_constant__ RaggedParams p, const __grid_constant__ CUtensorMap qmap,
                           const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  // The step's short requests stream in the grid's last CTAs: they fill the SMs as the
  // tiles run out.
  if (blockIdx.x >= p.tile_ctas) {
    if constexpr (MOD == kRaggedBias)
      ragged_stream_beside<HD, BF16>(p, &kmap, &vmap, blockIdx.x - p.tile_ctas);
    else
      ragged_stream_cta<HD, BF16, false>(p, &kmap, &vmap, blockIdx.x - p.tile_ctas);
    return;
  }
  using Cfg = RaggedTileCfg<HD>;
  const RaggedTiling& tl = p.tile;
  constexpr int NSUB = Cfg::kNSub;
  constexpr int BN = Cfg::kBN;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - raw_base);

  constexpr int MAXS = Cfg::kSoloSlots;  // barriers per ring
  const uint32_t q_smem0 = base;
  const uint32_t bars = base + Cfg::kBarOff;
  const uint32_t bar_q_full = bars;                             // [2]
  const uint32_t bar_k_full = bars + 16;                        // [MAXS] each
  const uint32_t bar_k_empty = bar_k_full + 8 * MAXS;
  const uint32_t bar_v_full = bar_k_empty + 8 * MAXS;
  const uint32_t bar_v_empty = bar_v_full + 8 * MAXS;
  const uint32_t bar_s_full = bar_v_empty + 8 * MAXS;           // [2]
  const uint32_t bar_p_full = bar_s_full + 16;                  // [2][kPParts]
  const uint32_t bar_o_final = bar_p_full + 16 * Cfg::kPParts;  // [2]
  const uint32_t bar_mma_done = bar_o_final + 16;
  uint32_t* tmem_base_ptr = reinterpret_cast<uint32_t*>(smem + Cfg::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kMiscOff + 4);

  // The work item, in shared memory: the softmax warps have no registers to spare, so its
  // fields are read where they are used.
  struct Work {
    int t0, nq, off_m0, len;  // first token's row, tokens, position of the first token, the request's keys
    int b, k_lo, k_hi;        // request; union of the rows' intervals
    int key0, nk, n_chunks;   // this CTA's first key, its 128-key tiles; chunks of the tile
    int unit;
  };
  volatile Work* const work = reinterpret_cast<volatile Work*>(smem + Cfg::kWorkOff);
  int* const scan_sums = reinterpret_cast<int*>(smem + Cfg::kWorkOff + 64);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const unsigned n_inner = (unsigned)(p.hkv * tl.nsplit);
  const int tile_id = (int)(blockIdx.x / n_inner);
  const int kvh = (int)((blockIdx.x % n_inner) / (unsigned)tl.nsplit);
  const int split = (int)(blockIdx.x % (unsigned)tl.nsplit);
  const int bm = tl.block_m >> 1;  // tokens per query tile

  if (tid == 0) {
    mbar_init(bar_q_full, 1);
    mbar_init(bar_q_full + 8, 1);
    for (int s = 0; s < 4 * MAXS; ++s) mbar_init(bar_k_full + 8 * s, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_s_full + 8 * i, 1);
      for (int h = 0; h < Cfg::kPParts; ++h) mbar_init(bar_p_full + 8 * (Cfg::kPParts * i + h), 128);
      mbar_init(bar_o_final + 8 * i, 1);
    }
    mbar_init(bar_mma_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  pdl_wait();
  pdl_trigger();

  // ---- which tile: count the tiles of every request that is this form's, and take number
  // (total - 1 - tile_id). Everything about a request is loaded at once, so that the thread
  // that finds the tile can describe it without another round trip.
  struct Request {
    int first, qn, len, off, prefix, tiles;  // off: position of the request's token 0 (see ragged_work_at)
  };
  auto load = [&](int b) -> Request {
    Request r{0, 0, 0, 0, 0, 0};
    if (b < p.n) {
      r.first = p.cu[b];
      r.qn = p.cu[b + 1];
      r.len = p.seq_lens[b];
      if (p.prefix) r.prefix = p.prefix[b];
      r.len = max(0, r.len);
      r.off = r.len - (r.qn - r.first);
      r.len = min(r.len, p.max_len);
      r.qn = min(r.qn, p.num_tokens) - r.first;
      if (r.first >= 0 && r.qn > 0 && (int64_t)r.qn * p.group >= tl.min_rows) r.tiles = (r.qn + tl.block_m - 1) / tl.block_m;
    }
    return r;
  };
  // The chunk's key range, from the union of the rows' intervals.
  auto set_keys = [&](int k_lo, int k_hi) {
    const int k_base = min(k_lo, k_hi) & ~(p.box - 1);  // where a box may start
    const int k_first = k_base + split * tl.chunk;
    const bool any = k_hi > k_lo;
    work->k_lo = k_lo;
    work->k_hi = k_hi;
    work->key0 = k_first;
    work->nk = any ? max(0, (min(k_first + tl.chunk, k_hi) - k_first + BN - 1) / BN) : 0;
    work->n_chunks = any ? (k_hi - k_base + tl.chunk - 1) / tl.chunk : 1;
  };
  {
    const int rounds = (p.n + 383) / 384;
    const Request mine = load(tid);
    int total = 0;
    for (int r = 0; r < rounds; ++r) {
      const int s = __reduce_add_sync(0xffffffffu, r ? load(r * 384 + tid).tiles : mine.tiles);
      if (r) __syncthreads();
      if (lane == 0) scan_sums[warp] = s;
      __syncthreads();
      for (int w = 0; w < 12; ++w) total += scan_sums[w];
    }
    const int want = total - 1 - tile_id;
    if (want < 0) return;  // the whole CTA, before TMEM
    if (warp == 8) {
      tmem_alloc(smem_u32(tmem_base_ptr), Cfg::kTmemCols);
      tmem_relinquish();
    }
    int before = 0;
    for (int r = 0; r < rounds; ++r) {
      const Request q = r ? load(r * 384 + tid) : mine;
      int incl = q.tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      if (rounds > 1) {  // one round: scan_sums still has the warps' sums
        __syncthreads();
        if (lane == 31) scan_sums[warp] = incl;
        __syncthreads();
      }
      int at = before;
      for (int w = 0; w < 12; ++w) {
        if (w < warp) at += scan_sums[w];
        before += scan_sums[w];
      }
      at += incl - q.tiles;
      if (want >= at && want < at + q.tiles) {
        const int m0 = (want - at) * tl.block_m, nq = min(tl.block_m, q.qn - m0);
        const int p_first = q.off + m0;
        int k_hi = q.len;
        if (p.causal) k_hi = max(0, min(k_hi, max(p_first + nq, q.prefix)));
        work->b = r * 384 + tid;
        work->t0 = q.first + m0;
        work->nq = nq;
        work->off_m0 = p_first;
        work->len = q.len;
        if (p.seq_lens[r * 384 + tid] > p.max_len) report_device_error(GQA_ERR_INVALID_ARG, 215);
        work->unit = (int)(blockIdx.x / (unsigned)tl.nsplit);
        set_keys(p.window > 0 ? max(0, p_first - p.window + 1) : 0, k_hi);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (p.key_starts) {
    if (warp == 0) {
      int s = INT_MAX;
      for (int i = lane; i < work->nq; i += 32) s = min(s, p.key_starts[work->t0 + i]);
      s = __reduce_min_sync(0xffffffffu, s);
      if (lane == 0) set_keys(max(work->k_lo, s), work->k_hi);
    }
    __syncthreads();
  }
  const uint32_t tmem_base = *tmem_base_ptr;
  if (split >= work->n_chunks) {
    if (warp == 8) tmem_dealloc(tmem_base, Cfg::kTmemCols);
    return;
  }
  const bool solo = work->nq <= bm;
  const int slots = solo ? MAXS : Cfg::kPairSlots;                       // of each ring
  const uint32_t k_ring = q_smem0 + (solo ? 1 : 2) * Cfg::kTileBytes;
  const uint32_t v_ring = k_ring + slots * Cfg::kTileBytes;

  // Register split as the dense prefill kernel's: 2 x 128 x 208 + 128 x 88 = 384 x 168.
  static_assert(Cfg::kSoftmaxRegs == 208 && Cfg::kControlRegs == 88, "keep the asm immediates in sync");
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
    if (warp == 9 || warp == 10) {
      // ============================================================== producers: K, V
      // Lane i brings box i / NSUB, 64 values of d at i % NSUB, of each tile. Boxes past the
      // last key get a block outside the cache: TMA fills them with zeros.
      const bool is_v = warp == 10;
      const CUtensorMap* map = is_v ? &vmap : &kmap;
      const uint32_t full0 = is_v ? bar_v_full : bar_k_full, empty0 = is_v ? bar_v_empty : bar_k_empty;
      const int nk = work->nk;
      if (nk > 0) {
        if (lane == 0) {
          tma_prefetch_desc(map);
          if (!is_v) {
            const int hq0 = kvh * p.group, t0 = work->t0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (i == 1 && solo) break;
              mbar_arrive_expect_tx(bar_q_full + 8 * i, (uint32_t)(bm * p.group) * 128u * NSUB);
#pragma unroll
              for (int s = 0; s < NSUB; ++s)
                tma_load_4d(q_smem0 + i * Cfg::kTileBytes + s * Cfg::kSubBytes, &qmap, bar_q_full + 8 * i, s * 64, hq0,
                            t0 + i * bm, 0);
            }
          }
        }
        const int box = p.box, nbox = BN / box;
        const int my_box = lane / NSUB, my_sub = lane % NSUB;
        const bool loads = my_box < nbox;
        const int k_hi = work->k_hi, key_first = work->key0 + my_box * box;
        const int* row_bt = p.block_table + (int64_t)work->b * p.bt_stride;
        const int mask = (1 << p.block_shift) - 1;
        const uint32_t dst0 = (is_v ? v_ring : k_ring) + my_sub * Cfg::kSubBytes + (uint32_t)(my_box * box) * 128u;
        int j = 0, slot = 0, use = 0;
        bool ok = true;
        for (; j < nk; ++j) {
          const int key = key_first + j * BN;
          // Looked up before the slot wait, so the table read overlaps it.
          const int pb = (loads && key < k_hi) ? row_bt[key >> p.block_shift] : p.num_blocks;
          if (use > 0) {
            ok = mbar_wait(empty0 + 8 * slot, (use - 1) & 1, abort_flag, 121);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          if (!withheld_load(2 * j + is_v)) {
            const uint32_t full = full0 + 8 * slot;
            if (lane == 0) mbar_arrive_expect_tx(full, Cfg::kTileBytes);
            __syncwarp();
            if (loads) tma_load_4d(dst0 + slot * Cfg::kTileBytes, map, full, my_sub * 64, kvh, key & mask, pb);
          }
          if (++slot == slots) {
            slot = 0;
            ++use;
          }
        }
        if (j < nk && lane == 0) {  // aborted: let in-flight loads land before teardown
          volatile int dummy = 0;
          for (int u = max(0, j - slots); u < j; ++u)
            if (!withheld_load(2 * u + is_v)) mbar_wait(full0 + 8 * (u % slots), (u / slots) & 1, &dummy, 122);
        }
      }
      __syncwarp();
    } else if (warp == 8) {
      // ============================================================== MMA issuer
      const int nk = work->nk;
      if (lane == 0 && nk > 0) {
        constexpr uint32_t idesc_qk = make_idesc_f16(128, BN, BF16, false);
        constexpr uint32_t idesc_pv = make_idesc_f16(128, HD, BF16, true);
        auto issue_qk = [&](int i, int slot) {
          const uint32_t tS = tmem_base + (i ? Cfg::kColS1 : Cfg::kColS0);
          const uint32_t qa = q_smem0 + (solo ? 0 : i) * Cfg::kTileBytes;
          const uint32_t kb = k_ring + slot * Cfg::kTileBytes;
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint32_t o = (k >> 2) * Cfg::kSubBytes + (k & 3) * 32;
            umma_ss(tS, desc_sw128_kmajor(qa + o), desc_sw128_kmajor(kb + o), idesc_qk, k > 0 ? 1u : 0u);
          }
        };
        auto issue_pv = [&](int i, int slot, int h, bool acc) {
          const uint32_t tS = tmem_base + (i ? Cfg::kColS1 : Cfg::kColS0);
          const uint32_t tO = tmem_base + (i ? Cfg::kColO1 : Cfg::kColO0);
          const uint32_t vb = v_ring + slot * Cfg::kTileBytes;
          constexpr int kPerPart = BN / 16 / Cfg::kPParts;
#pragma unroll
          for (int kk = 0; kk < kPerPart; ++kk) {
            const int k = h * kPerPart + kk;
            umma_ts(tO, tS + k * 8, desc_sw128_mnmajor(vb + k * 16 * 128, Cfg::kSubBytes), idesc_pv,
                    (acc || k > 0) ? 1u : 0u);
          }
        };
        bool ok = mbar_wait(bar_q_full, 0, abort_flag, 130) &&
                  (solo || mbar_wait(bar_q_full + 8, 0, abort_flag, 131)) && mbar_wait(bar_k_full, 0, abort_flag, 132);
        if (ok && !solo) {
          constexpr int S = Cfg::kPairSlots;
          tc_fence_after();
          issue_qk(0, 0);
          umma_commit(bar_s_full);
          issue_qk(1, 0);
          umma_commit(bar_s_full + 8);
          umma_commit(bar_k_empty);  // K_0 consumed
          for (int j = 0; j < nk; ++j) {
            const int sv = j % S, sk = (j + 1) % S;
            if (!mbar_wait(bar_v_full + 8 * sv, (j / S) & 1, abort_flag, 133)) break;
            bool pv_ok = true;
#pragma unroll
            for (int h = 0; h < Cfg::kPParts && pv_ok; ++h) {
              pv_ok = mbar_wait(bar_p_full + 8 * h, j & 1, abort_flag, h ? 138 : 134);
              if (pv_ok) {
                tc_fence_after();
                issue_pv(0, sv, h, h > 0 || j > 0);
              }
            }
            if (!pv_ok) break;
            const bool more = (j + 1 < nk);
            if (more) {
              if (!mbar_wait(bar_k_full + 8 * sk, ((j + 1) / S) & 1, abort_flag, 135)) break;
              tc_fence_after();
              issue_qk(0, sk);
              umma_commit(bar_s_full);
            } else {
              umma_commit(bar_o_final);
            }
#pragma unroll
            for (int h = 0; h < Cfg::kPParts && pv_ok; ++h) {
              pv_ok = mbar_wait(bar_p_full + 8 * (Cfg::kPParts + h), j & 1, abort_flag, h ? 139 : 136);
              if (pv_ok) {
                tc_fence_after();
                issue_pv(1, sv, h, h > 0 || j > 0);
              }
            }
            if (!pv_ok) break;
            umma_commit(bar_v_empty + 8 * sv);  // V_j consumed
            if (more) {
              issue_qk(1, sk);
              umma_commit(bar_s_full + 8);
              umma_commit(bar_k_empty + 8 * sk);  // K_{j+1} consumed
            } else {
              umma_commit(bar_o_final + 8);
            }
          }
        }
        if (ok && solo) {
          // Key tile j belongs to warpgroup j & 1, which owns S_i and O_i, i = j & 1. QK_0
          // and QK_1 go first, then PV_j and QK_{j + 2}.
          auto qk = [&](int j) -> bool {
            const int sl = j % MAXS;
            if (!mbar_wait(bar_k_full + 8 * sl, (j / MAXS) & 1, abort_flag, 135)) return false;
            tc_fence_after();
            issue_qk(j & 1, sl);
            umma_commit(bar_s_full + 8 * (j & 1));
            umma_commit(bar_k_empty + 8 * sl);  // K_j consumed
            return true;
          };
          bool go = qk(0) && (nk < 2 || qk(1));
          for (int j = 0; j < nk && go; ++j) {
            const int i = j & 1, sl = j % MAXS;
            go = mbar_wait(bar_v_full + 8 * sl, (j / MAXS) & 1, abort_flag, 133);
#pragma unroll
            for (int h = 0; h < Cfg::kPParts && go; ++h) {
              go = mbar_wait(bar_p_full + 8 * (Cfg::kPParts * i + h), (j >> 1) & 1, abort_flag, h ? 138 : 134);
              if (go) {
                tc_fence_after();
                issue_pv(i, sl, h, h > 0 || j > 1);
              }
            }
            if (!go) break;
            umma_commit(bar_v_empty + 8 * sl);  // V_j consumed
            if (j + 2 < nk)
              go = qk(j + 2);
            else
              umma_commit(bar_o_final + 8 * i);
          }
        }
        // Drain: every MMA issued above completes before TMEM is released.
        umma_commit(bar_mma_done);
        volatile int dummy = 0;
        mbar_wait(bar_mma_done, 0, &dummy, 137);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
    // ================================================================ softmax warpgroups
    const int wg = warp >> 2;  // query tile handled by this warpgroup
    const int row = tid & 127;  // packed row == TMEM lane
    const int wq = warp & 3;    // TMEM lane quarter of this warp
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + (wg ? Cfg::kColS1 : Cfg::kColS0);
    const uint32_t tO = tmem_base + lane_off + (wg ? Cfg::kColO1 : Cfg::kColO0);
    const uint32_t s_full = bar_s_full + 8 * wg;
    const uint32_t p_full = bar_p_full + 8 * Cfg::kPParts * wg;

    // This warpgroup's key tiles: all of them, or of a solo tile every other one.
    const int kstep = solo ? 2 * BN : BN;
    int key = work->key0 + (solo ? wg * BN : 0);  // first key of the step's tile
    const int n_steps = solo ? (work->nk + 1 - wg) >> 1 : work->nk;
    // The row's interval, counted from `key`: columns [low, rem) are visible. Idle rows
    // (past the tile's tokens, or of no head) count as seeing everything, so that they do
    // not put their warp on the masked path; whatever is in their rows of S and P reaches
    // their own rows of O alone, which are not stored.
    int low = INT_MIN / 2, rem = INT_MAX / 2;
    float dist = 0.f, slope = 0.f;  // position less that of column 0, with a distance bias
    const int m_row = row / p.group, i_row = (solo ? 0 : wg * bm) + m_row;
    const bool idle = m_row >= bm || i_row >= work->nq;
    if (!idle) {
      RaggedWork w;
      w.b = work->b;
      w.len = work->len;
      w.off = work->off_m0;
      w.m0 = 0;
      w.t0 = work->t0;
      int pos;
      ragged_row(p, w, i_row, pos, low, rem);
      if constexpr (MOD >= kRaggedBias) {
        slope = p.alibi[kvh * p.group + row % p.group] * 1.4426950408889634f;
        dist = (float)(pos - key);
      }
      low -= key;
      rem -= key;
    }
    const bool idle_warp = __all_sync(0xffffffffu, idle);  // only keeps the barriers going
    float m_run = -3.0e38f;
    float l_run = 0.f;
    bool ok = true;
    for (int n = 0; n < n_steps; ++n, key += kstep, rem -= kstep, low -= kstep) {
      ok = mbar_wait(s_full, n & 1, abort_flag, 140 + wg);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (key + BN > work->k_hi || key < work->k_lo) {
        // Keys of the tile that no row sees (past the last, or before the first in its
        // box) have P = 0, but their stale slots may hold NaN or Inf: each thread zeroes
        // its row of V, once V has landed and before P is published.
        const int j = (key - work->key0) / BN;
        ok = mbar_wait(bar_v_full + 8 * (j % slots), (j / slots) & 1, abort_flag, 144 + wg);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (key + row >= work->k_hi || key + row < work->k_lo) {
          const uint32_t vrow = v_ring + (j % slots) * Cfg::kTileBytes + row * 128;
#pragma unroll
          for (int c = 0; c < NSUB * 8; ++c)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vrow + (c >> 3) * Cfg::kSubBytes + (c & 7) * 16),
                         "r"(0u)
                         : "memory");
        }
        fence_proxy_async_smem();
      }
      if (idle_warp) {
#pragma unroll
        for (int h = 0; h < Cfg::kPParts; ++h) mbar_arrive(p_full + 8 * h);
        continue;
      }
      const bool cut_hi = __any_sync(0xffffffffu, rem < BN), cut_lo = __any_sync(0xffffffffu, low > 0);  // warp-uniform
      uint32_t sr[128];
      tmem_ld32(tS + 0, sr + 0);
      tmem_ld32(tS + 32, sr + 32);
      tmem_wait_ld();
      reg_fence_n<64>(sr);
      tmem_ld32(tS + 64, sr + 64);
      tmem_ld32(tS + 96, sr + 96);
      float mx;
      // With a bias: scores to log2 units in place, half a row at a time. Keys past the
      // token are only visible with a prefix (or without causal); otherwise the bias is
      // linear in the key, slope (c - distance of column 0).
      auto biased = [&](int c0) {
        const float d0 = dist - (float)(n * kstep);
        auto each = [&](auto score) {
#pragma unroll
          for (int c = c0; c < c0 + 64; ++c)
            sr[c] = __float_as_uint(fmaf(-slope, fabsf(d0 - (float)c), score(__uint_as_float(sr[c]))));
        };
        if constexpr (MOD == kRaggedCapBias) {
          float big = 0.f, big1 = 0.f;
#pragma unroll
          for (int c = c0; c < c0 + 64; c += 4) {
            big = max3_abs(big, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
            big1 = max3_abs(big1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
          }
          if (__all_sync(0xffffffffu, idle || fmaxf(big, big1) <= p.cap_most)) {  // the cap's polynomial holds
            const float2 a0 = make_float2(p.cap_a[0], p.cap_a[0]), a1 = make_float2(p.cap_a[1], p.cap_a[1]);
            const float2 a2 = make_float2(p.cap_a[2], p.cap_a[2]), a3 = make_float2(p.cap_a[3], p.cap_a[3]);
            auto pairs = [&](auto bias) {  // bias(c) of column c
#pragma unroll
              for (int c = c0; c < c0 + 64; c += 2) {
                const float2 s = make_float2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
                const float2 z = mul2(s, s);
                const float2 x = fma2(s, fma2(fma2(fma2(a3, z, a2), z, a1), z, a0), make_float2(bias(c), bias(c + 1)));
                sr[c] = __float_as_uint(x.x);
                sr[c + 1] = __float_as_uint(x.y);
              }
            };
            if (p.linear_bias) {
              const float b0 = -slope * d0;
              pairs([&](int c) { return fmaf(slope, (float)c, b0); });
            } else {
              pairs([&](int c) { return -slope * fabsf(d0 - (float)c); });
            }
          } else {
            each([&](float s) { return fmaf(-2.f * p.cap_out, fast_rcp(1.f + fast_exp2(s * p.cap_in)), p.cap_out); });
          }
        } else if (p.linear_bias) {
          const float b0 = -slope * d0;
#pragma unroll
          for (int c = c0; c < c0 + 64; ++c)
            sr[c] = __float_as_uint(fmaf(__uint_as_float(sr[c]), p.scale_log2, fmaf(slope, (float)c, b0)));
        } else {
          each([&](float s) { return s * p.scale_log2; });
        }
      };
      if constexpr (MOD >= kRaggedBias) biased(0);
      // With a cap and bf16 the largest magnitude, hidden scores' included, is all that a
      // tile needs: it says whether the polynomial holds, and its multiple by the
      // polynomial's slope at 0 bounds the row's scores and serves as their maximum. The
      // maximum itself is taken where the polynomial does not hold. (f16 has no exponents
      // for P that far below 1: maximum and magnitude both, 5 to 9 % slower.)
      constexpr bool kMagnitude = MOD == kRaggedCap && BF16;
      auto most = [&](float m, uint32_t a, uint32_t b) {
        if constexpr (kMagnitude) return max3_abs(m, __uint_as_float(a), __uint_as_float(b));
        else return max3(m, __uint_as_float(a), __uint_as_float(b));
      };
      float big = 0.f, big1 = 0.f;  // f16 with a cap: the largest magnitude, hidden scores' included
      auto magnitude = [&](int c0) {
#pragma unroll
        for (int c = c0; c < c0 + 64; c += 4) {
          big = max3_abs(big, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
          big1 = max3_abs(big1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
        }
      };
      auto mask = [&](int c0) {
        if (MOD == kRaggedCap && !kMagnitude && (cut_hi || cut_lo)) magnitude(c0);  // of other tiles later
        if (cut_hi) {
#pragma unroll
          for (int c = c0; c < c0 + 64; ++c) sr[c] = (c < rem) ? sr[c] : __float_as_uint(-INFINITY);
        }
        if (cut_lo) {
#pragma unroll
          for (int c = c0; c < c0 + 64; ++c) sr[c] = (c >= low) ? sr[c] : __float_as_uint(-INFINITY);
        }
      };
      if constexpr (!kMagnitude) mask(0);
      // Row max with three-input maxima, four independent chains.
      float mx0 = __uint_as_float(sr[0]), mx1 = __uint_as_float(sr[1]);
      float mx2 = __uint_as_float(sr[2]), mx3 = __uint_as_float(sr[3]);
#pragma unroll
      for (int c = 4; c < 60; c += 8) {
        mx0 = most(mx0, sr[c], sr[c + 1]);
        mx1 = most(mx1, sr[c + 2], sr[c + 3]);
        mx2 = most(mx2, sr[c + 4], sr[c + 5]);
        mx3 = most(mx3, sr[c + 6], sr[c + 7]);
      }
      mx0 = most(mx0, sr[60], sr[61]);
      mx1 = most(mx1, sr[62], sr[63]);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::"f"(mx0), "f"(mx1), "f"(mx2), "f"(mx3) : "memory");
      reg_fence_n<64>(sr + 64);
      if constexpr (MOD >= kRaggedBias) biased(64);
      if constexpr (!kMagnitude) mask(64);
#pragma unroll
      for (int c = 64; c < 128; c += 8) {
        mx0 = most(mx0, sr[c], sr[c + 1]);
        mx1 = most(mx1, sr[c + 2], sr[c + 3]);
        mx2 = most(mx2, sr[c + 4], sr[c + 5]);
        mx3 = most(mx3, sr[c + 6], sr[c + 7]);
      }
      mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
      bool small = false;  // kMagnitude: the polynomial holds for every score of the warp's rows
      if constexpr (kMagnitude) {
        small = __all_sync(0xffffffffu, idle || (mx <= p.cap_most && mx * p.cap_a[0] <= kBoundMost));
        mask(0);
        mask(64);
        if (small) {
          // |tanh y| <= |y|; hidden scores say nothing of a row that sees none of the tile.
          mx = max(low, 0) < min(rem, BN) ? mx * p.cap_a[0] : -INFINITY;
        } else {
          mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 128; c += 2) mx = max3(mx, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        }
      }
      if constexpr (MOD == kRaggedPlain) mx *= p.scale_log2;
      // A visible score may be -inf itself, and its cap is -cap: in the cap's MUFU form the
      // column says what is hidden, not the value.
      if (MOD == kRaggedCap && !small)
        mx = max(low, 0) >= min(rem, BN) ? -INFINITY : fmaf(-2.f * p.cap_out, fast_rcp(1.f + fast_exp2(mx * p.cap_in)), p.cap_out);
      const float m_new = fmaxf(m_run, mx);
      const bool need = !idle && m_new > m_run + 8.0f;
      if (n > 0 && __any_sync(0xffffffffu, need)) {
        const float alpha = need ? fast_exp2(m_run - m_new) : 1.0f;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t orr[32];
          tmem_ld32(tO + c * 32, orr);
          tmem_wait_ld();
          reg_fence(orr);
#pragma unroll
          for (int e = 0; e < 32; ++e) orr[e] = __float_as_uint(__uint_as_float(orr[e]) * alpha);
          tmem_st32(tO + c * 32, orr);
        }
        tmem_wait_st();
      }
      if (need) {
        l_run *= fast_exp2(m_run - m_new);
        m_run = m_new;
      }
      // P = exp2(x - m), written over S as packed 16-bit pairs in kPParts column parts.
      const float sc = MOD == kRaggedPlain ? p.scale_log2 : 1.0f;
      float2 sum2[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      constexpr int kPairs = 64 / Cfg::kPParts;
      auto publish = [&](auto shifted) {  // shifted(column, pair) = x - m of two neighbouring scores
#pragma unroll
        for (int h = 0; h < Cfg::kPParts; ++h) {
          uint32_t pk[kPairs];
#pragma unroll
          for (int c = 0; c < kPairs; ++c) {
            const int col = 2 * kPairs * h + 2 * c;
            const float2 x = shifted(col, make_float2(__uint_as_float(sr[col]), __uint_as_float(sr[col + 1])));
            const float2 pv = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sum2[c & 3] = add2(sum2[c & 3], pv);
            pk[c] = pack2<BF16>(pv.x, pv.y);
          }
          tmem_st32(tS + kPairs * h, pk);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(p_full + 8 * h);
        }
      };
      static_assert(kPairs == 32, "one 32-column store per part");
      const float2 nm2 = make_float2(-m_run, -m_run);
      if constexpr (MOD == kRaggedCap) {
        // The polynomial if every score of the warp's rows is small enough.
        const bool cut = cut_hi || cut_lo;
        if constexpr (!kMagnitude) {
          if (!cut) {
            magnitude(0);
            magnitude(64);
          }
          small = __all_sync(0xffffffffu, idle || fmaxf(big, big1) <= p.cap_most);
        }
        if (small) {
          const float2 a0 = make_float2(p.cap_a[0], p.cap_a[0]), a1 = make_float2(p.cap_a[1], p.cap_a[1]);
          const float2 a2 = make_float2(p.cap_a[2], p.cap_a[2]), a3 = make_float2(p.cap_a[3], p.cap_a[3]);
          auto capped = [&](float2 s) {
            const float2 z = mul2(s, s);
            return fma2(s, fma2(fma2(fma2(a3, z, a2), z, a1), z, a0), nm2);
          };
          if (!cut) {
            publish([&](int, float2 s) { return capped(s); });
          } else {
            publish([&](int, float2 s) {
              const float2 x = capped(s);
              return make_float2(s.x == -INFINITY ? s.x : x.x, s.y == -INFINITY ? s.y : x.y);
            });
          }
        } else {
          const float cin = p.cap_in, cout2 = -2.f * p.cap_out, off = p.cap_out - m_run;
          publish([&](int c, float2 s) {
            return make_float2(c < rem && c >= low ? fmaf(cout2, fast_rcp(1.f + fast_exp2(s.x * cin)), off) : -INFINITY,
                               c + 1 < rem && c + 1 >= low ? fmaf(cout2, fast_rcp(1.f + fast_exp2(s.y * cin)), off) : -INFINITY);
          });
        }
      } else {
        const float2 sc2 = make_float2(sc, sc);
        publish([&](int, float2 s) { return fma2(s, sc2, nm2); });
      }
      const float2 s01 = add2(sum2[0], sum2[1]);
      const float2 s23 = add2(sum2[2], sum2[3]);
      const float2 st = add2(s01, s23);
      l_run += st.x + st.y;
    }

    // ---- epilogue
    bool have_o = ok && n_steps > 0;
    if (have_o) {
      have_o = mbar_wait(bar_o_final + 8 * wg, 0, abort_flag, 142 + wg);
      have_o = __all_sync(0xffffffffu, have_o);
    }
    if (have_o) tc_fence_after();

    // What this thread writes of its row: all of it, or of a solo tile this warpgroup's
    // half of the columns, in chunks of 32.
    const int c_begin = solo ? wg * (HD / 64) : 0, c_end = solo ? c_begin + HD / 64 : HD / 32;
    const int prow = (solo ? 0 : wg * 128) + row;  // row of the tile's 256 packed rows
    float w_own = 1.f, w_other = 0.f;
    const float* other = nullptr;
    if (solo) {
      // The warpgroups' O, m and l of the same rows: each gives the other, through shared
      // memory ([warpgroup][column][row] floats, rows fastest, past the staging tile), the
      // half that the other writes. After the first barrier both are done with the ring.
      float* const xo = reinterpret_cast<float*>(smem + Cfg::kTileBytes);
      float* const xm = xo + HD * 128;
      asm volatile("bar.sync 3, 256;" ::: "memory");
      if (!idle_warp) {
        const int oc = (1 - wg) * (HD / 64);
        float* const to = xo + wg * (HD / 2) * 128 + row;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) {
          uint32_t orr[32];
          if (have_o) {
            tmem_ld32(tO + (oc + c) * 32, orr);
            tmem_wait_ld();
            reg_fence(orr);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) to[(c * 32 + e) * 128] = have_o ? __uint_as_float(orr[e]) : 0.f;
        }
        xm[wg * 256 + row] = m_run;
        xm[wg * 256 + 128 + row] = l_run;
      }
      asm volatile("bar.sync 3, 256;" ::: "memory");
      if (!idle_warp) {
        const float m1 = xm[(1 - wg) * 256 + row], l1 = xm[(1 - wg) * 256 + 128 + row];
        const float mx = fmaxf(m_run, m1);
        w_own = have_o ? fast_exp2(m_run - mx) : 0.f;
        w_other = fast_exp2(m1 - mx);
        // In the even tiles' warpgroup's order, so that both get the same sum.
        const float a = w_own * l_run, b = w_other * l1;
        l_run = wg ? b + a : a + b;
        m_run = mx;
        other = xo + (1 - wg) * (HD / 2) * 128 + row;
      }
    }

    const int n_chunks = work->n_chunks, unit = work->unit;
    float L = l_run, M = m_run;
    bool store = true;
    const uint32_t stage = q_smem0 + (solo ? 0 : wg) * Cfg::kTileBytes;
    auto stage_chunk = [&](int c, const uint32_t (&orr)[32], float inv) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int chunk = 4 * c + e;  // 16-byte chunk along d
#define GQA_OV(i) (__uint_as_float(orr[8 * e + (i)]) * inv)
        const uint32_t w0 = pack2<BF16>(GQA_OV(0), GQA_OV(1));
        const uint32_t w1 = pack2<BF16>(GQA_OV(2), GQA_OV(3));
        const uint32_t w2 = pack2<BF16>(GQA_OV(4), GQA_OV(5));
        const uint32_t w3 = pack2<BF16>(GQA_OV(6), GQA_OV(7));
#undef GQA_OV
        const uint32_t dst = stage + (chunk >> 3) * Cfg::kSubBytes + sw128_off(row, chunk & 7);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w0), "r"(w1), "r"(w2), "r"(w3)
                     : "memory");
      }
    };
    auto inverse = [](float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); };  // no key seen: 0; NaN stays NaN
    const int64_t pbase = (int64_t)unit * tl.nsplit * 256 + prow;
    if (!idle_warp) {
      // O of the chunk to the staging tile, or, if the tile has several chunks, its partial:
      // m, l [split][256 rows] and acc [split][d][256 rows].
      const float inv = inverse(l_run);
      float* acc_own = tl.ws_acc + ((int64_t)unit * tl.nsplit + split) * HD * 256 + prow;
#pragma unroll 1
      for (int c = c_begin; c < c_end; ++c) {
        uint32_t orr[32];
        if (have_o) {
          tmem_ld32(tO + c * 32, orr);
          tmem_wait_ld();
          reg_fence(orr);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) orr[e] = ok ? 0u : 0x7fc00000u;
        }
        if (solo) {
          const float* x = other + (c - c_begin) * 32 * 128;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            orr[e] = __float_as_uint(fmaf(w_other, x[e * 128], w_own * __uint_as_float(orr[e])));
        }
        if (n_chunks == 1) {
          stage_chunk(c, orr, inv);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) __stcg(acc_own + (c * 32 + e) * 256, __uint_as_float(orr[e]));
        }
      }
      if (n_chunks > 1 && c_begin == 0) {
        __stcg(tl.ws_m + pbase + (int64_t)split * 256, m_run);
        __stcg(tl.ws_l + pbase + (int64_t)split * 256, l_run);
      }
    }
    if (n_chunks > 1) {
      // The tile's last CTA (ticket) folds the chunks in their order.
      asm volatile("bar.sync 3, 256;" ::: "memory");
      uint32_t* last_slot = tmem_base_ptr + 2;
      if (tid == 0) {
        unsigned ticket;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(tl.ws_cnt + unit) : "memory");
        const bool last = ticket == (unsigned)(n_chunks - 1);
        *last_slot = last ? 1u : 0u;
        if (last) tl.ws_cnt[unit] = 0u;
      }
      asm volatile("bar.sync 3, 256;" ::: "memory");
      store = *last_slot != 0;
      if (store && !idle_warp) {
        // Every chunk's m and l at once (at most kMaxRaggedChunks), then their weights.
        float mv[kMaxRaggedChunks], lv[kMaxRaggedChunks];
#pragma unroll
        for (int i = 0; i < kMaxRaggedChunks; ++i) {
          const int64_t at = pbase + (int64_t)min(i, n_chunks - 1) * 256;
          mv[i] = __ldcg(tl.ws_m + at);
          lv[i] = __ldcg(tl.ws_l + at);
        }
#pragma unroll
        for (int i = 0; i < kMaxRaggedChunks; ++i) M = fmaxf(M, mv[i]);
        L = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxRaggedChunks; ++i)
          if (i < n_chunks) L += fast_exp2(mv[i] - M) * lv[i];
        const float inv = inverse(L);
#pragma unroll 1
        for (int c = c_begin; c < c_end; ++c) {
          // Four chunks per pass: 128 independent loads in flight per thread. An index past
          // the last chunk reads a valid partial at weight 0.
          uint32_t orr[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) orr[e] = 0u;
          for (int s0 = 0; s0 < n_chunks; s0 += 4) {
            float wt[4], x[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int si = min(s0 + i, n_chunks - 1);
              wt[i] = __ldcg(tl.ws_m + pbase + (int64_t)si * 256);
              const float* xi = tl.ws_acc + ((int64_t)unit * tl.nsplit + si) * HD * 256 + prow + c * 32 * 256;
#pragma unroll
              for (int e = 0; e < 32; ++e) x[i][e] = __ldcg(xi + e * 256);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              wt[i] = s0 + i < n_chunks ? fast_exp2(wt[i] - M) : 0.f;
#pragma unroll
              for (int e = 0; e < 32; ++e) orr[e] = __float_as_uint(fmaf(wt[i], x[i][e], __uint_as_float(orr[e])));
            }
          }
          stage_chunk(c, orr, inv);
        }
      }
    }
    // The staging tile is complete: one warpgroup's, or of a solo tile both's.
    if (solo)
      asm volatile("bar.sync 3, 256;" ::: "memory");
    else if (wg == 0)
      asm volatile("bar.sync 1, 128;" ::: "memory");
    else
      asm volatile("bar.sync 2, 128;" ::: "memory");
    if (store) {
      const int rows = max(0, min(work->nq - (solo ? 0 : wg * bm), bm)) * p.group;  // rows of real tokens
      const int tok0 = work->t0 + (solo ? 0 : wg * bm);
      if (p.lse && row < rows && c_begin == 0)
        p.lse[(int64_t)(tok0 + m_row) * p.hq + kvh * p.group + row % p.group] =
            L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
      // 16 bytes per thread, a row's pieces on neighbouring threads, `step` rows apart.
      constexpr int kPer = HD / 8;
      const int step = (solo ? 256 : 128) / kPer, chunk = tid % kPer;
      int r = (solo ? tid : row) / kPer;
      int tok = r / p.group, head = r - tok * p.group;
      const int d_tok = step / p.group, d_head = step - d_tok * p.group;
      uint16_t* const o0 = p.o + (int64_t)tok0 * p.o_st + (int64_t)kvh * p.group * p.o_sh + chunk * 8;
      const uint32_t s0 = stage + (chunk >> 3) * Cfg::kSubBytes;
      for (; r < rows; r += 4 * step) {
        uint4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (r + u * step < rows)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x[u].x), "=r"(x[u].y), "=r"(x[u].z), "=r"(x[u].w)
                         : "r"(s0 + sw128_off(r + u * step, chunk & 7))
                         : "memory");
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (r + u * step < rows) *reinterpret_cast<uint4*>(o0 + (int64_t)tok * p.o_st + (int64_t)head * p.o_sh) = x[u];
          tok += d_tok;
          head += d_head;
          if (head >= p.group) {
            head -= p.group;
            ++tok;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem_base, Cfg::kTmemCols);
}

}  // namespace gqa
