// Attention of a ragged step over the paged cache: request b's new tokens are rows
// cu[b] .. cu[b + 1] - 1 of the packed queries and the last of its seq_lens[b] cached
// positions. Row i of request b, at position p, sees an interval of its keys,
//
//   [lo, hi):  hi = min(len_b, max(p + 1, prefix_b))    (all of len_b without causal)
//              lo = max(0, p - window + 1, key_starts[token])
//
// which covers causal, prefix, window and document masks and their mixtures; a row whose
// interval is empty gives 0 (and log-sum-exp -inf). Keys that no row of a tile sees may hold
// anything; a NaN or infinite value of a key that some row sees may reach the tile's other
// rows too, as 0 x NaN. Scores, in log2 units:
//
//   x = s * scale * log2 e                                    or, capped,
//   x = cap * log2 e * tanh(s * scale / cap),  tanh y = 1 - 2 / (1 + 2^(2 y log2 e))
//   x -= slope_head * log2 e * |p - key|                      with a distance bias
//
// This file has the mask and score arithmetic and the streaming kernel, which takes tiles
// of few packed rows (tokens x the group's heads, token-major): up to kRaggedStreamRows of
// a 16-bit cache, up to 64 of an fp8 one, which has no other form. Like the dense
// streaming kernel it is bound by the keys' and values' bytes: one CTA streams one chunk
// of one (tile, kv head)'s keys through a 192 KB TMA ring, and the last CTA of a tile
// combines the chunks' partials. The key range of a tile is the union of its rows'
// intervals, so keys before a window or a document are not read at all. 48 requests of
// one token, 32 query and 8 kv heads of 128, up to 16384 bf16 keys (2.13 GB): 314 to 319
// us, 6.7 TB/s, where a plain copy, which writes as well, moves 6.5. The same over e4m3
// caches (1.06 GB): 213 us, 5.0 TB/s. A single short request is bound by latency: about
// 4 us for the launch, the lengths, the first loads and the join, then 0.7 us per 128
// keys of a chunk.
//
// Everything that depends on a length is read on the device: the host knows bounds only
// (tokens, the longest request's rows and keys), which size the grid; CTAs past the real
// work return at once.
#pragma once

#include <climits>

#include "gqa_common.cuh"
#include "gqa_stream.cuh"

namespace gqa {

// Requests of up to this many packed rows stream, longer ones take the tcgen05 form
// (16-bit caches). Measured with 8 kv heads of 128, bf16, causal, in us:
//                            32 rows               36 rows               64 rows
//   requests x keys     streamed  tcgen05     streamed  tcgen05     streamed  tcgen05
//    1 x 2048              14        20          20        20          27        20
//    4 x 8192              34        43          54        43          58        47
//   16 x 2048              27        36          48        36          49        36
//   48 x 2048              82        89         138        90         142        93
// Up to 32 rows the streaming CTA keeps the pace of its loads and starts sooner; four row
// groups of 16 need more than their registers. (Up to 512 keys streaming stays ahead to
// 64 rows, by 3 us at most; lengths are on the device, so the rule is on rows alone.)
constexpr int kRaggedStreamRows = 32;

// How one of the two forms cuts the step into tiles of block_m tokens of one request.
struct RaggedTiling {
  int block_m, rows;      // rows = packed rows of a tile at most (its partials' stride)
  int one_tile, slots;    // streaming form: every request has at most one tile, and slot b is
                          // request b's; otherwise slots are found by ragged_slot
  int min_rows, max_rows;  // packed rows of the requests that the form takes
  int nsplit, chunk;      // key chunks of a tile at most; keys per chunk (a multiple of 128)
  float* ws_m;            // partials [unit][nsplit][rows], unit = tile x kv head
  float* ws_l;
  float* ws_acc;
  unsigned* ws_cnt;       // tickets [unit], zero between calls
};

struct RaggedParams {
  const uint16_t* q;
  uint16_t* o;
  float* lse;             // (T, hq) natural log, or null
  int64_t q_st, q_sh;     // element strides (token, head)
  int64_t o_st, o_sh;
  const int* cu;          // (n + 1,)
  const int* seq_lens;    // (n,)
  const int* block_table;
  int bt_stride, block_shift, num_blocks;
  int box;                // keys per TMA box = min(64, block size)
  const float* alibi;     // (hq,) or null
  const int* prefix;      // (n,) or null
  const int* key_starts;  // (T,) or null
  int window;             // keys a row looks back over, itself included; 0: all
  int causal;
  int n, num_tokens, hq, hkv, group;
  int max_len;            // bound of seq_lens (longer ones are clipped to it)
  float scale_log2;       // scale * log2 e
  float cap_in, cap_out;  // 2 log2 e * scale / cap, cap * log2 e; cap_in 0: no cap
  float cap_a[4];         // the cap as s (a0 + a1 s^2 + a2 s^4 + a3 s^6), for |s| <= cap_most
  float cap_most;
  float v_scale;          // e4m3 values
  int mods;               // cap or bias present
  int linear_bias;        // no key past a token is visible to it
  RaggedTiling stream, tile;
  unsigned tile_ctas;     // CTAs of the tcgen05 form, the grid's first; the rest stream
};

// Request b's tiles take the slots cu[b] / block_m + b, +1, ...: it has at most
// cu[b + 1] / block_m - cu[b] / block_m + 1 of them, so the ranges do not overlap, and
// the last request whose first slot is not above `slot` is its owner, if any. A warp
// bisects 32 ways. Returns the request, or -1.
__device__ __forceinline__ int ragged_slot(const RaggedParams& p, const RaggedTiling& tl, int slot, int lane) {
  int lo = 0, n = p.n;  // the owner is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int i = lo + lane * step;
    const bool below = lane * step < n && p.cu[i] / tl.block_m + i <= slot;
    const unsigned m = __ballot_sync(0xffffffffu, below);
    if (m == 0) return -1;
    const int at = 31 - __clz(m);
    n = min(step, n - at * step);
    lo += at * step;
  }
  return lo;
}

// What one CTA works on, the same in every warp.
struct RaggedWork {
  int b, m0, t0, nq;       // request, first token of the tile in it, that token's row, tokens in the tile
  int len, off;            // the request's keys; position of its token i = off + i
  int k_lo, k_hi;          // union of the rows' key intervals (k_lo >= k_hi: none)
  int k_base, n_chunks;    // k_lo down to a box, chunks that hold keys (at least 1)
};

// The tile of request b that starts at its token m0: the union over its rows, by one warp.
// False: no such tile, or not this kernel's.
__device__ __forceinline__ bool ragged_work_at(const RaggedParams& p, const RaggedTiling& tl, int b, int m0, int lane,
                                               RaggedWork& w) {
  w.b = b;
  w.m0 = m0;
  const int first = p.cu[b], end = p.cu[b + 1];
  const int qn = min(end, p.num_tokens) - first;  // the rows that there are
  if (first < 0 || m0 < 0 || m0 >= qn) return false;
  const int64_t qrows = (int64_t)qn * p.group;
  if (qrows < tl.min_rows || qrows > tl.max_rows) return false;
  w.t0 = first + w.m0;
  w.nq = min(tl.block_m, qn - w.m0);
  const int len = max(0, p.seq_lens[w.b]);
  if (lane == 0) {  // bounds that do not hold
    if (tl.one_tile && qn > tl.block_m) report_device_error(GQA_ERR_INVALID_ARG, 214);  // rows past the tile stay unwritten
    if (len > p.max_len) report_device_error(GQA_ERR_INVALID_ARG, 215);
  }
  w.len = min(len, p.max_len);
  // Positions go by the request's own numbers: a step cut to fewer rows, or keys past the
  // bound, leave the other tokens where they are.
  w.off = len - (end - first);
  const int p_first = w.off + w.m0, p_last = p_first + w.nq - 1;
  w.k_hi = w.len;
  if (p.causal) {
    w.k_hi = p_last + 1;
    if (p.prefix) w.k_hi = max(w.k_hi, p.prefix[w.b]);
    w.k_hi = max(0, min(w.k_hi, w.len));
  }
  w.k_lo = p.window > 0 ? max(0, p_first - p.window + 1) : 0;
  if (p.key_starts) {
    int s = INT_MAX;
    for (int i = lane; i < w.nq; i += 32) s = min(s, p.key_starts[w.t0 + i]);
    w.k_lo = max(w.k_lo, __reduce_min_sync(0xffffffffu, s));
  }
  w.k_base = min(w.k_lo, w.k_hi) & ~(p.box - 1);
  w.n_chunks = w.k_hi > w.k_lo ? (w.k_hi - w.k_base + tl.chunk - 1) / tl.chunk : 1;
  return true;
}
__device__ __forceinline__ bool ragged_work(const RaggedParams& p, const RaggedTiling& tl, int slot, int lane,
                                            RaggedWork& w) {
  const int b = tl.one_tile ? slot : ragged_slot(p, tl, slot, lane);
  if (b < 0) return false;
  return ragged_work_at(p, tl, b, tl.one_tile ? 0 : (slot - (p.cu[b] / tl.block_m + b)) * tl.block_m, lane, w);
}

// The interval of the row of token t0 + i.
__device__ __forceinline__ void ragged_row(const RaggedParams& p, const RaggedWork& w, int i, int& pos, int& lo, int& hi) {
  pos = w.off + w.m0 + i;
  hi = w.len;
  if (p.causal) {
    hi = pos + 1;
    if (p.prefix) hi = max(hi, p.prefix[w.b]);
    hi = min(hi, w.len);
  }
  lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  if (p.key_starts) lo = max(lo, p.key_starts[w.t0 + i]);
}

__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Score in log2 units. 2 MUFU operations for the cap; exact at both ends (2^inf -> tanh 1,
// so a score of -inf is -cap).
struct RaggedScore {  // in registers: the parameters are not in constant memory of a function
  float scale, cap_in, cap_out;
  int mods;
};
__device__ __forceinline__ float ragged_score(const RaggedScore& sc, float s, float slope, int pos, int key) {
  float x = s * sc.scale;
  if (sc.cap_in != 0.f) x = fmaf(-2.f * sc.cap_out, fast_rcp(1.f + fast_exp2(s * sc.cap_in)), sc.cap_out);
  return fmaf(-slope, fabsf((float)(pos - key)), x);
}

#define GQA_CBAR() asm volatile("bar.sync 1, %0;" ::"n"(CT) : "memory")  // the compute warps

// The compute warps of one streaming CTA, for tiles of up to 16 RG packed rows. Template
// parameters as gqa_stream_kernel's: FP8 = e4m3 caches (HD 128, both MMAs in f16, to which
// bf16 queries are rounded: exact from 2^-14 to 65504, infinite above), NT = at
// most 8 rows, MMAs transposed. The scores and the accumulators are fp32; P is rounded to
// the values' 16-bit type for its MMA, as the dense kernels round it (relative error
// 2^-9, as large as the output's own rounding).
template <int HD, bool BF16, int RG, bool FP8, bool NT>
__device__ __forceinline__ void ragged_stream_compute(const RaggedParams& p, const RaggedWork& w, uint8_t* smem, uint32_t base,
                                                      int k_begin, int k_end, int n_stages, int unit, int split, int kvh) {
  static_assert(!FP8 || HD == 128, "fp8 K/V rows are 128 bytes");
  static_assert(!NT || RG == 1, "the transposed form is the one-row-group kernel");
  using Cfg = StreamCfg<FP8 ? 64 : HD>;
  constexpr bool MMA_BF16 = BF16 && !FP8;
  constexpr int NW = Cfg::kWarps;
  constexpr int KS = NW / RG;
  constexpr int NKW = Cfg::kBN / KS;
  constexpr int NNB = NKW / 8;
  constexpr int NDB = HD / 8;
  constexpr int NKS = HD / 16;
  constexpr int CT = NW * 32;
  constexpr int NACC = NT ? HD / 16 : NDB;
  const uint32_t bar_full = base + Cfg::kRingBytes;
  const uint32_t bar_empty = bar_full + Cfg::kStages * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kRingBytes + Cfg::kBarBytes);
  int* last_flag = reinterpret_cast<int*>(smem + Cfg::kRingBytes + Cfg::kBarBytes + 4);
  const RaggedTiling& tl = p.stream;
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int rg = warp % RG;
  const int ks = warp / RG;
  const int gr = lane >> 2;
  const int gc = lane & 3;
  const int n_valid = w.nq * p.group;  // packed rows of the tile: row r = token r / group, head r % group

  // Packed rows of this thread: rg*16 + gr and + 8 (NT: the softmax rows 2gc, 2gc + 1,
  // and Q row gr for the B fragments).
  int lo_r[2], hi_r[2], pos_r[2];
  float slope_r[2];
  const uint16_t* qrow[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int rl = NT ? 2 * gc + h : rg * 16 + gr + 8 * h;
    const int i = min(rl, n_valid - 1) / p.group;
    ragged_row(p, w, i, pos_r[h], lo_r[h], hi_r[h]);
    hi_r[h] = min(hi_r[h], k_end);
    slope_r[h] = p.alibi ? p.alibi[kvh * p.group + min(rl, n_valid - 1) % p.group] * 1.4426950408889634f : 0.f;
    const int rq = NT ? gr : rl;
    const bool valid = rq < n_valid && (!NT || h == 0);
    const int rc = min(rq, n_valid - 1);
    qrow[h] = valid ? p.q + (int64_t)(w.t0 + rc / p.group) * p.q_st + (int64_t)(kvh * p.group + rc % p.group) * p.q_sh
                    : nullptr;
  }

  // Q fragments (see gqa_stream_kernel for the three fragment orders).
  uint32_t qa[NKS][4];
#pragma unroll
  for (int kk = 0; kk < NKS; ++kk) {
    if constexpr (FP8) {
      const int d0 = kk * 16 + gc * 4;
      const uint2 z = make_uint2(0u, 0u);
      const uint2 q0 = qrow[0] ? *reinterpret_cast<const uint2*>(qrow[0] + d0) : z;
      const uint2 q1 = (!NT && qrow[1]) ? *reinterpret_cast<const uint2*>(qrow[1] + d0) : z;
      qa[kk][0] = to_f16x2<BF16>(q0.x);
      qa[kk][NT ? 1 : 2] = to_f16x2<BF16>(q0.y);
      qa[kk][NT ? 2 : 1] = to_f16x2<BF16>(q1.x);
      qa[kk][3] = to_f16x2<BF16>(q1.y);
    } else {
      const int d0 = kk * 16 + gc * 2;
      const uint32_t a0 = qrow[0] ? *reinterpret_cast<const uint32_t*>(qrow[0] + d0) : 0u;
      const uint32_t a1 = qrow[0] ? *reinterpret_cast<const uint32_t*>(qrow[0] + d0 + 8) : 0u;
      const uint32_t b0 = (!NT && qrow[1]) ? *reinterpret_cast<const uint32_t*>(qrow[1] + d0) : 0u;
      const uint32_t b1 = (!NT && qrow[1]) ? *reinterpret_cast<const uint32_t*>(qrow[1] + d0 + 8) : 0u;
      qa[kk][0] = a0;
      qa[kk][1] = NT ? a1 : b0;
      qa[kk][2] = NT ? b0 : a1;
      qa[kk][3] = b1;
    }
  }

  float acc[NACC][4];
#pragma unroll
  for (int i = 0; i < NACC; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY};
  float l_run[2] = {0.f, 0.f};
  const RaggedScore sc{p.scale_log2, p.cap_in, p.cap_out, p.mods};

  for (int t = 0; t < n_stages; ++t) {
    const int slot = t % Cfg::kStages;
    bool ok = mbar_wait(bar_full + 8 * slot, (t / Cfg::kStages) & 1, abort_flag, 113);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    const uint32_t kst = base + slot * Cfg::kStageBytes;
    const uint32_t vst = kst + Cfg::kTileBytes;
    const int key_w = k_begin + t * Cfg::kBN + ks * NKW;  // first key of this warp's block
    const bool work = key_w < k_end && key_w + NKW > w.k_lo;  // warp-uniform
    if (work && (key_w + NKW > k_end || key_w < w.k_lo)) {
      // Keys that no row of the tile sees -- past the end, or before the first interval in
      // the first box -- have P = 0, but their cache slots may hold stale NaN or Inf and
      // 0 x NaN would reach O through the MMA: this warp, their only reader, zeroes their
      // V rows. The fence orders the stores before the copy that refills the slot.
      constexpr int kRowChunks = Cfg::kNSub * 8;
      for (int i = lane; i < NKW * kRowChunks; i += 32) {
        const int r = i / kRowChunks, c = i % kRowChunks, key = key_w + r;
        if (key >= w.k_lo && key < k_end) continue;
        const uint32_t addr = vst + (c >> 3) * Cfg::kSubBytes + (ks * NKW + r) * 128 + (c & 7) * 16;
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0u) : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
    }
    if (work) {
      if constexpr (NT) {
        // ---- S^T = K Q^T: 16 keys (M) x 8 rows (N)
        float st[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        const int krow = ks * NKW + (lane & 7) + ((lane >> 3) & 1) * 8;
        if constexpr (FP8) {
#pragma unroll
          for (int c = 0; c < HD / 16; c += 2) {
            uint32_t r[4];
            ldsm_x4(kst + sw128_off(krow, c + (lane >> 4)), r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a[4] = {e4m3x2_to_f16x2(r[2 * h]), e4m3x2_to_f16x2(r[2 * h + 1]),
                                     e4m3x2_to_f16x2(r[2 * h] >> 16), e4m3x2_to_f16x2(r[2 * h + 1] >> 16)};
              mma_16816<false>(st[h], a, qa[c + h][0], qa[c + h][1]);
            }
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < NKS; ++kk) {
            const int chunk = 2 * kk + (lane >> 4);
            uint32_t a[4];
            ldsm_x4(kst + (chunk >> 3) * Cfg::kSubBytes + sw128_off(krow, chunk & 7), a[0], a[1], a[2], a[3]);
            mma_16816<MMA_BF16>(st[kk & 1], a, qa[kk][0], qa[kk][1]);
          }
        }
        // s[e]: key gr + 8 (e >> 1), row 2gc + (e & 1)
        float s[4], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key_w + gr + 8 * (e >> 1), h = e & 1;
          const float raw = st[0][e] + st[1][e];
          const float x = sc.mods ? ragged_score(sc, raw, slope_r[h], pos_r[h], key) : raw * sc.scale;
          s[e] = (key >= lo_r[h] && key < hi_r[h]) ? x : -INFINITY;
          mx[h] = fmaxf(mx[h], s[e]);
        }
        float alpha[2], mu[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 4));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 8));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 16));
          const float m_new = fmaxf(m_run[h], mx[h]);
          mu[h] = (m_new == -INFINITY) ? 0.f : m_new;
          alpha[h] = fast_exp2(m_run[h] - mu[h]);
          m_run[h] = m_new;
        }
        float lsum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[e] = fast_exp2(s[e] - mu[e & 1]);
          lsum[e & 1] += s[e];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) l_run[h] = l_run[h] * alpha[h] + lsum[h];
#pragma unroll
        for (int c = 0; c < NACC; ++c) {
          acc[c][0] *= alpha[0];
          acc[c][1] *= alpha[1];
          acc[c][2] *= alpha[0];
          acc[c][3] *= alpha[1];
        }
        // ---- O^T += V^T P^T
        const uint32_t pb0 = movmatrix_t(pack2<MMA_BF16>(s[0], s[1]));
        const uint32_t pb1 = movmatrix_t(pack2<MMA_BF16>(s[2], s[3]));
        if constexpr (FP8) {
#pragma unroll
          for (int c = 0; c < HD / 16; c += 2) {
            uint32_t r[4];
            ldsm_x4_t(vst + sw128_off(krow, c + (lane >> 4)), r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t lo = prmt(r[2 * h], 0u, 0x3120u);
              const uint32_t hi = prmt(r[2 * h + 1], 0u, 0x3120u);
              const uint32_t a[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi),
                                     e4m3x2_to_f16x2(hi >> 16)};
              mma_16816<false>(acc[c + h], a, pb0, pb1);
            }
          }
        } else {
          const int vrow = ks * NKW + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
          for (int c = 0; c < NACC; ++c) {
            const int chunk = 2 * c + ((lane >> 3) & 1);
            uint32_t a[4];
            ldsm_x4_t(vst + (chunk >> 3) * Cfg::kSubBytes + sw128_off(vrow, chunk & 7), a[0], a[1], a[2], a[3]);
            mma_16816<MMA_BF16>(acc[c], a, pb0, pb1);
          }
        }
      } else {
        // ---- S = Q K^T over this warp's NKW keys
        float s[NNB][4];
#pragma unroll
        for (int nb = 0; nb < NNB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
        if constexpr (FP8) {
#pragma unroll
          for (int kc = 0; kc < HD / 64; ++kc) {
#pragma unroll
            for (int nb = 0; nb < NNB; ++nb) {
              const int krow = ks * NKW + nb * 8 + (lane & 7);
              const int chunk = kc * 4 + (lane >> 3);
              uint32_t r[4];
              ldsm_x4(kst + sw128_off(krow, chunk), r[0], r[1], r[2], r[3]);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                mma_16816<false>(s[nb], qa[4 * kc + j], e4m3x2_to_f16x2(r[j]), e4m3x2_to_f16x2(r[j] >> 16));
            }
          }
        } else {
#pragma unroll
          for (int kc = 0; kc < HD / 32; ++kc) {
#pragma unroll
            for (int nb = 0; nb < NNB; ++nb) {
              const int krow = ks * NKW + nb * 8 + (lane & 7);
              const int chunk = kc * 4 + (lane >> 3);
              const uint32_t addr = kst + (chunk >> 3) * Cfg::kSubBytes + sw128_off(krow, chunk & 7);
              uint32_t b0, b1, b2, b3;
              ldsm_x4(addr, b0, b1, b2, b3);
              mma_16816<BF16>(s[nb], qa[2 * kc], b0, b1);
              mma_16816<BF16>(s[nb], qa[2 * kc + 1], b2, b3);
            }
          }
        }
        // ---- online softmax (log2 domain)
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nb = 0; nb < NNB; ++nb) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1;
            const int key = key_w + nb * 8 + gc * 2 + (e & 1);
            const float x = sc.mods ? ragged_score(sc, s[nb][e], slope_r[h], pos_r[h], key) : s[nb][e] * sc.scale;
            s[nb][e] = (key >= lo_r[h] && key < hi_r[h]) ? x : -INFINITY;
            mx[h] = fmaxf(mx[h], s[nb][e]);
          }
        }
        float alpha[2], mu[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
          const float m_new = fmaxf(m_run[h], mx[h]);
          mu[h] = (m_new == -INFINITY) ? 0.f : m_new;
          alpha[h] = fast_exp2(m_run[h] - mu[h]);
          m_run[h] = m_new;
        }
        float lsum[2] = {0.f, 0.f};
#pragma unroll
        for (int nb = 0; nb < NNB; ++nb) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pv = fast_exp2(s[nb][e] - mu[e >> 1]);
            s[nb][e] = pv;
            lsum[e >> 1] += pv;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) l_run[h] = l_run[h] * alpha[h] + lsum[h];
#pragma unroll
        for (int i = 0; i < NDB; ++i) {
          acc[i][0] *= alpha[0];
          acc[i][1] *= alpha[0];
          acc[i][2] *= alpha[1];
          acc[i][3] *= alpha[1];
        }
        // ---- O += P V
#pragma unroll
        for (int kk = 0; kk < NKW / 16; ++kk) {
          uint32_t pa[4];
          pa[0] = pack2<MMA_BF16>(s[2 * kk][0], s[2 * kk][1]);
          pa[1] = pack2<MMA_BF16>(s[2 * kk][2], s[2 * kk][3]);
          pa[2] = pack2<MMA_BF16>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
          pa[3] = pack2<MMA_BF16>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
          const int vrow = ks * NKW + kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
          if constexpr (FP8) {
#pragma unroll
            for (int c = 0; c < HD / 16; c += 2) {
              const int chunk = c + (lane >> 4);
              uint32_t r[4];
              ldsm_x4_t(vst + sw128_off(vrow, chunk), r[0], r[1], r[2], r[3]);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t lo = prmt(r[2 * h], 0u, 0x3120u);
                const uint32_t hi = prmt(r[2 * h + 1], 0u, 0x3120u);
                mma_16816<false>(acc[2 * (c + h)], pa, e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(hi));
                mma_16816<false>(acc[2 * (c + h) + 1], pa, e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi >> 16));
              }
            }
          } else {
#pragma unroll
            for (int dc = 0; dc < NDB; dc += 2) {
              const int chunk = dc + (lane >> 4);
              const uint32_t addr = vst + (chunk >> 3) * Cfg::kSubBytes + sw128_off(vrow, chunk & 7);
              uint32_t b0, b1, b2, b3;
              ldsm_x4_t(addr, b0, b1, b2, b3);
              mma_16816<BF16>(acc[dc], pa, b0, b1);
              mma_16816<BF16>(acc[dc + 1], pa, b2, b3);
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_empty + 8 * slot);
  }

  // Row sums are per-thread partials over the quad's columns (NT: over the lanes of one gc).
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (NT) {
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 4);
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 8);
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 16);
    } else {
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
    }
  }

  // ---- merge the KS warps of each row group through shared memory (paddings: see gqa_stream_kernel)
  GQA_CBAR();
  constexpr int AS = NT ? HD + 4 : HD + 8;
  float* mbuf = reinterpret_cast<float*>(smem);  // [NW][16]
  float* lbuf = mbuf + NW * 16;                  // [NW][16]
  float* abuf = lbuf + NW * 16;                  // [NW][16][AS]
  static_assert((2 * NW * 16 + NW * 16 * AS) * 4 <= Cfg::kRingBytes, "merge buffers fit the ring");
  {
    float* aw = abuf + warp * 16 * AS;
    const bool upper = rg * 16 + 8 < n_valid;  // warp-uniform
    if constexpr (NT && FP8) {
      const float vs = p.v_scale;
#pragma unroll
      for (int c = 0; c < NACC; ++c) {
        const int d = c * 16 + gr * 2;
        *reinterpret_cast<float2*>(aw + (2 * gc) * AS + d) = make_float2(acc[c][0] * vs, acc[c][2] * vs);
        *reinterpret_cast<float2*>(aw + (2 * gc + 1) * AS + d) = make_float2(acc[c][1] * vs, acc[c][3] * vs);
      }
    } else if constexpr (NT) {
#pragma unroll
      for (int c = 0; c < NACC; ++c) {
        const int d = c * 16 + gr;
        aw[(2 * gc) * AS + d] = acc[c][0];
        aw[(2 * gc + 1) * AS + d] = acc[c][1];
        aw[(2 * gc) * AS + d + 8] = acc[c][2];
        aw[(2 * gc + 1) * AS + d + 8] = acc[c][3];
      }
    } else if constexpr (FP8) {
      const float vs = p.v_scale;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        const int d = c * 16 + gc * 4;
        const float* e = acc[2 * c];
        const float* o = acc[2 * c + 1];
        *reinterpret_cast<float4*>(aw + gr * AS + d) = make_float4(e[0] * vs, o[0] * vs, e[1] * vs, o[1] * vs);
        if (upper)
          *reinterpret_cast<float4*>(aw + (gr + 8) * AS + d) =
              make_float4(e[2] * vs, o[2] * vs, e[3] * vs, o[3] * vs);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        const int d = i * 8 + gc * 2;
        *reinterpret_cast<float2*>(aw + gr * AS + d) = make_float2(acc[i][0], acc[i][1]);
        if (upper) *reinterpret_cast<float2*>(aw + (gr + 8) * AS + d) = make_float2(acc[i][2], acc[i][3]);
      }
    }
    if constexpr (NT) {
      if (gr == 0) {
        mbuf[warp * 16 + 2 * gc] = m_run[0];
        mbuf[warp * 16 + 2 * gc + 1] = m_run[1];
        lbuf[warp * 16 + 2 * gc] = l_run[0];
        lbuf[warp * 16 + 2 * gc + 1] = l_run[1];
      }
    } else if (gc == 0) {
      mbuf[warp * 16 + gr] = m_run[0];
      mbuf[warp * 16 + gr + 8] = m_run[1];
      lbuf[warp * 16 + gr] = l_run[0];
      lbuf[warp * 16 + gr + 8] = l_run[1];
    }
  }
  GQA_CBAR();

  struct RowMerge {
    float M, L;
    float4 a;
  };
  auto merge_row = [&](int r, int d) {
    const int g_rg = r / 16, rr = r % 16;
    float mk[KS];
    float M = -INFINITY;
#pragma unroll
    for (int k2 = 0; k2 < KS; ++k2) {
      mk[k2] = mbuf[(k2 * RG + g_rg) * 16 + rr];
      M = fmaxf(M, mk[k2]);
    }
    const float Mu = (M == -INFINITY) ? 0.f : M;
    RowMerge out{M, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
    for (int k2 = 0; k2 < KS; ++k2) {
      const int wp = k2 * RG + g_rg;
      const float wt = fast_exp2(mk[k2] - Mu);
      out.L += wt * lbuf[wp * 16 + rr];
      const float4 v = *reinterpret_cast<const float4*>(abuf + (wp * 16 + rr) * AS + d);
      out.a.x += wt * v.x;
      out.a.y += wt * v.y;
      out.a.z += wt * v.z;
      out.a.w += wt * v.w;
    }
    return out;
  };
  // O and the log-sum-exp of packed row r; a row that saw no key (L = 0) gives 0 and -inf.
  auto store_row = [&](int r, int d, float M, float L, float4 a) {
    const int tok = w.t0 + r / p.group, head = kvh * p.group + r % p.group;
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // a NaN sum stays NaN
    uint2 pk;
    pk.x = pack2<BF16>(a.x * inv, a.y * inv);
    pk.y = pack2<BF16>(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2*>(p.o + (int64_t)tok * p.o_st + (int64_t)head * p.o_sh + d) = pk;
    if (p.lse && d == 0)
      p.lse[(int64_t)tok * p.hq + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  };

  constexpr int per_row = HD / 4;
  if (w.n_chunks == 1) {
    for (int idx = tid; idx < n_valid * per_row; idx += CT) {
      const int r = idx / per_row, d = (idx - r * per_row) * 4;
      const RowMerge mr = merge_row(r, d);
      store_row(r, d, mr.M, mr.L, mr.a);
    }
    return;
  }

  // ---- publish this chunk's partial; the tile's last CTA combines them in chunk order.
  const int64_t ubase = (int64_t)unit * tl.nsplit * tl.rows;
  const int64_t wbase = ubase + (int64_t)split * tl.rows;
  for (int idx = tid; idx < n_valid * per_row; idx += CT) {
    const int r = idx / per_row, d = (idx - r * per_row) * 4;
    const RowMerge mr = merge_row(r, d);
    __stcg(reinterpret_cast<float4*>(tl.ws_acc + (wbase + r) * HD + d), mr.a);
    if (d == 0) {
      __stcg(tl.ws_m + wbase + r, mr.M);
      __stcg(tl.ws_l + wbase + r, mr.L);
    }
  }
  GQA_CBAR();
  if (tid == 0) {
    unsigned ticket;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(tl.ws_cnt + unit) : "memory");
    *last_flag = (ticket == (unsigned)(w.n_chunks - 1)) ? 1 : 0;
    if (*last_flag) tl.ws_cnt[unit] = 0u;
  }
  GQA_CBAR();
  if (!*last_flag) return;
  const int nc = w.n_chunks;
  float* sm_m = reinterpret_cast<float*>(smem);
  float* sm_l = sm_m + nc * n_valid;
  for (int i = tid; i < nc * n_valid; i += CT) {
    const int s2 = i / n_valid, r = i - s2 * n_valid;
    sm_m[i] = __ldcg(tl.ws_m + ubase + (int64_t)s2 * tl.rows + r);
    sm_l[i] = __ldcg(tl.ws_l + ubase + (int64_t)s2 * tl.rows + r);
  }
  GQA_CBAR();
  for (int idx = tid; idx < n_valid * per_row; idx += CT) {
    const int r = idx / per_row, d = (idx - r * per_row) * 4;
    float M = -INFINITY;
    for (int s2 = 0; s2 < nc; ++s2) M = fmaxf(M, sm_m[s2 * n_valid + r]);
    const float Mu = (M == -INFINITY) ? 0.f : M;
    float L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kBatch = 8;  // loads in flight before the first FMA
    for (int s0 = 0; s0 < nc; s0 += kBatch) {
      float4 v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        v[u] = __ldcg(reinterpret_cast<const float4*>(tl.ws_acc + (ubase + (int64_t)min(s0 + u, nc - 1) * tl.rows + r) * HD + d));
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (s0 + u < nc) {
          const float wt = fast_exp2(sm_m[(s0 + u) * n_valid + r] - Mu);
          L += wt * sm_l[(s0 + u) * n_valid + r];
          a.x += wt * v[u].x;
          a.y += wt * v[u].y;
          a.z += wt * v[u].z;
          a.w += wt * v[u].w;
        }
      }
    }
    store_row(r, d, M, L, a);
  }
}

#undef GQA_CBAR

// One CTA of the streaming form: at least 288 threads, warps 0-7 compute, warp 8 loads,
// any others only keep the barrier company. The tile's rows pick the compute form.
template <int HD, bool BF16, bool FP8>
__device__ __forceinline__ void ragged_stream_cta(const RaggedParams& p, const CUtensorMap* kmap, const CUtensorMap* vmap,
                                                  unsigned cta) {
  using Cfg = StreamCfg<FP8 ? 64 : HD>;
  constexpr int NW = Cfg::kWarps;
  constexpr int CT = NW * 32;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - raw_base);
  const uint32_t bar_full = base + Cfg::kRingBytes;
  const uint32_t bar_empty = bar_full + Cfg::kStages * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kRingBytes + Cfg::kBarBytes);

  const RaggedTiling& tl = p.stream;
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int split = (int)(cta % (unsigned)tl.nsplit);
  const int unit = (int)(cta / (unsigned)tl.nsplit);
  const int kvh = unit % p.hkv;
  const int slot_id = unit / p.hkv;
  if (tid == CT) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, NW);
    }
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(kmap);
    tma_prefetch_desc(vmap);
  }
  pdl_wait();
  pdl_trigger();
  RaggedWork w;
  if (!ragged_work(p, tl, slot_id, lane, w)) return;  // the same answer in every warp
  if (split >= w.n_chunks) return;
  const int k_begin = w.k_base + split * tl.chunk;
  const int k_end = min(k_begin + tl.chunk, w.k_hi);
  const int n_stages = (w.k_hi > w.k_lo) ? (k_end - k_begin + Cfg::kBN - 1) / Cfg::kBN : 0;
  __syncthreads();

  if (warp == NW) {
    // ---------------------------------------------------------------- producer
    // Lane i brings box i / NSUB, 64 values of d at i % NSUB, of each stage; its block is
    // looked up before the stage's slot is waited for. A table entry outside the cache
    // gives zeros (TMA's fill).
    constexpr int NSUB = Cfg::kNSub;
    const int box = p.box;
    const int nbox_full = Cfg::kBN / box;
    const uint32_t box_bytes = (uint32_t)box * 128u;
    const int* row_bt = p.block_table + (int64_t)w.b * p.bt_stride;
    const int mask = (1 << p.block_shift) - 1;
    const int my_box = lane / NSUB, my_sub = lane % NSUB;
    bool ok = true;
    int t = 0;
    for (; t < n_stages; ++t) {
      const int slot = t % Cfg::kStages;
      const uint32_t full = bar_full + 8 * slot;
      const int key0 = k_begin + t * Cfg::kBN;
      const int nbox = (min(Cfg::kBN, k_end - key0) + box - 1) / box;
      const int key = key0 + my_box * box;
      int pb = 0;
      if (my_box < nbox) pb = row_bt[key >> p.block_shift];
      if (t >= Cfg::kStages) {
        ok = mbar_wait(bar_empty + 8 * slot, (t / Cfg::kStages - 1) & 1, abort_flag, 111);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (withheld_load(t)) continue;
      if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)nbox * 2u * NSUB * box_bytes);
      __syncwarp();
      if (my_box < nbox && my_box < nbox_full) {
        const uint32_t o = base + slot * Cfg::kStageBytes + my_sub * Cfg::kSubBytes + my_box * box_bytes;
        tma_load_4d(o, kmap, full, my_sub * 64, kvh, key & mask, pb);
        tma_load_4d(o + Cfg::kTileBytes, vmap, full, my_sub * 64, kvh, key & mask, pb);
      }
    }
    // On abort, let the loads already issued land before the CTA exits.
    if (t < n_stages && lane == 0) {
      for (int u = max(0, t - Cfg::kStages); u < t; ++u) {
        volatile int dummy = 0;
        if (!withheld_load(u)) mbar_wait(bar_full + 8 * (u % Cfg::kStages), (u / Cfg::kStages) & 1, &dummy, 112);
      }
    }
    return;
  }
  if (warp > NW) return;
  const int n_valid = w.nq * p.group;
  if (n_valid <= 8) {
    ragged_stream_compute<HD, BF16, 1, FP8, true>(p, w, smem, base, k_begin, k_end, n_stages, unit, split, kvh);
  } else if (n_valid <= 16) {
    ragged_stream_compute<HD, BF16, 1, FP8, false>(p, w, smem, base, k_begin, k_end, n_stages, unit, split, kvh);
  } else if (n_valid <= 32) {
    ragged_stream_compute<HD, BF16, 2, FP8, false>(p, w, smem, base, k_begin, k_end, n_stages, unit, split, kvh);
  } else if constexpr (FP8) {  // 16-bit tiles have at most kRaggedStreamRows rows
    ragged_stream_compute<HD, BF16, 4, FP8, false>(p, w, smem, base, k_begin, k_end, n_stages, unit, split, kvh);
  }
}

// The streaming form as a function of its own, for the tcgen05 kernel with a distance bias,
// whose softmax warps otherwise spill more (two chunks beside 30 decodes, with bias and
// window: 229 us inlined, 213 so; heads of 64: 194 and 183). With a cap, inlined is ahead
// (16 capped drafts 55 us, 65 so), and plain steps do not care (305 us both).
template <int HD, bool BF16>
__device__ __noinline__ void ragged_stream_beside(const RaggedParams& p, const CUtensorMap* kmap, const CUtensorMap* vmap,
                                                  unsigned cta) {
  ragged_stream_cta<HD, BF16, false>(p, kmap, vmap, cta);
}

// Steps whose requests all stream.
template <int HD, bool BF16, bool FP8>
__global__ void __launch_bounds__(288, 1)
    gqa_ragged_stream_kernel(const __grid_constant__ RaggedParams p, const __grid_constant__ CUtensorMap kmap,
                             const __grid_constant__ CUtensorMap vmap) {
  ragged_stream_cta<HD, BF16, FP8>(p, &kmap, &vmap, blockIdx.x);
}

}  // namespace gqa
