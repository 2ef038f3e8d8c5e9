// Step plan of a ragged paged batch: from each request's new and cached token counts,
// the block-table entries it gains, the positions and cache slots of its new tokens and
// the packed token offsets, without the host seeing a length.
//
//   after_b = ceil((ctx_b + q_b) / block)       blocks the request needs in all
//   need_b  = max(0, after_b - held_b)          (0 when after_b exceeds the table's width)
//   upto_b  = need_0 + ... + need_b
//   granted_b = the table is wide enough and (need_b == 0 or upto_b <= free_count)
//   entry (b, held_b + j) = free_blocks[free_count - 1 - (upto_b - need_b) - j],  j < need_b
//   token i of request b: position ctx_b + i, slot entry(b, pos / block) * block + pos % block
//
// upto never falls, so the granted requests that need blocks are a prefix of those that
// do, and the blocks taken are the top of the free stack, without gaps. A refused
// request's tokens get slot -1 (paged writes skip it) and its length stays ctx_b.
//
// Integer work bound by latency: a few dependent loads and one scan. Every CTA scans the
// requests itself (1024 at a time), which costs less than a second launch or a grid-wide
// wait, and writes the tokens, table entries and per-request results of its own share. A
// new table entry is computed from the free stack rather than read back from the table, so
// no CTA depends on another's stores. Lengths come from the device unchecked, so both sums
// stay at 2^31 - 1 where they would pass it (which sums of any order agree on) and cannot
// come round to one that the step or the pool could serve. 8 requests of one token: 3.2 us;
// 1024 requests with 65536 new tokens: 4.4 us (5.5 with a loop over the warps' sums instead
// of a scan of them).
#pragma once

#include <climits>

#include "gqa_common.cuh"

namespace gqa {

struct StepPlanParams {
  const int* query_lens;    // (n,)
  const int* context_lens;  // (n,)
  const int* blocks_held;   // (n,)
  const int* free_blocks;   // (num_free,)
  const int* free_count;    // (1,)
  int* block_tables;        // (n, max_blocks), row stride bt_stride; new entries are written
  int* cu_query_lens;       // (n + 1,)
  int* seq_lens;            // (n,)
  int* positions;           // (max_tokens,)
  int64_t* slot_mapping;    // (max_tokens,)
  int* token_seqs;          // (max_tokens,)
  uint8_t* granted;         // (n,)
  int* blocks_held_out;     // (n,)
  int* free_count_out;      // (1,)
  int64_t bt_stride;
  int n, max_blocks, num_free, block_shift, max_tokens;
};

// Sum of two values up to 2^31 - 1, and no more than that.
__device__ __forceinline__ unsigned sum_to_limit(unsigned a, unsigned b) { return min(a + b, (unsigned)INT_MAX); }

// Inclusive sums of both over a warp.
__device__ __forceinline__ void scan_to_limit(unsigned& a, unsigned& b, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, a, d), z = __shfl_up_sync(0xffffffffu, b, d);
    if (lane >= d) {
      a = sum_to_limit(a, y);
      b = sum_to_limit(b, z);
    }
  }
}

__global__ void __launch_bounds__(1024) gqa_step_plan_kernel(const StepPlanParams p) {
  constexpr int kChunk = 1024;  // requests scanned at a time
  __shared__ int s_cu[kChunk + 1];  // first token of each request of the chunk
  __shared__ int s_ctx[kChunk];
  __shared__ int s_held[kChunk];
  __shared__ int s_off[kChunk];   // blocks taken by earlier requests
  __shared__ int s_need[kChunk];  // new blocks, -1: refused
  __shared__ uint2 s_warp[32];  // sums of q and need
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nthreads = blockDim.x, nwarps = nthreads >> 5;
  const int block = 1 << p.block_shift;
  const int free_count = max(0, min(min(*p.free_count, p.num_free), INT_MAX - 1));  // below a sum at its limit
  unsigned carry_q = 0, carry_need = 0;  // sums over the chunks before this one
  int taken = 0;                         // blocks taken so far (granted requests)
  for (int c0 = 0; c0 < p.n || c0 == 0; c0 += kChunk) {
    const int cn = min(kChunk, p.n - c0);
    int chunk_taken = 0;
    for (int i0 = 0; i0 < cn; i0 += nthreads) {  // one pass when the block has a thread per request
      const int i = i0 + tid, b = c0 + i;
      int q = 0, ctx = 0, held = 0, need = 0;
      bool fits = true;
      if (i < cn) {
        q = max(0, p.query_lens[b]);
        ctx = max(0, p.context_lens[b]);
        held = min(max(0, p.blocks_held[b]), p.max_blocks);
        const int64_t after = ((int64_t)ctx + q + block - 1) >> p.block_shift;
        fits = after <= p.max_blocks && (int64_t)ctx + q <= INT_MAX;
        need = fits ? max(0, (int)after - held) : 0;
      }
      unsigned first_q = q, upto = need;
      scan_to_limit(first_q, upto, lane);
      if (lane == 31) s_warp[warp] = make_uint2(first_q, upto);
      first_q = __shfl_up_sync(0xffffffffu, first_q, 1);  // the requests before this one
      if (lane == 0) first_q = 0;
      __syncthreads();
      // Every warp scans the warps' sums.
      uint2 y = lane < nwarps ? s_warp[lane] : make_uint2(0u, 0u);
      scan_to_limit(y.x, y.y, lane);
      const unsigned before_q = __shfl_sync(0xffffffffu, y.x, max(0, warp - 1));
      const unsigned before_need = __shfl_sync(0xffffffffu, y.y, max(0, warp - 1));
      first_q = sum_to_limit(first_q, sum_to_limit(carry_q, warp ? before_q : 0u));
      upto = sum_to_limit(upto, sum_to_limit(carry_need, warp ? before_need : 0u));
      const bool ok = fits && (need == 0 || upto <= (unsigned)free_count);
      if (i < cn) {
        s_cu[i] = (int)first_q;
        s_ctx[i] = ctx;
        s_held[i] = held;
        s_off[i] = (int)upto - need;
        s_need[i] = ok ? need : -1;
        if (ok && need > 0) chunk_taken = max(chunk_taken, (int)upto);
        if (blockIdx.x == 0) {
          p.cu_query_lens[b] = (int)first_q;
          p.seq_lens[b] = ok ? ctx + q : ctx;
          p.granted[b] = ok ? 1 : 0;
          p.blocks_held_out[b] = held + (ok ? need : 0);
        }
      }
      carry_q = sum_to_limit(carry_q, __shfl_sync(0xffffffffu, y.x, 31));
      carry_need = sum_to_limit(carry_need, __shfl_sync(0xffffffffu, y.y, 31));
      __syncthreads();
    }
    if (tid == 0) s_cu[max(cn, 0)] = (int)carry_q;
    if (blockIdx.x == 0) {
      // blocks taken: the largest running sum among the granted requests that need any
      const int m = __reduce_max_sync(0xffffffffu, chunk_taken);
      if (lane == 0) s_warp[warp].x = m;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0)
      for (int w = 0; w < nwarps; ++w) taken = max(taken, (int)s_warp[w].x);

    // New table entries: a warp per request, the requests dealt over the grid.
    for (int i = blockIdx.x + gridDim.x * warp; i < cn; i += gridDim.x * nwarps) {
      const int need = s_need[i];
      int* row = p.block_tables + (int64_t)(c0 + i) * p.bt_stride + s_held[i];
      const int* from = p.free_blocks + (free_count - 1 - s_off[i]);
      for (int j = lane; j < need; j += 32) row[j] = from[-j];
    }
    // Tokens of this chunk: a thread per token finds its request by bisection.
    const int t_end = min(p.max_tokens, s_cu[max(cn, 0)]);
    const int stride = gridDim.x * nthreads;
    // this thread's first token of its grid-strided share that is not before the chunk
    unsigned t = blockIdx.x * nthreads + tid;  // its last step may pass 2^31
    if (cn > 0) {
      const unsigned first = s_cu[0];
      if (t < first) t += (first - t + stride - 1) / stride * stride;
      for (; t < (unsigned)t_end; t += stride) {
        int lo = 0, hi = cn;  // the last request whose first token is <= t (the empty ones before it skipped)
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if ((unsigned)s_cu[mid] <= t) lo = mid; else hi = mid;
        }
        const int pos = (int)(s_ctx[lo] + (t - s_cu[lo]));  // a refused request's may wrap
        int64_t slot = -1;
        if (s_need[lo] >= 0) {
          const int col = pos >> p.block_shift, held = s_held[lo];
          const int id = col < held ? p.block_tables[(int64_t)(c0 + lo) * p.bt_stride + col]
                                    : p.free_blocks[free_count - 1 - s_off[lo] - (col - held)];
          slot = id < 0 ? -1 : ((int64_t)id << p.block_shift) + (pos & (block - 1));
        }
        p.positions[t] = pos;
        p.slot_mapping[t] = slot;
        p.token_seqs[t] = c0 + lo;
      }
    }
    __syncthreads();  // the shared arrays are free for the next chunk
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.cu_query_lens[p.n] = (int)carry_q;
    *p.free_count_out = free_count - taken;
    if (carry_q > (unsigned)p.max_tokens) report_device_error(GQA_ERR_INVALID_ARG, 211);
  }
  // Padding tokens past the step's own.
  for (unsigned t = blockIdx.x * nthreads + tid; t < (unsigned)p.max_tokens; t += gridDim.x * nthreads) {
    if (t < carry_q) continue;
    p.positions[t] = -1;
    p.slot_mapping[t] = -1;
    p.token_seqs[t] = -1;
  }
}

}  // namespace gqa
