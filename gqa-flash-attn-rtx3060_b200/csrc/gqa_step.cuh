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
// requests itself (1024 at a time, q in the low and need in the high half of one 64-bit
// sum), which costs less than a second launch or a grid-wide wait, and writes the
// tokens, table entries and per-request results of its own share. A new table entry is
// computed from the free stack rather than read back from the table, so no CTA depends
// on another's stores. 8 requests of one token: 3.4 us; 1024 requests with 65536 new
// tokens: 5.4 us, one scan longer.
#pragma once

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

__global__ void __launch_bounds__(1024) gqa_step_plan_kernel(const StepPlanParams p) {
  constexpr int kChunk = 1024;  // requests scanned at a time
  __shared__ int s_cu[kChunk + 1];  // first token of each request of the chunk
  __shared__ int s_ctx[kChunk];
  __shared__ int s_held[kChunk];
  __shared__ int s_off[kChunk];   // blocks taken by earlier requests
  __shared__ int s_need[kChunk];  // new blocks, -1: refused
  __shared__ unsigned long long s_warp[32];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nthreads = blockDim.x, nwarps = nthreads >> 5;
  const int block = 1 << p.block_shift;
  const int free_count = max(0, min(*p.free_count, p.num_free));
  unsigned long long carry = 0;  // sums over the chunks before this one
  int taken = 0;                 // blocks taken so far (granted requests)
  for (int c0 = 0; c0 < p.n || c0 == 0; c0 += kChunk) {
    const int cn = min(kChunk, p.n - c0);
    unsigned long long run = carry;
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
        fits = after <= p.max_blocks;
        need = fits ? max(0, (int)after - held) : 0;
      }
      unsigned long long x = ((unsigned long long)(unsigned)need << 32) | (unsigned)q;
      unsigned long long incl = x;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      if (lane == 31) s_warp[warp] = incl;
      __syncthreads();
      unsigned long long before = run, all = run;
      for (int w = 0; w < nwarps; ++w) {
        const unsigned long long y = s_warp[w];
        if (w < warp) before += y;
        all += y;
      }
      incl += before;
      const int upto = (int)(incl >> 32);
      const bool ok = fits && (need == 0 || upto <= free_count);
      if (i < cn) {
        s_cu[i] = (int)(unsigned)(incl - x);
        s_ctx[i] = ctx;
        s_held[i] = held;
        s_off[i] = upto - need;
        s_need[i] = ok ? need : -1;
        if (ok && need > 0) chunk_taken = max(chunk_taken, upto);
        if (blockIdx.x == 0) {
          p.cu_query_lens[b] = (int)(unsigned)(incl - x);
          p.seq_lens[b] = ok ? ctx + q : ctx;
          p.granted[b] = ok ? 1 : 0;
          p.blocks_held_out[b] = held + (ok ? need : 0);
        }
      }
      run = all;
      __syncthreads();
    }
    if (tid == 0) s_cu[max(cn, 0)] = (int)(unsigned)run;
    if (blockIdx.x == 0) {
      // blocks taken: the largest running sum among the granted requests that need any
      const int m = __reduce_max_sync(0xffffffffu, chunk_taken);
      if (lane == 0) s_warp[warp] = (unsigned long long)(unsigned)m;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0)
      for (int w = 0; w < nwarps; ++w) taken = max(taken, (int)s_warp[w]);

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
    int t = blockIdx.x * nthreads + tid;
    if (cn > 0) {
      const int first = s_cu[0];
      if (t < first) t += (int)(((int64_t)first - t + stride - 1) / stride) * stride;
      for (; t < t_end; t += stride) {
        int lo = 0, hi = cn;  // the last request whose first token is <= t (the empty ones before it skipped)
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_cu[mid] <= t) lo = mid; else hi = mid;
        }
        const int pos = s_ctx[lo] + (t - s_cu[lo]);
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
    carry = run;
    __syncthreads();  // the shared arrays are free for the next chunk
  }
  const int total = (int)(unsigned)carry;
  if (blockIdx.x == 0 && tid == 0) {
    p.cu_query_lens[p.n] = total;
    *p.free_count_out = free_count - taken;
    if (total > p.max_tokens) report_device_error(GQA_ERR_INVALID_ARG, 211);
  }
  // Padding tokens past the step's own.
  for (int t = blockIdx.x * nthreads + tid; t < p.max_tokens; t += gridDim.x * nthreads) {
    if (t < total) continue;
    p.positions[t] = -1;
    p.slot_mapping[t] = -1;
    p.token_seqs[t] = -1;
  }
}

}  // namespace gqa
