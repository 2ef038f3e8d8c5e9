// Verification of drafted tokens (speculative sampling), from given random numbers.
//
// Request b owns rows cu[b] .. cu[b + 1] - 1 of the target's probabilities: row i is the
// distribution after its first i drafts. Drafts are accepted in order while
//     u_i q_i(d_i) < p_i(d_i)
// and the token after the last accepted draft is drawn from the normalised
// max(p_i - q_i, 0) (from p_i after the last row) as
//     argmax_j max(p_i(j) - q_i(j), 0) / e_j,    e_j exponential numbers,
// an exponential race, whose winner is distributed as the weights: it needs no sum over
// the vocabulary, so nothing is normalised, and each score is one IEEE subtraction and one
// IEEE division of the inputs, so the token does not depend on how the row is split. Ties
// go to the lowest index. A row without a positive score gives the first largest
// probability.
//
// Bound by HBM for many requests (one row of p, q and e each) and by latency for few:
// the vocabulary is split over `nsplit` CTAs per request. Each walks the request's drafts
// itself (at most 64 gathers, in parallel) to learn the row, scans its part, and leaves
// its best in the workspace; the request's last CTA (a ticket, reset for the next call)
// picks among them.
#pragma once

#include "gqa_common.cuh"

namespace gqa {

struct VerifyParams {
  const int* draft_tokens;  // (n, k), row stride dt_st
  const void* target;       // (T, V), row stride t_st
  const void* draft;        // (n, k, V), strides d_sn, d_sk; null: the drafts are certain
  const float* uniforms;    // (n, k), row stride u_st
  const float* expo;        // (n, V), row stride e_st
  const int* cu;            // (n + 1,)
  int* tokens;              // (n, k + 1), contiguous
  int* num_tokens;          // (n,)
  int64_t dt_st, t_st, d_sn, d_sk, u_st, e_st;
  int n, k, vocab, num_rows, nsplit, part;  // part: vocabulary entries per CTA (a multiple of 8)
  float* ws_score;   // [units][nsplit]
  int* ws_index;     // [units][nsplit]
  unsigned* ws_cnt;  // [n], zero between calls
};

constexpr int kVerifyThreads = 512;
constexpr int kVerifyMaxDrafts = 64;

enum : int { kProbF32 = 0, kProbBf16 = 1, kProbF16 = 2 };

template <int DT>
struct ProbType;
template <>
struct ProbType<kProbF32> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float load(const T* p) { return *p; }
  static __device__ __forceinline__ void load_vec(const T* p, float (&f)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
};
template <bool BF16>
struct ProbType16 {
  using T = uint16_t;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float load(const T* p) {
    if constexpr (BF16) return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
    else return __half2float(*reinterpret_cast<const __half*>(p));
  }
  static __device__ __forceinline__ void load_vec(const T* p, float (&f)[4]) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f[0] = load(reinterpret_cast<const T*>(&v.x)); f[1] = load(reinterpret_cast<const T*>(&v.x) + 1);
    f[2] = load(reinterpret_cast<const T*>(&v.y)); f[3] = load(reinterpret_cast<const T*>(&v.y) + 1);
  }
};
template <>
struct ProbType<kProbBf16> : ProbType16<true> {};
template <>
struct ProbType<kProbF16> : ProbType16<false> {};

struct Best {
  float score;
  int index;
};
__device__ __forceinline__ Best better(Best a, Best b) {
  return (b.score > a.score || (b.score == a.score && b.index < a.index)) ? b : a;
}
__device__ __forceinline__ Best warp_best(Best x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Best y;
    y.score = __shfl_xor_sync(0xffffffffu, x.score, o);
    y.index = __shfl_xor_sync(0xffffffffu, x.index, o);
    x = better(x, y);
  }
  return x;
}
// Best over the CTA, in every thread.
__device__ __forceinline__ Best block_best(Best x) {
  __shared__ Best s_best[kVerifyThreads / 32];
  x = warp_best(x);
  __syncthreads();  // earlier readers of s_best are done
  if ((threadIdx.x & 31) == 0) s_best[threadIdx.x >> 5] = x;
  __syncthreads();
  Best r = s_best[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) r = better(r, s_best[w]);
  return r;
}

// The request's rows inside the target and its number of drafts; false: it has no row.
__device__ __forceinline__ bool verify_rows(const VerifyParams& p, int b, int& r0, int& drafts) {
  r0 = p.cu[b];
  const int rows = min(p.cu[b + 1], p.num_rows) - r0;
  drafts = min(rows - 1, p.k);
  return r0 >= 0 && rows > 0;
}

// Best of entries [j0, j1) of a row by `score(j)` / `score4(j, f)`: each thread takes
// its entries in rising order, so the first best is kept with a plain comparison.
template <typename S1, typename S4>
__device__ __forceinline__ Best scan_part(int j0, int j1, bool vec, S1 score, S4 score4, Best best) {
  if (vec) {
    const int jv = j0 + ((j1 - j0) & ~3);
#pragma unroll 4
    for (int j = j0 + 4 * (int)threadIdx.x; j < jv; j += 4 * (int)blockDim.x) {
      float f[4];
      score4(j, f);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f[e] > best.score) best = Best{f[e], j + e};
    }
    j0 = jv;
  }
#pragma unroll 8
  for (int j = j0 + (int)threadIdx.x; j < j1; j += (int)blockDim.x) {
    const float f = score(j);
    if (f > best.score) best = Best{f, j};
  }
  return best;
}

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) gqa_verify_kernel(const VerifyParams p) {
  using PT = ProbType<DT>;
  using T = typename PT::T;
  __shared__ int s_last;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / p.nsplit, split = blockIdx.x - b * p.nsplit;
  const int tid = threadIdx.x, lane = tid & 31;
  int r0, drafts;
  if (!verify_rows(p, b, r0, drafts)) {
    if (split == 0) {
      for (int i = tid; i <= p.k; i += blockDim.x) p.tokens[(int64_t)b * (p.k + 1) + i] = -1;
      if (tid == 0) p.num_tokens[b] = 0;
    }
    return;
  }
  const T* target = reinterpret_cast<const T*>(p.target);
  const T* draft = reinterpret_cast<const T*>(p.draft);
  // The accepted drafts: two per lane, the first refusal by ballot (every warp for itself).
  int accepted = drafts;
#pragma unroll
  for (int h = kVerifyMaxDrafts / 32 - 1; h >= 0; --h) {
    const int i = h * 32 + lane;
    bool ok = true;
    if (i < drafts) {
      const int d = p.draft_tokens[b * p.dt_st + i];
      ok = d >= 0 && d < p.vocab;
      if (ok) {
        const float pd = PT::load(target + (int64_t)(r0 + i) * p.t_st + d);
        const float qd = draft ? PT::load(draft + b * p.d_sn + i * p.d_sk + d) : 1.f;
        ok = __fmul_rn(p.uniforms[b * p.u_st + i], qd) < pd;
      }
    }
    const unsigned no = __ballot_sync(0xffffffffu, !ok);
    if (no) accepted = h * 32 + __ffs(no) - 1;
  }
  const bool refused = accepted < drafts;
  const T* prow = target + (int64_t)(r0 + accepted) * p.t_st;
  const T* drow = (refused && draft) ? draft + b * p.d_sn + accepted * p.d_sk : nullptr;
  const int hidden = (refused && !draft) ? p.draft_tokens[b * p.dt_st + accepted] : -1;  // a certain draft's whole weight
  const float* erow = p.expo + b * p.e_st;

  const int j0 = min(p.vocab, split * p.part), j1 = min(p.vocab, j0 + p.part);
  auto score_of = [&](float pj, float qj, float ej, int j) {
    const float w = fmaxf(__fsub_rn(pj, qj), 0.f);
    return (j == hidden) ? 0.f : __fdiv_rn(w, ej);
  };
  const bool vec = ((reinterpret_cast<uintptr_t>(prow) | reinterpret_cast<uintptr_t>(drow)) % (4 * sizeof(T))) == 0 &&
                   (reinterpret_cast<uintptr_t>(erow) & 15) == 0;
  Best best = scan_part(
      j0, j1, vec, [&](int j) { return score_of(PT::load(prow + j), drow ? PT::load(drow + j) : 0.f, erow[j], j); },
      [&](int j, float (&f)[4]) {
        float a[4], c[4] = {0.f, 0.f, 0.f, 0.f};
        PT::load_vec(prow + j, a);
        if (drow) PT::load_vec(drow + j, c);
        const float4 e = *reinterpret_cast<const float4*>(erow + j);
        f[0] = score_of(a[0], c[0], e.x, j);
        f[1] = score_of(a[1], c[1], e.y, j + 1);
        f[2] = score_of(a[2], c[2], e.z, j + 2);
        f[3] = score_of(a[3], c[3], e.w, j + 3);
      },
      Best{0.f, p.vocab});
  best = block_best(best);

  if (p.nsplit > 1) {
    if (tid == 0) {
      __stcg(p.ws_score + (int64_t)b * p.nsplit + split, best.score);
      __stcg(p.ws_index + (int64_t)b * p.nsplit + split, best.index);
      unsigned ticket;
      asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(p.ws_cnt + b) : "memory");
      s_last = ticket == (unsigned)(p.nsplit - 1);
      if (s_last) p.ws_cnt[b] = 0u;
    }
    __syncthreads();
    if (!s_last) return;
    best = Best{0.f, p.vocab};
    for (int i = tid; i < p.nsplit; i += blockDim.x)
      best = better(best, Best{__ldcg(p.ws_score + (int64_t)b * p.nsplit + i),
                               __ldcg(p.ws_index + (int64_t)b * p.nsplit + i)});
    best = block_best(best);
  }
  if (!(best.score > 0.f)) {
    // No weight is left (p and q agree where p is not zero, or the row holds NaN): the row's first largest.
    best = scan_part(
        0, p.vocab, false, [&](int j) { return PT::load(prow + j); }, [](int, float (&)[4]) {},
        Best{-INFINITY, p.vocab});
    best = block_best(best);
    if (best.index >= p.vocab) best.index = 0;
  }
  for (int i = tid; i <= p.k; i += blockDim.x)
    p.tokens[(int64_t)b * (p.k + 1) + i] =
        i < accepted ? p.draft_tokens[b * p.dt_st + i] : i == accepted ? best.index : -1;
  if (tid == 0) p.num_tokens[b] = accepted + 1;
}

// At temperature zero: a draft is accepted while it is the first largest entry of its
// row, and the next token is that of the row after it. Every row is read once: CTA
// (request, row, part) leaves its part's best; the request's last CTA walks the rows.
template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) gqa_verify_greedy_kernel(const VerifyParams p) {
  using PT = ProbType<DT>;
  using T = typename PT::T;
  __shared__ int s_last;
  __shared__ int s_token[kVerifyMaxDrafts + 1];
  pdl_wait();
  pdl_trigger();
  const int per = (p.k + 1) * p.nsplit;
  const int b = blockIdx.x / per, i = (blockIdx.x - b * per) / p.nsplit, split = blockIdx.x % p.nsplit;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int r0, drafts;
  if (!verify_rows(p, b, r0, drafts)) {
    if (i == 0 && split == 0) {
      for (int e = tid; e <= p.k; e += blockDim.x) p.tokens[(int64_t)b * (p.k + 1) + e] = -1;
      if (tid == 0) p.num_tokens[b] = 0;
    }
    return;
  }
  if (i > drafts) return;
  const T* row = reinterpret_cast<const T*>(p.target) + (int64_t)(r0 + i) * p.t_st;
  const int j0 = min(p.vocab, split * p.part), j1 = min(p.vocab, j0 + p.part);
  const bool vec = (reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T))) == 0;
  Best best = scan_part(
      j0, j1, vec, [&](int j) { return PT::load(row + j); }, [&](int j, float (&f)[4]) { PT::load_vec(row + j, f); },
      Best{-INFINITY, p.vocab});
  best = block_best(best);
  const int64_t unit = (int64_t)b * (p.k + 1);
  if (tid == 0) {
    __stcg(p.ws_score + (unit + i) * p.nsplit + split, best.score);
    __stcg(p.ws_index + (unit + i) * p.nsplit + split, best.index);
    unsigned ticket;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(p.ws_cnt + b) : "memory");
    s_last = ticket == (unsigned)((drafts + 1) * p.nsplit - 1);
    if (s_last) p.ws_cnt[b] = 0u;
  }
  __syncthreads();
  if (!s_last) return;
  for (int r = warp; r <= drafts; r += blockDim.x >> 5) {
    Best x{-INFINITY, p.vocab};
    for (int s = lane; s < p.nsplit; s += 32)
      x = better(x, Best{__ldcg(p.ws_score + (unit + r) * p.nsplit + s), __ldcg(p.ws_index + (unit + r) * p.nsplit + s)});
    x = warp_best(x);
    if (lane == 0) s_token[r] = x.index < p.vocab ? x.index : 0;  // no entry above -inf: the first
  }
  __syncthreads();
  if (warp == 0) {
    int accepted = drafts;
#pragma unroll
    for (int h = kVerifyMaxDrafts / 32 - 1; h >= 0; --h) {
      const int e = h * 32 + lane;
      const bool ok = e >= drafts || p.draft_tokens[b * p.dt_st + e] == s_token[e];
      const unsigned no = __ballot_sync(0xffffffffu, !ok);
      if (no) accepted = h * 32 + __ffs(no) - 1;
    }
    for (int e = lane; e <= p.k; e += 32) p.tokens[unit + e] = e <= accepted ? s_token[e] : -1;
    if (lane == 0) p.num_tokens[b] = accepted + 1;
  }
}

}  // namespace gqa
