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
// probability. Entries with NaN take no part in either.
//
// Bound by HBM for many requests (one row of p, q and e each) and by latency for few:
// the vocabulary is split over `nsplit` CTAs per request. Each walks the request's drafts
// itself (at most 64 gathers, in parallel) to learn the row, scans its part, and leaves
// its best in the workspace; the request's last CTA (a ticket, reset for the next call)
// picks among them. The division is only made for entries that can win: w / e > best
// needs w >= best e (1 - 2^-23) whatever the roundings, one product instead of a
// division that is slow for the many zero weights.
//
// Measured: 4 requests of a 32000-entry vocabulary 5.7 us; 64 requests of 131071 f32
// entries (100 MB; rows start at any word, and a request whose three rows are not all aligned
// reads each by words) 22 us, 0.70 of a plain copy's rate; the greedy form, 64 requests with
// up to 7 drafts of 131072 bf16 logits (91 MB), 20 us, 0.70. Five CTAs per SM of the race and eight of the comparison
// measured best.
#pragma once

#include <climits>
#include <type_traits>

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

constexpr int kVerifyThreads = 256;
constexpr int kVerifyMaxDrafts = 64;

enum : int { kProbF32 = 0, kProbBf16 = 1, kProbF16 = 2 };

// Probabilities or logits of one dtype; Vec = values per 16 bytes.
template <int DT>
struct ProbType {
  using T = uint16_t;
  static constexpr int Vec = 8;
  static __device__ __forceinline__ float value(T x) {
    if constexpr (DT == kProbBf16) return __uint_as_float((uint32_t)x << 16);
    else return __half2float(__ushort_as_half(x));
  }
  static __device__ __forceinline__ float load(const T* p) { return value(__ldg(p)); }
  static __device__ __forceinline__ void values(const uint4& v, float (&f)[Vec]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = value((T)w[i]);
      f[2 * i + 1] = value((T)(w[i] >> 16));
    }
  }
  // The largest of a piece, two values per instruction; NaN only if all are.
  static __device__ __forceinline__ float largest(const uint4& v) {
    using H2 = typename std::conditional<DT == kProbBf16, __nv_bfloat162, __half2>::type;
    auto h = [](const uint32_t& x) { return *reinterpret_cast<const H2*>(&x); };
    const H2 m = __hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w)));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
    return fmaxf(value((T)w), value((T)(w >> 16)));
  }
};
template <>
struct ProbType<kProbF32> {
  using T = float;
  static constexpr int Vec = 4;
  static __device__ __forceinline__ float load(const T* p) { return __ldg(p); }
  static __device__ __forceinline__ void values(const uint4& v, float (&f)[Vec]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    return fmaxf(max3(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z)), __uint_as_float(v.w));
  }
};

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

// Largest of entries [j0, j1) of a row. Each thread takes its 16-byte pieces in rising order
// and compares a piece's largest value with its best; only a piece that has a larger one,
// rare after the first few, is searched for the value's first place.
template <typename PT>
__device__ __forceinline__ Best scan_largest(const typename PT::T* row, int j0, int j1, bool vec) {
  constexpr int V = PT::Vec, U = 8;
  Best best{-INFINITY, INT_MAX};
  auto take = [&](float f, int j) {
    if (f > best.score) best = Best{f, j};
  };
  if (vec) {
    constexpr int step = V * kVerifyThreads;
    const int jv = j0 + (j1 - j0) / V * V;  // whole pieces; part boundaries are multiples of 8
    for (int j = j0 + V * (int)threadIdx.x; j < jv; j += U * step) {
      uint4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = __ldg(reinterpret_cast<const uint4*>(row + min(j + u * step, jv - V)));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float m = PT::largest(x[u]);
        if (m > best.score && j + u * step < jv) {
          float f[V];
          PT::values(x[u], f);
          int at = 0;
#pragma unroll
          for (int e = V - 1; e >= 0; --e) at = f[e] == m ? e : at;
          best = Best{m, j + u * step + at};
        }
      }
    }
    for (int j = jv + (int)threadIdx.x; j < j1; j += kVerifyThreads) take(PT::load(row + j), j);
    return best;
  }
  for (int j = j0 + (int)threadIdx.x; j < j1; j += U * kVerifyThreads) {
    float f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) f[u] = j + u * kVerifyThreads < j1 ? PT::load(row + j + u * kVerifyThreads) : -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) take(f[u], j + u * kVerifyThreads);
  }
  return best;
}

// First best of max(p - q, 0) / e over entries [j0, j1) (q null: of p / e), entry `hidden` left out.
template <typename PT>
__device__ __forceinline__ Best scan_race(const typename PT::T* prow, const typename PT::T* qrow, const float* erow, int hidden,
                                          int j0, int j1, bool vec) {
  constexpr int V = 4, U = 2, US = 4;
  Best best{0.f, INT_MAX};
  auto take = [&](float pj, float qj, float ej, int j) {
    const float w = __fsub_rn(pj, qj);
    if (w > 0.f && w >= best.score * ej * 0.9999995f && j != hidden) {  // 1 - 2^-21
      const float f = __fdiv_rn(w, ej);
      if (f > best.score) best = Best{f, j};
    }
  };
  if (vec) {
    const int step = V * kVerifyThreads;
    auto load4 = [&](const typename PT::T* p, float (&f)[V]) {
      if constexpr (sizeof(typename PT::T) == 4) {
        PT::values(__ldg(reinterpret_cast<const uint4*>(p)), f);
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        const typename PT::T h[4] = {(uint16_t)v.x, (uint16_t)(v.x >> 16), (uint16_t)v.y, (uint16_t)(v.y >> 16)};
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = PT::value(h[e]);
      }
    };
    for (int j = j0 + V * (int)threadIdx.x; j < j1; j += U * step) {
      float a[U][V], c[U][V], e4[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = j + u * step;
        if (at + V <= j1) {
          load4(prow + at, a[u]);
          if (qrow) load4(qrow + at, c[u]);
          const float4 e = __ldg(reinterpret_cast<const float4*>(erow + at));
          e4[u][0] = e.x; e4[u][1] = e.y; e4[u][2] = e.z; e4[u][3] = e.w;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = j + u * step;
        if (at + V <= j1) {
#pragma unroll
          for (int e = 0; e < V; ++e) take(a[u][e], qrow ? c[u][e] : 0.f, e4[u][e], at + e);
        } else {
          for (int e = at; e < j1; ++e) take(PT::load(prow + e), qrow ? PT::load(qrow + e) : 0.f, __ldg(erow + e), e);
        }
      }
    }
    return best;
  }
  // Rows of an odd vocabulary: one value per load, coalesced; the next US of each row are in
  // flight while these are compared.
  float a[US], c[US], e[US];
  auto load = [&](int j) {
#pragma unroll
    for (int u = 0; u < US; ++u) {
      const int at = min(j + u * kVerifyThreads, j1 - 1);
      a[u] = PT::load(prow + at);
      c[u] = qrow ? PT::load(qrow + at) : 0.f;
      e[u] = __ldg(erow + at);
    }
  };
  int j = j0 + (int)threadIdx.x;
  if (j < j1) load(j);
  while (j < j1) {
    float a1[US], c1[US], e1[US];
#pragma unroll
    for (int u = 0; u < US; ++u) {
      a1[u] = a[u];
      c1[u] = c[u];
      e1[u] = e[u];
    }
    const int next = j + US * kVerifyThreads;
    if (next < j1) load(next);
#pragma unroll
    for (int u = 0; u < US; ++u)
      if (j + u * kVerifyThreads < j1) take(a1[u], c1[u], e1[u], j + u * kVerifyThreads);
    j = next;
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
  const bool vec = ((reinterpret_cast<uintptr_t>(prow) | reinterpret_cast<uintptr_t>(drow)) % (4 * sizeof(T))) == 0 &&
                   (reinterpret_cast<uintptr_t>(erow) & 15) == 0;
  Best best = scan_race<PT>(prow, drow, erow, hidden, j0, j1, vec);
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
    best = Best{0.f, INT_MAX};
    for (int i = tid; i < p.nsplit; i += blockDim.x)
      best = better(best, Best{__ldcg(p.ws_score + (int64_t)b * p.nsplit + i),
                               __ldcg(p.ws_index + (int64_t)b * p.nsplit + i)});
    best = block_best(best);
  }
  if (!(best.score > 0.f)) {
    // No weight is left (p exceeds q nowhere, or only by NaN): the row's first largest.
    best = scan_largest<PT>(prow, 0, p.vocab, false);
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
  Best best = scan_largest<PT>(row, j0, j1, (reinterpret_cast<uintptr_t>(row) & 15) == 0);
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
    Best x{-INFINITY, INT_MAX};
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
