// Norm of each query and key head, the position rotation, and the write of K and V into
// the paged cache, in one pass over the projection's output.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                    (optional, per head of D values)
//   (a, b) -> (a cos - b sin, b cos + a sin)              for each pair f < rot / 2, with
//   cos, sin = table[position of f's axis][f]             a table of the caller's
//
// Pairs are (f, f + rot/2) or, interleaved, (2f, 2f + 1); values past `rot` pass through.
// With several position axes (time, height, width) the frequencies are dealt to the axes
// in consecutive sections.
//
// Bound by HBM: 2 x 2 B per value of q, k and v. One CTA per token; D / 8 lanes hold one
// head's row, 16 bytes per lane, and keep their cosines and sines in registers for all the
// token's heads, so the table is read once per token and lane group instead of once per
// head. Everything between the load and the one rounding of the store is fp32.
#pragma once

#include "gqa_cache.cuh"

namespace gqa {

constexpr int kMaxAxes = 4;

struct RopeParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // element strides (token, head); d stride 1
  const uint16_t* q_weight;  // (D,) or null
  const uint16_t* k_weight;
  const int* positions;  // axis a, token t at positions[a * pos_stride + t]
  int64_t pos_stride;
  const float* table;  // (max_pos, rot): cos | sin
  uint16_t* q_out;     // (T, hq, D), contiguous
  void* k_dst;         // the key cache (slots) or (T, hkv, D)
  void* v_dst;         // the value cache, or null: v is not written
  const int64_t* slots;  // (T,), or null: k_dst is indexed by token
  int64_t num_slots;
  int num_tokens, hq, hkv, rot, axes, max_pos, interleaved;
  int section_end[kMaxAxes];  // first frequency past each axis' section
  float eps, k_scale, v_scale;
};

// Eight 16-bit values as floats.
template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& x, float (&f)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = to_f32x2<BF16>(w[i]);
    f[2 * i] = y.x;
    f[2 * i + 1] = y.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]),
                    pack2<BF16>(f[6], f[7]));
}
// Eight floats over `scale`, as e4m3 (the cache write's rule: rounded to nearest even, saturated).
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], float scale) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f32x2_to_e4m3x2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale));
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(256) gqa_rope_kernel(const RopeParams p) {
  constexpr int LPR = D / 8;         // lanes per row
  constexpr int GROUPS = 256 / LPR;  // rows in flight per CTA
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int sub = threadIdx.x % LPR;  // 16-byte piece of the row
  const int grp = threadIdx.x / LPR;
  const int d0 = sub * 8;
  const int half = p.rot >> 1;
  const bool turned = d0 < p.rot;

  // A token whose position is negative is padding: its query is zero and nothing is
  // cached. One past the table is the same, and reported.
  bool valid = true;
  int pos[kMaxAxes];
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    pos[a] = a < p.axes ? p.positions[a * p.pos_stride + t] : 0;
    if (pos[a] < 0 || pos[a] >= p.max_pos) {
      if (pos[a] >= p.max_pos && threadIdx.x == 0) report_device_error(GQA_ERR_INVALID_ARG, 212);
      valid = false;
    }
  }
  int64_t dst = t;
  if (p.slots) {
    dst = p.slots[t];
    if (dst >= p.num_slots) {
      if (threadIdx.x == 0) report_device_error(GQA_ERR_INVALID_ARG, 213);
      dst = -1;
    }
    if (!valid) dst = -1;
  }
  const int rows = p.hq + 2 * p.hkv;
  if (!valid) {
    for (int r = grp; r < p.hq; r += GROUPS)
      *reinterpret_cast<uint4*>(p.q_out + ((int64_t)t * p.hq + r) * D + d0) = make_uint4(0u, 0u, 0u, 0u);
    if (!p.slots)
      for (int r = grp; r < p.hkv; r += GROUPS)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.k_dst) + ((int64_t)t * p.hkv + r) * D + d0) =
            make_uint4(0u, 0u, 0u, 0u);
    return;
  }

  // The lane's cosines and sines: value e turns with frequency (d0 + e) mod half, or, interleaved, (d0 + e) / 2.
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (turned) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int f = p.interleaved ? (d0 + e) >> 1 : (d0 + e < half ? d0 + e : d0 + e - half);
      int at = pos[0];
#pragma unroll
      for (int a = 1; a < kMaxAxes; ++a)
        if (a < p.axes && f >= p.section_end[a - 1]) at = pos[a];
      const float* row = p.table + (int64_t)at * p.rot;
      cs[e] = row[f];
      const float s = row[half + f];
      // the first of a pair takes -sin, the second +sin
      sn[e] = (p.interleaved ? (e & 1) == 0 : d0 < half) ? -s : s;
    }
  }
  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) wq[e] = wk[e] = 1.f;
  if (p.q_weight) unpack8<BF16>(*reinterpret_cast<const uint4*>(p.q_weight + d0), wq);
  if (p.k_weight) unpack8<BF16>(*reinterpret_cast<const uint4*>(p.k_weight + d0), wk);

  const int shift = half >> 3;  // lanes between the two values of a half-split pair
  const int lane = threadIdx.x & 31;
  const int base = lane - sub;
  const int src = (!p.interleaved && turned) ? base + (d0 < half ? sub + shift : sub - shift) : lane;

  const int n_iter = (rows + GROUPS - 1) / GROUPS;
  for (int it = 0; it < n_iter; ++it) {  // every lane runs every iteration: the shuffles are warp-wide
    const int r = it * GROUPS + grp;
    const bool is_q = r < p.hq, is_k = !is_q && r < p.hq + p.hkv, is_v = !is_q && !is_k && r < rows;
    const bool live = is_q || ((is_k || (is_v && p.v_dst)) && dst >= 0);
    const int h = is_q ? r : is_k ? r - p.hq : r - p.hq - p.hkv;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (live) {
      const uint16_t* x = is_q ? p.q + t * p.q_st + h * p.q_sh : is_k ? p.k + t * p.k_st + h * p.k_sh
                                                                      : p.v + t * p.v_st + h * p.v_sh;
      raw = *reinterpret_cast<const uint4*>(x + d0);
    }
    float f[8];
    unpack8<BF16>(raw, f);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!is_v) {
      const bool norm = is_q ? p.q_weight != nullptr : p.k_weight != nullptr;
      const float rs = norm ? rsqrtf(ss * (1.0f / D) + p.eps) : 1.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * rs * (is_q ? wq[e] : wk[e]);
    }
    float g[8];
    if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = f[e ^ 1];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = __shfl_sync(0xffffffffu, f[e], src);
    }
    if (!is_v && turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = fmaf(g[e], sn[e], f[e] * cs[e]);
    }
    if (!live) continue;
    if (is_q) {
      *reinterpret_cast<uint4*>(p.q_out + ((int64_t)t * p.hq + h) * D + d0) = pack8<BF16>(f);
    } else {
      void* to = is_k ? p.k_dst : p.v_dst;
      const int64_t at = (dst * p.hkv + h) * D + d0;
      if constexpr (FP8)
        *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(to) + at) = pack8_e4m3(f, is_k ? p.k_scale : p.v_scale);
      else
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(to) + at) = is_v ? raw : pack8<BF16>(f);
    }
  }
}

}  // namespace gqa
