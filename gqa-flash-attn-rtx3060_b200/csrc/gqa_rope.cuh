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
// Bound by HBM: 2 x 2 B per value of q, k and v. D / 8 lanes hold one head's row, 16 bytes
// per lane, and keep their cosines and sines in registers for all the token's heads that
// they take, so the table is read once per token and lane group instead of once per head.
// A token's heads are one item of work for a CTA (more than kRows per lane group: several
// items). CTAs stay resident and go from item to item with the next item's position and slot
// in flight, so that an item's rows and table entries leave together at its start; four
// CTAs per SM overlap one item's latency with another's arithmetic. ROPE_FIGURES Everything
// between the load and the one rounding of the store is fp32.
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
  int num_tokens, hq, hkv, rot, axes, max_pos;
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

// Rows are read once: no place in L1.
__device__ __forceinline__ uint4 ld_stream(const uint16_t* x) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(x)
               : "memory");
  return v;
}

constexpr int kRopeThreads = 256;
constexpr int kRopeCtas = 4;  // per SM
template <int D>
struct RopeCfg {
  static constexpr int kLanes = D / 8;                     // lanes per row
  static constexpr int kGroups = kRopeThreads / kLanes;    // lane groups per CTA
  static constexpr int kRows = D == 128 ? 3 : 2;           // rows per lane group and item
  static constexpr int kItemRows = kGroups * kRows;        // 48 or 64 heads
};

// INTER: neighbouring pairs (2f, 2f + 1) instead of (f, f + rot / 2).
template <int D, bool BF16, bool FP8, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) gqa_rope_kernel(const __grid_constant__ RopeParams p) {
  using Cfg = RopeCfg<D>;
  constexpr int R = Cfg::kRows;
  constexpr int NF = INTER ? 4 : 8;  // frequencies of a 16-byte piece
  pdl_wait();
  pdl_trigger();
  const int sub = threadIdx.x % Cfg::kLanes;  // 16-byte piece of the row
  const int grp = threadIdx.x / Cfg::kLanes;
  const int d0 = sub * 8;
  const int half = p.rot >> 1;
  const bool turned = d0 < p.rot;
  const bool second = d0 >= half;  // of a half-split pair (a piece lies in one half: rot % 16 == 0)
  const int f0 = INTER ? d0 >> 1 : (second ? d0 - half : d0);  // the piece's first frequency
  const int rows = p.hq + 2 * p.hkv;
  const int per_token = (rows + Cfg::kItemRows - 1) / Cfg::kItemRows;
  const int64_t items = (int64_t)p.num_tokens * per_token;
  auto axis_of = [&](int f) {
    int x = 0;
#pragma unroll
    for (int a = 1; a < kMaxAxes; ++a)
      if (a < p.axes && f >= p.section_end[a - 1]) x = a;
    return x;
  };
  const int axis = axis_of(f0);
  const bool one_axis = axis == axis_of(f0 + NF - 1);  // or the piece spans sections
  const int lane = threadIdx.x & 31;
  const int shift = half >> 3;  // lanes between the two values of a half-split pair
  const int src = (!INTER && turned) ? (second ? lane - shift : lane + shift) : lane;

  struct Place {  // of an item: token, position on the piece's (first) axis, slot
    int t, at;
    bool valid, past;
    int64_t slot;
  };
  auto place = [&](int64_t w) {
    Place x;
    x.t = (int)(w / per_token);
    x.valid = true;
    x.past = false;
    x.at = 0;
    for (int a = 0; a < p.axes; ++a) {
      const int pos = __ldg(p.positions + a * p.pos_stride + x.t);
      x.valid = x.valid && (unsigned)pos < (unsigned)p.max_pos;
      x.past = x.past || pos >= p.max_pos;
      if (a == axis) x.at = pos;
    }
    x.slot = p.slots ? __ldg(p.slots + x.t) : x.t;
    return x;
  };

  int64_t w = blockIdx.x;
  if (w >= items) return;
  Place next = place(w);
  for (; w < items; w += gridDim.x) {
    const Place it = next;
    const int r0 = (int)(w - (int64_t)it.t * per_token) * Cfg::kItemRows + grp;  // this lane group's first row
    uint4 raw[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + i * Cfg::kGroups;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      const uint16_t* x = nullptr;
      if (r < p.hq) x = p.q + it.t * p.q_st + r * p.q_sh;
      else if (r < p.hq + p.hkv) x = p.k + it.t * p.k_st + (r - p.hq) * p.k_sh;
      else if (r < rows && p.v_dst) x = p.v + it.t * p.v_st + (r - p.hq - p.hkv) * p.v_sh;
      if (x) raw[i] = ld_stream(x + d0);
    }
    // Frequency f0 + e turns value e of the piece, or, interleaved, values 2e and 2e + 1.
    float cs[NF], sn[NF];
#pragma unroll
    for (int e = 0; e < NF; ++e) {
      cs[e] = 1.f;
      sn[e] = 0.f;
    }
    if (turned && it.valid) {
      if (one_axis) {
        const float* row = p.table + (int64_t)it.at * p.rot + f0;
#pragma unroll
        for (int v = 0; v < NF / 4; ++v) {
          const float4 c = __ldg(reinterpret_cast<const float4*>(row) + v);
          const float4 s = __ldg(reinterpret_cast<const float4*>(row + half) + v);
          cs[4 * v] = c.x; cs[4 * v + 1] = c.y; cs[4 * v + 2] = c.z; cs[4 * v + 3] = c.w;
          sn[4 * v] = s.x; sn[4 * v + 1] = s.y; sn[4 * v + 2] = s.z; sn[4 * v + 3] = s.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < NF; ++e) {
          const float* row = p.table + (int64_t)__ldg(p.positions + axis_of(f0 + e) * p.pos_stride + it.t) * p.rot + f0 + e;
          cs[e] = __ldg(row);
          sn[e] = __ldg(row + half);
        }
      }
    }
    if (w + gridDim.x < items) next = place(w + gridDim.x);

    // A token whose position is negative is padding: its query is zero and nothing is
    // cached. One past the table is the same, and reported.
    if (it.past && threadIdx.x == 0) report_device_error(GQA_ERR_INVALID_ARG, 212);
    if (!it.valid) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = r0 + i * Cfg::kGroups;
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
        if (r < p.hq)
          *reinterpret_cast<uint4*>(p.q_out + ((int64_t)it.t * p.hq + r) * D + d0) = z;
        else if (r < p.hq + p.hkv && !p.slots)
          *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.k_dst) + ((int64_t)it.t * p.hkv + r - p.hq) * D + d0) = z;
      }
      continue;
    }
    int64_t dst = it.slot;
    if (p.slots && dst >= p.num_slots) {
      if (threadIdx.x == 0) report_device_error(GQA_ERR_INVALID_ARG, 213);
      dst = -1;
    }

#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + i * Cfg::kGroups;
      const bool is_q = r < p.hq, is_k = !is_q && r < p.hq + p.hkv, is_v = !is_q && !is_k;
      float f[8];
      unpack8<BF16>(raw[i], f);
      const uint16_t* weight = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
      if (weight) {  // uniform over the row's lanes
        float g[8], ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
        // All lanes of the row are here; other rows of the warp may not be.
        const unsigned mask = (Cfg::kLanes == 16 ? 0xffffu : 0xffu) << (lane & ~(Cfg::kLanes - 1));
#pragma unroll
        for (int o = 1; o < Cfg::kLanes; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float rs = rsqrtf(ss * (1.0f / D) + p.eps);
        unpack8<BF16>(__ldg(reinterpret_cast<const uint4*>(weight + d0)), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * rs * g[e];
      }
      // (a, b) -> (a c - b s, b c + a s): the first of a pair takes -s, the second +s.
      if constexpr (INTER) {
        if (!is_v) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = f[2 * e], b = f[2 * e + 1];
            f[2 * e] = fmaf(b, -sn[e], a * cs[e]);
            f[2 * e + 1] = fmaf(a, sn[e], b * cs[e]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float g = __shfl_sync(0xffffffffu, f[e], src);
          if (!is_v) f[e] = fmaf(g, second ? sn[e] : -sn[e], f[e] * cs[e]);
        }
      }
      if (is_q) {
        *reinterpret_cast<uint4*>(p.q_out + ((int64_t)it.t * p.hq + r) * D + d0) = pack8<BF16>(f);
      } else if (dst >= 0 && r < rows && (is_k || p.v_dst)) {
        void* to = is_k ? p.k_dst : p.v_dst;
        const int64_t at = (dst * p.hkv + (is_k ? r - p.hq : r - p.hq - p.hkv)) * D + d0;
        if constexpr (FP8)
          *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(to) + at) = pack8_e4m3(f, is_k ? p.k_scale : p.v_scale);
        else
          *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(to) + at) = is_v ? raw[i] : pack8<BF16>(f);
      }
    }
  }
}

}  // namespace gqa
