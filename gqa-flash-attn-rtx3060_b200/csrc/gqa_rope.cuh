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
// Bound by HBM (2 x 2 B per value of q, k and v) once it is not bound by instructions: the
// norm and the rotation of a 16-bit value leave about ten of them per 4 bytes moved. So
// D / 8 lanes hold one head's row as two 8-byte pieces, four values a and their four
// partners b (no shuffles; for neighbouring pairs and for values past `rot` the pieces are
// neighbours), arithmetic is packed two values at a time, and the work is cut into units
// of four rows of one token that share cosines and sines: four query heads, or the keys
// and values of two heads. Query and key-value units are different CTAs, so that a unit has
// no branches on what a row is, and a lane group goes through its units by additions. The
// next unit's position and slot are in flight while this one is turned, and its rows and
// table entries leave together. Everything between the load and the one rounding of the
// store is fp32.
//
// 16381 tokens of 32 query and 8 kv heads of 128, bf16, three axes: 79 to 83 us, 5.1 TB/s, 0.78
// of a plain copy (units of two rows 86 to 88 us, of eight 80 with three CTAs per SM; four CTAs
// are 64 registers a thread, three hide less latency and take 87, five and six spill; the
// next unit's rows fetched ahead 94). 16 tokens: 4.6 us, a launch and three dependent loads.
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
  int q_ctas;  // CTAs of query units, the grid's first; the rest take keys and values
  int section_end[kMaxAxes];  // first frequency past each axis' section
  float eps, k_scale, v_scale;
};

__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }

// A lane's two pieces of a row.
struct Piece {
  uint2 a, b;
};
// Rows are read once: no place in L1.
__device__ __forceinline__ Piece load_piece(const uint16_t* x, int da, int db) {
  Piece v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.a.x), "=r"(v.a.y) : "l"(x + da) : "memory");
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.b.x), "=r"(v.b.y) : "l"(x + db) : "memory");
  return v;
}
__device__ __forceinline__ void store_piece(uint16_t* x, int da, int db, const Piece& v) {
  *reinterpret_cast<uint2*>(x + da) = v.a;
  *reinterpret_cast<uint2*>(x + db) = v.b;
}
template <bool BF16>
__device__ __forceinline__ void unpack4(const uint2& x, float2 (&f)[2]) {
  f[0] = to_f32x2<BF16>(x.x);
  f[1] = to_f32x2<BF16>(x.y);
}
template <bool BF16>
__device__ __forceinline__ uint2 pack4(const float2 (&f)[2]) {
  return make_uint2(pack2<BF16>(f[0].x, f[0].y), pack2<BF16>(f[1].x, f[1].y));
}
// Four floats over `scale`, as e4m3 (the cache write's rule: rounded to nearest even, saturated).
__device__ __forceinline__ uint32_t pack4_e4m3(const float2 (&f)[2], float scale) {
  return f32x2_to_e4m3x2(__fdiv_rn(f[0].x, scale), __fdiv_rn(f[0].y, scale)) |
         (f32x2_to_e4m3x2(__fdiv_rn(f[1].x, scale), __fdiv_rn(f[1].y, scale)) << 16);
}
template <bool BF16, bool FP8>
__device__ __forceinline__ void store_cache(void* cache, int64_t at, int da, int db, const float2 (&a)[2], const float2 (&b)[2],
                                            float scale) {
  if constexpr (FP8) {
    uint8_t* const x = reinterpret_cast<uint8_t*>(cache) + at;
    *reinterpret_cast<uint32_t*>(x + da) = pack4_e4m3(a, scale);
    *reinterpret_cast<uint32_t*>(x + db) = pack4_e4m3(b, scale);
  } else {
    store_piece(reinterpret_cast<uint16_t*>(cache) + at, da, db, Piece{pack4<BF16>(a), pack4<BF16>(b)});
  }
}

constexpr int kRopeThreads = 256;
constexpr int kRopeCtas = 4;  // per SM
constexpr int kRopeRows = 4;  // of a unit
template <int D>
struct RopeCfg {
  static constexpr int kLanes = D / 8;                   // lanes per row
  static constexpr int kGroups = kRopeThreads / kLanes;  // lane groups per CTA
};

// A lane's place in a row, and its frequencies.
template <int D, bool INTER>
struct RopeLane {
  int da, db, f0, axis;
  bool turned, one_axis;
  unsigned mask;  // all lanes of the row; other rows of a warp may be of another token
};

// Norm (weights wa, wb; or none) and rotation of the lane's pieces a, b of one row.
template <int D, bool BF16, bool INTER>
__device__ __forceinline__ void rope_row(float2 (&a)[2], float2 (&b)[2], const RopeLane<D, INTER>& ln, bool norm, uint2 wa,
                                         uint2 wb, float eps, const float2 (&cs)[2], const float2 (&sn)[2]) {
  if (norm) {
    float2 sq = mul2(a[0], a[0]);
    sq = fma2(a[1], a[1], sq);
    sq = fma2(b[0], b[0], sq);
    sq = fma2(b[1], b[1], sq);
    float ss = sq.x + sq.y;
#pragma unroll
    for (int o = 1; o < RopeCfg<D>::kLanes; o <<= 1) ss += __shfl_xor_sync(ln.mask, ss, o);
    const float rs = rsqrtf(ss * (1.0f / D) + eps);
    const float2 rs2 = make_float2(rs, rs);
    float2 ga[2], gb[2];
    unpack4<BF16>(wa, ga);
    unpack4<BF16>(wb, gb);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      a[e] = mul2(mul2(a[e], rs2), ga[e]);
      b[e] = mul2(mul2(b[e], rs2), gb[e]);
    }
  }
  if (!ln.turned) return;  // past `rot`: as it is
  // (a, b) -> (a c - b s, b c + a s)
  if constexpr (INTER) {  // pairs (a0.x, a0.y), (a1.x, a1.y), (b0.x, b0.y), (b1.x, b1.y)
    float2* const v[4] = {&a[0], &a[1], &b[0], &b[1]};
    const float c[4] = {cs[0].x, cs[0].y, cs[1].x, cs[1].y}, s[4] = {sn[0].x, sn[0].y, sn[1].x, sn[1].y};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = *v[e];
      *v[e] = make_float2(fmaf(x.y, -s[e], x.x * c[e]), fmaf(x.x, s[e], x.y * c[e]));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 x = a[e];
      a[e] = fma2(b[e], neg2(sn[e]), mul2(x, cs[e]));
      b[e] = fma2(x, sn[e], mul2(b[e], cs[e]));
    }
  }
}

// The units of one kind, from `first` on, `step` apart: unit u is number u % per_token of
// token u / per_token.
template <int D, bool BF16, bool FP8, bool INTER, bool IS_Q>
__device__ __forceinline__ void rope_units(const RopeParams& p, const RopeLane<D, INTER>& ln, unsigned first, unsigned step,
                                           unsigned per_token) {
  int t = (int)(first / per_token), u = (int)(first % per_token);
  const int dt = (int)(step / per_token), du = (int)(step % per_token);
  const int half = p.rot >> 1;
  const uint16_t* const weight = IS_Q ? p.q_weight : p.k_weight;
  uint2 wa = make_uint2(0u, 0u), wb = wa;
  if (weight) {
    wa = __ldg(reinterpret_cast<const uint2*>(weight + ln.da));
    wb = __ldg(reinterpret_cast<const uint2*>(weight + ln.db));
  }
  struct Place {  // the token's position on the lane's (first) axis, and its slot
    int at;
    bool valid;
    int64_t slot;
  };
  auto place = [&](int tok) {
    Place x{0, true, tok};
    bool past = false;
    for (int a = 0; a < p.axes; ++a) {
      const int pos = __ldg(p.positions + a * p.pos_stride + tok);
      x.valid = x.valid && (unsigned)pos < (unsigned)p.max_pos;
      past = past || pos >= p.max_pos;
      if (a == ln.axis) x.at = pos;
    }
    if (past) report_device_error(GQA_ERR_INVALID_ARG, 212);
    if (!IS_Q && p.slots) x.slot = __ldg(p.slots + tok);
    return x;
  };
  if (t >= p.num_tokens) return;
  Place next = place(t);
  while (true) {
    const Place it = next;
    const int tok = t, un = u;
    // The unit's rows: query heads kRopeRows un and on, or the key and the value of heads
    // kRopeRows / 2 un and on; the last unit of a token may have fewer.
    constexpr int kHeads = IS_Q ? kRopeRows : kRopeRows / 2;
    const int h0 = kHeads * un, heads = min(kHeads, (IS_Q ? p.hq : p.hkv) - h0);
    Piece r[kRopeRows];
    if constexpr (IS_Q) {
      const uint16_t* x = p.q + tok * p.q_st + h0 * p.q_sh;
#pragma unroll
      for (int i = 0; i < kHeads; ++i, x += p.q_sh)
        if (i < heads) r[i] = load_piece(x, ln.da, ln.db);
    } else {
      const uint16_t* x = p.k + tok * p.k_st + h0 * p.k_sh;
      const uint16_t* y = p.v + tok * p.v_st + h0 * p.v_sh;
#pragma unroll
      for (int i = 0; i < kHeads; ++i, x += p.k_sh, y += p.v_sh)
        if (i < heads) {
          r[2 * i] = load_piece(x, ln.da, ln.db);
          if (p.v_dst) r[2 * i + 1] = load_piece(y, ln.da, ln.db);
        }
    }
    float2 cs[2], sn[2];
    if (ln.turned && it.valid) {
      if (ln.one_axis) {
        const float* row = p.table + (int64_t)it.at * p.rot + ln.f0;
        const float4 c = __ldg(reinterpret_cast<const float4*>(row));
        const float4 s = __ldg(reinterpret_cast<const float4*>(row + half));
        cs[0] = make_float2(c.x, c.y); cs[1] = make_float2(c.z, c.w);
        sn[0] = make_float2(s.x, s.y); sn[1] = make_float2(s.z, s.w);
      } else {
        float c[4], s[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          int axis = 0;
#pragma unroll
          for (int a = 1; a < kMaxAxes; ++a)
            if (a < p.axes && ln.f0 + e >= p.section_end[a - 1]) axis = a;
          const float* row = p.table + (int64_t)__ldg(p.positions + axis * p.pos_stride + tok) * p.rot + ln.f0 + e;
          c[e] = __ldg(row);
          s[e] = __ldg(row + half);
        }
        cs[0] = make_float2(c[0], c[1]); cs[1] = make_float2(c[2], c[3]);
        sn[0] = make_float2(s[0], s[1]); sn[1] = make_float2(s[2], s[3]);
      }
    }
    t += dt;
    u += du;
    if (u >= (int)per_token) {
      u -= (int)per_token;
      ++t;
    }
    const bool more = t < p.num_tokens;
    if (more) next = place(t);

    float2 a[2], b[2];
    if constexpr (IS_Q) {
      // A padding token's query is zero.
      uint16_t* o = p.q_out + ((int64_t)tok * p.hq + h0) * D;
#pragma unroll
      for (int i = 0; i < kHeads; ++i, o += D)
        if (i < heads) {
          Piece y{};
          if (it.valid) {
            unpack4<BF16>(r[i].a, a);
            unpack4<BF16>(r[i].b, b);
            rope_row<D, BF16, INTER>(a, b, ln, weight != nullptr, wa, wb, p.eps, cs, sn);
            y = Piece{pack4<BF16>(a), pack4<BF16>(b)};
          }
          store_piece(o, ln.da, ln.db, y);
        }
    } else {
      int64_t dst = it.slot;
      if (p.slots && (dst >= p.num_slots || !it.valid)) {
        if (dst >= p.num_slots) report_device_error(GQA_ERR_INVALID_ARG, 213);
        dst = -1;
      }
      if (dst >= 0) {
        int64_t at = (dst * p.hkv + h0) * D;
#pragma unroll
        for (int i = 0; i < kHeads; ++i, at += D)
          if (i < heads) {
            if (it.valid) {
              unpack4<BF16>(r[2 * i].a, a);
              unpack4<BF16>(r[2 * i].b, b);
              rope_row<D, BF16, INTER>(a, b, ln, weight != nullptr, wa, wb, p.eps, cs, sn);
            } else {  // padding without a cache: zero
              a[0] = a[1] = b[0] = b[1] = make_float2(0.f, 0.f);
            }
            store_cache<BF16, FP8>(p.k_dst, at, ln.da, ln.db, a, b, p.k_scale);
            if (p.v_dst) {
              if constexpr (FP8) {
                unpack4<BF16>(r[2 * i + 1].a, a);
                unpack4<BF16>(r[2 * i + 1].b, b);
                store_cache<BF16, FP8>(p.v_dst, at, ln.da, ln.db, a, b, p.v_scale);
              } else {
                store_piece(reinterpret_cast<uint16_t*>(p.v_dst) + at, ln.da, ln.db, r[2 * i + 1]);
              }
            }
          }
      }
    }
    if (!more) return;
  }
}

// INTER: neighbouring pairs (2f, 2f + 1) instead of (f, f + rot / 2).
template <int D, bool BF16, bool FP8, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) gqa_rope_kernel(const __grid_constant__ RopeParams p) {
  using Cfg = RopeCfg<D>;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, sub = threadIdx.x % Cfg::kLanes;
  RopeLane<D, INTER> ln;
  ln.f0 = 4 * sub;
  ln.turned = 8 * sub < p.rot;
  const bool split = !INTER && ln.turned;  // the pieces are half a rotation apart
  ln.da = split ? ln.f0 : 8 * sub;
  ln.db = split ? (p.rot >> 1) + ln.f0 : 8 * sub + 4;
  ln.axis = 0;
  int last = 0;
#pragma unroll
  for (int a = 1; a < kMaxAxes; ++a) {
    if (a < p.axes && ln.f0 >= p.section_end[a - 1]) ln.axis = a;
    if (a < p.axes && ln.f0 + 3 >= p.section_end[a - 1]) last = a;
  }
  ln.one_axis = ln.axis == last;  // or the lane's frequencies span sections
  ln.mask = (Cfg::kLanes == 16 ? 0xffffu : 0xffu) << (lane & ~(Cfg::kLanes - 1));
  const unsigned grp = threadIdx.x / Cfg::kLanes;
  if (blockIdx.x < (unsigned)p.q_ctas)
    rope_units<D, BF16, FP8, INTER, true>(p, ln, blockIdx.x * Cfg::kGroups + grp, p.q_ctas * Cfg::kGroups,
                                          (p.hq + kRopeRows - 1) / kRopeRows);
  else
    rope_units<D, BF16, FP8, INTER, false>(p, ln, (blockIdx.x - p.q_ctas) * Cfg::kGroups + grp,
                                           (gridDim.x - p.q_ctas) * Cfg::kGroups,
                                           (p.hkv + kRopeRows / 2 - 1) / (kRopeRows / 2));
}

}  // namespace gqa
