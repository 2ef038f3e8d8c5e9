// Host side of the ragged serving step's entry points (declared in include/gqa_sm100.h):
// argument checks, launch sizes and launches. Included at the end of gqa_sm100.cu, whose
// helpers it uses.
#pragma once

namespace gqa {
namespace {

// ----------------------------------------------------------------------------- ragged attention
// The ticket counters of these entry points have a fixed place at the workspace's start,
// so calls of any kind and shape share one workspace without zeroing it in between.
constexpr int kServingCounters = 16384;

template <int HD, bool BF, bool F8>
cudaError_t launch_ragged_stream_hd(const RaggedParams& p, unsigned grid, const CUtensorMap& km, const CUtensorMap& vm,
                                    cudaStream_t st) {
  using Cfg = StreamCfg<F8 ? 64 : HD>;
  if (p.rows <= 8)
    return launch_pdl(gqa_ragged_stream_kernel<HD, BF, 1, F8, true>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, km, vm);
  if (p.rows <= 16)
    return launch_pdl(gqa_ragged_stream_kernel<HD, BF, 1, F8, false>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, km, vm);
  if (p.rows <= 32)
    return launch_pdl(gqa_ragged_stream_kernel<HD, BF, 2, F8, false>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, km, vm);
  return launch_pdl(gqa_ragged_stream_kernel<HD, BF, 4, F8, false>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, km, vm);
}

cudaError_t prepare_ragged() {
  cudaError_t e = cudaSuccess;
  auto chk = [&](cudaError_t x) { if (x != cudaSuccess && e == cudaSuccess) e = x; };
#define GQA_SET_RAGGED(HD, BF, F8)                                                                        \
  chk(set_smem(gqa_ragged_stream_kernel<HD, BF, 1, F8, true>, StreamCfg<F8 ? 64 : HD>::kSmemBytes));      \
  chk(set_smem(gqa_ragged_stream_kernel<HD, BF, 1, F8, false>, StreamCfg<F8 ? 64 : HD>::kSmemBytes));     \
  chk(set_smem(gqa_ragged_stream_kernel<HD, BF, 2, F8, false>, StreamCfg<F8 ? 64 : HD>::kSmemBytes));     \
  chk(set_smem(gqa_ragged_stream_kernel<HD, BF, 4, F8, false>, StreamCfg<F8 ? 64 : HD>::kSmemBytes))
  GQA_SET_RAGGED(128, true, false); GQA_SET_RAGGED(128, false, false);
  GQA_SET_RAGGED(64, true, false); GQA_SET_RAGGED(64, false, false);
  GQA_SET_RAGGED(128, true, true); GQA_SET_RAGGED(128, false, true);
#undef GQA_SET_RAGGED
  return e;
}

template <int HD, bool BF>
cudaError_t launch_ragged_tile_hd(const RaggedParams& p, unsigned grid, const CUtensorMap& qm, const CUtensorMap& km,
                                  const CUtensorMap& vm, cudaStream_t st) {
  using Cfg = RaggedTileCfg<HD>;
  if (p.alibi)
    return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedBias>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
  if (p.cap_in != 0.f)
    return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedCap>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
  return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedPlain>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
}

// Shared memory opt-in, and the setmaxnreg split must fit the registers the launch holds.
int prepare_ragged_tile() {
  int rc = GQA_OK;
  auto prep = [&](auto kernel, int smem) {
    if (set_smem(kernel, smem) != cudaSuccess) rc = rc ? rc : GQA_ERR_CUDA;
    if (!rc) rc = check_reg_split(kernel, PrefillCfg<128>::kThreads, PrefillCfg<128>::kRegsNeeded);
  };
#define GQA_PREP_RAGGED(HD, BF)                                                           \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedPlain>, RaggedTileCfg<HD>::kSmemBytes);      \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedCap>, RaggedTileCfg<HD>::kSmemBytes);        \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedBias>, RaggedTileCfg<HD>::kSmemBytes)
  GQA_PREP_RAGGED(128, true); GQA_PREP_RAGGED(128, false); GQA_PREP_RAGGED(64, true); GQA_PREP_RAGGED(64, false);
#undef GQA_PREP_RAGGED
  return rc;
}

struct RaggedShape {
  int n, tokens, hq, hkv, group, max_q, max_len, head_dim, window, causal, prefix;
};

int check_ragged_shape(const gqa_ragged_args& a, RaggedShape* s) {
  if (a.num_seqs < 0 || a.num_tokens < 0 || a.num_heads <= 0 || a.num_kv_heads <= 0 || a.max_query_len < 0 ||
      a.max_seq_len < 0 || a.window < 0)
    return GQA_ERR_INVALID_ARG;
  if (a.num_heads % a.num_kv_heads != 0) return GQA_ERR_INVALID_ARG;
  if (a.head_dim != 64 && a.head_dim != 128) return GQA_ERR_UNSUPPORTED;
  if (a.num_heads / a.num_kv_heads > kStreamMaxRows) return GQA_ERR_UNSUPPORTED;
  *s = RaggedShape{a.num_seqs, a.num_tokens, a.num_heads, a.num_kv_heads, a.num_heads / a.num_kv_heads,
                   std::min(a.max_query_len, a.num_tokens), a.max_seq_len, a.head_dim, a.window, a.causal ? 1 : 0,
                   a.prefix_lens != nullptr};
  return GQA_OK;
}

struct RaggedPlan {
  int block_m, rows, one_tile, slots, nsplit, chunk;
};

// Tiles of the streaming kernel, and its key split. Only bounds are known here, so the
// chunk is chosen for the longest request; requests with fewer keys use fewer chunks.
RaggedPlan plan_ragged_stream(const RaggedShape& s, int sm_count) {
  RaggedPlan pl{};
  pl.block_m = std::max(1, std::min(s.max_q, kStreamMaxRows / s.group));
  pl.rows = s.group * pl.block_m;
  pl.one_tile = s.max_q <= pl.block_m;
  pl.slots = pl.one_tile ? s.n : s.tokens / pl.block_m + s.n;
  const int64_t tiles = pl.one_tile ? std::min(s.n, s.tokens) : std::min(pl.slots, s.tokens);
  const int64_t units = tiles * s.hkv;
  int span = s.max_len;  // keys of a tile at most
  if (s.window > 0 && s.causal && !s.prefix)
    span = (int)std::min<int64_t>(span, (int64_t)s.window + pl.block_m - 1 + 64);
  const int stages = std::max(1, (span + 127) / 128);
  pl.nsplit = 1;
  pl.chunk = stages * 128;
  if ((int64_t)pl.slots * s.hkv > kServingCounters / 2) return pl;
  constexpr double kFixedStages = 2.5;  // a CTA's fixed cost, in 128-key stages (plan_stream's, in 64-key ones, is 5)
  double best = 1e300;
  for (int ns = 1; ns <= std::min(stages, kMaxSplits); ++ns) {
    const int chunk_st = (stages + ns - 1) / ns;
    if ((stages + chunk_st - 1) / chunk_st != ns) continue;
    const double waves = std::ceil((double)units * ns / sm_count);
    const double cost = waves * (chunk_st + kFixedStages);
    if (cost < best - 1e-9) {
      best = cost;
      pl.nsplit = ns;
      pl.chunk = chunk_st * 128;
    }
  }
  return pl;
}

// Tiles of the tcgen05 kernel (pairs of 128-row query tiles) and its key split. At most
// tokens / block_m + (requests of more than kStreamMaxRows rows) tiles; when they are
// fewer than the SMs the keys are split, at least two 128-key tiles per chunk.
RaggedPlan plan_ragged_tile(const RaggedShape& s, int sm_count) {
  RaggedPlan pl{};
  pl.block_m = 2 * (128 / s.group);
  pl.rows = 256;
  const int64_t longest = std::min<int64_t>(s.n, (int64_t)s.tokens * s.group / (kStreamMaxRows + 1));
  pl.slots = (int)std::min<int64_t>((int64_t)s.tokens / pl.block_m + longest, INT_MAX);
  const int64_t units = (int64_t)pl.slots * s.hkv;
  int span = s.max_len;
  if (s.window > 0 && s.causal && !s.prefix)
    span = (int)std::min<int64_t>(span, (int64_t)s.window + pl.block_m - 1 + 64);
  const int nk = std::max(1, (span + 127) / 128);
  pl.nsplit = 1;
  if (units > 0 && units < sm_count && units <= kServingCounters / 2) {
    int ns = (int)std::min<int64_t>(sm_count / units, 16);
    while (ns > 1 && nk < 2 * ns) --ns;
    pl.nsplit = ns;
  }
  pl.chunk = (nk + pl.nsplit - 1) / pl.nsplit * 128;
  return pl;
}

// The streaming kernel takes the requests of up to kStreamMaxRows packed rows, the
// tcgen05 kernel the rest; e4m3 caches are the streaming kernel's alone.
bool ragged_uses_tile(const RaggedShape& s, bool fp8) { return !fp8 && (int64_t)s.max_q * s.group > kStreamMaxRows; }

RaggedShape stream_part(const RaggedShape& s, bool tile) {
  RaggedShape r = s;
  if (tile) r.max_q = kStreamMaxRows / s.group;
  return r;
}

size_t ragged_partial_bytes(const RaggedPlan& pl, const RaggedShape& s) {
  if (pl.nsplit <= 1) return 0;
  const size_t n = (size_t)pl.slots * s.hkv * pl.nsplit * pl.rows;
  return 2 * align256(n * 4) + align256(n * s.head_dim * 4);
}

// Counters first (half for each kernel), then the streaming kernel's partials, then the
// tcgen05 kernel's.
size_t ragged_ws_bytes(const RaggedPlan& stream, const RaggedPlan* tile, const RaggedShape& s) {
  const size_t n = ragged_partial_bytes(stream, s) + (tile ? ragged_partial_bytes(*tile, s) : 0);
  return n ? (size_t)kServingCounters * 4 + n : 0;
}

void ragged_ws_carve(const RaggedPlan& pl, const RaggedShape& s, uint8_t* counters, uint8_t* c, RaggedParams* p) {
  const size_t n = (size_t)pl.slots * s.hkv * pl.nsplit * pl.rows;
  p->ws_cnt = reinterpret_cast<unsigned*>(counters);
  p->ws_m = reinterpret_cast<float*>(c);
  c += align256(n * 4);
  p->ws_l = reinterpret_cast<float*>(c);
  c += align256(n * 4);
  p->ws_acc = reinterpret_cast<float*>(c);
}

void set_plan(RaggedParams& p, const RaggedPlan& pl) {
  p.block_m = pl.block_m;
  p.rows = pl.rows;
  p.one_tile = pl.one_tile;
  p.slots = pl.slots;
  p.nsplit = pl.nsplit;
  p.chunk = pl.chunk;
}

// 4-D map (d, kv head, position in block, block) of a paged cache with element strides
// (block, position, head), box {128 bytes of d, 1, box, 1}.
int make_cache_map(CUtensorMap* map, const void* cache, const int64_t* st, int num_blocks, int block_size, int hkv,
                   int d, int box, bool u8) {
  const int64_t bhsd[4] = {st[0], st[1], st[2], 1};  // make_map's (b, h, s, d) order: block, position, kv head, d
  return make_map(map, cache, bhsd, num_blocks, block_size, hkv, d, 1, box, u8);
}

int check_strides3(const void* ptr, const int64_t* st, int multiple) {
  if (!ptr || !st) return GQA_ERR_INVALID_ARG;
  if (!aligned16(ptr) || st[2] != 1) return GQA_ERR_ALIGNMENT;
  for (int i = 0; i < 2; ++i)
    if (st[i] < 0 || st[i] % multiple != 0) return GQA_ERR_ALIGNMENT;
  return GQA_OK;
}

int pow2_shift(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

}  // namespace
}  // namespace gqa

using namespace gqa;

extern "C" {

int gqa_step_plan(const gqa_step_plan_args* args, void* stream) {
  if (!args) return GQA_ERR_INVALID_ARG;
  const gqa_step_plan_args& a = *args;
  if (a.num_seqs < 0 || a.max_blocks < 0 || a.max_tokens < 0 || a.num_free < 0 || a.bt_stride < a.max_blocks)
    return GQA_ERR_INVALID_ARG;
  if (a.block_size < 1 || (a.block_size & (a.block_size - 1)) != 0) return GQA_ERR_UNSUPPORTED;
  if (!a.cu_query_lens || !a.free_count || !a.free_count_out || a.free_count == a.free_count_out) return GQA_ERR_INVALID_ARG;
  if (a.num_seqs > 0 && (!a.query_lens || !a.context_lens || !a.blocks_held || !a.seq_lens || !a.granted ||
                         !a.blocks_held_out || a.blocks_held == a.blocks_held_out || a.context_lens == a.seq_lens ||
                         (a.max_blocks > 0 && !a.block_tables)))
    return GQA_ERR_INVALID_ARG;
  if (a.max_tokens > 0 && (!a.positions || !a.slot_mapping || !a.token_seqs)) return GQA_ERR_INVALID_ARG;
  if (a.num_free > 0 && !a.free_blocks) return GQA_ERR_INVALID_ARG;
  int sm = 0;
  int rc = current_device(&sm);
  if (rc) return rc;
  StepPlanParams p{};
  p.query_lens = a.query_lens;
  p.context_lens = a.context_lens;
  p.blocks_held = a.blocks_held;
  p.free_blocks = a.free_blocks;
  p.free_count = a.free_count;
  p.block_tables = a.block_tables;
  p.cu_query_lens = a.cu_query_lens;
  p.seq_lens = a.seq_lens;
  p.positions = a.positions;
  p.slot_mapping = a.slot_mapping;
  p.token_seqs = a.token_seqs;
  p.granted = a.granted;
  p.blocks_held_out = a.blocks_held_out;
  p.free_count_out = a.free_count_out;
  p.bt_stride = a.bt_stride;
  p.n = a.num_seqs;
  p.max_blocks = a.max_blocks;
  p.num_free = a.num_free;
  p.block_shift = pow2_shift(a.block_size);
  p.max_tokens = a.max_tokens;
  const int threads = a.num_seqs > 256 ? 1024 : 256;
  const int grid = std::max(1, std::min(sm, (a.max_tokens + threads - 1) / threads));
  const cudaError_t e = launch_pdl(gqa_step_plan_kernel, dim3(grid), threads, 0, reinterpret_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

int gqa_qk_norm_rope(const gqa_qk_norm_rope_args* args, void* stream) {
  if (!args) return GQA_ERR_INVALID_ARG;
  const gqa_qk_norm_rope_args& a = *args;
  if (a.num_tokens < 0 || a.num_heads <= 0 || a.num_kv_heads <= 0 || a.max_positions < 0 || !(a.eps >= 0.f)) return GQA_ERR_INVALID_ARG;
  if (a.head_dim != 64 && a.head_dim != 128) return GQA_ERR_UNSUPPORTED;
  if (a.dtype != GQA_DTYPE_BF16 && a.dtype != GQA_DTYPE_F16) return GQA_ERR_UNSUPPORTED;
  if (a.axes < 1 || a.axes > kMaxAxes) return GQA_ERR_UNSUPPORTED;
  if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 16 != 0) return GQA_ERR_UNSUPPORTED;
  RopeParams p{};
  int end = 0;
  for (int i = 0; i < a.axes; ++i) {
    if (a.sections[i] < 0) return GQA_ERR_INVALID_ARG;
    end += a.sections[i];
    p.section_end[i] = end;
  }
  if (end != a.rotary_dim / 2) return GQA_ERR_INVALID_ARG;
  if (a.num_tokens == 0) return GQA_OK;
  const bool cached = a.slot_mapping != nullptr;
  if (!a.positions || !a.q_out || !a.k_dst || (a.rotary_dim > 0 && !a.cos_sin)) return GQA_ERR_INVALID_ARG;
  if (cached && (!a.v_dst || a.block_size <= 0 || a.num_blocks < 0)) return GQA_ERR_INVALID_ARG;
  if (!cached && (a.v_dst || a.cache_fp8)) return GQA_ERR_INVALID_ARG;
  if (a.cache_fp8 && !(a.k_scale > 0.f && a.v_scale > 0.f)) return GQA_ERR_INVALID_ARG;
  if (!aligned16(a.q_out) || !aligned16(a.k_dst) || !aligned16(a.v_dst) || !aligned16(a.q_weight) || !aligned16(a.k_weight))
    return GQA_ERR_ALIGNMENT;
  int rc = check_strides3(a.q, a.q_strides, 8);
  if (!rc) rc = check_strides3(a.k, a.k_strides, 8);
  if (!rc && cached) rc = check_strides3(a.v, a.v_strides, 8);
  if (rc) return rc;
  rc = current_device(nullptr);
  if (rc) return rc;
  p.q = reinterpret_cast<const uint16_t*>(a.q);
  p.k = reinterpret_cast<const uint16_t*>(a.k);
  p.v = reinterpret_cast<const uint16_t*>(a.v);
  p.q_st = a.q_strides[0]; p.q_sh = a.q_strides[1];
  p.k_st = a.k_strides[0]; p.k_sh = a.k_strides[1];
  if (cached) { p.v_st = a.v_strides[0]; p.v_sh = a.v_strides[1]; }
  p.q_weight = reinterpret_cast<const uint16_t*>(a.q_weight);
  p.k_weight = reinterpret_cast<const uint16_t*>(a.k_weight);
  p.positions = a.positions;
  p.pos_stride = a.pos_stride;
  p.table = a.cos_sin;
  p.q_out = reinterpret_cast<uint16_t*>(a.q_out);
  p.k_dst = a.k_dst;
  p.v_dst = a.v_dst;
  p.slots = a.slot_mapping;
  p.num_slots = (int64_t)a.num_blocks * a.block_size;
  p.num_tokens = a.num_tokens;
  p.hq = a.num_heads;
  p.hkv = a.num_kv_heads;
  p.rot = a.rotary_dim;
  p.axes = a.axes;
  p.max_pos = a.max_positions;
  p.interleaved = a.interleaved ? 1 : 0;
  p.eps = a.eps;
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a.dtype == GQA_DTYPE_BF16;
  const dim3 grid(a.num_tokens);
  cudaError_t e;
#define GQA_ROPE(D)                                                                    \
  e = a.cache_fp8 ? (bf ? launch_pdl(gqa_rope_kernel<D, true, true>, grid, 256, 0, st, p) \
                      : launch_pdl(gqa_rope_kernel<D, false, true>, grid, 256, 0, st, p)) \
                : (bf ? launch_pdl(gqa_rope_kernel<D, true, false>, grid, 256, 0, st, p) \
                      : launch_pdl(gqa_rope_kernel<D, false, false>, grid, 256, 0, st, p))
  if (a.head_dim == 128) { GQA_ROPE(128); } else { GQA_ROPE(64); }
#undef GQA_ROPE
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

size_t gqa_ragged_fwd_workspace_bytes(const gqa_ragged_args* args) {
  RaggedShape s;
  int sm = 0;
  if (!args || check_ragged_shape(*args, &s) || s.n == 0 || s.tokens == 0 || s.max_q == 0 || current_device(&sm)) return 0;
  const bool tile = ragged_uses_tile(s, args->cache_fp8 != 0);
  const RaggedPlan tp = plan_ragged_tile(s, sm);
  return ragged_ws_bytes(plan_ragged_stream(stream_part(s, tile), sm), tile ? &tp : nullptr, s);
}

int gqa_ragged_fwd(const gqa_ragged_args* args, void* stream) {
  RaggedShape s;
  if (!args) return GQA_ERR_INVALID_ARG;
  const gqa_ragged_args& a = *args;
  int rc = check_ragged_shape(a, &s);
  if (rc) return rc;
  if (a.dtype != GQA_DTYPE_BF16 && a.dtype != GQA_DTYPE_F16) return GQA_ERR_UNSUPPORTED;
  if (a.block_size < 16 || (a.block_size & (a.block_size - 1)) != 0 || a.num_blocks <= 0) return GQA_ERR_UNSUPPORTED;
  if (a.cache_fp8 && a.head_dim != 128) return GQA_ERR_UNSUPPORTED;
  if (a.cache_fp8 && !(a.k_scale > 0.f && a.v_scale > 0.f)) return GQA_ERR_INVALID_ARG;
  if (!(a.softcap >= 0.f) || !(a.scale > 0.f)) return GQA_ERR_INVALID_ARG;
  if (a.num_seqs == 0 || a.num_tokens == 0 || a.max_query_len == 0) return GQA_OK;
  if (!a.block_table || !a.cu_query_lens || !a.seq_lens || a.bt_stride <= 0) return GQA_ERR_INVALID_ARG;
  if (a.max_seq_len > (int64_t)a.bt_stride * a.block_size) return GQA_ERR_INVALID_ARG;
  if (!a.causal && (a.window > 0 || a.prefix_lens)) return GQA_ERR_INVALID_ARG;
  rc = check_strides3(a.q, a.q_strides, 8);
  if (!rc) rc = check_strides3(a.o, a.o_strides, 8);
  if (!rc) rc = (a.k_cache && a.v_cache) ? GQA_OK : GQA_ERR_INVALID_ARG;
  if (!rc && (a.k_strides[3] != 1 || a.v_strides[3] != 1 || !aligned16(a.k_cache) || !aligned16(a.v_cache))) rc = GQA_ERR_ALIGNMENT;
  if (rc) return rc;
  int sm = 0;
  rc = current_device(&sm);
  if (rc) return rc;

  RaggedParams p{};
  p.q = reinterpret_cast<const uint16_t*>(a.q);
  p.o = reinterpret_cast<uint16_t*>(a.o);
  p.lse = a.lse;
  p.q_st = a.q_strides[0]; p.q_sh = a.q_strides[1];
  p.o_st = a.o_strides[0]; p.o_sh = a.o_strides[1];
  p.cu = a.cu_query_lens;
  p.seq_lens = a.seq_lens;
  p.block_table = a.block_table;
  p.bt_stride = a.bt_stride;
  p.block_shift = pow2_shift(a.block_size);
  p.num_blocks = a.num_blocks;
  p.box = std::min(64, a.block_size);
  p.alibi = a.alibi_slopes;
  p.prefix = a.prefix_lens;
  p.key_starts = a.key_starts;
  p.window = a.window;
  p.causal = s.causal;
  p.n = a.num_seqs;
  p.num_tokens = a.num_tokens;
  p.hq = a.num_heads;
  p.hkv = a.num_kv_heads;
  p.group = s.group;
  p.max_len = a.max_seq_len;
  constexpr double kLog2e = 1.4426950408889634;
  const double sc = (double)a.scale * (a.cache_fp8 ? (double)a.k_scale : 1.0);
  p.scale_log2 = (float)(sc * kLog2e);
  p.cap_in = a.softcap > 0.f ? (float)(2.0 * kLog2e * sc / a.softcap) : 0.f;
  p.cap_out = a.softcap > 0.f ? (float)(a.softcap * kLog2e) : 0.f;
  if (a.softcap > 0.f) set_cap_polynomial(p, sc / a.softcap, a.softcap * kLog2e);
  p.v_scale = a.cache_fp8 ? a.v_scale : 1.f;
  p.mods = a.softcap > 0.f || a.alibi_slopes;

  const bool tile = ragged_uses_tile(s, a.cache_fp8 != 0);
  const RaggedShape ss = stream_part(s, tile);
  RaggedPlan sp = plan_ragged_stream(ss, sm), tp = plan_ragged_tile(s, sm);
  if (a.workspace) {
    if (!aligned16(a.workspace)) return GQA_ERR_ALIGNMENT;
    if (a.workspace_bytes < ragged_ws_bytes(sp, tile ? &tp : nullptr, s)) return GQA_ERR_WORKSPACE;
  } else {  // nowhere to leave partials: one CTA per tile
    sp.nsplit = tp.nsplit = 1;
    sp.chunk = tp.chunk = std::max(1, (a.max_seq_len + 127) / 128) * 128;
  }
  uint8_t* const counters = reinterpret_cast<uint8_t*>(a.workspace);
  uint8_t* const partials = counters + (size_t)kServingCounters * 4;
  CUtensorMap km, vm;
  rc = make_cache_map(&km, a.k_cache, a.k_strides, a.num_blocks, a.block_size, a.num_kv_heads, a.head_dim, p.box, a.cache_fp8);
  if (!rc) rc = make_cache_map(&vm, a.v_cache, a.v_strides, a.num_blocks, a.block_size, a.num_kv_heads, a.head_dim, p.box, a.cache_fp8);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a.dtype == GQA_DTYPE_BF16;
  cudaError_t e = cudaSuccess;

  if (tile) {
    RaggedParams t = p;
    set_plan(t, tp);
    t.min_rows = kStreamMaxRows + 1;
    t.max_rows = INT_MAX;
    if (tp.nsplit > 1)
      ragged_ws_carve(tp, s, counters + (size_t)kServingCounters * 2, partials + ragged_partial_bytes(sp, s), &t);
    // Queries (d, head, token): a tile is bm tokens of the group's heads, token-major rows.
    const int64_t bhsd[4] = {a.q_strides[0] * a.num_tokens, a.q_strides[0], a.q_strides[1], 1};
    CUtensorMap qm;
    rc = make_map(&qm, a.q, bhsd, 1, a.num_tokens, a.num_heads, a.head_dim, s.group, tp.block_m / 2);
    if (rc) return rc;
    const int64_t grid = (int64_t)tp.slots * a.num_kv_heads * tp.nsplit;
    if (grid > INT_MAX) return GQA_ERR_INVALID_ARG;
    if (a.head_dim == 128)
      e = bf ? launch_ragged_tile_hd<128, true>(t, (unsigned)grid, qm, km, vm, st)
             : launch_ragged_tile_hd<128, false>(t, (unsigned)grid, qm, km, vm, st);
    else
      e = bf ? launch_ragged_tile_hd<64, true>(t, (unsigned)grid, qm, km, vm, st)
             : launch_ragged_tile_hd<64, false>(t, (unsigned)grid, qm, km, vm, st);
    if (e != cudaSuccess) return GQA_ERR_CUDA;
  }

  set_plan(p, sp);
  p.min_rows = 0;
  p.max_rows = tile ? kStreamMaxRows : INT_MAX;
  if (sp.nsplit > 1) ragged_ws_carve(sp, s, counters, partials, &p);
  const int64_t grid = (int64_t)sp.slots * a.num_kv_heads * sp.nsplit;
  if (grid > INT_MAX) return GQA_ERR_INVALID_ARG;
  if (a.cache_fp8)
    e = bf ? launch_ragged_stream_hd<128, true, true>(p, (unsigned)grid, km, vm, st)
           : launch_ragged_stream_hd<128, false, true>(p, (unsigned)grid, km, vm, st);
  else if (a.head_dim == 128)
    e = bf ? launch_ragged_stream_hd<128, true, false>(p, (unsigned)grid, km, vm, st)
           : launch_ragged_stream_hd<128, false, false>(p, (unsigned)grid, km, vm, st);
  else
    e = bf ? launch_ragged_stream_hd<64, true, false>(p, (unsigned)grid, km, vm, st)
           : launch_ragged_stream_hd<64, false, false>(p, (unsigned)grid, km, vm, st);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"

// ----------------------------------------------------------------------------- draft verification
namespace gqa {
namespace {

struct VerifyPlan {
  int nsplit, part;
};

// CTAs per row: about one wave over the device, at least 1024 entries each. Four CTAs of
// the race fit an SM (registers), five of the greedy scan, of whose rows -- the most that
// the requests can have -- a good part is usually absent.
VerifyPlan plan_verify(int64_t rows, int vocab, int sm_count, bool greedy) {
  VerifyPlan pl;
  const int64_t want = (int64_t)sm_count * (greedy ? 8 : 4) / std::max<int64_t>(rows, 1);
  const int64_t most = std::max(1, vocab / 1024);
  pl.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
  pl.part = (((vocab + pl.nsplit - 1) / pl.nsplit) + 7) & ~7;
  return pl;
}

size_t verify_ws_bytes(int64_t units, const VerifyPlan& pl) {
  return (size_t)kServingCounters * 4 + 2 * align256((size_t)units * pl.nsplit * 4);
}

int verify_common(VerifyParams& p, int greedy, const gqa_verify_args& a, int* grid) {
  if (a.num_seqs < 0 || a.num_rows < 0 || a.max_drafts < 0 || a.vocab <= 0 || a.vocab > INT_MAX - 64)
    return GQA_ERR_INVALID_ARG;
  if (a.max_drafts > kVerifyMaxDrafts || a.num_seqs > kServingCounters) return GQA_ERR_UNSUPPORTED;
  if (a.dtype != GQA_DTYPE_BF16 && a.dtype != GQA_DTYPE_F16 && a.dtype != GQA_DTYPE_F32) return GQA_ERR_UNSUPPORTED;
  if (a.num_seqs == 0) return GQA_OK;
  if (!a.cu_query_lens || !a.tokens || !a.num_tokens || (a.max_drafts > 0 && !a.draft_tokens) ||
      (a.num_rows > 0 && !a.target) || a.target_stride < 0 || a.draft_token_stride < 0)
    return GQA_ERR_INVALID_ARG;
  int sm = 0;
  const int rc = current_device(&sm);
  if (rc) return rc;
  const int64_t units = (int64_t)a.num_seqs * (greedy ? a.max_drafts + 1 : 1);
  const VerifyPlan pl = plan_verify(units, a.vocab, sm, greedy != 0);
  if (!a.workspace || !aligned16(a.workspace) || a.workspace_bytes < verify_ws_bytes(units, pl)) return GQA_ERR_WORKSPACE;
  if (units * pl.nsplit > INT_MAX) return GQA_ERR_INVALID_ARG;
  p.draft_tokens = a.draft_tokens;
  p.dt_st = a.draft_token_stride;
  p.target = a.target;
  p.t_st = a.target_stride;
  p.cu = a.cu_query_lens;
  p.tokens = a.tokens;
  p.num_tokens = a.num_tokens;
  p.n = a.num_seqs;
  p.k = a.max_drafts;
  p.vocab = a.vocab;
  p.num_rows = a.num_rows;
  p.nsplit = pl.nsplit;
  p.part = pl.part;
  uint8_t* c = reinterpret_cast<uint8_t*>(a.workspace);
  p.ws_cnt = reinterpret_cast<unsigned*>(c);
  c += (size_t)kServingCounters * 4;
  p.ws_score = reinterpret_cast<float*>(c);
  c += align256((size_t)units * pl.nsplit * 4);
  p.ws_index = reinterpret_cast<int*>(c);
  *grid = (int)(units * pl.nsplit);
  return GQA_OK;
}

}  // namespace
}  // namespace gqa

extern "C" {

size_t gqa_verify_workspace_bytes(const gqa_verify_args* args, int greedy) {
  int sm = 0;
  if (!args || args->num_seqs <= 0 || args->max_drafts < 0 || args->vocab <= 0 || current_device(&sm)) return 0;
  const int64_t units = (int64_t)args->num_seqs * (greedy ? args->max_drafts + 1 : 1);
  return verify_ws_bytes(units, plan_verify(units, args->vocab, sm, greedy != 0));
}

int gqa_verify_drafts(const gqa_verify_args* args, void* stream) {
  if (!args) return GQA_ERR_INVALID_ARG;
  const gqa_verify_args& a = *args;
  if (a.num_seqs > 0 && (!a.exponentials || a.exponential_stride < 0 || (a.max_drafts > 0 && (!a.uniforms || a.uniform_stride < 0)) ||
                         a.draft_strides[0] < 0 || a.draft_strides[1] < 0))
    return GQA_ERR_INVALID_ARG;
  VerifyParams p{};
  int grid = 0;
  const int rc = verify_common(p, 0, a, &grid);
  if (rc || a.num_seqs == 0) return rc;
  p.draft = a.max_drafts > 0 ? a.draft_probs : nullptr;
  p.d_sn = a.draft_strides[0];
  p.d_sk = a.draft_strides[1];
  p.uniforms = a.uniforms;
  p.u_st = a.uniform_stride;
  p.expo = a.exponentials;
  p.e_st = a.exponential_stride;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e =
      a.dtype == GQA_DTYPE_F32    ? launch_pdl(gqa_verify_kernel<kProbF32>, dim3(grid), kVerifyThreads, 0, st, p)
      : a.dtype == GQA_DTYPE_BF16 ? launch_pdl(gqa_verify_kernel<kProbBf16>, dim3(grid), kVerifyThreads, 0, st, p)
                                  : launch_pdl(gqa_verify_kernel<kProbF16>, dim3(grid), kVerifyThreads, 0, st, p);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

int gqa_verify_greedy(const gqa_verify_args* args, void* stream) {
  if (!args) return GQA_ERR_INVALID_ARG;
  VerifyParams p{};
  int grid = 0;
  const int rc = verify_common(p, 1, *args, &grid);
  if (rc || args->num_seqs == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e =
      args->dtype == GQA_DTYPE_F32    ? launch_pdl(gqa_verify_greedy_kernel<kProbF32>, dim3(grid), kVerifyThreads, 0, st, p)
      : args->dtype == GQA_DTYPE_BF16 ? launch_pdl(gqa_verify_greedy_kernel<kProbBf16>, dim3(grid), kVerifyThreads, 0, st, p)
                                      : launch_pdl(gqa_verify_greedy_kernel<kProbF16>, dim3(grid), kVerifyThreads, 0, st, p);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"
