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

int check_ragged_shape(int n, int tokens, int hq, int hkv, int max_q, int max_len, int head_dim, int window,
                       RaggedShape* s) {
  if (n < 0 || tokens < 0 || hq <= 0 || hkv <= 0 || max_q < 0 || max_len < 0 || window < 0) return GQA_ERR_INVALID_ARG;
  if (hq % hkv != 0) return GQA_ERR_INVALID_ARG;
  if (head_dim != 64 && head_dim != 128) return GQA_ERR_UNSUPPORTED;
  if (hq / hkv > kStreamMaxRows) return GQA_ERR_UNSUPPORTED;
  *s = RaggedShape{n, tokens, hq, hkv, hq / hkv, std::min(max_q, tokens), max_len, head_dim, window, 1, 0};
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

int gqa_step_plan(const int* query_lens, const int* context_lens, int* block_tables, int64_t bt_stride,
                  const int* blocks_held, const int* free_blocks, int num_free, const int* free_count, int num_seqs,
                  int max_blocks, int block_size, int max_tokens, int* cu_query_lens, int* seq_lens, int* positions,
                  int64_t* slot_mapping, int* token_seqs, unsigned char* granted, int* blocks_held_out,
                  int* free_count_out, void* stream) {
  if (num_seqs < 0 || max_blocks < 0 || max_tokens < 0 || num_free < 0 || bt_stride < max_blocks) return GQA_ERR_INVALID_ARG;
  if (block_size < 1 || (block_size & (block_size - 1)) != 0) return GQA_ERR_UNSUPPORTED;
  if (!cu_query_lens || !free_count || !free_count_out || free_count == free_count_out) return GQA_ERR_INVALID_ARG;
  if (num_seqs > 0 && (!query_lens || !context_lens || !blocks_held || !seq_lens || !granted || !blocks_held_out ||
                       blocks_held == blocks_held_out || context_lens == seq_lens || (max_blocks > 0 && !block_tables)))
    return GQA_ERR_INVALID_ARG;
  if (max_tokens > 0 && (!positions || !slot_mapping || !token_seqs)) return GQA_ERR_INVALID_ARG;
  if (num_free > 0 && !free_blocks) return GQA_ERR_INVALID_ARG;
  int sm = 0;
  int rc = current_device(&sm);
  if (rc) return rc;
  StepPlanParams p{};
  p.query_lens = query_lens;
  p.context_lens = context_lens;
  p.blocks_held = blocks_held;
  p.free_blocks = free_blocks;
  p.free_count = free_count;
  p.block_tables = block_tables;
  p.cu_query_lens = cu_query_lens;
  p.seq_lens = seq_lens;
  p.positions = positions;
  p.slot_mapping = slot_mapping;
  p.token_seqs = token_seqs;
  p.granted = granted;
  p.blocks_held_out = blocks_held_out;
  p.free_count_out = free_count_out;
  p.bt_stride = bt_stride;
  p.n = num_seqs;
  p.max_blocks = max_blocks;
  p.num_free = num_free;
  p.block_shift = pow2_shift(block_size);
  p.max_tokens = max_tokens;
  const int threads = num_seqs > 256 ? 1024 : 256;
  const int grid = std::max(1, std::min(sm, (max_tokens + threads - 1) / threads));
  const cudaError_t e = launch_pdl(gqa_step_plan_kernel, dim3(grid), threads, 0, reinterpret_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

int gqa_qk_norm_rope(const void* q, const void* k, const void* v, const int64_t* q_strides3, const int64_t* k_strides3,
                     const int64_t* v_strides3, const void* q_weight, const void* k_weight, const int* positions,
                     int64_t pos_stride, int axes, const int* sections, const float* cos_sin, int max_positions,
                     int rotary_dim, int interleaved, void* q_out, void* k_dst, void* v_dst, const int64_t* slot_mapping,
                     int num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size, int num_blocks,
                     int dtype, int cache_fp8, float eps, float k_scale, float v_scale, void* stream) {
  if (num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || max_positions < 0 || !(eps >= 0.f)) return GQA_ERR_INVALID_ARG;
  if (head_dim != 64 && head_dim != 128) return GQA_ERR_UNSUPPORTED;
  if (dtype != GQA_DTYPE_BF16 && dtype != GQA_DTYPE_F16) return GQA_ERR_UNSUPPORTED;
  if (axes < 1 || axes > kMaxAxes) return GQA_ERR_UNSUPPORTED;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0) return GQA_ERR_UNSUPPORTED;
  RopeParams p{};
  int end = 0;
  for (int a = 0; a < axes; ++a) {
    const int size = sections ? sections[a] : (axes == 1 ? rotary_dim / 2 : -1);
    if (size < 0) return GQA_ERR_INVALID_ARG;
    end += size;
    p.section_end[a] = end;
  }
  if (end != rotary_dim / 2) return GQA_ERR_INVALID_ARG;
  if (num_tokens == 0) return GQA_OK;
  const bool cached = slot_mapping != nullptr;
  if (!positions || !q_out || !k_dst || (rotary_dim > 0 && !cos_sin)) return GQA_ERR_INVALID_ARG;
  if (cached && (!v_dst || block_size <= 0 || num_blocks < 0)) return GQA_ERR_INVALID_ARG;
  if (!cached && (v_dst || cache_fp8)) return GQA_ERR_INVALID_ARG;
  if (cache_fp8 && !(k_scale > 0.f && v_scale > 0.f)) return GQA_ERR_INVALID_ARG;
  if (!aligned16(q_out) || !aligned16(k_dst) || !aligned16(v_dst) || !aligned16(q_weight) || !aligned16(k_weight))
    return GQA_ERR_ALIGNMENT;
  int rc = check_strides3(q, q_strides3, 8);
  if (!rc) rc = check_strides3(k, k_strides3, 8);
  if (!rc && cached) rc = check_strides3(v, v_strides3, 8);
  if (rc) return rc;
  rc = current_device(nullptr);
  if (rc) return rc;
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.k = reinterpret_cast<const uint16_t*>(k);
  p.v = reinterpret_cast<const uint16_t*>(v);
  p.q_st = q_strides3[0]; p.q_sh = q_strides3[1];
  p.k_st = k_strides3[0]; p.k_sh = k_strides3[1];
  if (cached) { p.v_st = v_strides3[0]; p.v_sh = v_strides3[1]; }
  p.q_weight = reinterpret_cast<const uint16_t*>(q_weight);
  p.k_weight = reinterpret_cast<const uint16_t*>(k_weight);
  p.positions = positions;
  p.pos_stride = pos_stride;
  p.table = cos_sin;
  p.q_out = reinterpret_cast<uint16_t*>(q_out);
  p.k_dst = k_dst;
  p.v_dst = v_dst;
  p.slots = slot_mapping;
  p.num_slots = (int64_t)num_blocks * block_size;
  p.num_tokens = num_tokens;
  p.hq = num_heads;
  p.hkv = num_kv_heads;
  p.rot = rotary_dim;
  p.axes = axes;
  p.max_pos = max_positions;
  p.interleaved = interleaved ? 1 : 0;
  p.eps = eps;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == GQA_DTYPE_BF16;
  const dim3 grid(num_tokens);
  cudaError_t e;
#define GQA_ROPE(D)                                                                    \
  e = cache_fp8 ? (bf ? launch_pdl(gqa_rope_kernel<D, true, true>, grid, 256, 0, st, p) \
                      : launch_pdl(gqa_rope_kernel<D, false, true>, grid, 256, 0, st, p)) \
                : (bf ? launch_pdl(gqa_rope_kernel<D, true, false>, grid, 256, 0, st, p) \
                      : launch_pdl(gqa_rope_kernel<D, false, false>, grid, 256, 0, st, p))
  if (head_dim == 128) { GQA_ROPE(128); } else { GQA_ROPE(64); }
#undef GQA_ROPE
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

size_t gqa_ragged_fwd_workspace_bytes(int num_seqs, int num_tokens, int num_heads, int num_kv_heads, int max_query_len,
                                      int max_seq_len, int head_dim, int window, int cache_fp8) {
  RaggedShape s;
  int sm = 0;
  if (check_ragged_shape(num_seqs, num_tokens, num_heads, num_kv_heads, max_query_len, max_seq_len, head_dim, window, &s) ||
      num_seqs == 0 || num_tokens == 0 || max_query_len == 0 || current_device(&sm))
    return 0;
  const bool tile = ragged_uses_tile(s, cache_fp8 != 0);
  const RaggedPlan tp = plan_ragged_tile(s, sm);
  return ragged_ws_bytes(plan_ragged_stream(stream_part(s, tile), sm), tile ? &tp : nullptr, s);
}

int gqa_ragged_fwd(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse,
                   const int64_t* q_strides3, const int64_t* k_strides4, const int64_t* v_strides4,
                   const int64_t* o_strides3, const int* block_table, int bt_stride, const int* cu_query_lens,
                   const int* seq_lens, const float* alibi_slopes, const int* prefix_lens, const int* key_starts,
                   int num_seqs, int num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size,
                   int num_blocks, int max_query_len, int max_seq_len, float scale, float softcap, int window, int causal,
                   int dtype, int cache_fp8, float k_scale, float v_scale, void* workspace, size_t workspace_bytes,
                   void* stream) {
  RaggedShape s;
  int rc = check_ragged_shape(num_seqs, num_tokens, num_heads, num_kv_heads, max_query_len, max_seq_len, head_dim, window,
                              &s);
  if (rc) return rc;
  if (dtype != GQA_DTYPE_BF16 && dtype != GQA_DTYPE_F16) return GQA_ERR_UNSUPPORTED;
  if (block_size < 16 || (block_size & (block_size - 1)) != 0 || num_blocks <= 0) return GQA_ERR_UNSUPPORTED;
  if (cache_fp8 && head_dim != 128) return GQA_ERR_UNSUPPORTED;
  if (cache_fp8 && !(k_scale > 0.f && v_scale > 0.f)) return GQA_ERR_INVALID_ARG;
  if (!(softcap >= 0.f) || !(scale > 0.f)) return GQA_ERR_INVALID_ARG;
  if (num_seqs == 0 || num_tokens == 0 || max_query_len == 0) return GQA_OK;
  if (!block_table || !cu_query_lens || !seq_lens || bt_stride <= 0) return GQA_ERR_INVALID_ARG;
  if (max_seq_len > (int64_t)bt_stride * block_size) return GQA_ERR_INVALID_ARG;
  if (!causal && (window > 0 || prefix_lens)) return GQA_ERR_INVALID_ARG;
  rc = check_strides3(q, q_strides3, 8);
  if (!rc) rc = check_strides3(o, o_strides3, 8);
  if (!rc) rc = (k_cache && v_cache && k_strides4 && v_strides4) ? GQA_OK : GQA_ERR_INVALID_ARG;
  if (!rc && (k_strides4[3] != 1 || v_strides4[3] != 1 || !aligned16(k_cache) || !aligned16(v_cache))) rc = GQA_ERR_ALIGNMENT;
  if (rc) return rc;
  int sm = 0;
  rc = current_device(&sm);
  if (rc) return rc;
  s.causal = causal ? 1 : 0;
  s.prefix = prefix_lens != nullptr;

  RaggedParams p{};
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.o = reinterpret_cast<uint16_t*>(o);
  p.lse = lse;
  p.q_st = q_strides3[0]; p.q_sh = q_strides3[1];
  p.o_st = o_strides3[0]; p.o_sh = o_strides3[1];
  p.cu = cu_query_lens;
  p.seq_lens = seq_lens;
  p.block_table = block_table;
  p.bt_stride = bt_stride;
  p.block_shift = pow2_shift(block_size);
  p.num_blocks = num_blocks;
  p.box = std::min(64, block_size);
  p.alibi = alibi_slopes;
  p.prefix = prefix_lens;
  p.key_starts = key_starts;
  p.window = window;
  p.causal = s.causal;
  p.n = num_seqs;
  p.num_tokens = num_tokens;
  p.hq = num_heads;
  p.hkv = num_kv_heads;
  p.group = s.group;
  p.max_len = max_seq_len;
  constexpr double kLog2e = 1.4426950408889634;
  const double sc = (double)scale * (cache_fp8 ? (double)k_scale : 1.0);
  p.scale_log2 = (float)(sc * kLog2e);
  p.cap_in = softcap > 0.f ? (float)(2.0 * kLog2e * sc / softcap) : 0.f;
  p.cap_out = softcap > 0.f ? (float)(softcap * kLog2e) : 0.f;
  if (softcap > 0.f) set_cap_polynomial(p, sc / softcap, softcap * kLog2e);
  p.v_scale = cache_fp8 ? v_scale : 1.f;
  p.mods = softcap > 0.f || alibi_slopes;

  const bool tile = ragged_uses_tile(s, cache_fp8 != 0);
  const RaggedShape ss = stream_part(s, tile);
  RaggedPlan sp = plan_ragged_stream(ss, sm), tp = plan_ragged_tile(s, sm);
  const bool have_ws = workspace && aligned16(workspace) && workspace_bytes >= ragged_ws_bytes(sp, tile ? &tp : nullptr, s);
  if (!have_ws) {  // no room for the partials: one CTA per tile
    sp.nsplit = tp.nsplit = 1;
    sp.chunk = tp.chunk = std::max(1, (max_seq_len + 127) / 128) * 128;
  }
  uint8_t* const counters = reinterpret_cast<uint8_t*>(workspace);
  uint8_t* const partials = counters + (size_t)kServingCounters * 4;
  CUtensorMap km, vm;
  rc = make_cache_map(&km, k_cache, k_strides4, num_blocks, block_size, num_kv_heads, head_dim, p.box, cache_fp8);
  if (!rc) rc = make_cache_map(&vm, v_cache, v_strides4, num_blocks, block_size, num_kv_heads, head_dim, p.box, cache_fp8);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == GQA_DTYPE_BF16;
  cudaError_t e = cudaSuccess;

  if (tile) {
    RaggedParams t = p;
    set_plan(t, tp);
    t.min_rows = kStreamMaxRows + 1;
    t.max_rows = INT_MAX;
    if (tp.nsplit > 1)
      ragged_ws_carve(tp, s, counters + (size_t)kServingCounters * 2, partials + ragged_partial_bytes(sp, s), &t);
    // Queries (d, head, token): a tile is bm tokens of the group's heads, token-major rows.
    const int64_t bhsd[4] = {q_strides3[0] * num_tokens, q_strides3[0], q_strides3[1], 1};
    CUtensorMap qm;
    rc = make_map(&qm, q, bhsd, 1, num_tokens, num_heads, head_dim, s.group, tp.block_m / 2);
    if (rc) return rc;
    const int64_t grid = (int64_t)tp.slots * num_kv_heads * tp.nsplit;
    if (grid > INT_MAX) return GQA_ERR_INVALID_ARG;
    if (head_dim == 128)
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
  const int64_t grid = (int64_t)sp.slots * num_kv_heads * sp.nsplit;
  if (grid > INT_MAX) return GQA_ERR_INVALID_ARG;
  if (cache_fp8)
    e = bf ? launch_ragged_stream_hd<128, true, true>(p, (unsigned)grid, km, vm, st)
           : launch_ragged_stream_hd<128, false, true>(p, (unsigned)grid, km, vm, st);
  else if (head_dim == 128)
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

// CTAs per row: enough for two waves' worth of CTAs over the device, at least 2048
// entries each.
VerifyPlan plan_verify(int64_t rows, int vocab, int sm_count) {
  VerifyPlan pl;
  const int64_t want = (4 * (int64_t)sm_count + rows - 1) / std::max<int64_t>(rows, 1);
  const int64_t most = std::max(1, vocab / 2048);
  pl.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
  pl.part = (((vocab + pl.nsplit - 1) / pl.nsplit) + 7) & ~7;
  return pl;
}

size_t verify_ws_bytes(int64_t units, const VerifyPlan& pl) {
  return (size_t)kServingCounters * 4 + 2 * align256((size_t)units * pl.nsplit * 4);
}

int verify_common(VerifyParams& p, int greedy, const int* draft_tokens, int64_t draft_token_stride, const void* target,
                  int64_t target_stride, const int* cu_query_lens, int* tokens, int* num_tokens, int num_seqs,
                  int num_rows, int max_drafts, int vocab, int dtype, void* workspace, size_t workspace_bytes,
                  int* grid) {
  if (num_seqs < 0 || num_rows < 0 || max_drafts < 0 || vocab <= 0 || vocab > INT_MAX - 64) return GQA_ERR_INVALID_ARG;
  if (max_drafts > kVerifyMaxDrafts || num_seqs > kServingCounters) return GQA_ERR_UNSUPPORTED;
  if (dtype != GQA_DTYPE_BF16 && dtype != GQA_DTYPE_F16 && dtype != GQA_DTYPE_F32) return GQA_ERR_UNSUPPORTED;
  if (num_seqs == 0) return GQA_OK;
  if (!cu_query_lens || !tokens || !num_tokens || (max_drafts > 0 && !draft_tokens) || (num_rows > 0 && !target) ||
      target_stride < 0 || draft_token_stride < 0)
    return GQA_ERR_INVALID_ARG;
  int sm = 0;
  const int rc = current_device(&sm);
  if (rc) return rc;
  const int64_t units = (int64_t)num_seqs * (greedy ? max_drafts + 1 : 1);
  const VerifyPlan pl = plan_verify(units, vocab, sm);
  if (!workspace || !aligned16(workspace) || workspace_bytes < verify_ws_bytes(units, pl)) return GQA_ERR_WORKSPACE;
  if (units * pl.nsplit > INT_MAX) return GQA_ERR_INVALID_ARG;
  p.draft_tokens = draft_tokens;
  p.dt_st = draft_token_stride;
  p.target = target;
  p.t_st = target_stride;
  p.cu = cu_query_lens;
  p.tokens = tokens;
  p.num_tokens = num_tokens;
  p.n = num_seqs;
  p.k = max_drafts;
  p.vocab = vocab;
  p.num_rows = num_rows;
  p.nsplit = pl.nsplit;
  p.part = pl.part;
  uint8_t* c = reinterpret_cast<uint8_t*>(workspace);
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

size_t gqa_verify_workspace_bytes(int num_seqs, int max_drafts, int vocab, int greedy) {
  int sm = 0;
  if (num_seqs <= 0 || max_drafts < 0 || vocab <= 0 || current_device(&sm)) return 0;
  const int64_t units = (int64_t)num_seqs * (greedy ? max_drafts + 1 : 1);
  return verify_ws_bytes(units, plan_verify(units, vocab, sm));
}

int gqa_verify_drafts(const int* draft_tokens, int64_t draft_token_stride, const void* target_probs, int64_t target_stride,
                      const void* draft_probs, const int64_t* draft_strides2, const float* uniforms,
                      int64_t uniform_stride, const float* exponentials, int64_t exponential_stride,
                      const int* cu_query_lens, int* tokens, int* num_tokens, int num_seqs, int num_rows, int max_drafts,
                      int vocab, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  VerifyParams p{};
  int grid = 0;
  int rc = verify_common(p, 0, draft_tokens, draft_token_stride, target_probs, target_stride, cu_query_lens, tokens,
                         num_tokens, num_seqs, num_rows, max_drafts, vocab, dtype, workspace, workspace_bytes, &grid);
  if (rc || num_seqs == 0) return rc;
  if (!exponentials || exponential_stride < 0 || (max_drafts > 0 && (!uniforms || uniform_stride < 0)) ||
      (draft_probs && (!draft_strides2 || draft_strides2[0] < 0 || draft_strides2[1] < 0)))
    return GQA_ERR_INVALID_ARG;
  p.draft = max_drafts > 0 ? draft_probs : nullptr;
  if (draft_probs) { p.d_sn = draft_strides2[0]; p.d_sk = draft_strides2[1]; }
  p.uniforms = uniforms;
  p.u_st = uniform_stride;
  p.expo = exponentials;
  p.e_st = exponential_stride;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e =
      dtype == GQA_DTYPE_F32 ? launch_pdl(gqa_verify_kernel<kProbF32>, dim3(grid), kVerifyThreads, 0, st, p)
      : dtype == GQA_DTYPE_BF16 ? launch_pdl(gqa_verify_kernel<kProbBf16>, dim3(grid), kVerifyThreads, 0, st, p)
                                : launch_pdl(gqa_verify_kernel<kProbF16>, dim3(grid), kVerifyThreads, 0, st, p);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

int gqa_verify_greedy(const int* draft_tokens, int64_t draft_token_stride, const void* target, int64_t target_stride,
                      const int* cu_query_lens, int* tokens, int* num_tokens, int num_seqs, int num_rows, int max_drafts,
                      int vocab, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  VerifyParams p{};
  int grid = 0;
  const int rc = verify_common(p, 1, draft_tokens, draft_token_stride, target, target_stride, cu_query_lens, tokens,
                               num_tokens, num_seqs, num_rows, max_drafts, vocab, dtype, workspace, workspace_bytes, &grid);
  if (rc || num_seqs == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e =
      dtype == GQA_DTYPE_F32 ? launch_pdl(gqa_verify_greedy_kernel<kProbF32>, dim3(grid), kVerifyThreads, 0, st, p)
      : dtype == GQA_DTYPE_BF16 ? launch_pdl(gqa_verify_greedy_kernel<kProbBf16>, dim3(grid), kVerifyThreads, 0, st, p)
                                : launch_pdl(gqa_verify_greedy_kernel<kProbF16>, dim3(grid), kVerifyThreads, 0, st, p);
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"
