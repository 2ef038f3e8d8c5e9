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
static_assert(kServingCounters * 4 == GQA_SERVING_COUNTER_BYTES, "the part of a workspace that callers zero");

template <int HD, bool BF, bool F8>
cudaError_t launch_ragged_stream(const RaggedParams& p, unsigned grid, const CUtensorMap& km, const CUtensorMap& vm,
                                 cudaStream_t st) {
  using Cfg = StreamCfg<F8 ? 64 : HD>;
  return launch_pdl(gqa_ragged_stream_kernel<HD, BF, F8>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, km, vm);
}

template <int HD, bool BF>
cudaError_t launch_ragged_tile(const RaggedParams& p, unsigned grid, const CUtensorMap& qm, const CUtensorMap& km,
                                  const CUtensorMap& vm, cudaStream_t st) {
  using Cfg = RaggedTileCfg<HD>;
  if (p.alibi && p.cap_in != 0.f)
    return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedCapBias>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
  if (p.alibi)
    return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedBias>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
  if (p.cap_in != 0.f)
    return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedCap>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
  return launch_pdl(gqa_ragged_tile_kernel<HD, BF, kRaggedPlain>, grid, Cfg::kThreads, Cfg::kSmemBytes, st, p, qm, km, vm);
}

// Shared memory opt-in, and the tcgen05 form's setmaxnreg split must fit the registers the launch holds.
int prepare_ragged() {
  int rc = GQA_OK;
  auto prep = [&](auto kernel, int smem, int regs) {
    if (set_smem(kernel, smem) != cudaSuccess) rc = rc ? rc : GQA_ERR_CUDA;
    if (!rc && regs) rc = check_reg_split(kernel, RaggedTileCfg<128>::kThreads, regs);
  };
  constexpr int kRegs = RaggedTileCfg<128>::kRegsNeeded;
#define GQA_PREP_RAGGED(HD, BF)                                                              \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedPlain>, RaggedTileCfg<HD>::kSmemBytes, kRegs);  \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedCap>, RaggedTileCfg<HD>::kSmemBytes, kRegs);    \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedBias>, RaggedTileCfg<HD>::kSmemBytes, kRegs);   \
  prep(gqa_ragged_tile_kernel<HD, BF, kRaggedCapBias>, RaggedTileCfg<HD>::kSmemBytes, kRegs); \
  prep(gqa_ragged_stream_kernel<HD, BF, false>, StreamCfg<HD>::kSmemBytes, 0)
  GQA_PREP_RAGGED(128, true); GQA_PREP_RAGGED(128, false); GQA_PREP_RAGGED(64, true); GQA_PREP_RAGGED(64, false);
#undef GQA_PREP_RAGGED
  prep(gqa_ragged_stream_kernel<128, true, true>, StreamCfg<64>::kSmemBytes, 0);
  prep(gqa_ragged_stream_kernel<128, false, true>, StreamCfg<64>::kSmemBytes, 0);
  return rc;
}

// current_device() for the ragged attention: its kernels are loaded and checked at its own
// first call on the device, so that a caller of the dense entry points does not pay for them
// and cannot be refused because of them.
int current_device_ragged(int* sm_count) {
  const int rc = current_device(sm_count);
  if (rc) return rc;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return GQA_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lock(g_mutex);
  DeviceState& st = g_devices[dev];
  if (!st.ragged_ready) {
    st.ragged_status = prepare_ragged();
    st.ragged_ready = true;
  }
  return st.ragged_status;
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
                   std::min(a.max_query_len, a.num_tokens), a.max_seq_len, a.head_dim,
                   a.window < a.max_seq_len ? a.window : 0,  // a window of all keys is none, and its arithmetic may overflow
                   a.causal ? 1 : 0,
                   a.prefix_lens != nullptr};
  return GQA_OK;
}

// The launch: the two forms' tilings and their CTAs.
struct RaggedPlan {
  RaggedTiling stream, tile;
  int64_t stream_ctas, tile_ctas;
};

int64_t tiling_units(const RaggedTiling& t, int hkv) { return (int64_t)t.slots * hkv; }

// Keys that a tile of block_m tokens sees at most.
int ragged_span(const RaggedShape& s, int block_m) {
  int64_t span = s.max_len;
  if (s.window > 0 && s.causal && !s.prefix) span = std::min<int64_t>(span, (int64_t)s.window + block_m - 1 + 64);
  return (int)std::max<int64_t>(1, span);
}

// Key split of `units` tiles that see up to `span` keys each, `keys` at a time (a stage),
// for one CTA per SM: the split of the fewest wave-stages, a CTA's fixed cost (set-up,
// pipeline ramp, merge, partials) counting `fixed` stages. Only the longest request's
// bound is known; shorter ones use fewer chunks and their CTAs return at once.
void split_keys(RaggedTiling& t, int64_t units, int span, int keys, int sm_count, double fixed, int most) {
  const int stages = (span + keys - 1) / keys;
  t.nsplit = 1;
  t.chunk = stages * keys;
  double best = 1e300;
  for (int ns = 1; ns <= std::min(stages, most); ++ns) {
    const int chunk = (stages + ns - 1) / ns;
    if ((stages + chunk - 1) / chunk != ns) continue;
    const double cost = std::ceil((double)units * ns / sm_count) * (chunk + fixed);
    if (cost < best - 1e-9) {
      best = cost;
      t.nsplit = ns;
      t.chunk = chunk * keys;
    }
  }
}

RaggedPlan plan_ragged(const RaggedShape& s, bool fp8, int sm_count) {
  RaggedPlan pl{};
  const int stream_rows = fp8 ? kStreamMaxRows : kRaggedStreamRows;
  const bool tile = !fp8 && (int64_t)s.max_q * s.group > stream_rows;
  // A single request of which the bounds allow the tcgen05 form takes it, whatever its length.
  const bool stream = !tile || (s.group <= stream_rows && s.n > 1);
  if (tile) {
    // Pairs of 128-row query tiles: at most tokens / block_m + (requests of the form) of them.
    RaggedTiling& t = pl.tile;
    t.block_m = 2 * (128 / s.group);
    t.rows = 256;
    t.min_rows = stream ? stream_rows + 1 : 0;
    t.max_rows = INT_MAX;
    const int64_t longest = std::min<int64_t>(s.n, (int64_t)s.tokens * s.group / std::max(1, t.min_rows));
    t.slots = (int)std::min<int64_t>((int64_t)s.tokens / t.block_m + longest, INT_MAX);
    const int64_t units = tiling_units(t, s.hkv);
    const int keys = s.head_dim == 128 ? RaggedTileCfg<128>::kBN : RaggedTileCfg<64>::kBN;
    const int span = ragged_span(s, t.block_m) + keys;
    const int most = (units < sm_count && units <= kServingCounters / 2) ? std::max(1, std::min(kMaxRaggedChunks, span / (2 * keys))) : 1;
    split_keys(t, units, span, keys, sm_count, 12.0, most);
    pl.tile_ctas = units * t.nsplit;
  }
  if (stream) {
    RaggedTiling& t = pl.stream;
    const int max_q = tile ? stream_rows / s.group : s.max_q;
    t.block_m = std::max(1, std::min(max_q, stream_rows / s.group));
    t.rows = s.group * t.block_m;
    t.one_tile = max_q <= t.block_m;
    t.slots = t.one_tile ? s.n : s.tokens / t.block_m + s.n;
    t.min_rows = 0;
    t.max_rows = tile ? stream_rows : INT_MAX;
    const int64_t tiles = t.one_tile ? std::min(s.n, s.tokens) : std::min(t.slots, s.tokens);
    split_keys(t, tiles * s.hkv, ragged_span(s, t.block_m), 128, sm_count, 4.0,
               tiling_units(t, s.hkv) <= kServingCounters / 2 ? kMaxSplits : 1);
    pl.stream_ctas = tiling_units(t, s.hkv) * t.nsplit;
  }
  return pl;
}

size_t ragged_partial_bytes(const RaggedTiling& t, const RaggedShape& s) {
  if (t.nsplit <= 1) return 0;
  const size_t n = (size_t)tiling_units(t, s.hkv) * t.nsplit * t.rows;
  return 2 * align256(n * 4) + align256(n * s.head_dim * 4);
}

// Counters first (half for each form), then the streaming form's partials, then the other's.
size_t ragged_ws_bytes(const RaggedPlan& pl, const RaggedShape& s) {
  const size_t n = ragged_partial_bytes(pl.stream, s) + ragged_partial_bytes(pl.tile, s);
  return n ? (size_t)kServingCounters * 4 + n : 0;
}

void carve_partials(RaggedTiling& t, const RaggedShape& s, uint8_t* counters, uint8_t* c) {
  const size_t n = (size_t)tiling_units(t, s.hkv) * t.nsplit * t.rows;
  t.ws_cnt = reinterpret_cast<unsigned*>(counters);
  t.ws_m = reinterpret_cast<float*>(c);
  c += align256(n * 4);
  t.ws_l = reinterpret_cast<float*>(c);
  c += align256(n * 4);
  t.ws_acc = reinterpret_cast<float*>(c);
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
  if (!aligned16(a.q_out) || !aligned16(a.cos_sin) || !aligned16(a.k_dst) || !aligned16(a.v_dst) || !aligned16(a.q_weight) || !aligned16(a.k_weight))
    return GQA_ERR_ALIGNMENT;
  int rc = check_strides3(a.q, a.q_strides, 8);
  if (!rc) rc = check_strides3(a.k, a.k_strides, 8);
  if (!rc && cached) rc = check_strides3(a.v, a.v_strides, 8);
  if (rc) return rc;
  int sm = 0;
  rc = current_device(&sm);
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
  p.eps = a.eps;
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a.dtype == GQA_DTYPE_BF16;
  // Both kinds of units get CTAs in proportion, at most what fits the device at once.
  const int groups = a.head_dim == 128 ? RopeCfg<128>::kGroups : RopeCfg<64>::kGroups;
  const int64_t q_units = (int64_t)a.num_tokens * ((a.num_heads + kRopeRows - 1) / kRopeRows);
  const int64_t kv_units = (int64_t)a.num_tokens * ((a.num_kv_heads + kRopeRows / 2 - 1) / (kRopeRows / 2));
  if (q_units > INT_MAX / 2 || kv_units > INT_MAX / 2) return GQA_ERR_INVALID_ARG;
  const int64_t q_need = (q_units + groups - 1) / groups, kv_need = (kv_units + groups - 1) / groups;
  const int64_t fit = (int64_t)kRopeCtas * sm;
  int64_t q_ctas = q_need, kv_ctas = kv_need;
  if (q_need + kv_need > fit) {
    kv_ctas = std::max<int64_t>(1, std::min(kv_need, fit * kv_units / (q_units + kv_units)));
    q_ctas = std::min(q_need, fit - kv_ctas);
  }
  p.q_ctas = (int)q_ctas;
  const dim3 grid((unsigned)(q_ctas + kv_ctas));
  cudaError_t e;
#define GQA_ROPE(D, BF, F8)                                                                                     \
  e = a.interleaved ? launch_pdl(gqa_rope_kernel<D, BF, F8, true>, grid, kRopeThreads, 0, st, p)                \
                    : launch_pdl(gqa_rope_kernel<D, BF, F8, false>, grid, kRopeThreads, 0, st, p)
#define GQA_ROPE_D(D)                                                                                           \
  if (a.cache_fp8) { if (bf) { GQA_ROPE(D, true, true); } else { GQA_ROPE(D, false, true); } }                  \
  else { if (bf) { GQA_ROPE(D, true, false); } else { GQA_ROPE(D, false, false); } }
  if (a.head_dim == 128) { GQA_ROPE_D(128) } else { GQA_ROPE_D(64) }
#undef GQA_ROPE_D
#undef GQA_ROPE
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

size_t gqa_ragged_fwd_workspace_bytes(const gqa_ragged_args* args) {
  RaggedShape s;
  int sm = 0;
  if (!args || check_ragged_shape(*args, &s) || s.n == 0 || s.tokens == 0 || s.max_q == 0 || current_device(&sm)) return 0;
  return ragged_ws_bytes(plan_ragged(s, args->cache_fp8 != 0, sm), s);
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
  rc = current_device_ragged(&sm);
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
  p.alibi = a.alibi_slopes;
  p.prefix = a.prefix_lens;
  p.key_starts = a.key_starts;
  p.window = s.window;
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
  p.linear_bias = a.causal && !a.prefix_lens;

  RaggedPlan pl = plan_ragged(s, a.cache_fp8 != 0, sm);
  if (a.workspace) {
    if (!aligned16(a.workspace)) return GQA_ERR_ALIGNMENT;
    if (a.workspace_bytes < ragged_ws_bytes(pl, s)) return GQA_ERR_WORKSPACE;
    uint8_t* const counters = reinterpret_cast<uint8_t*>(a.workspace);
    uint8_t* const partials = counters + (size_t)kServingCounters * 4;
    if (pl.stream.nsplit > 1) carve_partials(pl.stream, s, counters, partials);
    if (pl.tile.nsplit > 1)
      carve_partials(pl.tile, s, counters + (size_t)kServingCounters * 2, partials + ragged_partial_bytes(pl.stream, s));
  } else {  // nowhere to leave partials: one CTA per tile
    pl.stream_ctas /= std::max(1, pl.stream.nsplit);
    pl.tile_ctas /= std::max(1, pl.tile.nsplit);
    pl.stream.nsplit = pl.tile.nsplit = 1;
    pl.stream.chunk = pl.tile.chunk = INT_MAX / 2 / 640 * 640;  // one chunk, a multiple of both forms' stages
  }
  if (pl.tile_ctas + pl.stream_ctas > INT_MAX) return GQA_ERR_INVALID_ARG;
  const unsigned grid = (unsigned)(pl.tile_ctas + pl.stream_ctas);
  p.stream = pl.stream;
  p.tile = pl.tile;
  p.tile_ctas = (unsigned)pl.tile_ctas;
  p.box = std::min(64, a.block_size);

  CUtensorMap km, vm;
  rc = make_cache_map(&km, a.k_cache, a.k_strides, a.num_blocks, a.block_size, a.num_kv_heads, a.head_dim, p.box, a.cache_fp8);
  if (!rc) rc = make_cache_map(&vm, a.v_cache, a.v_strides, a.num_blocks, a.block_size, a.num_kv_heads, a.head_dim, p.box, a.cache_fp8);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a.dtype == GQA_DTYPE_BF16;
  cudaError_t e = cudaSuccess;
  if (pl.tile_ctas > 0) {
    // Queries (d, head, token): a tile is tokens of the group's heads, token-major rows.
    const int64_t bhsd[4] = {a.q_strides[0] * a.num_tokens, a.q_strides[0], a.q_strides[1], 1};
    CUtensorMap qm;
    rc = make_map(&qm, a.q, bhsd, 1, a.num_tokens, a.num_heads, a.head_dim, s.group, pl.tile.block_m / 2);
    if (rc) return rc;
    if (a.head_dim == 128)
      e = bf ? launch_ragged_tile<128, true>(p, grid, qm, km, vm, st) : launch_ragged_tile<128, false>(p, grid, qm, km, vm, st);
    else
      e = bf ? launch_ragged_tile<64, true>(p, grid, qm, km, vm, st) : launch_ragged_tile<64, false>(p, grid, qm, km, vm, st);
  } else if (a.cache_fp8) {
    e = bf ? launch_ragged_stream<128, true, true>(p, grid, km, vm, st) : launch_ragged_stream<128, false, true>(p, grid, km, vm, st);
  } else if (a.head_dim == 128) {
    e = bf ? launch_ragged_stream<128, true, false>(p, grid, km, vm, st) : launch_ragged_stream<128, false, false>(p, grid, km, vm, st);
  } else {
    e = bf ? launch_ragged_stream<64, true, false>(p, grid, km, vm, st) : launch_ragged_stream<64, false, false>(p, grid, km, vm, st);
  }
  return e == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // extern "C"

// ----------------------------------------------------------------------------- draft verification
namespace gqa {
namespace {

struct VerifyPlan {
  int nsplit, part;
};

// CTAs per row: about one wave over the device, at least 1024 entries each. Five CTAs fit
// an SM (registers); of the greedy scan's rows -- the most that the requests can have -- a
// good part is usually absent.
VerifyPlan plan_verify(int64_t rows, int vocab, int sm_count, bool greedy) {
  VerifyPlan pl;
  const int64_t want = (int64_t)sm_count * (greedy ? 8 : 5) / std::max<int64_t>(rows, 1);
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
