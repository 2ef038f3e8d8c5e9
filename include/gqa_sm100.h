/*
 * gqa_sm100.h -- C ABI of libgqa_sm100.so, the B200 (sm_100a) GQA
 * flash-attention forward.
 *
 * Conventions shared by every entry point:
 *   - All pointers are device pointers owned by the caller; the library never
 *     allocates device memory. Kernels that need scratch take a caller-owned
 *     workspace (see *_workspace_bytes).
 *   - Tensors use the reference layout: Q/O (batch, num_heads, seq_q, head_dim),
 *     K/V (batch, num_kv_heads, seq_kv, head_dim). Strides are in ELEMENTS, in
 *     dimension order (b, h, s, d). The d stride must be 1 and every other
 *     stride a multiple of 8 elements (16 bytes); base pointers 16-byte aligned.
 *   - dtype: GQA_DTYPE_F16 or GQA_DTYPE_BF16 (q, k, v and o share it).
 *   - scale_log2 = head_dim^-0.5 * log2(e); the softmax is evaluated with exp2.
 *   - causal = 1: query row i (in key coordinates i + seq_kv - seq_q) attends
 *     to keys [0, i + seq_kv - seq_q] (bottom-right alignment). A row with no
 *     visible key produces NaN, as the reference does.
 *   - Work is enqueued on `stream` (a cudaStream_t; NULL = legacy default);
 *     no entry point synchronises. Return 0 on success or a GQA_ERR_* code;
 *     gqa_strerror() turns a code into text.
 *   - Entry points are stateless and re-entrant; per-device attributes are
 *     cached once under a mutex.
 */
#ifndef GQA_SM100_H_
#define GQA_SM100_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GQA_OK 0
#define GQA_ERR_INVALID_ARG 1   /* bad shape, null pointer, negative size      */
#define GQA_ERR_UNSUPPORTED 2   /* head_dim not 64/128, group size not 2^k ... */
#define GQA_ERR_ALIGNMENT 3     /* stride or base pointer not 16-byte aligned  */
#define GQA_ERR_CUDA 4          /* a CUDA runtime/driver call failed           */
#define GQA_ERR_TIMEOUT 5       /* a bounded in-kernel wait expired            */
#define GQA_ERR_WORKSPACE 6     /* workspace missing or too small              */
#define GQA_ERR_NO_DEVICE 7     /* no sm_100 device current                    */
#define GQA_ERR_SCRATCH_LIMIT 8 /* problem needs more than the static scratch  */
#define GQA_ERR_DEBUG_CHECK 9   /* a debug build's address/coordinate check failed (device error word) */

#define GQA_DTYPE_F16 0
#define GQA_DTYPE_BF16 1
#define GQA_DTYPE_F32 2 /* gqa_verify_* only */

/* Text for a status code (static storage). */
const char* gqa_strerror(int code);

/* Library version, major*10000 + minor*100 + patch (0.1.0 -> 100). */
int gqa_version(void);

/*
 * Single-pass GQA forward: O = softmax(Q K^T * scale) V with the group's
 * query heads packed into the M dimension of each tile.
 * Replaces the launch of gqa_fwd_kernel in gqa_kernels/dispatch.py:50-61
 * (kernel body gqa_kernels/gqa_fwd.py:33-109).
 * Packed rows (group_size * seq_q) >= 128 run the tcgen05/TMEM prefill
 * kernel; fewer run the HBM-streaming kernel, which may split the key range
 * across CTAs when `workspace` is large enough
 * (gqa_fwd_workspace_bytes) -- the combine is fused into the same launch.
 */
size_t gqa_fwd_workspace_bytes(int batch, int num_heads, int num_kv_heads, int seq_q, int seq_kv,
                               int head_dim);
int gqa_fwd(const void* q, const void* k, const void* v, void* o, const int64_t* q_strides4,
            const int64_t* k_strides4, const int64_t* v_strides4, const int64_t* o_strides4, int batch,
            int num_heads, int num_kv_heads, int seq_q, int seq_kv, int head_dim, float scale_log2,
            int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Split-KV first pass: per-(row, split) partial softmax statistics over key
 * chunk [s*ceil(seq_kv/splits), min((s+1)*ceil(seq_kv/splits), seq_kv)).
 * m_p, l_p: float32 (batch, num_heads, seq_q, splits) with strides p_strides4;
 * acc_p: float32 (batch, num_heads, seq_q, splits, head_dim), strides a_strides5.
 * m is in log2 units (already multiplied by scale_log2), l = sum exp2(s - m),
 * acc = sum exp2(s - m) v (unnormalised). An empty chunk gives (-inf, 0, 0).
 * Replaces gqa_split_first_kernel, gqa_kernels/gqa_split.py:26-112, launched at :168-183.
 */
int gqa_split_first(const void* q, const void* k, const void* v, float* m_p, float* l_p, float* acc_p,
                    const int64_t* q_strides4, const int64_t* k_strides4, const int64_t* v_strides4,
                    const int64_t* p_strides4, const int64_t* a_strides5, int batch, int num_heads,
                    int num_kv_heads, int seq_q, int seq_kv, int head_dim, float scale_log2, int causal,
                    int splits, int dtype, void* stream);

/*
 * Split-KV second pass: log-sum-exp combine of the partials above into O.
 * Replaces gqa_split_reduce_kernel, gqa_kernels/gqa_split.py:115-147, launched at :185-193.
 */
int gqa_split_reduce(const float* m_p, const float* l_p, const float* acc_p, void* o,
                     const int64_t* p_strides4, const int64_t* a_strides5, const int64_t* o_strides4,
                     int batch, int num_heads, int seq_q, int head_dim, int splits, int dtype, void* stream);

/*
 * One-launch split-KV forward: the key range is split into chunks sized for
 * the device's SM count and the last CTA of each (batch, kv_head, q-block)
 * combines the chunk partials in-kernel (atomic ticket, no second launch).
 * Same result as split_kv_forward, gqa_kernels/gqa_split.py:153-194.
 * The workspace must hold gqa_split_fused_workspace_bytes() bytes and its
 * ticket counters must be zero before the first call; every call leaves them
 * zero again. Calls sharing a workspace must be ordered on one stream.
 */
size_t gqa_split_fused_workspace_bytes(int batch, int num_heads, int num_kv_heads, int seq_q, int seq_kv,
                                       int head_dim);
int gqa_split_fused(const void* q, const void* k, const void* v, void* o, const int64_t* q_strides4,
                    const int64_t* k_strides4, const int64_t* v_strides4, const int64_t* o_strides4,
                    int batch, int num_heads, int num_kv_heads, int seq_q, int seq_kv, int head_dim,
                    float scale_log2, int causal, int dtype, void* workspace, size_t workspace_bytes,
                    void* stream);

/*
 * gqa_split_fused without a workspace argument, for callers that cannot
 * allocate device memory -- e.g. a host bound to this C ABI through an FFI
 * (Go, Java, Rust) that owns no CUDA allocator, or an engine that reserves all
 * of HBM for its own pool up front, where a cudaMalloc would fail or stall the
 * device in the middle of a decode step. The scratch lives in a static
 * __device__ array of GQA_NOALLOC_SCRATCH_BYTES that every GPU loading the
 * library holds until the process exits; the library calls no cudaMalloc,
 * cudaFree or allocating routine here. Problems whose scratch would exceed it
 * return GQA_ERR_SCRATCH_LIMIT (gqa_split_fused_workspace_bytes gives the
 * need). The first call on a device looks up the array's device address
 * (cudaGetSymbolAddress) with that device current; make that first call
 * before any stream capture. All calls share the one array: calls that
 * overlap on the GPU (other streams, other threads) race and must be ordered
 * by the caller. No counterpart in the reference.
 */
#define GQA_NOALLOC_SCRATCH_BYTES (4u << 20)
int gqa_split_fused_noalloc(const void* q, const void* k, const void* v, void* o, const int64_t* q_strides4,
                            const int64_t* k_strides4, const int64_t* v_strides4, const int64_t* o_strides4,
                            int batch, int num_heads, int num_kv_heads, int seq_q, int seq_kv, int head_dim,
                            float scale_log2, int causal, int dtype, void* stream);

/*
 * Partial attention over one shard of the key axis, for a key range split
 * across GPUs. k and v hold keys [kv_offset, kv_offset + seq_kv_local) of a
 * sequence of seq_kv_total keys; causal masking uses global key positions.
 * Outputs are float32, contiguous: m_out/l_out (batch, num_heads, seq_q),
 * acc_out (batch, num_heads, seq_q, head_dim), with the meaning of
 * gqa_split_first's (m, l, acc) for this shard. seq_kv_local may be 0 (a rank
 * whose share of the keys is empty): the outputs are then (-inf, 0, 0) for every
 * row, which gqa_lse_combine weighs 0, and k/v are not read.
 * No reference counterpart (the reference is single-GPU); the partial
 * definition follows gqa_kernels/gqa_split.py:102-112.
 */
size_t gqa_partial_workspace_bytes(int batch, int num_heads, int num_kv_heads, int seq_q, int seq_kv_local,
                                   int head_dim);
int gqa_partial(const void* q, const void* k, const void* v, float* m_out, float* l_out, float* acc_out,
                const int64_t* q_strides4, const int64_t* k_strides4, const int64_t* v_strides4, int batch,
                int num_heads, int num_kv_heads, int seq_q, int seq_kv_local, int kv_offset, int seq_kv_total,
                int head_dim, float scale_log2, int causal, int dtype, void* workspace, size_t workspace_bytes,
                void* stream);

/*
 * Log-sum-exp combine of `nparts` partial sets (e.g. one per GPU). Part s
 * holds, for row r = (b*num_heads + h)*seq_q + i, the values
 * m_parts[s*ml_part_stride + r], l_parts[s*ml_part_stride + r] and
 * acc_parts[s*acc_part_stride + r*head_dim + d] (float32), i.e. gqa_partial's
 * outputs stacked along a leading axis -- either as three stacked arrays or as
 * one packed [m | l | acc] buffer per part, as an all-gather produces.
 * Algebra of gqa_kernels/gqa_split.py:137-144, applied across parts.
 */
int gqa_lse_combine(const float* m_parts, const float* l_parts, const float* acc_parts, int nparts,
                    int64_t ml_part_stride, int64_t acc_part_stride, void* o, const int64_t* o_strides4, int batch,
                    int num_heads, int seq_q, int head_dim, int dtype, void* stream);

/*
 * Peer exchange: the key-sharded combine across the GPUs of one node without a
 * collective library. gqa_partial's outputs go straight from the partial kernel
 * into every rank's receive buffer (plain stores, over NVLink for the other
 * ranks), and each rank's combine waits for them in-kernel. It replaces
 * gqa_partial + an all-gather + gqa_lse_combine with two launches and no
 * collective call. No reference counterpart (the reference is single-GPU); the
 * algebra is gqa_kernels/gqa_split.py:137-144's across ranks.
 *
 * Each rank holds one exchange buffer (gqa_exchange_alloc, zeroed; it allocates
 * and synchronises, a setup call): [2 parities][nranks slots][slot_floats
 * floats] of packed partials [m | l | pad to 16 B | acc] (the layout of
 * gqa_lse_combine's packed form), then nranks uint64 counters (one per source
 * rank), then one uint64 call counter (the epoch). Every rank maps the other
 * ranks' buffers once: gqa_ipc_handle exports this process's buffer as a
 * GQA_IPC_HANDLE_BYTES handle, gqa_ipc_open maps another process's (CUDA IPC,
 * same node; never a multicast mapping), gqa_ipc_close unmaps it.
 *
 * Per call, on every rank, in this order on one stream:
 *   gqa_epoch_bump(epoch)       one thread: epoch += 1
 *   gqa_partial_peer(...)       writes this rank's partial into slot `rank`
 *                               of parity (epoch & 1) of every rank's buffer,
 *                               then adds 1 per unit to that rank's counter
 *                               for this source (system-scope release)
 *   gqa_lse_combine_peer(...)   waits (bounded) until every source's counter
 *                               reaches epoch x units, then combines into o
 * Every rank makes the same calls with the same shapes (so the epochs and unit
 * counts agree; gqa_partial_units gives the count), and every rank must hold at
 * least one key (seq_kv_local > 0; else GQA_ERR_UNSUPPORTED: use the all-gather
 * form, which accepts empty shards). Two parities let a rank start its next
 * call while another still reads this one: a rank cannot reach the call after
 * next before every rank has finished this call's combine. A source that never
 * arrives ends the combine's wait after the wait limit with GQA_ERR_TIMEOUT in
 * the device error word (gqa_device_error) and o unwritten.
 * peer_bases[i] / peer_cnts[i] are rank i's buffer and counters as this
 * process maps them (its own for i == rank); npeer <= 8.
 */
#define GQA_IPC_HANDLE_BYTES 64
int gqa_exchange_alloc(size_t bytes, void** ptr);
int gqa_exchange_free(void* ptr);
int gqa_ipc_handle(const void* ptr, void* handle);
int gqa_ipc_open(const void* handle, void** ptr);
int gqa_ipc_close(void* ptr);
int gqa_epoch_bump(unsigned long long* epoch, void* stream);
int gqa_partial_units(int batch, int num_heads, int num_kv_heads, int seq_q, int head_dim, int* units);
int gqa_partial_peer(const void* q, const void* k, const void* v, const int64_t* q_strides4, const int64_t* k_strides4,
                     const int64_t* v_strides4, int batch, int num_heads, int num_kv_heads, int seq_q,
                     int seq_kv_local, int kv_offset, int seq_kv_total, int head_dim, float scale_log2, int causal,
                     int dtype, float* const* peer_bases, unsigned long long* const* peer_cnts, int npeer, int rank,
                     const unsigned long long* epoch, int64_t slot_floats, int64_t parity_floats, void* workspace,
                     size_t workspace_bytes, void* stream);
int gqa_lse_combine_peer(const float* recv, const unsigned long long* cnt, const unsigned long long* epoch,
                         int nparts, int64_t slot_floats, int64_t parity_floats, int units, void* o,
                         const int64_t* o_strides4, int batch, int num_heads, int seq_q, int head_dim, int dtype,
                         void* stream);

/*
 * Paged decode: one new query token per sequence attends to that sequence's
 * cached keys, read from a paged K/V cache in the layout vLLM uses,
 * k_cache/v_cache (num_blocks, block_size, num_kv_heads, head_dim), contiguous.
 * Sequence b holds seq_lens[b] keys; its key k lives in physical block
 * block_table[b * bt_stride + k / block_size] at position k % block_size.
 * q/o are (num_seqs, num_heads, head_dim) with element strides q_strides3 /
 * o_strides3 (seq, head, d; d stride 1). block_size must be a power of two
 * >= 64; block_table and seq_lens are int32 device arrays; max_seq_len bounds
 * every seq_lens[b] and sizes the key split (the workspace query takes it).
 * A sequence with no key gives NaN, as the dense path does. The split
 * combine is fused into the launch when the workspace (zeroed before first
 * use; every call leaves it zero) holds gqa_paged_decode_workspace_bytes().
 * No reference counterpart: the reference's roadmap names a vLLM-shaped
 * interface (README.md:144); the attention is gqa_kernels/gqa_split.py's.
 */
size_t gqa_paged_decode_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads, int max_seq_len,
                                        int head_dim);
int gqa_paged_decode(const void* q, const void* k_cache, const void* v_cache, void* o, const int64_t* q_strides3,
                     const int64_t* o_strides3, const int* block_table, int bt_stride, const int* seq_lens,
                     int num_seqs, int num_heads, int num_kv_heads, int head_dim, int block_size, int num_blocks,
                     int max_seq_len, float scale_log2, int dtype, void* workspace, size_t workspace_bytes,
                     void* stream);

/*
 * Paged forward (chunked prefill over a paged cache): each sequence's seq_q new
 * query tokens attend to its cached keys, read from the same vLLM-layout caches
 * as gqa_paged_decode. q/o are (num_seqs, num_heads, seq_q, head_dim) with
 * element strides q_strides / o_strides (the gqa_fwd convention). The queries
 * of sequence b are its last seq_q positions: with `causal`, query i sees keys
 * [0, seq_lens[b] - seq_q + i] (bottom-right alignment per sequence, the dense
 * path's rule); without, all seq_lens[b] keys. Rows that see no key give NaN.
 * Short chunks (group * seq_q <= 64) run the streaming kernel, longer ones the
 * tcgen05 prefill kernel, whose producer reads K/V tiles through the block
 * table. Cache slots past seq_lens[b] in a sequence's last block are read but
 * never reach O (their V rows are zeroed in shared memory before the PV MMA), so
 * stale or non-finite values there are harmless.
 * The key split is sized by max_seq_len; its workspace (zeroed before first
 * use; every call leaves it zero) is gqa_paged_fwd_workspace_bytes(). Called
 * with seq_q = 1 and causal = 0 this is gqa_paged_decode.
 * No reference counterpart: the roadmap's vLLM-shaped interface (README.md:144)
 * over the attention of gqa_kernels/gqa_fwd.py.
 */
size_t gqa_paged_fwd_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads, int seq_q, int max_seq_len,
                                     int head_dim);
int gqa_paged_fwd(const void* q, const void* k_cache, const void* v_cache, void* o, const int64_t* q_strides,
                  const int64_t* o_strides, const int* block_table, int bt_stride, const int* seq_lens,
                  int num_seqs, int num_heads, int num_kv_heads, int seq_q, int head_dim, int block_size,
                  int num_blocks, int max_seq_len, float scale_log2, int causal, int dtype, void* workspace,
                  size_t workspace_bytes, void* stream);

/*
 * gqa_paged_fwd over fp8 caches: k_cache/v_cache hold e4m3 values (one byte
 * each, same layout), and key = stored key x k_scale, value = stored value x
 * v_scale (vLLM's fp8 KV-cache convention; both scales > 0). q/o keep `dtype`
 * (bf16 or fp16). head_dim must be 128 and group * seq_q <= 64 (decode and
 * short chunks: the streaming kernel, whose K/V fragments are converted exactly
 * from e4m3 to f16 in registers; both MMAs run in f16, so |q| must stay within
 * the f16 range). Otherwise GQA_ERR_UNSUPPORTED. The workspace is
 * gqa_paged_fwd_workspace_bytes(). Halves the bytes streamed per key against
 * 16-bit caches.
 * No reference counterpart: the reference's K/V are bf16 or fp16 only.
 */
int gqa_paged_fwd_kv8(const void* q, const void* k_cache, const void* v_cache, void* o, const int64_t* q_strides,
                      const int64_t* o_strides, const int* block_table, int bt_stride, const int* seq_lens,
                      int num_seqs, int num_heads, int num_kv_heads, int seq_q, int head_dim, int block_size,
                      int num_blocks, int max_seq_len, float scale_log2, float k_scale, float v_scale, int causal,
                      int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Cache write of the paged interface (vLLM's reshape_and_cache_flash): token t's K
 * and V rows, key/value (num_tokens, num_kv_heads, head_dim) with element strides
 * k_strides3 / v_strides3 (d stride 1, the others multiples of 8 elements), go to
 * slot slot_mapping[t] (int64; block = slot / block_size, position = slot %
 * block_size) of the (num_blocks, block_size, num_kv_heads, head_dim) caches. A
 * negative slot is a padding token and is skipped. 16-bit caches (dtype) receive the
 * rows unchanged; with cache_fp8 the caches are e4m3 and receive x / k_scale (x /
 * v_scale) rounded to nearest even and saturated to +-448, vLLM's convention (real
 * value = stored value x scale; scales > 0). A slot >= num_blocks * block_size is not
 * written: its row is skipped and GQA_ERR_INVALID_ARG is recorded in the device error
 * word (site 201; gqa_device_error). Tokens must map to distinct slots.
 * No reference counterpart: the cache-write half of the roadmap's vLLM-shaped
 * interface (README.md:144).
 */
int gqa_paged_kv_append(const void* key, const void* value, const int64_t* k_strides3, const int64_t* v_strides3,
                        void* k_cache, void* v_cache, const int64_t* slot_mapping, int num_tokens, int num_kv_heads,
                        int head_dim, int block_size, int num_blocks, int dtype, int cache_fp8, float k_scale,
                        float v_scale, void* stream);

/*
 * The ragged serving step (its entry points take their arguments in a struct, which is
 * only read during the call; strides are in elements): requests of any number of new tokens each (one for a
 * decode, a few drafted ones, a prompt or a chunk of one) planned, rotated, cached,
 * attended and verified without the host reading a length. No reference counterpart
 * (the roadmap's vLLM-shaped interface, README.md:144); the attention's definition is
 * gqa_kernels/gqa_fwd.py's with more masks.
 *
 * gqa_step_plan: from query_lens[b] new and context_lens[b] cached tokens of each
 * request, the blocks it gains, and its tokens' positions and cache slots. Request b
 * holds blocks_held[b] entries of its row of block_tables (row stride bt_stride >=
 * max_blocks); it needs ceil((context + query) / block_size) in all. Requests are granted
 * in order while the pool's free_count[0] ids on top of the stack free_blocks
 * (num_free long) last; the j-th block handed out is free_blocks[free_count - 1 - j]. A
 * request that the pool or the table's width refuses gets granted 0, slots of -1 and
 * seq_lens[b] = context_lens[b]. Outputs: cu_query_lens (num_seqs + 1), seq_lens,
 * granted and blocks_held_out (num_seqs), free_count_out (1), and per token, packed by
 * request, positions, slot_mapping and token_seqs (max_tokens; -1 past the step's
 * tokens). New table entries are written into block_tables. The inputs blocks_held,
 * free_count and context_lens must not be the outputs of the same name. More tokens than
 * max_tokens are dropped and reported (GQA_ERR_INVALID_ARG, site 211); cu_query_lens
 * counts them, and stays at 2^31 - 1 if they are more. block_size: a power of two.
 */
typedef struct {
  const int* query_lens;
  const int* context_lens;
  int* block_tables;
  const int* blocks_held;
  const int* free_blocks;
  const int* free_count;
  int* cu_query_lens;
  int* seq_lens;
  int* positions;
  int64_t* slot_mapping;
  int* token_seqs;
  unsigned char* granted;
  int* blocks_held_out;
  int* free_count_out;
  int64_t bt_stride;
  int num_seqs, max_blocks, num_free, block_size, max_tokens;
} gqa_step_plan_args;
int gqa_step_plan(const gqa_step_plan_args* args, void* stream);

/*
 * gqa_qk_norm_rope: RMS norm of every query and key head (weights of head_dim values in
 * the tensors' dtype, or NULL: no norm), the position rotation, and the cache write.
 * q (num_tokens, num_heads, head_dim), k and v (num_tokens, num_kv_heads, head_dim), element
 * strides of three dimensions (d stride 1, the others multiples of 8). Positions: axis
 * a of token t at positions[a * pos_stride + t]; the rotary_dim / 2 frequencies belong to
 * the axes (1 to 4) in consecutive sections[a]. cos_sin is float32
 * (max_positions, rotary_dim), cosines then sines; rotary_dim a multiple of 16 up to
 * head_dim. Pairs are (f, f + rotary_dim / 2), interleaved: (2f, 2f + 1). q_out is
 * (num_tokens, num_heads, head_dim), contiguous. With slot_mapping, k and v go to the
 * contiguous caches k_dst / v_dst (num_blocks, block_size, num_kv_heads, head_dim) as
 * gqa_paged_kv_append writes them (negative slots skipped; slots past the cache skipped
 * and reported at site 213; e4m3 with cache_fp8); without, k goes to k_dst
 * (num_tokens, num_kv_heads, head_dim) and v is not read. A token with a negative
 * position (padding) gives zero rows and caches nothing; one with a position past the
 * table too, and is reported (site 212). Arithmetic is fp32 with one rounding.
 */
typedef struct {
  const void* q;
  const void* k;
  const void* v;
  const void* q_weight;
  const void* k_weight;
  const int* positions;
  const float* cos_sin;
  void* q_out;
  void* k_dst;
  void* v_dst;
  const int64_t* slot_mapping;
  int64_t q_strides[3], k_strides[3], v_strides[3];
  int64_t pos_stride;
  int sections[4];
  int axes, max_positions, rotary_dim, interleaved;
  int num_tokens, num_heads, num_kv_heads, head_dim, block_size, num_blocks, dtype, cache_fp8;
  float eps, k_scale, v_scale;
} gqa_qk_norm_rope_args;
int gqa_qk_norm_rope(const gqa_qk_norm_rope_args* args, void* stream);

/*
 * gqa_ragged_fwd: attention of request b's new tokens, rows cu_query_lens[b] ..
 * cu_query_lens[b + 1] - 1 of q / o (num_tokens, num_heads, head_dim; element strides of
 * three dimensions), over its seq_lens[b] cached keys, the new tokens' own being the
 * last. The caches are (num_blocks, block_size, num_kv_heads, head_dim) with element
 * strides of four dimensions (d stride 1, the others multiples of 16 bytes), block_size
 * a power of two >= 16. Token i of request b, at position p = seq_lens[b] - (its query
 * length) + i, sees keys [max(0, p - window + 1, key_starts[token]),
 * min(seq_lens[b], max(p + 1, prefix_lens[b]))): window 0, key_starts NULL and
 * prefix_lens NULL leave those terms out; without `causal` it sees all seq_lens[b] keys
 * from key_starts on (window and prefix_lens are then errors). Scores are
 * s = q.k * scale, then softcap * tanh(s / softcap) if softcap > 0, then
 * - alibi_slopes[head] * |p - key| if given. A token that sees no key gives 0 (unlike
 * gqa_fwd's NaN, which is the reference's rule) and lse -inf. lse (num_tokens,
 * num_heads), float32, natural log, may be NULL. Groups of up to 64 heads, any number.
 * e4m3 caches (cache_fp8, scales and range of q as gqa_paged_fwd_kv8) need head_dim 128. max_query_len
 * and max_seq_len bound the lengths and must hold: a request with more tokens may have
 * rows unwritten (reported: GQA_ERR_INVALID_ARG, site 214), keys past max_seq_len are not
 * seen (reported, site 215).
 * Workspace: gqa_ragged_fwd_workspace_bytes of the same arguments (workspace and
 * pointers are not looked at), its first GQA_SERVING_COUNTER_BYTES zeroed before its
 * first use; every call leaves these counters zero, whatever its shape, so calls of all
 * shapes on one stream share one workspace. After a device error they are to be zeroed
 * again. A captured graph should have one of its own that it zeroes itself: one that other
 * graphs or streams use at the same time gives wrong results. Too little gives
 * GQA_ERR_WORKSPACE; NULL leaves the key axis unsplit.
 */
#define GQA_SERVING_COUNTER_BYTES 65536
typedef struct {
  void* workspace;
  size_t workspace_bytes;
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  float* lse;
  const int* block_table;
  const int* cu_query_lens;
  const int* seq_lens;
  const float* alibi_slopes;
  const int* prefix_lens;
  const int* key_starts;
  int64_t q_strides[3], k_strides[4], v_strides[4], o_strides[3];
  int bt_stride, num_seqs, num_tokens, num_heads, num_kv_heads, head_dim, block_size, num_blocks;
  int max_query_len, max_seq_len, window, causal, dtype, cache_fp8;
  float scale, softcap, k_scale, v_scale;
} gqa_ragged_args;
size_t gqa_ragged_fwd_workspace_bytes(const gqa_ragged_args* args);
int gqa_ragged_fwd(const gqa_ragged_args* args, void* stream);

/*
 * gqa_verify_drafts: request b owns rows cu_query_lens[b] .. of the target's
 * probabilities (num_rows, vocab); row i is the distribution after its first i drafted
 * tokens draft_tokens[b][0 ..] (at most max_drafts <= 64, one fewer than its rows). Draft i
 * is accepted while uniforms[b][i] * draft_probs[b][i][d] < target[i][d] (draft_probs
 * NULL: 1 * uniforms); the token after the accepted ones is the argmax over j of
 * max(target[i][j] - draft_probs[b][i][j], 0) / exponentials[b][j] (of target[i][j] /
 * exponentials[b][j] after the last draft; without draft_probs the refused token's
 * weight is 0), ties to the lowest index, NaN left out, or, if no weight is positive, the
 * row's first largest probability. tokens (num_seqs, max_drafts + 1): accepted drafts, then that
 * token, then -1; num_tokens (num_seqs): how many. A request without rows gives 0
 * tokens. Probabilities share dtype (GQA_DTYPE_F32, _BF16 or _F16); uniforms and
 * exponentials are float32. Strides in elements, the vocabulary's is 1. A draft outside
 * [0, vocab) is refused. gqa_verify_greedy: draft i is accepted while it is row i's
 * first largest entry, and the next token is that of the row after; `target` may hold
 * logits. At most 16384 requests.
 * The workspace (gqa_verify_workspace_bytes) may be gqa_ragged_fwd's: its counters
 * have the same place and are left zero too.
 */
typedef struct {
  void* workspace;
  size_t workspace_bytes;
  const int* draft_tokens;
  const void* target;
  const void* draft_probs;   /* gqa_verify_drafts only, as the next two */
  const float* uniforms;
  const float* exponentials;
  const int* cu_query_lens;
  int* tokens;
  int* num_tokens;
  int64_t draft_token_stride, target_stride, draft_strides[2], uniform_stride, exponential_stride;
  int num_seqs, num_rows, max_drafts, vocab, dtype;
} gqa_verify_args;
size_t gqa_verify_workspace_bytes(const gqa_verify_args* args, int greedy);
int gqa_verify_drafts(const gqa_verify_args* args, void* stream);
int gqa_verify_greedy(const gqa_verify_args* args, void* stream);

/*
 * The tcgen05 prefill path's launch plan for a shape on `sm_count` SMs, without
 * launching (host only; needs no GPU). plan[0..4] = units (query pairs x batch x
 * kv heads), nsplit (CTAs per unit; > 1 when the units are fewer than the SMs),
 * key tiles per split, head-major unit order (0/1), grid size.
 * No reference counterpart (the reference launches one program per query block).
 */
int gqa_prefill_plan(int batch, int num_heads, int num_kv_heads, int seq_q, int seq_kv, int head_dim, int causal,
                     int sm_count, int* plan);

/*
 * Reads (and clears, if `clear` is nonzero) the device error word of the
 * current device: 0, or GQA_ERR_TIMEOUT when a bounded in-kernel wait expired.
 * `site` (optional) receives the wait site id. Synchronises the current device.
 * No reference counterpart (the reference has no in-kernel waits).
 */
int gqa_device_error(int* code, int* site, int clear);

/* Number of SMs of the current device as used for split sizing. */
int gqa_sm_count(void);

/*
 * Test hooks of the checked build (libgqa_sm100_debug.so, build.py --debug); the
 * release library returns GQA_ERR_UNSUPPORTED from both. No reference counterpart:
 * they exist to test this library's failure detection and arithmetic on the GPU.
 *
 * gqa_debug_inject: the TMA producer of CTA `cta` withholds its load number `load`
 * (prefill: the K/V tile load index, K and V alternating; streaming kernel: the
 * stage index) in every following launch, and every bounded in-kernel wait gives up
 * after wait_limit_ns (<= 0 restores the default). The consumer's wait on the
 * withheld load then expires: the kernel records GQA_ERR_TIMEOUT in the device error
 * word, aborts the CTA (its other waits end, issued copies land, TMEM is freed) and
 * returns. cta = -1 withholds nothing. Applies to the current device.
 *
 * gqa_debug_exp2_poly2: y[i] = the kernels' FMA-pipe exp2 (the polynomial the prefill
 * softmax uses for one column pair in eight) of x[i], for i < n; device pointers.
 */
int gqa_debug_inject(int cta, int load, long long wait_limit_ns);
int gqa_debug_exp2_poly2(const float* x, float* y, int n, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GQA_SM100_H_ */
