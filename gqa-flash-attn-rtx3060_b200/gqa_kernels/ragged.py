"""Attention of a ragged step over the paged cache.

`paged_ragged_attention` attends every request's own number of new tokens in one call:
decodes, drafted tokens and chunks of prompts side by side, which paged_decode and
paged_prefill (one chunk length per call) cannot. The lengths stay on the GPU. Scores can
be capped by a tanh or biased by distance, and each token's visible keys are an interval
that combines the causal rule, a window, a prefix that every token sees, and documents
packed into one request.

`RaggedPagedAttention` ties the step's operators together as one attention layer.
"""
import torch

from . import _serving
from .qk_rope import qk_norm_rope_append

__all__ = ["paged_ragged_attention", "RaggedPagedAttention"]


def paged_ragged_attention(query, key_cache, value_cache, block_tables, cu_query_lens, seq_lens, max_query_len=None,
                           max_seq_len=None, scale=None, causal=True, softcap=0.0, alibi_slopes=None, window=None,
                           prefix_lens=None, key_starts=None, k_scale=1.0, v_scale=1.0, return_lse=False, out=None):
    """Attention of each request's new tokens over its cached keys.

    Args:
        query: (num_tokens, num_heads, head_dim), bf16 or fp16, the requests' tokens one
            after the other; head_dim 64 or 128, d stride 1.
        key_cache, value_cache: (num_blocks, block_size, num_kv_heads, head_dim), d stride 1,
            block_size a power of two >= 16; query's dtype, or float8_e4m3fn (head_dim 128)
            with key = stored key * k_scale and value = stored value * v_scale (the products
            then run in f16: |query| must stay within its range, 65504). num_heads is any
            multiple (up to 64) of num_kv_heads.
        block_tables: int32 (num_seqs, max_blocks); request b's key k is in block
            block_tables[b, k // block_size] at position k % block_size.
        cu_query_lens: int32 (num_seqs + 1,); request b's tokens are rows
            cu_query_lens[b] .. cu_query_lens[b + 1] - 1 of query. Rows past the last
            request's (padding) are not written.
        seq_lens: int32 (num_seqs,), cached keys of each request, its new tokens' included:
            token i of q new ones is at position seq_lens[b] - q + i.
        max_query_len, max_seq_len: upper bounds of the query lengths and of seq_lens, which
            size the launch; they must hold. Keys past max_seq_len are not seen, and rows past
            max_query_len may stay unwritten; both are reported through the device error
            word (gqa_kernels.check_device_error()). Defaults: num_tokens and the tables'
            capacity.
        scale: softmax scale; defaults to head_dim ** -0.5.
        causal: a token sees the keys up to its own position; False: all of the request's.
        softcap: scores become softcap * tanh(score / softcap); 0: not.
        alibi_slopes: float32 (num_heads,): slope * |distance| is taken off the (capped) score.
        window: a token sees at most this many keys back, its own included.
        prefix_lens: int32 (num_seqs,): the first prefix_lens[b] keys are seen by every token
            of request b (within its window).
        key_starts: int32 (num_tokens,): the first key that each token sees, e.g. where its
            document begins.
        return_lse: also return the log-sum-exp of each row's scores.
        out: optional output of query's shape and dtype, d stride 1.

    Returns:
        (num_tokens, num_heads, head_dim) in query's dtype, and with return_lse float32
        (num_tokens, num_heads). A token that sees no key gives zeros and -inf (where
        gqa_flash_attn and paged_prefill give NaN, the reference's rule: here masks that
        leave a row empty are ordinary). Cache slots that no token sees may hold anything; a
        NaN or infinite value that some token of a request sees may reach the request's
        other tokens as well. Asynchronous on the current stream.
    """
    return (_serving._ext or _serving.load()).ragged(
        query, key_cache, value_cache, block_tables, cu_query_lens, seq_lens, max_query_len, max_seq_len, scale, causal, softcap,
        alibi_slopes, window, prefix_lens, key_starts, k_scale, v_scale, return_lse, out)


class RaggedPagedAttention:
    """The attention layer of a ragged step: forward(qkv, plan, ...) normalises and rotates
    the heads, writes K and V into the layer's cache and attends.

    Args:
        num_heads, num_kv_heads, head_dim: the layer's heads.
        cos_sin: the rotation table (qk_rope.rope_table).
        q_weight, k_weight, eps: the heads' RMS norm (None: no norm).
        sections, interleaved: see qk_norm_rope_append.
        scale, softcap, window, alibi_slopes: see paged_ragged_attention.
        kv_cache_dtype, k_scale, v_scale: "auto" (the model's dtype) or "fp8_e4m3".
    """

    def __init__(self, num_heads, num_kv_heads, head_dim, cos_sin, q_weight=None, k_weight=None, eps=1e-6, sections=None,
                 interleaved=False, scale=None, softcap=0.0, window=None, alibi_slopes=None, kv_cache_dtype="auto",
                 k_scale=1.0, v_scale=1.0):
        if num_heads % num_kv_heads:
            raise ValueError("num_heads must be a multiple of num_kv_heads")
        if kv_cache_dtype not in ("auto", "fp8_e4m3"):
            raise ValueError("kv_cache_dtype must be 'auto' or 'fp8_e4m3'")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.cos_sin, self.q_weight, self.k_weight, self.eps = cos_sin, q_weight, k_weight, eps
        self.sections, self.interleaved = sections, interleaved
        self.scale, self.softcap, self.window, self.alibi_slopes = scale, softcap, window, alibi_slopes
        self.kv_cache_dtype, self.k_scale, self.v_scale = kv_cache_dtype, k_scale, v_scale

    def allocate_kv_cache(self, num_blocks, block_size, dtype, device):
        """A zeroed (2, num_blocks, block_size, num_kv_heads, head_dim) cache: [0] keys, [1] values."""
        dt = torch.float8_e4m3fn if self.kv_cache_dtype == "fp8_e4m3" else dtype
        return torch.zeros(2, num_blocks, block_size, self.num_kv_heads, self.head_dim, dtype=dt, device=device)

    def forward(self, qkv, kv_cache, plan, block_tables, max_query_len, max_seq_len=None, positions=None, prefix_lens=None,
                key_starts=None):
        """qkv (num_tokens, (num_heads + 2 num_kv_heads) * head_dim), the fused projection of the
        packed tokens; plan a StepPlan of at least num_tokens. positions defaults to the
        plan's (pass (axes, num_tokens) for several axes). Returns (num_tokens, num_heads *
        head_dim); rows of padding tokens are undefined, and those of a request that the plan
        did not grant (its keys are not cached) mean nothing and have to be left unused."""
        t = qkv.shape[0]
        x = qkv.view(t, self.num_heads + 2 * self.num_kv_heads, self.head_dim)
        q = x[:, :self.num_heads]
        k = x[:, self.num_heads:self.num_heads + self.num_kv_heads]
        v = x[:, self.num_heads + self.num_kv_heads:]
        positions = plan.positions[:t] if positions is None else positions
        q = qk_norm_rope_append(q, k, v, positions, self.cos_sin, kv_cache[0], kv_cache[1], plan.slot_mapping[:t],
                                self.q_weight, self.k_weight, self.eps, self.sections, self.interleaved,
                                k_scale=self.k_scale, v_scale=self.v_scale)
        o = paged_ragged_attention(q, kv_cache[0], kv_cache[1], block_tables, plan.cu_query_lens, plan.seq_lens,
                                   max_query_len, max_seq_len, self.scale, True, self.softcap, self.alibi_slopes, self.window,
                                   prefix_lens, key_starts, self.k_scale, self.v_scale)
        return o.view(t, self.num_heads * self.head_dim)
