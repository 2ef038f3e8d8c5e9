"""Norm of query and key heads, the position rotation and the cache write, in one pass.

Between the projection and the attention of a layer, models normalise each query and
key head, rotate it by its token's position (or, for pictures and video, by several:
time, height and width), and write the keys and values into the cache. Done apart, each
step reads and writes the activations once; `qk_norm_rope_append` does all of it in one
kernel, straight from the projection's output into the paged caches that
`paged_ragged_attention`, `paged_decode` and `paged_prefill` read. `qk_norm_rope` is
the same without a cache: it returns the rotated keys, for gqa_flash_attn and
PrefixKVCache.
"""
import torch

from . import _serving

__all__ = ["rope_table", "qk_norm_rope", "qk_norm_rope_append"]


def rope_table(max_positions, rotary_dim, base=10000.0, device="cuda"):
    """float32 (max_positions, rotary_dim): cosines, then sines, of position x
    base^(-2 f / rotary_dim) for the rotary_dim / 2 frequencies, computed in 64 bits."""
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device)


def qk_norm_rope(q, k, positions, cos_sin, q_weight=None, k_weight=None, eps=1e-6, sections=None, interleaved=False):
    """Normalises and rotates query and key heads; see qk_norm_rope_append for the arguments.

    Returns:
        (q, k) rotated, contiguous, in q's dtype.
    """
    return (_serving._ext or _serving.load()).norm_rope(q, k, None, positions, cos_sin, None, None, None, q_weight, k_weight, eps,
                                                        sections, interleaved, None, 1.0, 1.0)


def qk_norm_rope_append(q, k, v, positions, cos_sin, key_cache, value_cache, slot_mapping, q_weight=None, k_weight=None,
                        eps=1e-6, sections=None, interleaved=False, out=None, k_scale=1.0, v_scale=1.0):
    """Normalises and rotates query and key heads and writes K and V into the paged caches.

    Args:
        q: (num_tokens, num_heads, head_dim), bf16 or fp16, e.g. a slice of the fused
            projection's output; head_dim 64 or 128.
        k, v: (num_tokens, num_kv_heads, head_dim), q's dtype.
        positions: int32 (num_tokens,), or (axes, num_tokens) for up to four position axes.
            A token with a negative position is padding: its row of the result is zero and
            it is not cached. A position past the table is treated so too and reported
            through the device error word (gqa_kernels.check_device_error()).
        cos_sin: float32 (max_positions, rotary_dim), cosines then sines (see rope_table);
            the head's values past rotary_dim are not rotated.
        key_cache, value_cache: (num_blocks, block_size, num_kv_heads, head_dim), contiguous;
            q's dtype, or float8_e4m3fn (stored = x / scale rounded and saturated, as
            paged_kv_append stores it).
        slot_mapping: int64 (num_tokens,), as paged_kv_append's: negative slots are not
            written, slots past the cache are not written and are reported.
        q_weight, k_weight: (head_dim,) weights of the heads' RMS norm in q's dtype; None:
            no norm.
        eps: the norm's epsilon.
        sections: how many of the rotary_dim / 2 frequencies each axis has, in order.
        interleaved: rotate neighbouring pairs (2f, 2f + 1) instead of (f, f + rotary_dim / 2).
        out: optional contiguous result tensor.

    Returns:
        the rotated queries, (num_tokens, num_heads, head_dim). The arithmetic is fp32,
        rounded once. Asynchronous on the current stream.
    """
    return (_serving._ext or _serving.load()).norm_rope(q, k, v, positions, cos_sin, key_cache, value_cache, slot_mapping, q_weight,
                                                        k_weight, eps, sections, interleaved, out, k_scale, v_scale)
