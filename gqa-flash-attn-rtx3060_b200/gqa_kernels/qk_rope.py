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

from . import _lib, _serving

__all__ = ["rope_table", "qk_norm_rope", "qk_norm_rope_append"]


def rope_table(max_positions, rotary_dim, base=10000.0, device="cuda"):
    """float32 (max_positions, rotary_dim): cosines, then sines, of position x
    base^(-2 f / rotary_dim) for the rotary_dim / 2 frequencies, computed in 64 bits."""
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device)


def _launch(q, k, v, positions, cos_sin, k_dst, v_dst, slots, block_size, num_blocks, q_weight, k_weight, eps, sections,
            interleaved, out, k_scale, v_scale):
    num_tokens, num_heads, head_dim = q.shape
    if k.dim() != 3 or k.shape[0] != num_tokens or k.shape[2] != head_dim:
        raise ValueError("q and k must be (num_tokens, heads, head_dim) of the same tokens and head_dim")
    if head_dim != 128 and head_dim != 64:
        raise ValueError(f"unsupported head_dim {head_dim}")
    dt = q.dtype
    dtype = _lib.dtype_code(q)
    if k.dtype != dt:
        raise TypeError("q and k must share one dtype")
    if positions.dtype != torch.int32 or positions.dim() not in (1, 2) or positions.shape[-1] != num_tokens:
        raise ValueError("positions must be int32 (num_tokens,) or (axes, num_tokens)")
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.data_ptr() & 15:
        raise ValueError("cos_sin must be a contiguous, 16-byte aligned float32 (max_positions, rotary_dim)")
    max_positions, rotary_dim = cos_sin.shape
    if rotary_dim > head_dim or rotary_dim % 16:
        raise ValueError("rotary_dim must be a multiple of 16, at most head_dim")
    if axes == 1:
        sec = (rotary_dim // 2, 0, 0, 0)
        if sections is not None and tuple(sections) != sec[:1]:
            raise ValueError("one position axis has all of the rotary_dim / 2 frequencies")
    else:
        if not 1 < axes <= 4:
            raise ValueError("1 to 4 position axes are supported")
        if sections is None or len(sections) != axes or sum(sections) * 2 != rotary_dim or min(sections) < 0:
            raise ValueError("sections must give each position axis its share of the rotary_dim / 2 frequencies")
        sec = (*sections, 0, 0)[:4]
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (head_dim,) or w.dtype != dt or w.stride(0) != 1 or w.data_ptr() & 15):
            raise ValueError("norm weights must be contiguous (head_dim,) tensors of q's dtype, 16-byte aligned")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != dt or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape and dtype")
    index = _serving.device_index(q, k, v, positions, cos_sin, k_dst, v_dst, slots, q_weight, k_weight, out)
    if not _lib.tma_compatible(q):
        q = q.contiguous()
    if not _lib.tma_compatible(k):
        k = k.contiguous()
    if v is None:
        vp = vd = sp = vs0 = vs1 = vs2 = 0
    else:
        if not _lib.tma_compatible(v):
            v = v.contiguous()
        vp, vd, sp = v.data_ptr(), v_dst.data_ptr(), slots.data_ptr()
        vs0, vs1, vs2 = v.stride()
    if positions.stride(-1) != 1 and num_tokens > 1:
        positions = positions.contiguous()
    _serving.call("gqa_qk_norm_rope", _serving.QK_NORM_ROPE(
        q.data_ptr(), k.data_ptr(), vp, 0 if q_weight is None else q_weight.data_ptr(),
        0 if k_weight is None else k_weight.data_ptr(), positions.data_ptr(), cos_sin.data_ptr(), out.data_ptr(),
        k_dst.data_ptr(), vd, sp, *q.stride(), *k.stride(), vs0, vs1, vs2, positions.stride(0) if axes > 1 else 0,
        *sec, axes, max_positions, rotary_dim, 1 if interleaved else 0, num_tokens, num_heads, k.shape[1], head_dim, block_size,
        num_blocks, dtype, 1 if k_dst.dtype == torch.float8_e4m3fn else 0, eps, k_scale, v_scale), index)
    return out


def qk_norm_rope(q, k, positions, cos_sin, q_weight=None, k_weight=None, eps=1e-6, sections=None, interleaved=False):
    """Normalises and rotates query and key heads; see qk_norm_rope_append for the arguments.

    Returns:
        (q, k) rotated, contiguous, in q's dtype.
    """
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    return _launch(q, k, None, positions, cos_sin, k_out, None, None, 0, 0, q_weight, k_weight, eps, sections, interleaved,
                   None, 1.0, 1.0), k_out


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
    num_blocks, block_size, hkv, hd = cache = key_cache.shape
    if v.shape != k.shape or v.dtype != k.dtype or value_cache.shape != cache or k.shape != (q.shape[0], hkv, hd):
        raise ValueError("k/v must be (num_tokens, num_kv_heads, head_dim) of one dtype and the caches "
                         "(num_blocks, block_size, num_kv_heads, head_dim)")
    fp8 = key_cache.dtype == torch.float8_e4m3fn
    if value_cache.dtype != key_cache.dtype or not (fp8 or key_cache.dtype == k.dtype):
        raise TypeError("the caches share q's dtype, or are both float8_e4m3fn")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("the caches must be contiguous")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (q.shape[0],):
        raise TypeError("slot_mapping must be int64 (num_tokens,)")
    if slot_mapping.shape[0] > 1 and slot_mapping.stride(0) != 1:
        slot_mapping = slot_mapping.contiguous()
    if fp8 and not (k_scale > 0 and v_scale > 0):
        raise ValueError("fp8 caches need positive k_scale and v_scale")
    return _launch(q, k, v, positions, cos_sin, key_cache, value_cache, slot_mapping, block_size, num_blocks, q_weight,
                   k_weight, eps, sections, interleaved, out, k_scale, v_scale)
