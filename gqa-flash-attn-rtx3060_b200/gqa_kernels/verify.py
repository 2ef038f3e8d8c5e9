"""Verification of drafted tokens (speculative decoding).

A draft model (or an n-gram table) proposes a few tokens per request; one ragged step
of the target scores them all, and verification keeps the longest run that leaves the
target's distribution unchanged, plus one token of the target's own. Random numbers are
inputs, so a result can be reproduced, and nothing is read back to the host.
"""
import torch

from . import _lib, _serving

__all__ = ["verify_drafts", "verify_drafts_greedy"]

_CODES = {torch.float16: _lib.GQA_DTYPE_F16, torch.bfloat16: _lib.GQA_DTYPE_BF16, torch.float32: _lib.GQA_DTYPE_F32}


def _common(draft_tokens, target, cu_query_lens, out, *others):
    """Shapes and types first, the device last; the outputs are made here."""
    n, k = draft_tokens.shape
    dtype = _CODES.get(target.dtype)
    if dtype is None:
        raise TypeError(f"float32, bfloat16 or float16 targets are supported, got {target.dtype}")
    if draft_tokens.dtype != torch.int32 or cu_query_lens.dtype != torch.int32:
        raise TypeError("draft_tokens and cu_query_lens must be int32")
    if cu_query_lens.shape != (n + 1,):
        raise ValueError("cu_query_lens must be (num_seqs + 1,)")
    if k > 64:
        raise ValueError("at most 64 drafted tokens are supported")
    index = _serving.device_index(target, draft_tokens, cu_query_lens, *others)
    if draft_tokens.stride(1) != 1 and k > 1:
        draft_tokens = draft_tokens.contiguous()
    if target.stride(1) != 1:
        target = target.contiguous()
    if not cu_query_lens.is_contiguous():
        cu_query_lens = cu_query_lens.contiguous()
    if out is None:
        dev = target.device
        out = (torch.empty((n, k + 1), dtype=torch.int32, device=dev), torch.empty((n,), dtype=torch.int32, device=dev))
    else:
        tokens, num = out
        if tokens.shape != (n, k + 1) or num.shape != (n,) or tokens.dtype != torch.int32 or num.dtype != torch.int32 \
                or not (tokens.is_contiguous() and num.is_contiguous()):
            raise ValueError("out must be contiguous int32 (num_seqs, max_drafts + 1) and (num_seqs,)")
        _serving.device_index(target, tokens, num)
    return draft_tokens, target, cu_query_lens, out, dtype, index


def _race_bytes(lib, args):
    return lib.gqa_verify_workspace_bytes(args, 0)


def _greedy_bytes(lib, args):
    return lib.gqa_verify_workspace_bytes(args, 1)


def verify_drafts(draft_tokens, target_probs, draft_probs, uniforms, exponentials, cu_query_lens, out=None):
    """Speculative sampling of each request's drafted tokens.

    Args:
        draft_tokens: int32 (num_seqs, max_drafts), the proposals after the request's last
            token; request b has one fewer than its rows of the target (at most 64).
        target_probs: (num_rows, vocab), float32, bf16 or fp16: row cu_query_lens[b] + i is
            the target's distribution after request b's first i drafts.
        draft_probs: (num_seqs, max_drafts, vocab), target_probs' dtype, the distributions
            that the drafts were drawn from; None: proposals that were not drawn at random.
        uniforms: float32 (num_seqs, max_drafts) in [0, 1).
        exponentials: float32 (num_seqs, vocab), positive (torch's exponential_()).
        cu_query_lens: int32 (num_seqs + 1,), the step's packed offsets (StepPlan's).
        out: optional (tokens, num_tokens) to write.

    Returns:
        tokens int32 (num_seqs, max_drafts + 1): the accepted drafts, then one token drawn
        from what is left of the target's distribution (from its next one when all were
        accepted), then -1; and num_tokens int32 (num_seqs,), how many there are (0 for a
        request without rows). Draft i is accepted while uniforms * draft_prob <
        target_prob; the drawn token is the first argmax of weight / exponentials.
        Asynchronous on the current stream.
    """
    if draft_tokens.dim() != 2 or target_probs.dim() != 2:
        raise ValueError("draft_tokens must be (num_seqs, max_drafts) and target_probs (num_rows, vocab)")
    n, k = draft_tokens.shape
    num_rows, vocab = target_probs.shape
    if uniforms.shape != (n, k) or exponentials.shape != (n, vocab):
        raise ValueError("uniforms must be (num_seqs, max_drafts) and exponentials (num_seqs, vocab)")
    if uniforms.dtype != torch.float32 or exponentials.dtype != torch.float32:
        raise TypeError("uniforms and exponentials must be float32")
    if draft_probs is not None:
        if draft_probs.shape != (n, k, vocab):
            raise ValueError("draft_probs must be (num_seqs, max_drafts, vocab)")
        if draft_probs.dtype != target_probs.dtype:
            raise TypeError("draft_probs must have target_probs' dtype")
    draft_tokens, target, cu, (tokens, num), dtype, index = _common(draft_tokens, target_probs, cu_query_lens, out, uniforms,
                                                                    exponentials, draft_probs)
    d_ptr = d_sn = d_sk = 0
    if draft_probs is not None:
        if draft_probs.stride(2) != 1:
            draft_probs = draft_probs.contiguous()
        d_ptr, (d_sn, d_sk, _) = draft_probs.data_ptr(), draft_probs.stride()
    if uniforms.stride(1) != 1 and k > 1:
        uniforms = uniforms.contiguous()
    if exponentials.stride(1) != 1:
        exponentials = exponentials.contiguous()
    _serving.call_with_workspace("gqa_verify_drafts", _serving.VERIFY(
        draft_tokens.data_ptr(), target.data_ptr(), d_ptr, uniforms.data_ptr(), exponentials.data_ptr(), cu.data_ptr(),
        tokens.data_ptr(), num.data_ptr(), draft_tokens.stride(0), target.stride(0), d_sn, d_sk, uniforms.stride(0),
        exponentials.stride(0), n, num_rows, k, vocab, dtype), index, _race_bytes)
    return tokens, num


def verify_drafts_greedy(draft_tokens, target, cu_query_lens, out=None):
    """Verification at temperature zero: a draft is accepted while it is the target's first
    largest entry, and the next token is that of the row after it.

    Args:
        draft_tokens, cu_query_lens, out: see verify_drafts.
        target: (num_rows, vocab) logits or probabilities, float32, bf16 or fp16. NaN entries
            are never the largest.

    Returns:
        (tokens, num_tokens), as verify_drafts.
    """
    if draft_tokens.dim() != 2 or target.dim() != 2:
        raise ValueError("draft_tokens must be (num_seqs, max_drafts) and the target (num_rows, vocab)")
    draft_tokens, target, cu, (tokens, num), dtype, index = _common(draft_tokens, target, cu_query_lens, out)
    n, k = draft_tokens.shape
    num_rows, vocab = target.shape
    _serving.call_with_workspace("gqa_verify_greedy", _serving.VERIFY(
        draft_tokens.data_ptr(), target.data_ptr(), 0, 0, 0, cu.data_ptr(), tokens.data_ptr(), num.data_ptr(),
        draft_tokens.stride(0), target.stride(0), 0, 0, 0, 0, n, num_rows, k, vocab, dtype), index, _greedy_bytes)
    return tokens, num
