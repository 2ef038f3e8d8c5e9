"""Verification of drafted tokens (speculative decoding).

A draft model (or an n-gram table) proposes a few tokens per request; one ragged step
of the target scores them all, and verification keeps the longest run that leaves the
target's distribution unchanged, plus one token of the target's own. Random numbers are
inputs, so a result can be reproduced, and nothing is read back to the host.
"""
from . import _serving

__all__ = ["verify_drafts", "verify_drafts_greedy"]


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
        target_prob; the drawn token is the first argmax of weight / exponentials (entries
        with NaN never are).
        Asynchronous on the current stream.
    """
    return (_serving._ext or _serving.load()).verify(draft_tokens, target_probs, draft_probs, uniforms, exponentials, cu_query_lens,
                                                     out, False)


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
    return (_serving._ext or _serving.load()).verify(draft_tokens, target, None, None, None, cu_query_lens, out, True)
