"""The plan of a ragged serving step, built on the GPU from the requests' lengths.

A scheduler that keeps its requests' lengths on the GPU (speculative decoding does: only
the device knows how many drafts were accepted) cannot build block tables, positions
and slot mappings on the host without waiting for it. `plan_step` builds them in one
kernel: it hands blocks of the paged cache's pool to the requests in order, and writes
the packed offsets, positions and cache slots that `qk_norm_rope_append`,
`paged_kv_append`, `paged_ragged_attention` and `verify_drafts` take.

A plan changes nothing but the new entries of `block_tables`, so planning the same step
twice gives the same plan; the step takes effect when the caller goes on with the plan's
`blocks_held` and `free_count`.
"""
from dataclasses import dataclass

import torch

from . import _serving

__all__ = ["StepPlan", "plan_step"]


@dataclass
class StepPlan:
    """What `plan_step` writes (all on the lengths' device).

    cu_query_lens: int32 (n + 1,), first packed token of each request, and their number.
    seq_lens: int32 (n,), cached tokens after the step (unchanged where not granted).
    positions: int32 (max_tokens,), each packed token's position; -1 past the step's.
    slot_mapping: int64 (max_tokens,), its cache slot; -1 past the step's tokens and for
        requests that were not granted.
    token_seqs: int32 (max_tokens,), its request; -1 past the step's.
    granted: bool (n,), whether the pool and the table had room for the request. The tokens of
        one that was not are still packed, so that the offsets fit the step's rows, but what
        later operators make of them is not to be used.
    blocks_held: int32 (n,), entries in use of each table row after the step.
    free_count: int32 (1,), free blocks left after the step.
    """
    cu_query_lens: torch.Tensor
    seq_lens: torch.Tensor
    positions: torch.Tensor
    slot_mapping: torch.Tensor
    token_seqs: torch.Tensor
    granted: torch.Tensor
    blocks_held: torch.Tensor
    free_count: torch.Tensor

    @classmethod
    def empty(cls, num_seqs, max_tokens, device="cuda"):
        """Unwritten buffers for plans of num_seqs requests and at most max_tokens tokens."""
        def i32(n):
            return torch.empty(n, dtype=torch.int32, device=device)
        max_tokens = max(0, max_tokens)
        return cls(i32(num_seqs + 1), i32(num_seqs), i32(max_tokens),
                   torch.empty(max_tokens, dtype=torch.int64, device=device), i32(max_tokens),
                   torch.empty(num_seqs, dtype=torch.bool, device=device), i32(num_seqs), i32(1))


def plan_step(query_lens, context_lens, block_tables, blocks_held, free_blocks, free_count, block_size, max_tokens, out=None):
    """Plans one step.

    Args:
        query_lens: int32 (n,), new tokens of each request (0 allowed).
        context_lens: int32 (n,), its cached tokens.
        block_tables: int32 (n, max_blocks), each row contiguous; row b's first
            blocks_held[b] entries are in use. The entries that the step adds are written.
        blocks_held: int32 (n,).
        free_blocks: int32 (num_free,), a stack of free block ids, of which the first
            free_count[0] count; blocks are handed out from its top.
        free_count: int32 (1,).
        block_size: tokens per block, a power of two.
        max_tokens: size of the per-token outputs; a step with more tokens is cut and
            reported through the device error word (gqa_kernels.check_device_error()).
        out: a StepPlan of buffers to write (of this n and max_tokens); must not be the
            plan whose tensors are passed as inputs.

    Returns:
        a StepPlan. Requests are granted in order; one that needs more blocks than are
        left, or more than its row has entries, is refused for this step, and so is every
        later one that needs any. Asynchronous on the current stream.
    """
    if out is None:
        out = StepPlan.empty(query_lens.shape[0], max_tokens, query_lens.device)
    (_serving._ext or _serving.load()).step_plan(
        query_lens, context_lens, block_tables, blocks_held, free_blocks, free_count, block_size, max_tokens, out.cu_query_lens,
        out.seq_lens, out.positions, out.slot_mapping, out.token_seqs, out.granted, out.blocks_held, out.free_count)
    return out
