"""B200 (sm_100a) GQA flash-attention forward with the reference's public API.

`gqa_flash_attn(q, k, v, causal=True)` keeps the signature, layout and routing
of tonbistudio/gqa-flash-attn-rtx3060 (gqa_kernels/__init__.py:1-4); the work
runs in hand-written sm_100a CUDA behind the C ABI of include/gqa_sm100.h.

The ragged serving step's operators are exported here too: plan_step,
qk_norm_rope_append (and qk_norm_rope, rope_table), paged_ragged_attention,
RaggedPagedAttention, verify_drafts and verify_drafts_greedy.
"""
from .dispatch import gqa_flash_attn, set_nvtx_ranges
from ._lib import device_error as check_device_error
from .qk_rope import qk_norm_rope, qk_norm_rope_append, rope_table
from .ragged import RaggedPagedAttention, paged_ragged_attention
from .step_plan import StepPlan, plan_step
from .verify import verify_drafts, verify_drafts_greedy

__all__ = ["gqa_flash_attn", "check_device_error", "set_nvtx_ranges", "StepPlan", "plan_step", "rope_table",
           "qk_norm_rope", "qk_norm_rope_append", "paged_ragged_attention", "RaggedPagedAttention", "verify_drafts",
           "verify_drafts_greedy"]
__version__ = "0.1.0"
