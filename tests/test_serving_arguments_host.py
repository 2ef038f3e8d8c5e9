"""Calls of the ragged step that would compute something else than their name says are refused."""
import pytest
import torch

from gqa_kernels import qk_norm_rope_append


@pytest.mark.parametrize("missing", [("key_cache", "value_cache", "slot_mapping"), ("key_cache",), ("key_cache", "value_cache"),
                                     ("slot_mapping",), ("value_cache",)])
def test_append_without_its_cache(lib_path, missing):
    def bf(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16)
    a = dict(q=bf(3, 8, 128), k=bf(3, 2, 128), v=bf(3, 2, 128), positions=torch.zeros(3, dtype=torch.int32), cos_sin=torch.zeros(10, 128),
             key_cache=bf(4, 16, 2, 128), value_cache=bf(4, 16, 2, 128), slot_mapping=torch.zeros(3, dtype=torch.int64))
    a.update({k: None for k in missing})
    with pytest.raises(ValueError, match="cache"):
        qk_norm_rope_append(**a)
