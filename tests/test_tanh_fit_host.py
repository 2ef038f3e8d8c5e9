"""The ragged kernels' score cap (csrc/gqa_ragged_tile.cuh): its polynomial is the output of
tests/tanh_fit.py's fit, rounded to float32, and the float32 emulation of the kernel's
evaluation stays within the bound that the kernel's comment states."""
import os
import re

import numpy as np

from tests import tanh_fit as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = os.path.join(ROOT, "gqa-flash-attn-rtx3060_b200", "csrc", "gqa_ragged_tile.cuh")


def kernel_constants():
    got = {k: float(v) for k, v in re.findall(r"\bkTanh(C[0-3]|Range)\s*=\s*([0-9.eE+-]+)f", open(SOURCE).read())}
    return got.pop("Range"), np.array([got[f"C{i}"] for i in range(4)], dtype=np.float32)


def test_kernel_constants_are_the_fit():
    most, c = kernel_constants()
    assert np.float32(most) == np.float32(F.RANGE)
    assert np.array_equal(c, F.fit().astype(np.float32))


def test_emulated_evaluation_meets_the_stated_bound():
    assert F.max_error(kernel_constants()[1]) < 7e-7
