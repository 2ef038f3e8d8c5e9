"""What the dense entry points wait for on their first call does not include the ragged step."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_devices_set_up_leaves_the_ragged_kernels_to_their_first_call():
    with open(os.path.join(ROOT, "gqa-flash-attn-rtx3060_b200", "csrc", "gqa_sm100.cu")) as f:
        body = re.search(r"\nint init_device\(int dev\) \{\n(.*?)\n\}\n", f.read(), re.S).group(1)
    assert "gqa_stream_kernel" in body and "ragged" not in body
