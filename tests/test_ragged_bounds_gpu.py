"""Ragged attention where a step's numbers and its bounds disagree: rows that were cut off,
lengths past a bound, and bounds at the ends of their type."""
import pytest
import torch

from gqa_kernels import check_device_error, paged_ragged_attention
from tests._serving import attention64, check_attention, paged_batch

pytestmark = pytest.mark.gpu
GQA_ERR_INVALID_ARG = 1


@pytest.fixture(autouse=True)
def _lib_ready(cuda_lib):
    check_device_error()
    yield
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)


def slopes(hq):
    return torch.exp2(-8.0 / hq * torch.arange(1, hq + 1, dtype=torch.float32, device="cuda"))


@pytest.mark.parametrize("reqs,rows", [
    ([(1, 50), (8, 300)], 6),               # streamed
    ([(1, 50), (200, 300)], 131),           # tcgen05
    ([(70, 0), (1, 50), (200, 300)], 75),   # both; the cut request streams what is left of it
    ([(150, 40), (90, 0), (3, 20)], 200),   # a request without rows after the cut one
])
@pytest.mark.parametrize("case", ["causal", "window", "alibi", "prefix"])
def test_a_step_cut_to_fewer_rows_keeps_its_positions(reqs, rows, case):
    """The packed offsets count more tokens than there are rows: each remaining row sees what
    it sees in the whole step. The dropped tokens' cache slots were never written."""
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 16, torch.bfloat16, rows, float("nan"))
    prefix = torch.tensor([min(30, c) for _, c in reqs], dtype=torch.int32, device="cuda")
    kw = {"causal": {}, "window": dict(window=40), "alibi": dict(alibi_slopes=slopes(8)),
          "prefix": dict(window=500, prefix_lens=prefix)}[case]
    ref = {"window": kw.get("window"), "alibi": kw.get("alibi_slopes"), "prefix": kw.get("prefix_lens")}
    o, _, a = attention64(q, kc.nan_to_num(0), vc.nan_to_num(0), bt, reqs, **ref)
    at = 0
    for b, (qn, c) in enumerate(reqs):
        for i in range(qn):
            if at + i >= rows:
                kc[bt[b, (c + i) // 16], (c + i) % 16] = float("nan")
                vc[bt[b, (c + i) // 16], (c + i) % 16] = float("nan")
        at += qn
    out = paged_ragged_attention(q[:rows], kc, vc, bt, cu, lens, **kw)
    check_attention(out, o[:rows], a[:rows], torch.bfloat16)
