"""Ragged attention with infinite scores under a cap: cap * tanh(-inf / cap) is -cap, an
ordinary score, in every form (streamed, tcgen05, with and without hidden keys in a tile)."""
import pytest
import torch

from gqa_kernels import check_device_error, paged_ragged_attention
from tests._serving import attention64, check_attention, paged_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reqs", [[(2, 60), (1, 300)], [(200, 30)], [(150, 800), (3, 20)], [(40, 3000)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", ["cap", "window", "bias", "full"])
def test_capped_infinite_scores(cuda_lib, reqs, dtype, d, case):
    check_device_error()
    hq, hkv, block = 8, 2, 16
    q, kc, vc, bt, _, lens = paged_batch(reqs, hq, hkv, d, block, dtype, 31, 0.0)
    q = q.abs() + 0.1  # so that a key's infinity decides its score
    for b, (qn, c) in enumerate(reqs):
        for k in range(qn + c):
            row = kc[bt[b, k // block], k % block]
            if k < 5 or k % 7 == 0 or k > qn + c - 40:  # among them all that some rows see
                row[..., k % d] = float("-inf")
            elif k % 11 == 0:
                row[..., k % d] = float("inf")
    kw = {"cap": {}, "window": dict(window=33), "bias": dict(alibi_slopes=torch.full((hq,), 0.01, device="cuda")),
          "full": dict(causal=False)}[case]
    ref = dict(kw)
    if "alibi_slopes" in ref:
        ref["alibi"] = ref.pop("alibi_slopes")
    cu = torch.tensor([0] + torch.tensor([x for x, _ in reqs]).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    for cap in (2.0, 20.0):
        out, lse = paged_ragged_attention(q, kc, vc, bt, cu, lens, softcap=cap, return_lse=True, **kw)
        o, l64, a = attention64(q, kc, vc, bt, reqs, softcap=cap, **ref)
        assert torch.isfinite(l64).all()
        check_attention(out, o, a, dtype)
        # as the other tests of the log-sum-exp
        assert ((lse.double() - l64).abs() <= 2e-4 + 1e-6 * l64.abs()).all()
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)
