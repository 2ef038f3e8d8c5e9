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


@pytest.mark.parametrize("fp8", [False, True])
def test_a_request_longer_than_its_bound_is_reported(fp8):
    """Streamed requests have as many tiles as max_query_len needs: more tokens than it says
    are left out, and the error word says so."""
    reqs = [(1, 50), (9, 100), (2, 7)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, torch.bfloat16, 1)
    if fp8:
        kc, vc = kc.to(torch.float8_e4m3fn), vc.to(torch.float8_e4m3fn)
    out = paged_ragged_attention(q, kc, vc, bt, cu, lens, max_query_len=9)
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)
    got = torch.full_like(q, 7.0)
    paged_ragged_attention(q, kc, vc, bt, cu, lens, max_query_len=2, out=got)
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 214)
    kept = torch.ones(12, dtype=torch.bool, device="cuda")
    kept[3:10] = False
    assert ((got.float() - out.float())[kept].abs() <= 0.02 * out.float().abs().max()).all() and (got[~kept] == 7.0).all()


@pytest.mark.parametrize("reqs", [[(1, 700), (2, 90)], [(200, 500), (2, 90)]])  # streamed, tcgen05
def test_a_length_past_its_bound_is_reported(reqs):
    """Keys past max_seq_len are not seen; tokens keep their positions."""
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 16, torch.bfloat16, 2)
    bound = 600
    out = paged_ragged_attention(q, kc, vc, bt, cu, lens, max_seq_len=bound, alibi_slopes=slopes(8))
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 215)
    first, n = 0, sum(reqs[0])
    assert n > bound
    k, v = (x[bt[0].long()].flatten(0, 1)[:bound].double().repeat_interleave(4, 1) for x in (kc, vc))
    pos = torch.arange(reqs[0][1], n, device="cuda")[:, None]
    key = torch.arange(bound, device="cuda")
    x = torch.einsum("qhd,khd->hqk", q[:reqs[0][0]].double(), k) * 128 ** -0.5 - slopes(8).double()[:, None, None] * (pos - key).abs()
    p = x.masked_fill(key > pos, float("-inf")).softmax(-1)
    check_attention(out[:reqs[0][0]], torch.einsum("hqk,khd->qhd", p, v), torch.einsum("hqk,khd->qhd", p, v.abs()), torch.bfloat16)


@pytest.mark.parametrize("reqs,lens", [([(6, 0), (1, 40)], [3, 41]), ([(150, 0), (2, 40)], [130, 42])])  # streamed, tcgen05
@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 100, 1 << 20])
def test_a_window_of_everything(reqs, lens, window):
    """With a window past all keys a request's mask is the causal one, also where its first
    rows lie before position 0 (fewer cached keys than new tokens)."""
    q, kc, vc, bt, cu, _ = paged_batch(reqs, 8, 2, 128, 16, torch.bfloat16, 3)
    out, lse = paged_ragged_attention(q, kc, vc, bt, cu, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window,
                                      return_lse=True)
    o, l64, a = attention64(q, kc, vc, bt, reqs, lens=lens)
    check_attention(out, o, a, torch.bfloat16)
    assert torch.equal(torch.isinf(lse), torch.isinf(l64))
