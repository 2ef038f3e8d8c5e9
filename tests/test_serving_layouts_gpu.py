"""Layouts that the ragged step's operators copy or that do not matter to them: bases that are
not 16-byte aligned, and odd strides of dimensions of size 1 (one token of a projection
with padded rows, one kv head)."""
import pytest
import torch

from gqa_kernels import check_device_error, paged_ragged_attention, qk_norm_rope, qk_norm_rope_append, rope_table
from tests._serving import attention64, check_attention, paged_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib_ready(cuda_lib):
    check_device_error()
    yield
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)


def shifted(x, by):
    """x's values, contiguous on a base `by` elements past an aligned one."""
    buf = torch.empty(x.numel() + by, dtype=x.dtype, device=x.device)
    y = buf[by:].view(x.shape)
    y.copy_(x)
    return y


def odd_strides(x, last_of_one):
    """x's values with an odd stride in every dimension of size 1 but the last."""
    st = [s if n != 1 or i == x.dim() - 1 else last_of_one for i, (n, s) in enumerate(zip(x.shape, x.stride()))]
    return torch.as_strided(x, x.shape, st, x.storage_offset())


@pytest.mark.parametrize("reqs", [[(1, 70)], [(3, 90), (1, 20)], [(90, 10)]])
@pytest.mark.parametrize("by", [1, 4])
def test_attention_of_queries_on_an_unaligned_base(reqs, by):
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 16, torch.bfloat16, by)
    o, _, a = attention64(q, kc, vc, bt, reqs)
    check_attention(paged_ragged_attention(shifted(q, by), kc, vc, bt, cu, lens), o, a, torch.bfloat16)


@pytest.mark.parametrize("reqs,hq,hkv,d", [([(1, 70)], 8, 1, 128), ([(1, 300)], 1, 1, 64), ([(33, 40)], 4, 1, 128)])
def test_attention_of_size_one_dimensions(reqs, hq, hkv, d):
    q, kc, vc, bt, cu, lens = paged_batch(reqs, hq, hkv, d, 16, torch.float16, d + hq)
    o, _, a = attention64(q, kc, vc, bt, reqs)
    out = odd_strides(torch.empty_like(q), 3)
    got = paged_ragged_attention(odd_strides(q, 5), odd_strides(kc, 7), odd_strides(vc, 9), bt, cu, lens, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_attention(got, o, a, torch.float16)
    wide = torch.zeros(reqs[0][0], hq * d + 2 * hkv * d + 3, dtype=torch.float16, device="cuda")  # a projection with padded rows
    wide[:, :hq * d] = q.view(-1, hq * d)
    check_attention(paged_ragged_attention(wide[:, :hq * d].view(-1, hq, d), kc, vc, bt, cu, lens), o, a, torch.float16)


@pytest.mark.parametrize("t,hq,hkv,d", [(1, 8, 2, 128), (1, 1, 1, 64), (7, 4, 1, 64)])
def test_rotation(t, hq, hkv, d):
    g = torch.Generator(device="cuda").manual_seed(t + d)
    q, k, v = (torch.randn(t, h, d, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv))
    pos = torch.randint(0, 50, (t,), generator=g, device="cuda", dtype=torch.int32)
    table = rope_table(50, d)
    want_q, want_k = qk_norm_rope(q, k, pos, table)
    for f in (lambda x: shifted(x, 1), lambda x: shifted(x, 4), lambda x: odd_strides(x, 3)):
        got_q, got_k = qk_norm_rope(f(q), f(k), pos, table)
        assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
        kc, vc = (torch.zeros(2, 16, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        got = qk_norm_rope_append(f(q), f(k), f(v), pos, table, kc, vc, torch.arange(t, device="cuda"))
        assert torch.equal(got, want_q) and torch.equal(kc.view(-1, hkv, d)[:t], want_k) and torch.equal(vc.view(-1, hkv, d)[:t], v)
