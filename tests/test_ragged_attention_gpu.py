"""Ragged attention over the paged cache against its definition in 64 bits: every length
from an absent request to long ones, head layouts, block sizes, masks and score
transforms, and the places where a mask, a stale slot or a stride can go wrong."""
import pytest
import torch

from gqa_kernels import check_device_error, paged_ragged_attention
from gqa_kernels.paged import paged_prefill
from tests._serving import attention64, attention_bound, check_attention, cu_of, paged_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib_ready(cuda_lib):
    check_device_error()
    yield
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)


def run(reqs, hq, hkv, d, block, dtype, seed=0, poison=float("nan"), q_scale=1.0, **kw):
    q, kc, vc, bt, cu, lens = paged_batch(reqs, hq, hkv, d, block, dtype, seed, poison, q_scale=q_scale)
    bounds = dict(max_query_len=max(x for x, _ in reqs), max_seq_len=max(sum(r) for r in reqs))
    ref_kw = {"alibi": kw.get("alibi_slopes"), "prefix": kw.get("prefix_lens"), "starts": kw.get("key_starts")}
    ref_kw.update({k: v for k, v in kw.items() if k in ("scale", "causal", "softcap", "window")})
    out, lse = paged_ragged_attention(q, kc, vc, bt, cu, lens, return_lse=True, **bounds, **kw)
    kz, vz = kc.nan_to_num(0, 0, 0), vc.nan_to_num(0, 0, 0)
    o, l64, a = attention64(q, kz, vz, bt, reqs, **ref_kw)
    check_attention(out, o, a, dtype)
    empty = torch.isinf(l64)
    assert torch.equal(torch.isinf(lse), empty)
    # the sum of n exponentials good to 1e-4 relative; the scores' own error in it
    assert ((lse.double() - l64)[~empty].abs() <= 2e-4 + 1e-6 * l64[~empty].abs()).all()
    return out


MIXES = {
    "one_token": [(1, 0)],
    "decodes": [(1, 0), (1, 1), (1, 62), (1, 63), (1, 64), (1, 700)],
    "absent": [(0, 0), (1, 5), (0, 40), (3, 9), (0, 0)],
    "drafts": [(5, 100), (1, 1), (9, 640), (2, 126), (8, 0)],
    "chunks": [(130, 0), (1, 300), (70, 250), (257, 3), (0, 7), (33, 1)],
    "long_context": [(1, 9000), (3, 4100), (40, 5000)],
}


@pytest.mark.parametrize("mix", sorted(MIXES))
@pytest.mark.parametrize("hq,hkv,d,block,dtype", [
    (8, 2, 128, 64, torch.bfloat16), (4, 4, 64, 16, torch.float16), (14, 2, 128, 32, torch.float16),
    (5, 1, 64, 128, torch.bfloat16), (16, 1, 128, 16, torch.bfloat16), (64, 1, 64, 64, torch.float16)])
def test_causal(mix, hq, hkv, d, block, dtype):
    run(MIXES[mix], hq, hkv, d, block, dtype, seed=hq + d)


def slopes(hq):
    return torch.exp2(-8.0 / hq * torch.arange(1, hq + 1, dtype=torch.float32, device="cuda"))


@pytest.mark.parametrize("mix", ["drafts", "chunks", "long_context"])
@pytest.mark.parametrize("d,block,dtype", [(128, 64, torch.bfloat16), (64, 16, torch.float16)])
@pytest.mark.parametrize("case", ["cap", "cap_hard", "alibi", "window", "window_1", "prefix", "all", "full"])
def test_masks_and_scores(mix, d, block, dtype, case):
    reqs, hq, hkv = MIXES[mix], 8, 2
    prefix = torch.tensor([min(sum(r), 90) for r in reqs], dtype=torch.int32, device="cuda")
    kw = {"cap": dict(softcap=20.0), "cap_hard": dict(softcap=1.5, q_scale=6.0), "alibi": dict(alibi_slopes=slopes(hq)),
          "window": dict(window=77), "window_1": dict(window=1), "prefix": dict(prefix_lens=prefix),
          "all": dict(softcap=30.0, alibi_slopes=slopes(hq), window=200, prefix_lens=prefix),
          "full": dict(causal=False, scale=0.2)}[case]
    run(reqs, hq, hkv, d, block, dtype, seed=3, **kw)


@pytest.mark.parametrize("mix", ["drafts", "chunks", "long_context"])
@pytest.mark.parametrize("softcap", [0.0, 25.0])
def test_documents(mix, softcap):
    """Documents packed into a request, of one to hundreds of tokens."""
    reqs = MIXES[mix]
    g = torch.Generator().manual_seed(1)
    starts = []
    for qn, c in reqs:
        at, left = 0, 0
        for p in range(qn + c):
            if left == 0:
                at, left = p, int(torch.randint(1, 120, (1,), generator=g)) if p % 3 else 1
            left -= 1
            if p >= c:
                starts.append(at)
    run(reqs, 8, 2, 128, 16, torch.bfloat16, seed=4, softcap=softcap,
        key_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("first,n", [(100, 256), (200, 200 + 33), (64, 1000)])
def test_low_scores_after_hidden_small_ones(first, n):
    """A document whose scores are all far below 0, after one with scores near 0 that it does
    not see: what it does not see sets no scale for it."""
    d, block, cap = 128, 16, 1000.0
    q, kc, vc, bt, cu, lens = paged_batch([(n, 0)], 8, 2, d, block, torch.bfloat16, 21, 0.0)
    q += 20.0
    for k in range(n):
        row = kc[bt[0, k // block], k % block]
        row.copy_(row * 0.05 - 1.3 if k >= first else row * 0.01)
    starts = torch.zeros(n, dtype=torch.int32, device="cuda")
    starts[first:] = first
    out = paged_ragged_attention(q, kc, vc, bt, cu, lens, softcap=cap, key_starts=starts)
    o, _, a = attention64(q, kc, vc, bt, [(n, 0)], softcap=cap, starts=starts)
    check_attention(out, o, a, torch.bfloat16)


def test_rows_that_see_nothing_are_zero():
    """Key starts past the token, at the end of the keys, and a request whose cache is
    shorter than its new tokens: zero rows and -inf, their neighbours untouched."""
    for reqs in ([(4, 60), (130, 20), (1, 0)], [(1, 7), (1, 2000)]):
        q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, torch.bfloat16, 5, float("inf"))
        t = q.shape[0]
        starts = torch.zeros(t, dtype=torch.int32, device="cuda")
        starts[::3] = 1 << 30
        out, lse = paged_ragged_attention(q, kc, vc, bt, cu, lens, key_starts=starts, return_lse=True)
        assert (out[::3] == 0).all() and torch.isneginf(lse[::3]).all()
        o, l64, a = attention64(q, kc.nan_to_num(0, 0, 0), vc.nan_to_num(0, 0, 0), bt, reqs, starts=starts)
        check_attention(out, o, a, torch.bfloat16)
        # lengths below the query lengths: the first rows lie before position 0
        short = [max(0, x - 3) if x > 1 else 0 for x, _ in reqs]
        out, lse = paged_ragged_attention(q, kc, vc, bt, cu, torch.tensor(short, dtype=torch.int32, device="cuda"),
                                          return_lse=True)
        o, l64, a = attention64(q, kc.nan_to_num(0, 0, 0), vc.nan_to_num(0, 0, 0), bt, reqs, lens=short)
        check_attention(out, o, a, torch.bfloat16)
        assert torch.equal(torch.isinf(lse), torch.isinf(l64))


@pytest.mark.parametrize("block", [16, 64])
def test_freed_blocks_before_a_window_are_not_seen(block):
    """Blocks that a window has left behind may be gone (-1) or hold another request's
    values, not numbers among them; keys of the first block before the window too."""
    reqs, window = [(1, 800), (5, 700), (150, 900)], 100
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, block, torch.bfloat16, 6, float("nan"))
    o, _, a = attention64(q, kc.nan_to_num(0), vc.nan_to_num(0), bt, reqs, window=window)
    bt = bt.clone()
    for b, (qn, c) in enumerate(reqs):
        first = c - window + 1
        for j in range(first // block):
            kc[bt[b, j]] = float("nan")
            vc[bt[b, j]] = float("inf")
            if j % 2:
                bt[b, j] = -1
        kc[bt[b, first // block], :first % block] = float("nan")
        vc[bt[b, first // block], :first % block] = float("nan")
    out = paged_ragged_attention(q, kc, vc, bt, cu, lens, window=window)
    check_attention(out, o, a, torch.bfloat16)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 2, 64)])
def test_strides(hq, hkv, d):
    """Queries as a slice of a fused projection, caches interleaved per block, an output
    with padded rows, and arrays that are not contiguous."""
    reqs = [(3, 90), (140, 33), (1, 400)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, hq, hkv, d, 64, torch.bfloat16, 7)
    t = q.shape[0]
    fused = torch.randn(t, hq + 2 * hkv, d, device="cuda").to(torch.bfloat16)
    fused[:, :hq] = q
    both = torch.stack([kc, vc], dim=1)  # (num_blocks, 2, block, hkv, d)
    wide = torch.full((t, hq, d + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    bt2 = torch.stack([bt, bt], dim=2)[:, :, 0]
    out = paged_ragged_attention(fused[:, :hq], both[:, 0], both[:, 1], bt2, cu, lens, out=wide[:, :, :d])
    o, _, a = attention64(q, kc, vc, bt, reqs)
    check_attention(out, o, a, torch.bfloat16)
    assert (wide[:, :, d:] == 7.0).all()
    odd = torch.zeros(t, hq, d + 3, dtype=torch.bfloat16, device="cuda")  # rows not 16-byte aligned: copied
    odd[:, :, :d] = q
    check_attention(paged_ragged_attention(odd[:, :, :d], kc, vc, bt, cu, lens), o, a, torch.bfloat16)


def test_padding_rows_are_left_alone():
    reqs = [(2, 50), (1, 9)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, torch.float16, 8)
    padded = torch.cat([q, torch.full((5, 8, 128), float("nan"), dtype=torch.float16, device="cuda")])
    out = torch.full_like(padded, 3.0)
    paged_ragged_attention(padded, kc, vc, bt, cu, lens, out=out)
    o, _, a = attention64(q, kc, vc, bt, reqs)
    check_attention(out[:3], o, a, torch.float16)
    assert (out[3:] == 3.0).all()


def test_nothing_to_do():
    q, kc, vc, bt, cu, lens = paged_batch([(1, 3)], 8, 2, 128, 64, torch.bfloat16, 9)
    assert paged_ragged_attention(q[:0], kc, vc, bt, cu_of([0]), lens).shape == (0, 8, 128)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged_ragged_attention(q[:0], kc, vc, bt[:0], cu_of([]), empty).shape == (0, 8, 128)


@pytest.mark.parametrize("reqs", [[(1, 500), (1, 70), (1, 4000)], [(4, 200), (1, 77), (9, 1000)], [(90, 120), (1, 5)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_e4m3_caches(reqs, dtype, softcap):
    """Against 64 bits on the values that the caches stand for. Both MMAs run in f16, so
    P's rounding is f16's; bf16 queries are exact in f16 at these sizes or round to 2^-11."""
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, dtype, 10)
    ks, vs = 0.5, 0.25
    k8, v8 = (kc.float() / ks).to(torch.float8_e4m3fn), (vc.float() / vs).to(torch.float8_e4m3fn)
    out = paged_ragged_attention(q, k8, v8, bt, cu, lens, softcap=softcap, k_scale=ks, v_scale=vs)
    o, _, a = attention64(q, k8.double() * ks, v8.double() * vs, bt, reqs, softcap=softcap)
    check_attention(out, o, a, dtype)


def test_agrees_with_equal_chunks():
    """A batch of equal chunks is what paged_prefill computes."""
    reqs = [(64, 300 + 64 * i) for i in range(5)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 32, 8, 128, 64, torch.bfloat16, 11)
    out = paged_ragged_attention(q, kc, vc, bt, cu, lens)
    same = paged_prefill(q.view(5, 64, 32, 128).transpose(1, 2), kc, vc, bt, lens).transpose(1, 2).reshape(q.shape)
    o, _, a = attention64(q, kc, vc, bt, reqs)
    assert ((out.double() - same.double()).abs() <= 2 * attention_bound(o, a, torch.bfloat16)).all()


def test_many_requests_and_wide_bounds():
    """Hundreds of requests with bounds far above the lengths, as a captured step has."""
    g = torch.Generator().manual_seed(12)
    reqs = [(int(torch.randint(0, 4, (1,), generator=g)), int(torch.randint(0, 150, (1,), generator=g))) for _ in range(700)]
    reqs[350] = (200, 10)
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 4, 1, 64, 16, torch.float16, 12)
    wide = torch.zeros(700, 512, dtype=torch.int32, device="cuda")
    wide[:, :bt.shape[1]] = bt
    o, _, a = attention64(q, kc, vc, bt, reqs)
    check_attention(paged_ragged_attention(q, kc, vc, wide, cu, lens), o, a, torch.float16)


def test_repeats_bit_for_bit_and_on_another_stream():
    reqs = [(1, 12000), (7, 3000), (300, 2000), (1, 30)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, torch.bfloat16, 13)
    first = paged_ragged_attention(q, kc, vc, bt, cu, lens, softcap=30.0)
    for _ in range(3):
        assert torch.equal(paged_ragged_attention(q, kc, vc, bt, cu, lens, softcap=30.0), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_ragged_attention(q, kc, vc, bt, cu, lens, softcap=30.0)
    side.synchronize()
    assert torch.equal(other, first)


def test_captured_step_follows_its_lengths():
    """A step captured once, replayed after the lengths on the device changed."""
    reqs = [(2, 600), (1, 100), (3, 900)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, torch.bfloat16, 14)
    out = torch.empty_like(q)
    paged_ragged_attention(q, kc, vc, bt, cu, lens, max_query_len=8, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_ragged_attention(q, kc, vc, bt, cu, lens, max_query_len=8, out=out)
    for change in ([(2, 600), (1, 100), (3, 900)], [(1, 90), (2, 30), (3, 511)], [(5, 5), (0, 0), (1, 0)]):
        cu.copy_(cu_of([x for x, _ in change]))
        lens.copy_(torch.tensor([sum(r) for r in change], dtype=torch.int32))
        graph.replay()
        o, _, a = attention64(q, kc, vc, bt, change)
        check_attention(out, o, a, torch.bfloat16)


def test_cache_offsets_past_32_bits():
    """Blocks whose first element lies past 2^31 elements (2^32 bytes) of the cache."""
    hkv, d, block = 8, 128, 64
    num_blocks = (1 << 31) // (hkv * d * block) + 40
    reqs = [(2, 130), (140, 60), (1, 700)]
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 16, hkv, d, block, torch.bfloat16, 15, spare=0)
    big_k = torch.empty(num_blocks, block, hkv, d, dtype=torch.bfloat16, device="cuda")
    big_v = torch.empty_like(big_k)
    far = num_blocks - kc.shape[0]
    big_k[far:], big_v[far:] = kc, vc
    out = paged_ragged_attention(q, big_k, big_v, bt + far, cu, lens)
    o, _, a = attention64(q, kc, vc, bt, reqs)
    check_attention(out, o, a, torch.bfloat16)
