"""The ragged step's other operators on the GPU: the plan against a token-by-token
restatement (equal), norm + rotation + cache write against 64 bits, verification
against a request-by-request restatement (equal)."""
import pytest
import torch

from gqa_kernels import (StepPlan, check_device_error, plan_step, qk_norm_rope, qk_norm_rope_append, rope_table,
                         verify_drafts, verify_drafts_greedy)
from gqa_kernels.paged import paged_kv_append
from tests._serving import UNIT, cu_of, plan64, rope64, verify64

pytestmark = pytest.mark.gpu
GQA_ERR_INVALID_ARG = 1


@pytest.fixture(autouse=True)
def _lib_ready(cuda_lib):
    check_device_error()
    yield
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------------------- plan
def plan_case(n, seed, block, width, q_most, ctx_most, free_share, extra_held=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, q_most + 1, (n,), generator=g).tolist()
    c = torch.randint(0, ctx_most + 1, (n,), generator=g).tolist()
    held = [min(width, -(-x // block) + (extra_held if i % 3 == 0 else 0)) for i, x in enumerate(c)]
    need = sum(max(0, -(-(a + b) // block) - h) for a, b, h in zip(q, c, held))
    ids = torch.randperm(sum(held) + need + 5, generator=g).tolist()
    table, at = [[-7] * width for _ in range(n)], 0
    for b in range(n):
        for j in range(held[b]):
            table[b][j] = ids[at]
            at += 1
    free = ids[at:]
    return q, c, table, held, free, int(need * free_share)


@pytest.mark.parametrize("n,block,width,q_most,ctx_most,free_share,extra", [
    (1, 16, 8, 1, 50, 1.0, 0), (1, 64, 4, 200, 0, 1.0, 0), (5, 1, 40, 3, 20, 1.0, 1), (33, 16, 32, 9, 300, 1.0, 2),
    (300, 32, 16, 40, 200, 0.6, 1), (1024, 64, 8, 3, 400, 0.9, 0), (1025, 16, 64, 70, 500, 0.5, 3), (2500, 16, 24, 5, 300, 1.0, 0),
    (64, 16, 6, 60, 90, 1.0, 0)])  # the last: rows too short for some requests
def test_plan(n, block, width, q_most, ctx_most, free_share, extra):
    q, c, table, held, free, count = plan_case(n, n, block, width, q_most, ctx_most, free_share, extra)
    max_tokens = sum(q) + 13
    want, want_table, left = plan64(q, c, table, held, free, count, block, max_tokens)
    bt = i32(table)
    args = (i32(q), i32(c), bt, i32(held), i32(free), i32([count]), block, max_tokens)
    p = plan_step(*args)
    for _ in range(2):  # a plan can be made again: it advances nothing
        assert p.cu_query_lens.tolist() == want["cu"] and p.seq_lens.tolist() == want["seq"]
        assert p.granted.tolist() == want["granted"] and p.blocks_held.tolist() == want["held"]
        assert p.positions.tolist() == want["pos"] and p.slot_mapping.tolist() == want["slot"]
        assert p.token_seqs.tolist() == want["seqs"] and p.free_count.tolist() == [left]
        assert bt.tolist() == want_table
        p = plan_step(*args, out=p)


def test_plan_of_nothing_and_strided_table():
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    p = plan_step(e, e, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), e, i32([3, 4]), i32([2]), 16, 5)
    assert p.cu_query_lens.tolist() == [0] and p.positions.tolist() == [-1] * 5 and p.free_count.tolist() == [2]
    wide = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    p = plan_step(i32([1, 20, 2]), i32([0, 0, 0]), wide[:, 2:6], i32([0, 0, 0]), i32([9, 8, 7, 6]), i32([4]), 16, 23)
    assert wide.tolist() == [[-1, -1, 6] + [-1] * 7, [-1, -1, 7, 8] + [-1] * 6, [-1, -1, 9] + [-1] * 7]
    assert p.slot_mapping[:2].tolist() == [6 * 16, 7 * 16] and p.free_count.tolist() == [0]


def test_plan_with_too_many_tokens_is_cut_and_reported():
    p = plan_step(i32([5, 6]), i32([0, 0]), torch.zeros(2, 2, dtype=torch.int32, device="cuda"), i32([0, 0]), i32([1, 2]), i32([2]),
                  16, 8)
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 211)
    assert p.cu_query_lens.tolist() == [0, 5, 11] and p.positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2]


def test_plan_output_may_not_be_its_input():
    args = [i32([1]), i32([0]), torch.zeros(1, 2, dtype=torch.int32, device="cuda"), i32([0]), i32([1, 2]), i32([2])]
    p = plan_step(*args, 16, 4)
    for at, name in ((3, "blocks_held"), (5, "free_count"), (1, "seq_lens")):
        bad = list(args)
        bad[at] = getattr(p, name)
        with pytest.raises(ValueError):
            plan_step(*bad, 16, 4, out=p)
    assert plan_step(args[0], p.seq_lens, args[2], p.blocks_held, args[4], p.free_count, 16, 4).seq_lens.tolist() == [2]


# ----------------------------------------------------------------------------- norm, rotation, cache write
def rope_inputs(t, hq, hkv, d, rot, axes, dtype, seed, max_pos=3000):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(t, hq + 2 * hkv, d, generator=g, device="cuda").mul_(2.0).to(dtype)
    pos = torch.randint(0, max_pos, (axes, t), generator=g, device="cuda", dtype=torch.int32)
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device="cuda")).to(dtype)
    table = rope_table(max_pos, rot)
    half = rot // 2
    sizes = [half] if axes == 1 else [half - (axes - 1) * (half // 4 + 1)] + [half // 4 + 1] * (axes - 1)
    axis = torch.repeat_interleave(torch.arange(axes), torch.tensor(sizes)).cuda()
    at = pos.long()[axis].t()
    f = torch.arange(half, device="cuda")
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], pos, w, table, sizes, table[at, f], table[at, half + f]


def close(got, want, dtype):
    """One rounding to dtype, and fp32 arithmetic of a norm and two products (a few 2^-24
    of the row's largest value; f16's smallest steps are 2^-24)."""
    tol = UNIT[dtype] * want.abs() * (1 + 2.0 ** -10) + 2e-6 * want.abs().amax(-1, keepdim=True) + 2.0 ** -24
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("t,hq,hkv,d,rot,axes,norm,inter,dtype", [
    (1, 8, 2, 128, 128, 1, True, False, torch.bfloat16), (1, 1, 1, 64, 64, 1, False, True, torch.float16),
    (37, 7, 1, 128, 64, 1, True, False, torch.float16), (300, 32, 8, 128, 128, 3, True, False, torch.bfloat16),
    (65, 10, 5, 64, 32, 2, True, True, torch.bfloat16), (20, 4, 4, 64, 64, 4, False, False, torch.float16),
    (9, 64, 1, 128, 16, 1, True, True, torch.bfloat16), (5, 3, 3, 128, 0, 1, True, False, torch.float16)])
def test_rope(t, hq, hkv, d, rot, axes, norm, inter, dtype):
    q, k, v, pos, w, table, sizes, cos, sin = rope_inputs(t, hq, hkv, d, rot, axes, dtype, t + d)
    qw, kw = (w[0], w[1]) if norm else (None, None)
    kwargs = dict(q_weight=qw, k_weight=kw, eps=1e-5, sections=sizes, interleaved=inter)
    positions = pos if axes > 1 else pos[0]
    q64, k64 = rope64(q, qw, 1e-5, cos, sin, inter), rope64(k, kw, 1e-5, cos, sin, inter)
    qo, ko = qk_norm_rope(q, k, positions, table, **kwargs)
    close(qo, q64, dtype)
    close(ko, k64, dtype)
    # and into the cache: the same keys, the values as they are, every other slot untouched
    block, blocks = 16, t // 16 + 3
    g = torch.Generator().manual_seed(t)
    slots = torch.randperm(blocks * block, generator=g)[:t].cuda()
    slots[::4] = -1
    kc = torch.full((blocks, block, hkv, d), 5.0, dtype=dtype, device="cuda")
    vc = torch.full_like(kc, 6.0)
    qa = qk_norm_rope_append(q, k, v, positions, table, kc, vc, slots, **kwargs)
    assert torch.equal(qa, qo)
    ek, ev = torch.full_like(kc, 5.0).view(-1, hkv, d), torch.full_like(vc, 6.0).view(-1, hkv, d)
    keep = slots >= 0
    ek[slots[keep]], ev[slots[keep]] = ko[keep], v[keep]
    assert torch.equal(kc.view(-1, hkv, d), ek) and torch.equal(vc.view(-1, hkv, d), ev)


@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_rope_into_e4m3_caches(d, dtype):
    t, hq, hkv, ks, vs = 90, 8, 2, 0.25, 0.125
    q, k, v, pos, w, table, sizes, cos, sin = rope_inputs(t, hq, hkv, d, d, 1, dtype, 3)
    slots = torch.randperm(128, generator=torch.Generator().manual_seed(1))[:t].cuda()
    kc = torch.zeros(8, 16, hkv, d, dtype=torch.float8_e4m3fn, device="cuda")
    vc, vw = torch.zeros_like(kc), torch.zeros_like(kc)
    qk_norm_rope_append(q, k, v, pos[0], table, kc, vc, slots, w[0], w[1], k_scale=ks, v_scale=vs)
    paged_kv_append(k, v, torch.zeros_like(kc), vw, slots, ks, vs)
    assert torch.equal(vc.view(torch.uint8), vw.view(torch.uint8))
    got = kc.view(-1, hkv, d)[slots].double() * ks
    want = rope64(k, w[1], 1e-6, cos, sin, False)
    # e4m3 keeps 4 bits: half a unit is 2^-4 of the value; its smallest step is 2^-9
    assert ((got - want).abs() <= want.abs() * 2.0 ** -4 * 1.001 + ks * 2.0 ** -10 * 1.001).all()


def test_rope_padding_and_bad_positions_and_slots():
    t, hq, hkv, d = 6, 4, 2, 128
    q, k, v, pos, w, table, _, cos, sin = rope_inputs(t, hq, hkv, d, d, 1, torch.bfloat16, 5)
    p = pos[0].clone()
    p[2] = -1
    kc = torch.zeros(2, 16, hkv, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    slots = torch.tensor([0, 1, 2, -1, 4, 5], device="cuda")
    out = qk_norm_rope_append(q, k, v, p, table, kc, vc, slots)
    assert (out[2] == 0).all() and (out[3] != 0).any() and (kc[0, 2] == 0).all() and (vc[0, 2:4] == 0).all()
    assert torch.equal(vc[0, 4], v[4])
    qo, ko = qk_norm_rope(q, k, p, table)
    assert torch.equal(qo, out) and (ko[2] == 0).all()
    p[4] = table.shape[0]
    out = qk_norm_rope_append(q, k, v, p, table, kc, vc, slots)
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 212) and (out[4] == 0).all()
    guard_k, guard_v = torch.zeros(3, 16, hkv, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(
        3, 16, hkv, d, dtype=torch.bfloat16, device="cuda")
    slots[5] = 32
    qk_norm_rope_append(q, k, v, pos[0], table, guard_k[:2], guard_v[:2], slots)
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 213) and (guard_k[2] == 0).all() and (guard_v[2] == 0).all()


def test_rope_nonfinite_rows_stay_their_own():
    q, k, v, pos, w, table, _, cos, sin = rope_inputs(4, 4, 2, 128, 128, 1, torch.float16, 6)
    q, k = q.clone(), k.clone()
    q[1, 2, 5], k[3, 1, 0] = float("nan"), float("inf")
    qo, ko = qk_norm_rope(q, k, pos[0], table, w[0], w[1])
    assert torch.isnan(qo[1, 2]).all() and torch.isnan(ko[3, 1]).any()
    qo[1, 2], ko[3, 1] = 0, 0
    assert torch.isfinite(qo).all() and torch.isfinite(ko).all()


def test_rope_slots_past_32_bits():
    hkv, d, block = 8, 128, 16
    blocks = (1 << 31) // (hkv * d * block) + 2
    q, k, v, pos, w, table, _, cos, sin = rope_inputs(3, 8, hkv, d, d, 1, torch.bfloat16, 7)
    kc = torch.empty(blocks, block, hkv, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    slots = torch.tensor([blocks * block - 1, blocks * block - 9, 3], device="cuda")
    qk_norm_rope_append(q, k, v, pos[0], table, kc, vc, slots)
    assert torch.equal(vc.view(-1, hkv, d)[slots], v)
    assert torch.equal(kc.view(-1, hkv, d)[slots], qk_norm_rope(q, k, pos[0], table)[1])


# ----------------------------------------------------------------------------- verification
def verify_inputs(rows, k, vocab, dtype, seed, tied=False):
    g = torch.Generator().manual_seed(seed)
    n, total = len(rows), sum(rows)
    logits = torch.randn(total, vocab, generator=g) * 2
    if tied:
        logits = logits.round()  # many equal entries
    target = logits.softmax(-1).to(dtype)
    near = torch.randn(n, k, vocab, generator=g) * 2
    at = 0
    for b, r in enumerate(rows):
        m = min(k, r)
        near[b, :m] = logits[at:at + m] + 0.5 * near[b, :m]
        at += r
    draft = near.softmax(-1).to(dtype)
    tokens = torch.multinomial(draft.float().view(-1, vocab) + 1e-9, 1, generator=g).view(n, k).int() if n * k else \
        torch.zeros(n, k, dtype=torch.int32)
    uni = torch.rand(n, k, generator=g)
    expo = torch.empty(n, vocab).exponential_(generator=g)
    return target, draft, tokens, uni, expo, cu_of(rows, "cpu")


@pytest.mark.parametrize("rows,k,vocab,dtype", [
    ([1], 0, 11, torch.float32), ([1, 1, 1], 3, 1000, torch.float32), ([5, 1, 0, 3, 5], 4, 5003, torch.float32),
    ([65, 40], 64, 257, torch.float32), ([3] * 40, 2, 32001, torch.float32), ([4, 2, 4], 3, 50000, torch.bfloat16),
    ([4, 2, 4], 3, 49999, torch.float16), ([2, 9], 3, 8, torch.float32), ([3] * 200, 2, 333, torch.float32)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(rows, k, vocab, dtype, certain):
    target, draft, tokens, uni, expo, cu = verify_inputs(rows, k, vocab, dtype, len(rows) + vocab)
    if k and len(rows) > 1:
        tokens[1, 0] = vocab + 5  # out of the vocabulary: refused
    want, num = verify64(tokens.tolist(), target, None if certain else draft, uni, expo, cu.tolist())
    for _ in range(2):
        got, gn = verify_drafts(tokens.cuda(), target.cuda(), None if certain else draft.cuda(), uni.cuda(), expo.cuda(), cu.cuda())
        assert gn.tolist() == num and got.tolist() == want


def test_verify_without_weight_left_and_strides():
    """p == q with a refused draft of probability zero leaves no weight: the row's first
    largest probability. Inputs as slices of wider arrays."""
    vocab, n, k = 4100, 6, 2
    target, draft, tokens, uni, expo, cu = verify_inputs([3] * n, k, vocab, torch.float32, 1)
    for b in range(n):
        draft[b, 0] = target[3 * b]
        target[3 * b, 17] = draft[b, 0, 17] = 0.0
        tokens[b, 0] = 17
    want, num = verify64(tokens.tolist(), target, draft, uni, expo, cu.tolist())
    wt = torch.zeros(3 * n, vocab + 3, device="cuda")
    wt[:, 1:vocab + 1] = target.cuda()
    wd = torch.zeros(n, k + 1, vocab + 2, device="cuda")
    wd[:, :k, :vocab] = draft.cuda()
    we = torch.ones(n, vocab + 1, device="cuda")
    we[:, 1:] = expo.cuda()
    wide = torch.zeros(n, k + 5, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + k] = tokens.cuda()
    got, gn = verify_drafts(wide[:, 2:2 + k], wt[:, 1:vocab + 1], wd[:, :k, :vocab], uni.cuda(), we[:, 1:], cu.cuda())
    assert gn.tolist() == num == [1] * n and got.tolist() == want


def test_verify_keeps_the_targets_distribution():
    """Over many requests of one draft, the first emitted token is distributed as the
    target, whatever the draft: each frequency within 5 standard deviations."""
    n, vocab = 16000, 12
    g = torch.Generator().manual_seed(2)
    p = torch.rand(vocab, generator=g).softmax(-1)
    q = (2 * torch.rand(vocab, generator=g)).softmax(-1)
    drafts = torch.multinomial(q, n, replacement=True, generator=g).int()[:, None]
    target = p.expand(2 * n, vocab).contiguous()
    got, _ = verify_drafts(drafts.cuda(), target.cuda(), q.expand(n, 1, vocab).contiguous().cuda(),
                           torch.rand(n, 1, generator=g).cuda(), torch.empty(n, vocab).exponential_(generator=g).cuda(),
                           cu_of([2] * n))
    freq = torch.bincount(got[:, 0].cpu(), minlength=vocab) / n
    assert ((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all()


@pytest.mark.parametrize("rows,k,vocab,dtype", [
    ([1], 0, 9, torch.float32), ([5, 1, 0, 3, 5], 4, 5003, torch.bfloat16), ([65, 2], 64, 300, torch.float16),
    ([4] * 30, 3, 40001, torch.float32), ([2, 9], 3, 8, torch.bfloat16), ([3] * 300, 2, 128, torch.float32)])
def test_verify_greedy(rows, k, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(sum(rows), vocab, generator=g) * 4).round().to(dtype)  # ties in most rows
    best = [int(torch.nonzero(r == r.max())[0]) for r in logits.float()]
    cu = cu_of(rows, "cpu").tolist()
    tokens = torch.randint(0, vocab, (len(rows), k), generator=g, dtype=torch.int32)
    want, num = [], []
    for b, r in enumerate(rows):
        m = min(r - 1, k)
        for i in range(max(0, m)):
            if torch.rand(1, generator=g) < 0.8:
                tokens[b, i] = best[cu[b] + i]
        i = 0
        while i < m and int(tokens[b, i]) == best[cu[b] + i]:
            i += 1
        want.append(tokens[b, :i].tolist() + [best[cu[b] + i]] + [-1] * (k - i) if r else [-1] * (k + 1))
        num.append(i + 1 if r else 0)
    for _ in range(2):
        got, gn = verify_drafts_greedy(tokens.cuda(), logits.cuda(), cu_of(rows))
        assert got.tolist() == want and gn.tolist() == num


def test_verify_greedy_odd_rows():
    logits = torch.full((3, 70), float("-inf"))
    logits[1, 3] = float("nan")
    logits[2, 60] = float("inf")
    got, num = verify_drafts_greedy(torch.zeros(3, 0, dtype=torch.int32, device="cuda"), logits.cuda(), cu_of([1, 1, 1]))
    assert got.tolist() == [[0], [0], [60]] and num.tolist() == [1, 1, 1]


def test_workspace_shared_by_calls_of_all_shapes():
    """Verification and attention of changing shapes in one workspace: counters stay zero."""
    for seed, (rows, k, vocab) in enumerate([([3] * 50, 2, 40000), ([2], 1, 90000), ([4] * 7, 3, 1000), ([3] * 50, 2, 40000)]):
        target, draft, tokens, uni, expo, cu = verify_inputs(rows, k, vocab, torch.float32, seed)
        want, num = verify64(tokens.tolist(), target, draft, uni, expo, cu.tolist())
        got, gn = verify_drafts(tokens.cuda(), target.cuda(), draft.cuda(), uni.cuda(), expo.cuda(), cu.cuda())
        assert got.tolist() == want and gn.tolist() == num
        verify_drafts_greedy(tokens.cuda(), target.cuda(), cu.cuda())


def test_plan_buffers_are_reused():
    out = StepPlan.empty(2, 10)
    args = (i32([2, 3]), i32([0, 4]), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), i32([0, 1]), i32([5, 6, 7]), i32([3]))
    p = plan_step(*args, 4, 10, out=out)
    assert p is out and p.seq_lens.tolist() == [2, 7] and p.slot_mapping.tolist()[:5] == [28, 29, 24, 25, 26]
