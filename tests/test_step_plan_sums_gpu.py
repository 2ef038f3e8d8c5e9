"""The step plan where its sums pass 32 bits: token offsets stay at 2^31 - 1, the step is
reported as cut, and a request is granted what the pool has, not what a wrapped sum says."""
import pytest
import torch

from gqa_kernels import check_device_error, plan_step
from tests._serving import plan64

pytestmark = pytest.mark.gpu
GQA_ERR_INVALID_ARG = 1
MOST = (1 << 31) - 1


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def _lib_ready(cuda_lib):
    check_device_error()
    yield
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)


@pytest.mark.parametrize("max_tokens", [0, 7, 64])
@pytest.mark.parametrize("huge", [[MOST, MOST], [MOST] * 5, [MOST, 3, MOST - 2]])
def test_tokens_past_32_bits(huge, max_tokens):
    small = [5, 0, 19, 3]
    q = small + huge + small
    n, table = len(q), torch.full((len(q), 4), -9, dtype=torch.int32, device="cuda")
    p = plan_step(i32(q), i32([0] * n), table, i32([0] * n), i32(list(range(20))), i32([20]), 16, max_tokens)
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 211)
    # as if the huge requests were only too long for their rows: 100 tokens are so too
    few = [min(x, 100) for x in q]
    want, want_table, left = plan64(few, [0] * n, [[-9] * 4 for _ in range(n)], [0] * n, list(range(20)), 20, 16, max_tokens)
    cu = [0]
    for x in q:
        cu.append(min(MOST, cu[-1] + x))
    assert p.cu_query_lens.tolist() == cu and p.granted.tolist() == want["granted"] and table.tolist() == want_table
    assert p.seq_lens.tolist() == [x if ok else 0 for x, ok in zip(q, want["granted"])]
    assert p.blocks_held.tolist() == want["held"] and p.free_count.tolist() == [left]
    pos, slot, seqs = p.positions.tolist(), p.slot_mapping.tolist(), p.token_seqs.tolist()
    for t in range(max_tokens):
        b = max(i for i in range(n) if cu[i] <= t and q[i])
        assert seqs[t] == b and pos[t] == t - cu[b]
        assert slot[t] == (want_table[b][pos[t] // 16] * 16 + pos[t] % 16 if want["granted"][b] else -1)


def test_lengths_that_overflow_are_refused():
    p = plan_step(i32([5, MOST, 2]), i32([MOST - 2, 9, 1]), torch.zeros(3, 8, dtype=torch.int32, device="cuda"), i32([8, 8, 0]), i32([1, 2]),
                  i32([2]), 1 << 30, 8)
    torch.cuda.synchronize()
    assert check_device_error() == (GQA_ERR_INVALID_ARG, 211)
    assert p.granted.tolist() == [False, False, True] and p.seq_lens.tolist() == [MOST - 2, 9, 3]


@pytest.mark.parametrize("n", [700, 1030])
def test_blocks_past_32_bits(n):
    """Rows of 2^22 blocks, all of which every request needs: their sum passes 2^31 (2^32)."""
    width = 1 << 22
    table = torch.empty(n, width, dtype=torch.int32, device="cuda")
    q, free = [1] * n, list(range(2 * n))
    ctx = [0 if b % 10 == 3 else width - 1 for b in range(n)]
    held = [width if b % 10 == 7 else 0 for b in range(n)]
    p = plan_step(i32(q), i32(ctx), table, i32(held), i32(free), i32([2 * n]), 1, n)
    upto, granted, left = 0, [], 2 * n
    for b in range(n):
        need = max(0, ctx[b] + 1 - held[b])
        upto += need
        granted.append(need == 0 or upto <= 2 * n)
        left -= need if granted[-1] else 0
    assert p.granted.tolist() == granted and p.free_count.tolist() == [left]
    assert p.seq_lens.tolist() == [c + 1 if ok else c for c, ok in zip(ctx, granted)]
    assert all((s == -1) == (not ok) for s, ok, h in zip(p.slot_mapping.tolist(), granted, held) if not h)
