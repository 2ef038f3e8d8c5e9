"""The example's server with a pool that runs out: a refused request emits nothing, keeps
the token that it goes on from, and continues from it once the pool has blocks again."""
import pytest
import torch

from gqa_kernels import check_device_error
from tests.test_speculative_serving_gpu import dense_logits, example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafts,block,spare", [(3, 16, 5), (0, 16, 3), (5, 32, 1), (3, 16, 0)])
def test_refused_requests_go_on_where_they_were(example, drafts, block, spare):  # noqa: F811
    check_device_error()
    model = example.TinyDecoder(vocab=400, seed=drafts + block)
    prompts = [([7 * b + 1, 7 * b + 2, 5] * 12)[:30] for b in range(6)]
    held = 6 * -(-30 // block)
    total = held + 6 * 8
    server = example.Server(model, 6, num_blocks=total, block_size=block, max_blocks=8)
    server.free_count = torch.tensor([held + spare], dtype=torch.int32, device="cuda")
    first = server.prefill(prompts)
    own = [[t] for t in first.tolist()]
    last, refused = first, 0
    for phase in range(3):
        before = server.context_lens.tolist()
        out = server.decode(last, 8, drafts).tolist()
        counts = server.counts.tolist()
        for b in range(6):
            for tokens, n in zip(out[b], counts[b]):
                assert all(t >= 0 for t in tokens[:max(n, 1)]) and all(t == -1 for t in tokens[max(n, 1):])
                if n:
                    own[b] += tokens[:n]
                else:
                    refused += 1
                    assert tokens[0] == own[b][-1]
            assert int(server.context_lens[b]) == before[b] + sum(counts[b])
        last = torch.tensor([x[-1] for x in own], dtype=torch.int32, device="cuda")
        at, more = int(server.free_count), 2 + 4 * phase  # the pool gains blocks
        server.free_blocks[at:at + more] = torch.arange(total - more, total, dtype=torch.int32, device="cuda")
        total -= more
        server.free_count = server.free_count + more
    assert refused and check_device_error() == (0, 0)
    for b, prompt in enumerate(prompts):
        logits = dense_logits(model, prompt + own[b][:-1])[len(prompt) - 1:]
        chosen = logits.gather(1, torch.tensor(own[b], device="cuda")[:, None])[:, 0]
        # as the example's other test: bf16 activations, 2^-8 relative per layer step of logits of a few units
        assert float((logits.amax(1) - chosen).max()) <= 0.05 * float(logits.std()) + 0.02 * float(logits.abs().max())


def test_prompts_that_the_pool_cannot_hold_are_refused(example):  # noqa: F811
    model = example.TinyDecoder(vocab=100, layers=1, seed=1)
    with pytest.raises(ValueError):
        example.Server(model, 2, num_blocks=3, block_size=16, max_blocks=8).prefill([[1] * 30, [2] * 30])
    with pytest.raises(ValueError):
        example.Server(model, 2, num_blocks=9, block_size=16, max_blocks=2).prefill([[1] * 30, [2] * 33])
