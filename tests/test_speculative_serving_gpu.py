"""The example that runs the ragged step's operators together (examples/speculative_serving.py).

Every token that speculative decoding emits at temperature zero must be the model's own
best next token: the whole sequence is scored once by a dense fp32 restatement of the
model, and each emitted token's logit has to reach the largest one up to what bf16
activations are off by."""
import importlib.util
import os

import pytest
import torch

from gqa_kernels import check_device_error

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(cuda_lib):
    spec = importlib.util.spec_from_file_location("speculative_serving", os.path.join(ROOT, "examples", "speculative_serving.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def dense_logits(model, ids):
    """The model in fp32, without a cache, on one sequence."""
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    n = len(ids)
    x = model.embedding[torch.tensor(ids, device="cuda")].float()
    for attention, qkv, out, up, down in model.layers:
        hq, hkv, d = attention.num_heads, attention.num_kv_heads, attention.head_dim
        y = (norm(x) @ qkv.float().t()).view(n, hq + 2 * hkv, d)
        q, k, v = norm(y[:, :hq]), norm(y[:, hq:hq + hkv]), y[:, hq + hkv:]
        c, s = attention.cos_sin[:n, None, :d // 2], attention.cos_sin[:n, None, d // 2:]

        def turn(z):
            a, b = z[..., :d // 2], z[..., d // 2:]
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k = turn(q).transpose(0, 1), turn(k).repeat_interleave(hq // hkv, 1).transpose(0, 1)
        p = q @ k.transpose(1, 2) * d ** -0.5
        if attention.softcap:
            p = attention.softcap * torch.tanh(p / attention.softcap)
        i = torch.arange(n, device="cuda")
        hidden = i[None] > i[:, None]
        if attention.window:
            hidden = hidden | (i[None] <= i[:, None] - attention.window)
        p = p.masked_fill(hidden, float("-inf")).softmax(-1)
        o = (p @ v.repeat_interleave(hq // hkv, 1).transpose(0, 1)).transpose(0, 1).reshape(n, hq * d)
        x = x + o @ out.float().t()
        x = x + torch.nn.functional.silu(norm(x) @ up.float().t()) @ down.float().t()
    return norm(x) @ model.embedding.float().t()


@pytest.mark.parametrize("drafts,softcap,window,block", [(4, 0.0, None, 16), (1, 20.0, None, 64), (7, 0.0, 40, 16), (0, 0.0, None, 32)])
def test_greedy_speculation_emits_the_models_tokens(example, drafts, softcap, window, block):
    check_device_error()
    model = example.TinyDecoder(vocab=512, softcap=softcap, window=window, seed=drafts)
    g = torch.Generator().manual_seed(drafts)
    prompts = [(torch.randint(0, 512, (int(torch.randint(1, 20, (1,), generator=g)),), generator=g).tolist() * 9)[:m] for m in (3, 90, 41, 17, 64)]
    server = example.Server(model, 5, num_blocks=5 * 40, block_size=block, max_blocks=40)
    first = server.prefill(prompts)
    out = server.decode(first, 12, drafts)
    assert check_device_error() == (0, 0)
    first, out = first.tolist(), out.tolist()
    for b, prompt in enumerate(prompts):
        own = [first[b]] + [t for step in out[b] for t in step if t >= 0]
        assert len(own) >= 13
        # everything but the last token is cached
        assert int(server.context_lens[b]) == len(prompt) + len(own) - 1
        logits = dense_logits(model, prompt + own[:-1])[len(prompt) - 1:]
        chosen = logits.gather(1, torch.tensor(own, device="cuda")[:, None])[:, 0]
        # bf16 activations: 2^-8 relative per layer step of logits of a few units
        assert float((logits.amax(1) - chosen).max()) <= 0.05 * float(logits.std()) + 0.02 * float(logits.abs().max())


def test_sampling_and_a_pool_that_runs_out(example):
    """At temperature one the emitted tokens are in the vocabulary and lengths add up; a pool
    too small for all requests refuses some, whose lengths then stand still."""
    check_device_error()
    model = example.TinyDecoder(vocab=300, seed=9)
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [[i + 1] * 30 for i in range(6)]
    server = example.Server(model, 6, num_blocks=6 * 2 + 5, block_size=16, max_blocks=8)
    first = server.prefill(prompts, 1.0, gen)
    before = server.context_lens.tolist()
    assert before == [30] * 6
    out = server.decode(first, 10, 3, 1.0, gen)
    assert check_device_error() == (0, 0)
    assert ((out >= -1) & (out < 300)).all() and (out[:, :, 0] >= 0).all()
    lens, held = server.context_lens.tolist(), server.blocks_held.tolist()
    assert sum(held) + int(server.free_count) == 17 and all(x <= 16 * h for x, h in zip(lens, held))
    assert min(lens) < max(lens)  # the pool ran out for the later requests
