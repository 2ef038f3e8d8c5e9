"""Speculative decoding of many requests over a paged cache, without the host reading a length.

    python examples/speculative_serving.py [--requests 16] [--steps 48] [--drafts 4] [--temperature 0]

Every step takes all requests, each with its own number of new tokens: whole prompts
first, then the last token and a few drafted ones. Per step

    plan_step                   blocks, positions and cache slots from the device's lengths
    RaggedPagedAttention        per layer: norm + rotation + cache write, ragged attention
    verify_drafts(_greedy)      the drafts that stand, and one token of the model's own

and the lengths, block tables and free list move on by what was accepted, on the device.
Drafts come from what followed the same token earlier in the same request (a table on the
device, no draft model). The model is a small decoder with random weights.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gqa-flash-attn-rtx3060_b200"))
from gqa_kernels import (RaggedPagedAttention, StepPlan, check_device_error, plan_step, rope_table, verify_drafts,  # noqa: E402
                         verify_drafts_greedy)


class TinyDecoder:
    """Embedding, layers of (attention, MLP) with RMS norms, and a tied output head; random weights."""

    def __init__(self, vocab=4096, layers=2, num_heads=8, num_kv_heads=2, head_dim=64, max_positions=4096, softcap=0.0,
                 window=None, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vocab, self.width, self.dtype = vocab, num_heads * head_dim, dtype

        def w(*shape, gain=1.0):
            return (torch.randn(*shape, generator=g, device="cuda") * gain * shape[-1] ** -0.5).to(dtype)
        self.embedding = w(vocab, self.width, gain=self.width ** 0.5)
        table = rope_table(max_positions, head_dim)
        ones = torch.ones(head_dim, dtype=dtype, device="cuda")
        self.layers = []
        for _ in range(layers):
            attention = RaggedPagedAttention(num_heads, num_kv_heads, head_dim, table, q_weight=ones, k_weight=ones,
                                             softcap=softcap, window=window)
            self.layers.append((attention, w((num_heads + 2 * num_kv_heads) * head_dim, self.width), w(self.width, self.width),
                                w(4 * self.width, self.width), w(self.width, 4 * self.width)))

    def allocate(self, num_blocks, block_size):
        return [layer[0].allocate_kv_cache(num_blocks, block_size, self.dtype, "cuda") for layer in self.layers]

    @staticmethod
    def norm(x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, ids, caches, plan, block_tables, max_query_len, max_seq_len):
        """Logits (tokens, vocab) of the step's packed tokens."""
        x = self.embedding[ids]
        for (attention, qkv, out, up, down), cache in zip(self.layers, caches):
            y = attention.forward(self.norm(x) @ qkv.t(), cache, plan, block_tables, max_query_len, max_seq_len)
            x = x + y @ out.t()
            x = x + torch.nn.functional.silu(self.norm(x) @ up.t()) @ down.t()
        return (self.norm(x) @ self.embedding.t()).float()


class Server:
    """Requests in slots 0 .. n - 1 of a paged cache; all state on the device."""

    def __init__(self, model, num_requests, num_blocks, block_size=16, max_blocks=256):
        n, dev = num_requests, "cuda"
        self.model, self.n, self.block_size = model, n, block_size
        self.caches = model.allocate(num_blocks, block_size)
        self.block_tables = torch.zeros(n, max_blocks, dtype=torch.int32, device=dev)
        self.context_lens = torch.zeros(n, dtype=torch.int32, device=dev)
        self.blocks_held = torch.zeros(n, dtype=torch.int32, device=dev)
        self.free_blocks = torch.arange(num_blocks, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([num_blocks], dtype=torch.int32, device=dev)
        # what followed a token; one column more for what is not to be remembered
        self.successor = torch.zeros(n, model.vocab + 1, dtype=torch.int32, device=dev)
        self.max_len = max_blocks * block_size
        self.counts = None  # of the last decode()

    def step(self, ids, query_lens, max_query_len, drafts, temperature, generator):
        """One step: ids the packed new tokens, query_lens (n,) how many each request has, drafts
        (n, k) the drafted ones among them. Returns (tokens (n, k + 1), num_tokens (n,)): -1 and 0
        for a request that the pool refused."""
        plan = plan_step(query_lens, self.context_lens, self.block_tables, self.blocks_held, self.free_blocks, self.free_count,
                         self.block_size, ids.shape[0])
        logits = self.model.forward(ids, self.caches, plan, self.block_tables, max_query_len, self.max_len)
        # the rows that score the drafts and the token after them: each request's last k + 1
        k = drafts.shape[1]
        last = plan.cu_query_lens[1:, None] - (k + 1) + torch.arange(k + 1, device=ids.device)
        scores = logits[last.long().flatten()]
        cu = torch.arange(0, (self.n + 1) * (k + 1), k + 1, dtype=torch.int32, device=ids.device)
        if temperature == 0:
            tokens, num = verify_drafts_greedy(drafts, scores, cu)
        else:
            probs = torch.softmax(scores / temperature, dim=-1)
            uniforms = torch.rand(self.n, k, generator=generator, device=ids.device)
            exponentials = torch.empty(self.n, probs.shape[1], device=ids.device).exponential_(generator=generator)
            tokens, num = verify_drafts(drafts, probs, None, uniforms, exponentials, cu)
        # The tokens of a request that the pool refused have no slots: their keys were not cached,
        # and what was computed from their rows means nothing.
        tokens = torch.where(plan.granted[:, None], tokens, -1)
        num = torch.where(plan.granted, num, 0)
        # What is cached and stands: everything but the refused drafts.
        stands = query_lens - (k + 1) + num
        self.context_lens = torch.where(plan.granted, self.context_lens + stands, self.context_lens)
        self.blocks_held, self.free_count = plan.blocks_held, plan.free_count
        return tokens, num

    def prefill(self, prompts, temperature=0, generator=None):
        """All prompts in one ragged step; returns each request's first own token."""
        lens = [len(p) for p in prompts]
        blocks = [-(-x // self.block_size) for x in lens]
        if sum(blocks) > self.free_blocks.numel() or max(blocks) > self.block_tables.shape[1]:
            raise ValueError("the pool or a row of the block tables is too small for the prompts")
        ids = torch.tensor([t for p in prompts for t in p], device="cuda")
        for b, p in enumerate(prompts):
            if len(p) > 1:
                t = torch.tensor(p, device="cuda")
                self.successor[b, t[:-1]] = t[1:].int()
        none = torch.zeros(self.n, 0, dtype=torch.int32, device="cuda")
        tokens, _ = self.step(ids, torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), none, temperature, generator)
        return tokens[:, 0]

    def decode(self, last, steps, num_drafts, temperature=0, generator=None):
        """`steps` steps from the requests' last tokens; returns the emitted tokens (n, steps, k + 1),
        -1 where a draft was refused, without waiting for the device. `counts` (n, steps) holds how
        many of each step's are new: 0 for a request that the pool refused, which stays where
        it is and whose first entry is the token that it goes on from, again."""
        emitted, counts = [], []
        rows = torch.arange(self.n, device="cuda")
        lens = torch.full((self.n,), num_drafts + 1, dtype=torch.int32, device="cuda")
        for _ in range(steps):
            chain = [last]
            for _ in range(num_drafts):
                chain.append(self.successor[rows, chain[-1].long()])
            ids = torch.stack(chain, 1)  # (n, k + 1): the last token and its drafts
            tokens, num = self.step(ids.flatten().long(), lens, num_drafts + 1, ids[:, 1:].int().contiguous(), temperature, generator)
            # remember what followed what: the accepted tokens, each after the one before it
            before = torch.cat([last[:, None], tokens[:, :-1]], 1)
            self.successor[rows[:, None], torch.where(tokens >= 0, before, self.model.vocab).long()] = tokens
            tokens[:, 0] = torch.where(num > 0, tokens[:, 0], last)
            last = tokens.gather(1, (num - 1).clamp(min=0)[:, None].long())[:, 0]
            emitted.append(tokens)
            counts.append(num)
        self.counts = torch.stack(counts, 1)
        return torch.stack(emitted, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--steps", type=int, default=48)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    model = TinyDecoder()
    g = torch.Generator(device="cuda").manual_seed(1)
    cpu = torch.Generator().manual_seed(2)
    prompts = []
    for _ in range(a.requests):  # prompts that repeat themselves, of mixed lengths
        phrase = torch.randint(0, model.vocab, (int(torch.randint(3, 40, (1,), generator=cpu)),), generator=cpu).tolist()
        prompts.append((phrase * 8)[:int(torch.randint(20, 200, (1,), generator=cpu))])
    server = Server(model, a.requests, num_blocks=a.requests * 64)
    last = server.prefill(prompts, a.temperature, g)
    server.decode(last, 2, a.drafts, a.temperature, g)  # warm-up
    server = Server(model, a.requests, num_blocks=a.requests * 64)
    last = server.prefill(prompts, a.temperature, g)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    server.decode(last, a.steps, a.drafts, a.temperature, g)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - t0
    kept = int(server.counts.sum())
    print(f"{a.requests} requests, {a.steps} steps of 1 + {a.drafts} tokens: {kept} tokens, {kept / (a.requests * a.steps):.2f} per "
          f"request and step, {kept / seconds:.0f} tokens/s; device error word {check_device_error()}")


if __name__ == "__main__":
    main()
