"""What one step of ragged paged serving costs: the cases that its operators are timed on.

A serving step takes a batch of requests, each with its own number of new tokens (one
for a plain decode, a few drafted ones for speculative decoding, thousands for a prompt
or a chunk of one) and its own cached length:

  plan      block tables, positions and cache slots of the step's tokens, from the
            requests' lengths and the pool's free blocks
  rope      norms of each query and key head, the position rotation (one or several
            position axes), and the write of K and V into the paged cache
  attn      attention of the step's tokens over the paged cache: causal per request,
            with a tanh cap on the scores, a bias by distance, a window, a prefix that
            every token sees, or documents that do not see one another
  verify    drafted tokens accepted or replaced by the target's probabilities (from
            given random numbers), or by the target's best token

`run` computes them in their plain form, or, where `own` is set, by the framework's
kernels. `exact` computes them in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # The smallest step of a server: eight requests decode one token each.
        dict(name="plan_decode_8", op="plan", n=8, tokens=8, ctx=4096, block=64, max_blocks=256, lens=1),
        # A full scheduler tick: prompts and decodes of many requests, small blocks.
        dict(name="plan_mixed_1024", op="plan", n=1024, tokens=65536, ctx=8192, block=16, max_blocks=1024, lens=2),
        # One decode step of a small batch: latency of the rotation and the cache write.
        dict(name="rope_decode_16", op="rope", tokens=16, hq=32, hkv=8, d=128, rot=128, axes=1, norm=True,
             interleaved=False, pos=16384, block=64, dtype="bf16"),
        # A long prompt of text and pictures: three position axes, an odd token count.
        dict(name="rope_prompt_3axis", op="rope", tokens=16381, hq=32, hkv=8, d=128, rot=128, axes=3, norm=True,
             interleaved=False, pos=16384, block=64, dtype="bf16"),
        # Ragged decode of a busy server, one token per request, lengths up to 16K.
        dict(name="attn_decode_48", op="attn", n_short=48, q_short=1, ctx_short=16384, n_long=0, q_long=0, ctx_long=0,
             hq=32, hkv=8, d=128, block=64, dtype="bf16", cap=0.0, alibi=False, window=0, prefix=False, docs=0, lens=3),
        # A speculative step: up to eight drafted tokens per request, capped scores.
        dict(name="attn_drafts_cap", op="attn", n_short=16, q_short=9, ctx_short=4096, n_long=0, q_long=0, ctx_long=0,
             hq=32, hkv=8, d=128, block=64, dtype="bf16", cap=30.0, alibi=False, window=0, prefix=False, docs=0, lens=4),
        # Chunked prefill beside decodes, a sliding window and a distance bias, small blocks.
        dict(name="attn_mixed_window", op="attn", n_short=30, q_short=1, ctx_short=8192, n_long=2, q_long=2048,
             ctx_long=4096, hq=32, hkv=4, d=128, block=16, dtype="f16", cap=0.0, alibi=True, window=2048, prefix=False,
             docs=0, lens=5),
        # A prompt packed of documents that do not see one another, 64-wide heads.
        dict(name="attn_documents", op="attn", n_short=0, q_short=0, ctx_short=0, n_long=1, q_long=16384, ctx_long=0,
             hq=32, hkv=8, d=64, block=64, dtype="bf16", cap=0.0, alibi=False, window=0, prefix=False, docs=1500, lens=6),
        # Prompts with a prefix that sees itself whole, chunks against long contexts, capped scores.
        dict(name="attn_chunks_prefix", op="attn", n_short=0, q_short=0, ctx_short=0, n_long=2, q_long=4096,
             ctx_long=12288, hq=32, hkv=8, d=128, block=64, dtype="bf16", cap=50.0, alibi=False, window=0, prefix=True,
             docs=0, lens=7),
        # Verification for a few users.
        dict(name="verify_4", op="verify", n=4, k=4, vocab=32000, greedy=False, dtype="f32", lens=8),
        # Verification for many users over a large odd-sized vocabulary.
        dict(name="verify_64", op="verify", n=64, k=7, vocab=131071, greedy=False, dtype="f32", lens=9),
        # The same at temperature zero: the best token of every row of logits.
        dict(name="verify_greedy_64", op="verify", n=64, k=7, vocab=131072, greedy=True, dtype="bf16", lens=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    lens = rng.randrange(1 << 30)
    op = rng.choice(["plan", "rope", "attn", "attn", "attn", "verify"])
    if op == "plan":
        n = _log(rng, 1, 1024)
        return dict(op=op, n=n, tokens=min(65536, n * _log(rng, 1, 512)), ctx=_log(rng, 1, 8192),
                    block=rng.choice([16, 32, 64, 128]), max_blocks=1024, lens=lens)
    if op == "rope":
        hkv = rng.choice([1, 2, 4, 8])
        d = rng.choice([64, 128])
        return dict(op=op, tokens=_log(rng, 1, 16384), hq=hkv * rng.choice([1, 2, 4, 5, 7, 8]) if hkv < 8 else 32, hkv=hkv,
                    d=d, rot=rng.choice([d, d, d // 2]), axes=rng.choice([1, 1, 2, 3]), norm=rng.random() < 0.7,
                    interleaved=rng.random() < 0.3, pos=16384, block=rng.choice([16, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]))
    if op == "verify":
        return dict(op=op, n=_log(rng, 1, 64), k=rng.randint(0, 7), vocab=_log(rng, 1000, 131072),
                    greedy=rng.random() < 0.4, dtype=rng.choice(["f32", "bf16"]), lens=lens)
    hkv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, n_short=0, q_short=0, ctx_short=0, n_long=0, q_long=0, ctx_long=0,
             hq=hkv * rng.choice([1, 2, 4, 5, 7, 8]) if hkv < 8 else 32, hkv=hkv, d=rng.choice([64, 128, 128]),
             block=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16"]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
             alibi=rng.random() < 0.3, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), prefix=False, docs=0, lens=lens)
    if rng.random() < 0.7:
        c["n_short"], c["q_short"], c["ctx_short"] = _log(rng, 1, 48), rng.choice([1, 1, rng.randint(2, 9)]), _log(rng, 16, 16384)
    if rng.random() < 0.5 or not c["n_short"]:
        c["n_long"], c["q_long"], c["ctx_long"] = rng.randint(1, 2), _log(rng, 17, 4096), _log(rng, 1, 12288)
    extra = rng.random()
    if extra < 0.25:
        c["prefix"] = True
    elif extra < 0.5:
        c["docs"] = _log(rng, 8, 2048)
    return c


# --------------------------------------------------------------------------- lengths and masks
def _requests(case):
    """The new tokens and the cached tokens of each request, from the case alone."""
    r = random.Random(case["lens"])
    if case["op"] == "plan":
        left, q = case["tokens"], []
        for i in range(case["n"]):
            rest = case["n"] - 1 - i
            mean = left / (rest + 1)
            take = left if not rest else max(0, min(left, int(round(r.uniform(0.2, 1.8) * mean))))
            q.append(take)
            left -= take
        return [(x, r.randint(0, case["ctx"])) for x in q]
    if case["op"] == "verify":
        return [(r.randint(max(1, case["k"] // 2), case["k"] + 1), 0) for _ in range(case["n"])]
    out = [(r.randint(1, case["q_short"]), r.randint(case["ctx_short"] // 4, case["ctx_short"])) for _ in range(case["n_short"])]
    out += [(r.randint(max(17, case["q_long"] * 3 // 4), max(17, case["q_long"])), r.randint(0, case["ctx_long"]))
            for _ in range(case["n_long"])]
    r.shuffle(out)
    return out


def _masks(case, requests):
    """The prefix length of each request and the first visible key of each token (or None)."""
    r = random.Random(case["lens"] + 1)
    prefix = [r.randint(0, c + q) for q, c in requests] if case["prefix"] else None
    starts = None
    if case["docs"]:
        starts = []
        for q, c in requests:
            at, nxt, seen = 0, 0, []
            for p in range(c + q):
                if p == nxt:
                    at, nxt = p, p + max(1, int(r.expovariate(1.0 / case["docs"])))
                seen.append(at)
            starts += seen[c:]
    return prefix, starts


def _spans(case):
    """(first key, one past the last key) that each token of the step sees, per request."""
    requests = _requests(case)
    prefix, starts = _masks(case, requests)
    spans, t = [], 0
    for b, (q, c) in enumerate(requests):
        rows = []
        for i in range(q):
            p = c + i
            hi = max(p + 1, min(prefix[b], c + q)) if prefix else p + 1
            lo = max(0, p - case["window"] + 1) if case["window"] else 0
            if starts:
                lo = max(lo, starts[t])
            rows.append((lo, max(lo, hi)))
            t += 1
        spans.append(rows)
    return requests, spans


def work(case):
    op = case["op"]
    if op == "plan":
        reqs = _requests(case)
        bs = case["block"]
        new = sum(max(0, -(-(q + c) // bs) - -(-c // bs)) for q, c in reqs)
        used = sum(-(-(q + c) // bs) - c // bs for q, c in reqs if q)
        return {"bytes": 4 * (3 * case["n"] + 2 * new + used - new) + 4 * (3 * case["n"] + 2) + case["n"] + 16 * (case["tokens"] + case["tokens"] // 8),
                "flops": 0}
    if op == "rope":
        t, d, es = case["tokens"], case["d"], 2
        heads = case["hq"] + 2 * case["hkv"]
        # the rotation table: one row per token and axis, of which each axis reads its part
        return {"bytes": 2 * es * t * heads * d + 4 * t * case["rot"] + t * (4 * case["axes"] + 8), "flops": 8 * t * (case["hq"] + case["hkv"]) * d}
    if op == "verify":
        reqs = _requests(case)
        es = 4 if case["dtype"] == "f32" else 2
        rows = sum(q for q, _ in reqs)
        if case["greedy"]:
            return {"bytes": es * rows * case["vocab"] + 4 * rows, "flops": rows * case["vocab"]}
        return {"bytes": case["n"] * case["vocab"] * (2 * es + 4) + rows * (2 * es + 8), "flops": 3 * case["n"] * case["vocab"]}
    reqs, spans = _spans(case)
    pairs = sum(hi - lo for rows in spans for lo, hi in rows)
    tokens = sum(q for q, _ in reqs)
    keys = 0
    for rows in spans:
        end = -1  # the union of the rows' spans
        for lo, hi in sorted(rows):
            keys += max(0, hi - max(lo, end))
            end = max(end, hi)
    return {"bytes": 4 * tokens * case["hq"] * case["d"] + 4 * keys * case["hkv"] * case["d"], "flops": 4 * pairs * case["hq"] * case["d"]}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


_imported = None


def _kernels():
    global _imported
    if _imported is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gqa-flash-attn-rtx3060_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import gqa_kernels
        _imported = gqa_kernels
    return _imported


def prepare(case, seed):
    g = _gen(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn, "verify": _prepare_verify}[case["op"]](case, g)


def _prepare_plan(case, g):
    reqs = _requests(case)
    bs, n = case["block"], case["n"]
    held = [-(-c // bs) for _, c in reqs]
    total = sum(-(-(q + c) // bs) for q, c in reqs)
    pool = torch.randperm(total + total // 8 + 1, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n, case["max_blocks"]), -1, dtype=torch.int32, device="cuda")
    have = torch.arange(case["max_blocks"], device="cuda") < _i32(held)[:, None]
    table[have] = pool[:sum(held)]
    free = pool[sum(held):].contiguous()
    return dict(op="plan", block=bs, out=None, tokens=case["tokens"] + case["tokens"] // 8,  # room, as a captured step has
                query_lens=_i32([q for q, _ in reqs]), context_lens=_i32([c for _, c in reqs]), block_tables=table,
                blocks_held=_i32(held), free_blocks=free,
                # the step may need a little more than the pool holds: the last requests then wait
                free_count=_i32([min(free.numel(), (total - sum(held)) * 31 // 32 + 1)]))


def _table(positions, rot, base=10000.0):
    """cos | sin of positions x base^(-2 i / rot), float32."""
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _sections(axes, half):
    """How many of the `half` rotation frequencies each position axis has (time first)."""
    side = half // 4 + half // 8 if axes == 3 else half // 2
    return [half] if axes == 1 else [half - (axes - 1) * side] + [side] * (axes - 1)


def _prepare_rope(case, g):
    t, hq, hkv, d, dt = case["tokens"], case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    qkv = torch.randn(t, hq + 2 * hkv, d, generator=g, device="cuda").mul_(1.5).to(dt)  # the projection's output
    blocks = -(-t // case["block"]) + 2
    slots = torch.randperm(blocks * case["block"], generator=g, device="cuda")[:t]
    slots[t // 3:t // 3 + t // 50] = -1  # padding tokens
    pos = torch.randint(0, case["pos"], (case["axes"], t), generator=g, device="cuda", dtype=torch.int32)
    cache = torch.randn(2, blocks, case["block"], hkv, d, generator=g, device="cuda").to(dt)
    w = (1 + 0.2 * torch.randn(2, d, generator=g, device="cuda")).to(dt)
    return dict(op="rope", q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], positions=pos if case["axes"] > 1 else pos[0],
                slots=slots, key_cache=cache[0], value_cache=cache[1], cos_sin=_table(case["pos"], case["rot"]),
                q_weight=w[0] if case["norm"] else None, k_weight=w[1] if case["norm"] else None,
                sections=_sections(case["axes"], case["rot"] // 2), interleaved=case["interleaved"])


def _prepare_attn(case, g):
    reqs = _requests(case)
    prefix, starts = _masks(case, reqs)
    dt, bs = DTYPES[case["dtype"]], case["block"]
    total = sum(q for q, _ in reqs)
    lens = [q + c for q, c in reqs]
    nb = [-(-x // bs) for x in lens]
    pool = torch.randperm(sum(nb) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(reqs), max(nb), dtype=torch.int32, device="cuda")
    table[torch.arange(max(nb), device="cuda") < _i32(nb)[:, None]] = pool[:sum(nb)]
    q = torch.randn(total, case["hq"], case["d"], generator=g, device="cuda")
    if case["cap"]:
        q *= case["cap"] / 10  # scores that the cap bends
    shape = (sum(nb) + 3, bs, case["hkv"], case["d"])
    kc = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
    vc = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
    cu = [0]
    for x, _ in reqs:
        cu.append(cu[-1] + x)
    slopes = torch.exp2(-8.0 / case["hq"] * torch.arange(1, case["hq"] + 1, dtype=torch.float32, device="cuda"))
    return dict(op="attn", q=q.to(dt), key_cache=kc, value_cache=vc, block_tables=table, cu=_i32(cu), seq_lens=_i32(lens),
                reqs=reqs, max_q=max(x for x, _ in reqs), max_len=max(lens), cap=case["cap"],
                alibi=slopes if case["alibi"] else None, window=case["window"] or None,
                prefix=_i32(prefix) if prefix else None, starts=_i32(starts) if starts else None)


def _prepare_verify(case, g):
    reqs = _requests(case)
    n, k, v, dt = case["n"], case["k"], case["vocab"], DTYPES[case["dtype"]]
    rows = sum(q for q, _ in reqs)
    cu = [0]
    for x, _ in reqs:
        cu.append(cu[-1] + x)
    logits = torch.randn(rows, v, generator=g, device="cuda").mul_(3.0)
    s = dict(op="verify", greedy=case["greedy"], cu=_i32(cu), k=k)
    # the draft model sees what the target sees, less well: row i of request b, nudged
    at = (_i32(cu[:-1]).long()[:, None] + torch.arange(max(k, 1), device="cuda")).clamp(max=rows - 1)
    near = logits[at] + 0.7 * torch.randn(n, max(k, 1), v, generator=g, device="cuda")
    if case["greedy"]:
        best = logits[at].argmax(-1)
        other = near.argmax(-1)
        pick = torch.rand(n, max(k, 1), generator=g, device="cuda") < 0.7
        s["target"], s["draft_tokens"] = logits.to(dt), torch.where(pick, best, other).to(torch.int32)[:, :k].contiguous()
        return s
    dp = near.softmax(-1)
    tokens = torch.multinomial(dp.view(-1, v), 1, generator=g).view(n, -1)
    s["target"], s["draft_probs"] = logits.softmax(-1).to(dt), dp.to(dt)[:, :k].contiguous()
    s["draft_tokens"] = tokens.to(torch.int32)[:, :k].contiguous()
    s["uniforms"] = torch.rand(n, max(k, 1), generator=g, device="cuda")[:, :k].contiguous()
    s["exponentials"] = torch.empty(n, v, device="cuda").exponential_(generator=g)
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    forms = {"plan": (_plan, _own_plan), "rope": (_rope, _own_rope), "attn": (_attn, _own_attn), "verify": (_verify, _own_verify)}
    return forms[state["op"]][1 if own else 0](state)


def _own_plan(s):
    p = _kernels().plan_step(s["query_lens"], s["context_lens"], s["block_tables"], s["blocks_held"], s["free_blocks"],
                             s["free_count"], s["block"], s["tokens"], out=s["out"])
    s["out"] = p  # a server plans every step into the same buffers
    return [p.cu_query_lens, p.seq_lens, p.positions, p.slot_mapping, p.token_seqs, p.granted, p.blocks_held, p.free_count,
            s["block_tables"]]


def _own_rope(s):
    q = _kernels().qk_norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["key_cache"], s["value_cache"],
                                       s["slots"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                                       sections=s["sections"], interleaved=s["interleaved"])
    return [q, s["key_cache"], s["value_cache"]]


def _own_attn(s):
    return _kernels().paged_ragged_attention(s["q"], s["key_cache"], s["value_cache"], s["block_tables"], s["cu"], s["seq_lens"],
                                             max_query_len=s["max_q"], max_seq_len=s["max_len"], softcap=s["cap"],
                                             alibi_slopes=s["alibi"], window=s["window"], prefix_lens=s["prefix"],
                                             key_starts=s["starts"])


def _own_verify(s):
    k = _kernels()
    if s["greedy"]:
        return list(k.verify_drafts_greedy(s["draft_tokens"], s["target"], s["cu"]))
    return list(k.verify_drafts(s["draft_tokens"], s["target"], s["draft_probs"], s["uniforms"], s["exponentials"], s["cu"]))


# --------------------------------------------------------------------------- the plain forms
def _plan(s):
    bs, table = s["block"], s["block_tables"]
    q, ctx, held = s["query_lens"], s["context_lens"], s["blocks_held"]
    after = (ctx + q + bs - 1) // bs
    fits = after <= table.shape[1]
    need = torch.where(fits, (after - held).clamp(min=0), torch.zeros_like(held))
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= s["free_count"]))
    take = torch.where(granted, need, torch.zeros_like(need))
    cu = torch.zeros(q.numel() + 1, dtype=torch.int32, device=q.device)
    cu[1:] = q.cumsum(0)
    col = torch.arange(table.shape[1], device=q.device)
    new = (col >= held[:, None]) & (col < (held + take)[:, None])
    at = (s["free_count"] - 1 - (upto - need)[:, None] - (col - held[:, None])).clamp(min=0, max=s["free_blocks"].numel() - 1)
    table = torch.where(new, s["free_blocks"][at], table)
    t = torch.arange(s["tokens"], device=q.device, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], t, right=True).clamp(max=q.numel() - 1)
    valid = t < cu[-1]
    pos = ctx[seq] + t - cu[seq]
    slot = table[seq, (pos // bs).clamp(max=table.shape[1] - 1)].long() * bs + pos % bs
    none = torch.full_like(t, -1)
    return [cu, ctx + torch.where(granted, q, torch.zeros_like(q)), torch.where(valid, pos, none),
            torch.where(valid & granted[seq], slot, none.long()), torch.where(valid, seq.int(), none), granted, held + take,
            s["free_count"] - take.sum().int(), table]


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


def _angles(s, table):
    """cos and sin of each token, (tokens, 1, rot / 2)."""
    half = table.shape[1] // 2
    pos = s["positions"].long()
    if pos.dim() == 1:
        both = table[pos]
        return both[:, None, :half], both[:, None, half:]
    axis = torch.repeat_interleave(torch.arange(pos.shape[0], device="cuda"), torch.tensor(s["sections"], device="cuda"))
    at = pos[axis].t()  # tokens x half
    f = torch.arange(half, device="cuda")
    return table[at, f][:, None], table[at, half + f][:, None]


def _turned(x, cos, sin, interleaved):
    half = cos.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, d = a * cos - b * sin, b * cos + a * sin
    both = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([both, x[..., 2 * half:]], -1)


def _rope(s):
    cos, sin = _angles(s, s["cos_sin"])
    dt = s["q"].dtype
    q = _turned(_normed(s["q"], s["q_weight"]), cos, sin, s["interleaved"]).to(dt)
    k = _turned(_normed(s["k"], s["k_weight"]), cos, sin, s["interleaved"]).to(dt)
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["key_cache"].view(-1, *k.shape[1:])[at] = k[keep]
    s["value_cache"].view(-1, *k.shape[1:])[at] = s["v"][keep]
    return [q, s["key_cache"], s["value_cache"]]


def _batches(reqs, hq):
    """Requests of few tokens go as one padded batch, longer ones one by one, in blocks of
    rows whose scores fit a gigabyte: (requests, first row, one past the last row)."""
    short = [b for b, (q, _) in enumerate(reqs) if q <= 16]
    out = [(short, 0, max(reqs[b][0] for b in short))] if short else []
    for b in range(len(reqs)):
        q, c = reqs[b]
        if q > 16:
            rows = max(1, (1 << 28) // (hq * (q + c)))
            out += [([b], r, min(q, r + rows)) for r in range(0, q, rows)]
    return out


def _attn(s):
    q, kc, vc = s["q"], s["key_cache"], s["value_cache"]
    t, hq, d = q.shape
    bs, hkv = kc.shape[1:3]
    out = torch.zeros(t, hq, d, dtype=q.dtype, device=q.device)
    for bb, r0, r1 in _batches(s["reqs"], hq):
        length = max(sum(s["reqs"][b]) for b in bb)
        nb = -(-length // bs)
        b = torch.tensor(bb, device=q.device)
        blocks = s["block_tables"][b, :nb].long()
        k = kc[blocks].flatten(1, 2)[:, :length].float()  # requests, keys, kv heads, d
        v = vc[blocks].flatten(1, 2)[:, :length].float()
        lens, qlens = s["seq_lens"][b].long()[:, None], (s["cu"][b + 1] - s["cu"][b]).long()[:, None]
        i = torch.arange(r0, r1, device=q.device)
        rows = s["cu"][b].long()[:, None] + i
        real = i < qlens
        rows = torch.where(real, rows, torch.zeros_like(rows))
        pos = lens - qlens + i  # requests, rows
        hi, lo = pos + 1, torch.zeros_like(pos)
        if s["prefix"] is not None:
            hi = torch.maximum(hi, torch.minimum(s["prefix"][b].long()[:, None], lens))
        if s["window"] is not None:
            lo = torch.maximum(lo, pos - s["window"] + 1)
        if s["starts"] is not None:
            lo = torch.maximum(lo, s["starts"][rows].long())
        key = torch.arange(length, device=q.device)
        seen = (key >= lo[..., None]) & (key < hi[..., None]) & (key < lens[..., None])
        qf = q[rows].float().view(len(bb), r1 - r0, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
        x = torch.matmul(qf, k.permute(0, 2, 3, 1)[:, :, None]) * d ** -0.5  # requests, kv heads, group, rows, keys
        if s["cap"]:
            x = s["cap"] * torch.tanh(x / s["cap"])
        if s["alibi"] is not None:
            x = x - s["alibi"].view(1, hkv, hq // hkv, 1, 1) * (key - pos[..., None]).abs()[:, None, None].float()
        x = x.masked_fill(~seen[:, None, None], float("-inf"))
        p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
        p = p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
        o = torch.matmul(p, v.transpose(1, 2)[:, :, None]).permute(0, 3, 1, 2, 4).reshape(len(bb), r1 - r0, hq, d)
        out[rows[real]] = o[real].to(q.dtype)
    return out


def _first_best(x):
    """The lowest index of the largest value of each row."""
    best = x.amax(-1, keepdim=True)
    at = torch.arange(x.shape[-1], device=x.device, dtype=torch.int32)
    return torch.where(x == best, at, torch.full_like(at, x.shape[-1] - 1)).amin(-1)


def _verify(s):
    d, cu, k, target = s["draft_tokens"], s["cu"].long(), s["k"], s["target"]
    n = cu.numel() - 1
    step = torch.arange(k + 1, device=d.device)
    kept_rows = (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + step).clamp(max=target.shape[0] - 1)  # n, k + 1
    if s["greedy"]:
        best = _first_best(target.float())[rows]
        ok = best[:, :k] == d
    else:
        p = target[rows[:, :k], d.long()].float()
        q = torch.gather(s["draft_probs"], 2, d.long()[..., None])[..., 0].float()
        ok = s["uniforms"] * q < p
    ok = ok & (step[:k] < kept_rows - 1)
    accepted = ok.int().cumprod(1).sum(1) if k else torch.zeros(n, dtype=torch.int64, device=d.device)
    if s["greedy"]:
        last = best.gather(1, accepted[:, None])[:, 0]
    else:
        pr = target[rows.gather(1, accepted[:, None])[:, 0]].float()
        rest = pr
        if k:
            dr = s["draft_probs"][torch.arange(n, device=d.device), accepted.clamp(max=k - 1)].float()
            rest = torch.where((accepted < kept_rows[:, 0] - 1)[:, None], (pr - dr).clamp(min=0), pr)
        score = rest / s["exponentials"]
        last = torch.where(score.amax(-1) > 0, _first_best(score), _first_best(pr))
    none = torch.full((n, k + 1), -1, dtype=torch.int32, device=d.device)
    padded = torch.cat([d, none[:, :1]], 1)
    tokens = torch.where(step < accepted[:, None], padded, torch.where(step == accepted[:, None], last.int()[:, None], none))
    return [tokens, (accepted + 1).int()]


# --------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] in ("plan", "verify"):
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_rope(s, case) if case["op"] == "rope" else _exact_attn(s, case)


def _exact_rope(s, case):
    """Each pair of numbers as a complex one, turned by a unit number of its angle's table entry."""
    half = case["rot"] // 2
    pos = s["positions"].long().view(case["axes"], -1)
    table = s["cos_sin"].double()
    turn, f = [], 0
    for a, size in enumerate(s["sections"]):
        turn.append(torch.complex(table[pos[a], f:f + size], table[pos[a], half + f:half + f + size]))
        f += size
    turn = torch.cat(turn, 1)[:, None]

    def heads(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * w.double()
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    k = heads(s["k"], s["k_weight"])
    kc, vc = s["key_cache"].double(), s["value_cache"].double()
    flat_k, flat_v = kc.view(-1, *k.shape[1:]), vc.view(-1, *k.shape[1:])
    keep = torch.nonzero(s["slots"] >= 0)[:, 0]
    flat_k[s["slots"][keep]] = k[keep]
    flat_v[s["slots"][keep]] = s["v"][keep].double()
    return [heads(s["q"], s["q_weight"]), kc, vc]


def _exact_attn(s, case):
    """Request by request, head by head, from the spans of keys that each token sees."""
    reqs, spans = _spans(case)
    if sum((q + c) * q for q, c in reqs) * case["hq"] * case["d"] > 4e13:
        return None
    d, group, bs = case["d"], case["hq"] // case["hkv"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (q, c) in enumerate(reqs):
        blocks = s["block_tables"][b, :-(-(q + c) // bs)].long()
        lo_hi = torch.tensor(spans[b], device="cuda")
        key = torch.arange(q + c, device="cuda")
        for h in range(case["hkv"]):
            kh = s["key_cache"][blocks, :, h].reshape(-1, d)[:q + c].double()
            vh = s["value_cache"][blocks, :, h].reshape(-1, d)[:q + c].double()
            step = max(1, (1 << 27) // (group * (q + c)))
            for r in range(0, q, step):
                e = min(q, r + step)
                qh = s["q"][first + r:first + e, h * group:(h + 1) * group].double()
                x = torch.einsum("rgd,kd->rgk", qh, kh) / math.sqrt(d)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                if case["alibi"]:
                    slope = s["alibi"][h * group:(h + 1) * group].double()
                    x = x - slope[None, :, None] * (torch.arange(c + r, c + e, device="cuda")[:, None] - key).abs()[:, None]
                hide = (key < lo_hi[r:e, :1]) | (key >= lo_hi[r:e, 1:])
                x = x.masked_fill(hide[:, None], -1e300)
                w = torch.softmax(x, -1).masked_fill(hide[:, None], 0.0)
                out[first + r:first + e, h * group:(h + 1) * group] = torch.einsum("rgk,kd->rgd", w, vh)
        first += q
    return out
