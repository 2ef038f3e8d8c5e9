"""64-bit restatements of the ragged serving step's operators, and its test inputs."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # one rounding's relative error: half a unit of the last of 8 (11) bits


def cu_of(lens, device="cuda"):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def paged_batch(reqs, hq, hkv, d, block, dtype, seed=0, poison=None, spare=3, q_scale=1.0):
    """Queries, caches, a shuffled block table and lengths of requests (new, cached).
    Slots past each request's length hold `poison`, as do the spare blocks."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = [q + c for q, c in reqs]
    nb = [-(-x // block) for x in lens]
    total = sum(nb) + spare
    kc = torch.randn(total, block, hkv, d, generator=g, device="cuda").to(dtype)
    vc = torch.randn(total, block, hkv, d, generator=g, device="cuda").to(dtype)
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    bt = torch.full((len(reqs), max(nb + [1])), perm[-1], dtype=torch.int32)
    used = torch.zeros(total, block, dtype=torch.bool)
    at = 0
    for b, x in enumerate(lens):
        for j in range(nb[b]):
            bt[b, j] = perm[at]
            used[perm[at], :min(block, x - j * block)] = True
            at += 1
    if poison is not None:
        kc[~used.cuda()] = poison
        vc[~used.cuda()] = poison
    q = torch.randn(sum(x for x, _ in reqs), hq, d, generator=g, device="cuda").mul_(q_scale).to(dtype)
    return q, kc, vc, bt.cuda(), cu_of([x for x, _ in reqs]), torch.tensor(lens, dtype=torch.int32, device="cuda")


def attention64(q, kc, vc, bt, reqs, scale=None, causal=True, softcap=0.0, alibi=None, window=None, prefix=None, starts=None,
                lens=None):
    """(o, lse, a): the attention, its log-sum-exp and sum_j p_j |v_j|, in 64 bits. Rows
    that see no key: 0, -inf, 0. `lens` overrides the requests' cached lengths."""
    t, hq, d = q.shape
    block, hkv = kc.shape[1:3]
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    first = 0
    for b, (qn, c) in enumerate(reqs):
        n = qn + c if lens is None else lens[b]
        if qn and n:
            ids = bt[b, :-(-n // block)].long()
            k = kc[ids].flatten(0, 1)[:n].double()
            v = vc[ids].flatten(0, 1)[:n].double()
            pos = torch.arange(n - qn, n, device=q.device)[:, None]
            key = torch.arange(n, device=q.device)
            hi = torch.full_like(pos, n)
            lo = torch.zeros_like(pos)
            if causal:
                hi = pos + 1
                if prefix is not None:
                    hi = hi.clamp(min=int(prefix[b]))
            if window is not None:
                lo = pos - window + 1
            if starts is not None:
                lo = torch.maximum(lo, starts[first:first + qn, None].long())
            seen = (key >= lo) & (key < hi)
            for h in range(hq):
                x = q[first:first + qn, h].double() @ k[:, h // group].t() * scale
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                if alibi is not None:
                    x = x - alibi[h].double() * (pos - key).abs()
                x = x.masked_fill(~seen, -math.inf)
                m = x.amax(1, keepdim=True).clamp(min=-1e300)
                e = torch.exp(x - m)
                s = e.sum(1, keepdim=True)
                p = e / s.clamp(min=1e-300)
                vh = torch.where(seen.any(0)[:, None], v[:, h // group], torch.zeros_like(v[:, h // group]))
                o[first:first + qn, h] = p @ vh
                a[first:first + qn, h] = p @ vh.abs()
                lse[first:first + qn, h] = (m + torch.log(s))[:, 0]
        first += qn
    return o, lse, a


def attention_bound(o, a, dtype):
    """What the kernels may be off by: the output's rounding, P's rounding to the values'
    type (one rounding each of o and of sum p |v|), and scores and exponentials that are good
    to 1e-4 relative (fp32 sums of 128 products, the cap's 2^-23 times cap log2 e); the
    smallest f16 probabilities underflow by 2^-25 of the largest at most."""
    u = UNIT[dtype]
    return 1.05 * u * (o.abs() + a) + 1e-4 * a + 2e-5


def check_attention(out, o, a, dtype):
    err = (out.double() - o).abs()
    bad = ~(err <= attention_bound(o, a, dtype))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((err - attention_bound(o, a, dtype)).max()):.3e} over"


def rope64(x, w, eps, cos, sin, interleaved):
    """x (t, heads, d) normalised and rotated in 64 bits; cos, sin (t, rot / 2)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    half = cos.shape[1]
    y = y.clone()
    for f in range(half):
        i, j = (2 * f, 2 * f + 1) if interleaved else (f, f + half)
        a, b = y[..., i].clone(), y[..., j].clone()
        c, s = cos[:, f, None].double(), sin[:, f, None].double()
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


def plan64(query_lens, context_lens, table, held, free, free_count, block, max_tokens):
    """The step plan request by request and token by token, on the host."""
    n, width = len(query_lens), len(table[0]) if table else 0
    table = [list(r) for r in table]
    left, blocked = free_count, False
    out = dict(cu=[0], seq=[], pos=[], slot=[], seqs=[], granted=[], held=[])
    upto = 0
    for b in range(n):
        q, c = max(0, query_lens[b]), context_lens[b]
        after = -(-(c + q) // block)
        need = max(0, after - held[b]) if after <= width else 0
        upto += need
        ok = after <= width and (need == 0 or upto <= free_count)
        if ok:
            for j in range(need):
                left -= 1
                table[b][held[b] + j] = free[left]
        out["granted"].append(ok)
        out["held"].append(held[b] + (need if ok else 0))
        out["seq"].append(c + q if ok else c)
        out["cu"].append(out["cu"][-1] + q)
        for i in range(q):
            p = c + i
            out["pos"].append(p)
            out["slot"].append(table[b][p // block] * block + p % block if ok else -1)
            out["seqs"].append(b)
    for k in ("pos", "slot", "seqs"):
        out[k] = out[k][:max_tokens] + [-1] * (max_tokens - len(out[k]))
    return out, table, left


def verify64(drafts, target, draft, uniforms, expo, cu):
    """Speculative sampling request by request, on the host, with fp32's own products,
    differences and quotients (torch's, element by element)."""
    n, k = len(drafts), len(drafts[0]) if drafts else 0
    tokens, num = [], []
    for b in range(n):
        rows = cu[b + 1] - cu[b]
        if rows <= 0:
            tokens.append([-1] * (k + 1))
            num.append(0)
            continue
        m = min(rows - 1, k)
        i = 0
        while i < m:
            d = drafts[b][i]
            if not 0 <= d < target.shape[1]:
                break
            q = draft[b, i, d].float() if draft is not None else torch.tensor(1.0)
            if not bool(uniforms[b, i] * q < target[cu[b] + i, d].float()):
                break
            i += 1
        p = target[cu[b] + i].float()
        w = p
        if i < m:
            if draft is not None:
                w = (p - draft[b, i].float()).clamp(min=0)
            else:
                w = p.clone()
                if 0 <= drafts[b][i] < len(w):
                    w[drafts[b][i]] = 0
        s = w / expo[b]
        best = int(torch.nonzero(s == s.max())[0]) if float(s.max()) > 0 else int(torch.nonzero(p == p.max())[0])
        tokens.append(drafts[b][:i] + [best] + [-1] * (k - i))
        num.append(i + 1)
    return tokens, num
