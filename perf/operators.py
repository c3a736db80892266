"""What a program that generates or scores text with a trained model asks of the framework, as measured cases: the plan of a step over a
paged key / value cache, keys and values appended to that cache in 8 bits, attention over it, and log probabilities of tokens.

``run`` makes the framework's calls where ``own`` is true and computes the same in elementary torch operations where it is false; ``exact``
computes it again in 64 bits.  Shapes are those of the models this repository configures (32 query / 2 KV heads of 128, 16 / 8 heads of 64 or
128, vocabularies of 32000 and 151936) or generic.

The cache: pages of P tokens.  ``k`` is uint8 (pages, Hkv, P/2, D/64, 2, 64): token 2i+e, columns 64j..64j+63 of a head at [:, :, i, j, e];
``v`` is uint8 (pages, Hkv, P/16, D, 16): 16 tokens of a column side by side.  A code u stands for (u - 128) * scale with one fp32 scale for each
page, head and side (``scale``, (pages, Hkv, 2)): the smallest power of two 2^e, e in -60..60, for which no value of the page exceeds 127 steps.
Appending to a page that holds tokens may raise its scale; the codes that are there are then rounded to the new step (half to even).
``table`` (B, W) int32 lists the pages of each sequence, ``free`` / ``free_count`` are a stack of free pages.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
HEADS = [(32, 2, 128), (16, 8, 128), (32, 8, 128), (16, 8, 64), (16, 2, 128), (8, 2, 64), (12, 4, 128), (16, 16, 64)]


def listed():
    return [
        # one generated token for each of 64 running requests: pages and slots of the step
        dict(name="plan_decode", kind="plan", B=64, P=64, longest=8192, prompts=0, prompt=1, short=False),
        # a mixed step: 16 new prompts of up to 8192 tokens among 496 requests that generate or idle
        dict(name="plan_mixed", kind="plan", B=512, P=16, longest=4096, prompts=16, prompt=8192, short=False),
        # the keys and values of one token of each of 64 requests go into pages that are in use, and the pages are read back
        dict(name="append_decode", kind="append", B=64, P=64, longest=8192, most=1, Hkv=2, D=128),
        # prompts of odd lengths, about 32768 tokens together, and all of their pages read back
        dict(name="append_prompt", kind="append", B=8, P=64, longest=100, most=7777, Hkv=8, D=128),
        # one request, a short context: the smallest call, latency alone counts
        dict(name="attend_one", kind="attend", B=1, P=16, shortest=300, longest=300, most=1, Hq=16, Hkv=8, D=64, window=0),
        # one token of each of 64 requests with contexts of 1 to 8192 tokens
        dict(name="attend_decode", kind="attend", B=64, P=64, shortest=1, longest=8192, most=1, Hq=32, Hkv=2, D=128, window=0),
        # up to eight drafted tokens of each of 32 requests are verified at once
        dict(name="attend_draft", kind="attend", B=32, P=32, shortest=8, longest=12000, most=8, Hq=32, Hkv=8, D=128, window=0),
        # few requests with long contexts
        dict(name="attend_long", kind="attend", B=8, P=128, shortest=60000, longest=65536, most=1, Hq=32, Hkv=2, D=128, window=0),
        # the log probability of each sampled token with its 20 best alternatives, a step of 64 requests
        dict(name="logprobs_step", kind="logprobs", N=64, V=151936, k=20, fp32=False, train=False),
        # scoring of given text: fp32 logits of a vocabulary of odd size
        dict(name="logprobs_score", kind="logprobs", N=511, V=50257, k=5, fp32=True, train=False),
        # scoring of given text: log probability and entropy of each token, and the likeliest token
        dict(name="logprobs_eval", kind="logprobs", N=8192, V=32000, k=1, fp32=False, train=False),
        # training on log probabilities, entropies and the best alternatives (policy gradients, distillation): forward and backward
        dict(name="logprobs_train", kind="logprobs", N=4096, V=151936, k=8, fp32=False, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    P = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        B = _log(rng, 1, 512)
        return dict(kind=kind, B=B, P=P, longest=_log(rng, 16, 8192), prompts=rng.randint(0, min(B, 16)), prompt=_log(rng, 16, 8192),
                    short=rng.random() < 0.2)
    Hq, Hkv, D = rng.choice(HEADS)
    if kind == "append":
        most = rng.choice([1, 1, 5, _log(rng, 16, 7777)])
        return dict(kind=kind, B=_log(rng, 1, 64 if most < 16 else 8), P=P, longest=_log(rng, 1, 4096), most=most, Hkv=Hkv, D=D)
    if kind == "attend":
        most = rng.choice([1, 1, 1, 4, 8, rng.randint(1, 8)])
        longest = _log(rng, 16, 65536)
        B = _log(rng, 1, 64)
        while B > 1 and B * longest * Hkv * D > 8 * 65536 * 256:
            B //= 2
        if longest * Hkv * D > 8 * 65536 * 256 // max(B, 1):
            longest = 8 * 65536 * 256 // (Hkv * D)
        return dict(kind=kind, B=B, P=P, shortest=max(most, rng.choice([1, longest // 2, longest])), longest=max(most, longest), most=most, Hq=Hq,
                    Hkv=Hkv, D=D, window=rng.choice([0, 0, 0, 512, 1000]))
    V = rng.choice([32000, 151936, 50257, _log(rng, 1000, 160000)])
    N = min(_log(rng, 1, 8192), 4096 * 151936 // V)
    return dict(kind=kind, N=N, V=V, k=rng.choice([0, 1, 5, 8, 20]), fp32=rng.random() < 0.3 and N * V < 1 << 28, train=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------ inputs
def _order(g, n):
    return torch.rand(n, device=DEV, generator=g).argsort().to(torch.int32)


def _whole(g, lo, hi, n):
    """n whole numbers of lo..hi."""
    return torch.randint(lo, hi + 1, (n,), device=DEV, generator=g, dtype=torch.int32)


def _sizes(case):
    """The generator of a case's lengths: those are the same for every seed, in another order."""
    return torch.Generator(DEV).manual_seed(sum((i + 1) * x for i, x in enumerate(v for v in case.values() if type(v) is int)))


def _ceil(a, b):
    return (a + b - 1) // b


def _starts(n):
    return torch.nn.functional.pad(n.cumsum(0), (1, 0)).to(torch.int32)


def _tables(g, held, W):
    """(table, pages): the pages of sequences that hold ``held`` pages each, in a random order, -1 behind them, and how many there are."""
    pages = int(held.sum())
    have = torch.arange(W, device=DEV) < held[:, None]
    table = torch.full(have.shape, -1, dtype=torch.int32, device=DEV)
    table[have] = _order(g, pages)
    return table, pages


def _activations(g, *shape):
    """Keys or values: normal numbers whose columns differ in size, a few columns much larger."""
    size = torch.rand(shape[-1], device=DEV, generator=g) * 1.5 + 0.25
    size[torch.randint(0, shape[-1], (2,), device=DEV, generator=g)] = 8.0
    return (torch.randn(shape, device=DEV, generator=g) * size).to(BF)


def _step(amax):
    """The smallest power of two of which no value up to amax needs more than 127, 2^-60 at least."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 127 / 128, e - 6, e - 7).clamp(-60, 60)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -60)))


def _pack(k, v):
    """Codes (pages, P, Hkv, D) of both sides in the cache's order."""
    n, P, H, D = k.shape
    k = k.view(n, P // 2, 2, H, D // 64, 64).permute(0, 3, 1, 4, 2, 5)
    v = v.view(n, P // 16, 16, H, D).permute(0, 3, 1, 4, 2)
    return k.contiguous(), v.contiguous()


def _filled(g, pages, P, Hkv, D, kept=None):
    """A cache whose pages hold ``kept`` tokens each (all of them P where it is None): (k, v, scale)."""
    codes, scales = [], []
    for _ in "kv":
        x = _activations(g, pages, P, Hkv, D).float()
        if kept is not None:
            x *= (torch.arange(P, device=DEV) < kept[:, None])[:, :, None, None]
        s = _step(x.abs().amax((1, 3)))
        codes.append(((x / s[:, None, :, None]).round() + 128).to(torch.uint8))
        scales.append(s)
    return (*_pack(*codes), torch.stack(scales, -1).contiguous())


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    kind, s = case["kind"], dict(case)
    if kind == "logprobs":
        N, V, k = case["N"], case["V"], case["k"]
        x = torch.randn(N, V, device=DEV, generator=g).mul_(2.5)
        x += torch.randn(V, device=DEV, generator=g) * 1.5
        x[:, torch.randint(0, V, (max(1, V // 200),), device=DEV, generator=g)] = float("-inf")        # tokens that may not be produced
        tokens = torch.randint(0, V, (N,), device=DEV, generator=g)
        tokens[::7] = -100                                                                             # positions that do not count
        s.update(logits=x if case["fp32"] else x.to(BF), tokens=tokens)
        if case["train"]:
            s.update(dlogprob=torch.randn(N, device=DEV, generator=g), dentropy=torch.randn(N, device=DEV, generator=g) * 0.1,
                     dtop=torch.randn(N, k, device=DEV, generator=g) * 0.3)
            bad = torch.isneginf(x.gather(1, tokens.clamp(min=0)[:, None]))[:, 0]
            s["dlogprob"][bad] = 0
        return s
    B, P, fixed = case["B"], case["P"], _sizes(case)
    mix = _order(g, B).long()
    if kind == "plan":
        lengths = _whole(fixed, 0, case["longest"], B)
        new = (torch.rand(B, device=DEV, generator=fixed) < 0.9).to(torch.int32)
        lengths[:case["prompts"]] = 0
        new[:case["prompts"]] = _whole(fixed, 1, case["prompt"], case["prompts"])
        lengths, new = lengths[mix], new[mix]
        W = _ceil(case["longest"] + case["prompt"] + 1, P)
        held = _ceil(lengths, P)
        table, pages = _tables(g, held, W)
        need = int((_ceil(lengths + new, P) - held).sum())
        spare = need // 2 if case["short"] else need + 100
        free = _order(g, spare) + pages if spare else torch.zeros(1, dtype=torch.int32, device=DEV)
        s.update(lengths=lengths, new=new, table=table, free=free, free_count=torch.tensor([spare], dtype=torch.int32, device=DEV),
                 num_tokens=int(new.sum()))
        return s
    Hkv, D, most = case["Hkv"], case["D"], case["most"]
    if kind == "append":
        past = _whole(fixed, 0, case["longest"], B)
        past[0] = case["longest"] // P * P + P - 1                         # the last place of a page
        new = _whole(fixed, max(1, most // 10), most, B)
        if B > 2:
            new[2] = 0                                                     # a request that idles
        past, new = past[mix], new[mix]
        lengths = past + new
        table, pages = _tables(g, _ceil(lengths, P), _ceil(int(lengths.max()), P) + 1)
        n = int(new.sum())
        at = torch.arange(table.shape[1], device=DEV)
        touched = (at >= (past // P)[:, None]) & (at < _ceil(lengths, P)[:, None]) & (new > 0)[:, None]
        kept = torch.zeros(pages, dtype=torch.int32, device=DEV)
        kept[table[table >= 0].long()] = (past[:, None] - at * P).clamp(0, P)[table >= 0].to(torch.int32)
        k, v, scale = _filled(g, pages, P, Hkv, D, kept)
        s.update(k=k, v=v, scale=scale, table=table, lengths=lengths, query_start=_starts(new), ids=table[touched],
                 k_new=_activations(g, n, Hkv, D) * 1.5, v_new=_activations(g, n, Hkv, D) * 1.5)
        return s
    new = _whole(fixed, 1, most, B)
    lengths = torch.maximum(_whole(fixed, case["shortest"], case["longest"], B), new)
    lengths[-1] = case["longest"]
    new, lengths = new[mix], lengths[mix]
    table, pages = _tables(g, _ceil(lengths, P), _ceil(case["longest"], P) + 1)
    k, v, scale = _filled(g, pages, P, Hkv, D)
    s.update(k=k, v=v, scale=scale, table=table, lengths=lengths, query_start=_starts(new),
             q=_activations(g, int(new.sum()), case["Hq"], D))
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_own if own else _plain)[s["kind"]](s)


def _own_plan(s):
    from nsa_optim_b200 import ops
    p = ops.cache_plan(s["lengths"], s["new"], s["table"], s["free"], s["free_count"], s["num_tokens"], s["P"])
    return dict(query_start=p.query_start, lengths=p.lengths, slots=p.slots, positions=p.positions, free_count=p.free_count,
                shortfall=p.shortfall, table=s["table"])


def _own_append(s):
    from nsa_optim_b200 import ops
    pages = ops.KVPages(s["k"], s["v"], s["scale"])
    ops.cache_append(pages, s["k_new"], s["v_new"], s["table"], s["query_start"], s["lengths"])
    k, v = ops.cache_values(pages, s["ids"])
    return dict(k=k, v=v, scale=s["scale"])


def _own_attend(s):
    from nsa_optim_b200 import ops
    pages = ops.KVPages(s["k"], s["v"], s["scale"])
    return ops.cache_attention(s["q"], pages, s["table"], s["query_start"], s["lengths"], window=s["window"], max_new=s["most"])


def _own_logprobs(s):
    from nsa_optim_b200 import ops
    x = s["logits"].detach().requires_grad_() if s["train"] else s["logits"]
    r = ops.token_logprobs(x, s["tokens"], s["k"])
    out = dict(logprob=r.logprob, entropy=r.entropy, top_logprob=r.top_logprob, top_index=r.top_index)
    if s["train"]:
        outs, grads = [r.logprob, r.entropy], [s["dlogprob"], s["dentropy"]]
        if s["k"]:
            outs.append(r.top_logprob)
            grads.append(s["dtop"])
        out["dlogits"], = torch.autograd.grad(outs, x, grads)
        out = {n: t.detach() for n, t in out.items()}
    return out


_own = dict(plan=_own_plan, append=_own_append, attend=_own_attend, logprobs=_own_logprobs)


def _token_rows(query_start, lengths, n):
    """(sequence, position) of n packed tokens; those behind the last sequence's get sequence B."""
    i = torch.arange(n, device=DEV)
    b = torch.searchsorted(query_start[1:].contiguous(), i.to(torch.int32), right=True)
    start, new = query_start[:-1], query_start[1:] - query_start[:-1]
    c = b.clamp(max=lengths.numel() - 1)
    return b, (lengths - new)[c] + i - start[c]


def _plain_plan(s):
    P, n, table, free, count = s["P"], s["num_tokens"], s["table"], s["free"], s["free_count"]
    W = table.shape[1]
    start = _starts(s["new"]).clamp(max=n)
    lengths = s["lengths"] + (start[1:] - start[:-1])
    held, need = _ceil(s["lengths"], P), _ceil(lengths, P)
    take = need.clamp(max=W) - held.clamp(max=W)
    first = _starts(take)
    at = torch.arange(W, device=DEV)
    fresh = (at >= held[:, None]) & (at < need[:, None])
    order = (first[:-1, None] + at - held[:, None])[fresh]
    given = torch.where(order < count, free[(count - 1 - order).clamp(min=0).long()], -1)
    table[fresh] = given.to(torch.int32)
    b, pos = _token_rows(start, lengths, n)
    page = torch.where(pos // P < W, table[b, (pos // P).clamp(max=W - 1)], -1)
    slots = torch.where(page >= 0, page.long() * P + pos % P, -1)
    got = torch.minimum(first[-1:], count)
    return dict(query_start=start, lengths=lengths, slots=slots, positions=pos.long(), free_count=count - got,
                shortfall=((need - held).sum().view(1) - got).to(torch.int32), table=table)


def _codes(k, v):
    """The cache's codes as whole numbers in fp32, (pages, P, Hkv, D) for each side."""
    n, H, P2, J = k.shape[:4]
    kc = k.permute(0, 2, 4, 1, 3, 5).reshape(n, 2 * P2, H, 64 * J)
    vc = v.permute(0, 2, 4, 1, 3).reshape(n, 2 * P2, H, 64 * J)
    return kc.float() - 128, vc.float() - 128


def _plain_append(s):
    P, Hkv, D, table, scale = s["P"], s["Hkv"], s["D"], s["table"], s["scale"]
    n = s["k_new"].shape[0]
    b, pos = _token_rows(s["query_start"], s["lengths"], n)
    ids = s["ids"].long()
    place = torch.empty(s["k"].shape[0], dtype=torch.long, device=DEV)
    place[ids] = torch.arange(ids.numel(), device=DEV)
    at = place[table[b, pos // P].long()]                                    # each token's place among the pages that are touched
    kept = torch.full((ids.numel(),), P, device=DEV).scatter_reduce(0, at, pos % P, "amin")     # tokens that a page held
    pair, codes = s["scale"][ids], _codes(s["k"][ids], s["v"][ids])
    out, new_codes = [], []
    for side, x in enumerate((s["k_new"], s["v_new"])):
        x = x.float()
        amax = torch.zeros(ids.numel(), Hkv, device=DEV).scatter_reduce(0, at[:, None].expand(-1, Hkv), x.abs().amax(-1), "amax")
        before = pair[..., side]
        step = torch.where((kept > 0)[:, None], torch.maximum(before, _step(amax)), _step(amax))
        held = torch.arange(P, device=DEV) < kept[:, None]
        c = torch.where(held[:, :, None, None], (codes[side] * (before / step)[:, None, :, None]).round(), codes[side])
        c[at, pos % P] = (x / step[at][..., None]).round()
        scale[ids, :, side] = step
        new_codes.append((c + 128).to(torch.uint8))
        out.append((c * step[:, None, :, None]).to(BF))
    k, v = _pack(*new_codes)
    s["k"][ids] = k
    s["v"][ids] = v
    return dict(k=out[0], v=out[1], scale=scale)


def _plain_attend(s):
    P, Hkv, D, window, most = s["P"], s["Hkv"], s["D"], s["window"], s["most"]
    table, lengths, start = s["table"], s["lengths"], s["query_start"]
    B, n, G = lengths.numel(), s["q"].shape[0], s["Hq"] // Hkv
    W = _ceil(int(s["longest"]), P)
    pages = table[:, :W].clamp(min=0).long()
    kc, vc = _codes(s["k"], s["v"])
    k = (kc * s["scale"][:, None, :, None, 0])[pages].reshape(B, W * P, Hkv, D)
    v = (vc * s["scale"][:, None, :, None, 1])[pages].reshape(B, W * P, Hkv, D)
    b, pos = _token_rows(start, lengths, n)
    t = torch.arange(n, device=DEV) - start[b]
    q = torch.zeros(B, most, Hkv, G, D, device=DEV)
    q[b, t] = s["q"].float().view(n, Hkv, G, D)
    x = torch.einsum("bthgd,blhd->bhtgl", q, k) * D ** -0.5
    at = torch.arange(W * P, device=DEV)
    own_pos = torch.zeros(B, most, dtype=torch.long, device=DEV)
    own_pos[b, t] = pos.long()
    seen = at <= own_pos[..., None]
    if window:
        seen &= at > own_pos[..., None] - window
    x = x.masked_fill(~seen[:, None, :, None], float("-inf"))
    p = (x - x.amax(-1, keepdim=True)).exp()
    o = torch.einsum("bhtgl,blhd->bthgd", p, v) / p.sum(-1).permute(0, 2, 1, 3)[..., None]
    return o[b, t].reshape(n, s["Hq"], D).to(BF)


def _plain_logprobs(s):
    N, V, k = s["N"], s["V"], s["k"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    lse = m + e.sum(-1, keepdim=True).log()
    p = e / e.sum(-1, keepdim=True)
    logp = x - lse
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    counts = s["tokens"] >= 0
    chosen = logp.gather(1, s["tokens"].clamp(min=0)[:, None])[:, 0]
    bits = (x + 0.0).view(torch.int32)                                       # -0 is 0
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() * (1 << 18) + torch.arange(V - 1, -1, -1, device=DEV)   # ties: the lower index
    top = key.topk(k, -1).indices
    top_logp = logp.gather(1, top)
    out = dict(logprob=torch.where(counts, chosen, 0.0), entropy=entropy, top_logprob=top_logp, top_index=top)
    if s["train"]:
        g = torch.where(counts, s["dlogprob"], 0.0)
        d = -p * (g + s["dtop"].sum(-1))[:, None] - s["dentropy"][:, None] * (plogp + p * entropy[:, None])
        d.scatter_add_(1, top, s["dtop"])
        d.scatter_add_(1, s["tokens"].clamp(min=0)[:, None], g[:, None])
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


_plain = dict(plan=_plain_plan, append=_plain_append, attend=_plain_attend, logprobs=_plain_logprobs)


# ------------------------------------------------------------------------------------------------ what a pass has to move and compute
def work(case):
    kind = case["kind"]
    if kind == "plan":
        n = case["prompts"] * (case["prompt"] + 1) // 2 + case["B"]
        return {"bytes": 24 * case["B"] + 16 * n + 8 * _ceil(n, case["P"]), "flops": 0}
    if kind == "logprobs":
        n, each = case["N"] * case["V"], 4 if case["fp32"] else 2
        return {"bytes": n * each * (3 if case["train"] else 1) + case["N"] * (16 + 12 * case["k"]), "flops": n * (16 if case["train"] else 8)}
    if kind == "append":
        tokens = case["B"] * (case["most"] + max(1, case["most"] // 10)) // 2
        pages = case["B"] * (1 + (case["most"] - 1) // (2 * case["P"]))
        values = pages * case["P"] * case["Hkv"] * case["D"] * 2
        return {"bytes": 4 * tokens * case["Hkv"] * case["D"] + 3 * values + values * (case["most"] == 1), "flops": 6 * values}
    tokens = case["B"] * (case["most"] + 1) / 2
    keys = case["B"] * (case["shortest"] + case["longest"]) / 2
    if case["window"]:
        keys = min(keys, case["B"] * (case["window"] + case["most"]))
    return {"bytes": int(2 * keys * case["Hkv"] * case["D"] + 4 * tokens * case["Hq"] * case["D"]),
            "flops": int(4 * keys * (case["most"] + 1) / 2 * case["Hq"] * case["D"])}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_codes(s):
    """Values of whole pages in 64 bits, (pages, P, Hkv, D) for each side, from the layout's definition."""
    P, D = s["P"], s["D"]
    t, d = torch.arange(P, device=DEV)[:, None], torch.arange(D, device=DEV)
    k = s["k"][:, :, t // 2, d // 64, t % 2, d % 64].transpose(1, 2)
    v = s["v"][:, :, t // 16, d, t % 16].transpose(1, 2)
    return [(c.double() - 128) * s["scale"][:, None, :, None, i].double() for i, c in enumerate((k, v))]


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](s)


def _exact_plan(s):
    P, n = s["P"], s["num_tokens"]
    lengths, new, table, free = (s[x].tolist() for x in ("lengths", "new", "table", "free"))
    left, lacking = int(s["free_count"]), 0
    start, slots, positions = [0], [], []
    for b in range(len(lengths)):
        for _ in range(new[b]):
            if len(slots) == n:
                break
            pos = lengths[b]
            j, off = divmod(pos, P)
            if off == 0:
                page = -1
                if j < len(table[b]) and left:
                    left -= 1
                    page = free[left]
                lacking += page < 0
                if j < len(table[b]):
                    table[b][j] = page
            page = table[b][j] if j < len(table[b]) else -1
            slots.append(page * P + off if page >= 0 else -1)
            positions.append(pos)
            lengths[b] += 1
        start.append(len(slots))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(query_start=i32(start), lengths=i32(lengths), slots=torch.tensor(slots, device=DEV, dtype=torch.long),
                positions=torch.tensor(positions, device=DEV, dtype=torch.long), free_count=i32([left]), shortfall=i32([lacking]), table=i32(table))


def _exact_append(s):
    P, scale, values = s["P"], s["scale"].double(), _exact_codes(s)
    start, lengths, table, ids = (s[x].tolist() for x in ("query_start", "lengths", "table", "ids"))
    x = [s["k_new"].double(), s["v_new"].double()]
    for b, (lo, hi) in enumerate(zip(start, start[1:])):
        pos = lengths[b] - (hi - lo)
        while lo < hi:
            m, off, page = min(hi - lo, P - pos % P), pos % P, table[b][pos // P]
            for i in (0, 1):
                part = x[i][lo:lo + m]
                need = part.abs().amax((0, 2)) / 127
                step = 2.0 ** torch.ceil(torch.log2(need.clamp(min=2.0 ** -60)))
                step = torch.where(step / 2 >= need, step / 2, step).clamp(min=2.0 ** -60)
                if off:
                    step = torch.maximum(step, scale[page, :, i])
                values[i][page, :off] = (values[i][page, :off] / step[:, None]).round() * step[:, None]
                values[i][page, off:off + m] = (part / step[:, None]).round() * step[:, None]
                scale[page, :, i] = step
            lo, pos = lo + m, pos + m
    return dict(k=values[0][ids], v=values[1][ids], scale=scale)


def _exact_attend(s):
    if s["scale"].shape[0] * s["P"] * s["Hkv"] * s["D"] > 1 << 28:
        return None
    P, G, D = s["P"], s["Hq"] // s["Hkv"], s["D"]
    k, v = _exact_codes(s)
    start, lengths = s["query_start"].tolist(), s["lengths"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.double, device=DEV)
    for b, (lo, hi) in enumerate(zip(start, start[1:])):
        L = lengths[b]
        ids = s["table"][b, :_ceil(L, P)].long()
        kb, vb = (t[ids].flatten(0, 1)[:L] for t in (k, v))
        for i in range(lo, hi):
            end = L - (hi - i) + 1
            first = max(0, end - s["window"]) if s["window"] else 0
            q = s["q"][i].double().view(s["Hkv"], G, D)
            p = torch.softmax(torch.einsum("hgd,lhd->hgl", q, kb[first:end]) / math.sqrt(D), -1)
            out[i] = torch.einsum("hgl,lhd->hgd", p, vb[first:end]).flatten(0, 1)
    return out


def _exact_logprobs(s):
    N, V, k = s["N"], s["V"], s["k"]
    out = {n: [] for n in ("logprob", "entropy", "top_logprob", "dlogits")}
    rows = max(1, (1 << 27) // V)
    for lo in range(0, N, rows):
        x, tok = s["logits"][lo:lo + rows].double(), s["tokens"][lo:lo + rows]
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        h = -torch.special.xlogy(p, p).sum(-1)
        counts = tok >= 0
        row = torch.arange(x.shape[0], device=DEV)
        out["logprob"].append(torch.where(counts, logp[row, tok.clamp(min=0)], 0.0))
        out["entropy"].append(h)
        top = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k] if s["train"] else None
        out["top_logprob"].append(torch.topk(logp, k, -1).values)
        if s["train"]:
            g, gt, gh = (s[n][lo:lo + rows].double() for n in ("dlogprob", "dtop", "dentropy"))
            d = torch.zeros_like(x)
            d[row, tok.clamp(min=0)] += torch.where(counts, g, 0.0)
            d.scatter_add_(1, top, gt)
            d -= p * d.sum(-1, keepdim=True)
            d -= gh[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            out["dlogits"].append(d)
    r = {n: torch.cat(t) for n, t in out.items() if t}
    r["top_index"] = None
    if not s["train"]:
        r.pop("dlogits", None)
    return r
