"""Generation and scoring with a trained dense transformer, Mamba-2 model or hybrid of both, over a paged key / value cache in 8 bits and the mixers' states.

    cache = PagedCache(model, requests=8, tokens=8 * 2048)
    out = generate(model, prompts, max_new_tokens=128, cache=cache)      # tokens, their log probabilities and the alternatives
    lp = score(model, input_ids)                                         # log probability and entropy of every token of a text

A step takes any mix of prompts, single tokens and idle requests, packed one request after another: ``ops.cache_plan`` finds pages and
slots, each attention layer turns queries and keys by their positions and appends keys and values (``ops.cache_append_rope``) and attends over the pages
(``ops.cache_attention``), each Mamba-2 layer continues its convolution and its scan from the requests' states (``ops.conv1d_cached``, ``ops.ssd_scan_cached``), and
``ops.token_logprobs`` turns the logits into the chosen tokens' log probabilities.  Nothing but the end of a request (an end token) makes the host wait
for a bf16 model on a GPU; models of other types append and attend in PyTorch there, which waits in every layer.
The reference decodes with a concatenated cache (models/transformer.py:104-118 there); that path is still ``use_cache=True``.

    python -m nsa_optim_b200.generation --requests 16 --prompt_length 512 --max_new_tokens 64 [--block_pattern MMA]
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import ops
from .models.base import CausalLMBase
from .models.hybrid import AttentionBlock
from .models.mamba import Mamba2Mixer
from .models.transformer import DenseAttention


def _attention_of(layer):
    """The module of a layer that attends densely, None where there is none."""
    a = getattr(layer, "self_attn", layer)
    return a if type(a) is DenseAttention or (type(a) is AttentionBlock and not a.sparse) else None


class PagedCache:
    """Pages of every attention layer of a model for up to ``requests`` requests at once, ``tokens`` tokens together (each request's last page counts
    whole), and the states of every Mamba-2 layer; a model of these alone takes requests of any length.  ``table``, ``lengths``, ``free`` and ``free_count`` are
    those of :mod:`nsa_optim_b200.ops.cache`."""

    def __init__(self, model: CausalLMBase, requests: int, tokens: int, page_size: int = 64, device=None):
        first = next(model.parameters())
        device = device or first.device
        attention = [_attention_of(layer) for layer in model.layers]
        mixers = [layer.mixer if type(getattr(layer, "mixer", None)) is Mamba2Mixer else None for layer in model.layers]
        if any(a is None and m is None for a, m in zip(attention, mixers)):
            raise ValueError("the paged cache serves dense attention and Mamba-2 mixers; sparse layers of transformers decode with use_cache=True")
        self.paged, self.has_states = any(a is not None for a in attention), any(m is not None for m in mixers)
        pages = -(-tokens // page_size) + requests if self.paged else 0
        self.page_size, self.requests = page_size, requests
        self.layers = [ops.cache_pages(pages, a.num_kv_heads, a.head_dim, page_size, device=device) if m is None else
                       ops.scan_states(requests, m.nheads, m.headdim, m.d_state, m.conv_dim, m.d_conv, device=device, dtype=first.dtype)
                       for a, m in zip(attention, mixers)]
        self.table = torch.full((requests, max(pages, 1)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.held = [0] * requests                           # the lengths as the host knows them

    def step(self, new: Sequence[int]) -> "CacheStep":
        """Makes room for ``new[b]`` tokens of each request; the result goes to the model as ``past_key_values``.  A step for which there are too few
        pages is refused and changes nothing."""
        if len(new) != self.requests or min(new) < 0:
            raise ValueError(f"a count of new tokens for each of {self.requests} requests is needed")
        need, pages = sum(-(-(a + b) // self.page_size) for a, b in zip(self.held, new)), self.free.numel()
        if self.paged and need > pages:
            raise ValueError(f"the step needs {need} pages of {self.page_size} tokens, the cache has {pages}")
        counts = torch.tensor(list(new), dtype=torch.int32).to(self.lengths.device, non_blocking=True)
        plan = ops.cache_plan(self.lengths, counts, self.table, self.free, self.free_count, sum(new), self.page_size)
        self.lengths, self.free_count = plan.lengths, plan.free_count
        self.held = [a + b for a, b in zip(self.held, new)]
        return CacheStep(self, plan, max(max(new), 1))

    def release(self, finished: Sequence[bool]) -> None:
        """Gives the pages of finished requests back."""
        mask = torch.tensor(list(finished), dtype=torch.bool).to(self.lengths.device, non_blocking=True)
        self.lengths, self.free_count = ops.cache_release(mask, self.lengths, self.table, self.free, self.free_count, self.page_size)
        self.held = [0 if f else n for f, n in zip(finished, self.held)]

    def take_back(self, tokens: Sequence[int]) -> None:
        """Takes the last ``tokens[b]`` tokens of each request back (drafted ones that were rejected) and frees the pages behind what is left.  A page that
        stays keeps the scale that they may have raised.  The states of Mamba-2 layers cannot be taken back: models that have any refuse it."""
        if self.has_states:
            raise ValueError("the states of Mamba-2 layers hold no earlier tokens to go back to")
        if len(tokens) != self.requests or any(not 0 <= t <= n for t, n in zip(tokens, self.held)):
            raise ValueError(f"a count of each request's tokens to take back is needed, of {self.held} at most")
        left = [n - t for n, t in zip(self.held, tokens)]
        keep, had = ([-(-n // self.page_size) for n in counts] for counts in (left, self.held))
        there = lambda numbers, dtype: torch.tensor(numbers, dtype=dtype).to(self.lengths.device, non_blocking=True)  # noqa: E731
        # the pages to free as requests of their own: each row of the table from the first of them on
        W = self.table.shape[1]
        at, first = torch.arange(W, device=self.table.device), there(keep, torch.long)[:, None]
        tail = self.table.gather(1, (at + first).clamp(max=W - 1))
        _, self.free_count = ops.cache_release(there([h > k for h, k in zip(had, keep)], torch.bool),
                                               there([(h - k) * self.page_size for h, k in zip(had, keep)], torch.int32), tail, self.free, self.free_count,
                                               self.page_size)
        self.table.masked_fill_(at >= first, -1)
        self.lengths, self.held = there(left, torch.int32), left


class CacheStep:
    """One step's view of a :class:`PagedCache`: ``step[i]`` is what layer i appends to and attends over, or continues from."""

    def __init__(self, cache: PagedCache, plan: ops.CachePlan, max_new: int):
        self.cache, self.plan, self.max_new = cache, plan, max_new
        self.limit = max(cache.held)                         # above all of the plan's positions, whatever leaves the cache later
        self._rotary: dict = {}
        self._tables: dict = {}

    def __getitem__(self, layer: int):
        state = self.cache.layers[layer]
        return MixerStep(self, state) if isinstance(state, ops.ScanStates) else LayerStep(self, state)

    def last_rows(self) -> Tensor:
        """Row of each request's last token in the packed step (that of the token before it where it has none)."""
        return (self.plan.query_start[1:] - 1).clamp(min=0).long()

    def rotary(self, emb) -> Tuple[Tensor, Tensor]:
        """Cosines and sines of the step's positions, looked up once for all layers: for queries and keys that are turned outside of ``attend``."""
        key = self._angles(emb)
        if key not in self._rotary:
            self._rotary[key] = emb.rows(self.plan.positions, self.limit)
        return self._rotary[key]

    def tables(self, emb) -> Tuple[Tensor, Tensor]:
        """Tables that reach as far as the step, those of the first layer for all layers of the same angles: the others build none."""
        key = self._angles(emb)
        if key not in self._tables:
            self._tables[key] = emb.tables(self.limit, self.plan.positions.device)
        return self._tables[key]

    @staticmethod
    def _angles(emb):
        return emb.dim, emb.base, getattr(emb, "scaling", None)


class LayerStep:
    def __init__(self, step: CacheStep, pages: ops.KVPages):
        self.step, self.pages = step, pages
        self.rotary = step.rotary

    def attend(self, q: Tensor, k: Tensor, v: Tensor, rotary=None) -> Tensor:
        """Attention of the step's packed queries (1, N, Hq, D) over their requests, to which k and v (1, N, Hkv, D) are appended first; queries and keys are turned
        by their positions' rows of ``rotary``'s tables, or come as they are (None)."""
        c, p = self.step.cache, self.step.plan
        q, k, v = q[0], k[0], v[0]
        if rotary is None:
            ops.cache_append(self.pages, k, v, c.table, p.query_start, p.lengths)
        else:
            cos, sin = self.step.tables(rotary)
            q = ops.cache_append_rope(self.pages, q, k, v, cos, sin, c.table, p.query_start, p.lengths, rotary.interleaved)
        return ops.cache_attention(q, self.pages, c.table, p.query_start, p.lengths, max_new=self.step.max_new).unsqueeze(0)


class MixerStep:
    def __init__(self, step: CacheStep, states: ops.ScanStates):
        self.step, self.states = step, states

    def convolve(self, x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tensor:
        """The short convolution of the step's packed inputs (N, C), after those that its requests had before."""
        return ops.conv1d_cached(x, weight, bias, self.states.conv, self.step.plan.query_start, self.step.plan.lengths)

    def scan(self, x: Tensor, dt: Tensor, A_log: Tensor, Bm: Tensor, Cm: Tensor, D: Tensor, dt_bias: Tensor) -> Tensor:
        """The scan of the step's packed tokens from its requests' states on."""
        p = self.step.plan
        return ops.ssd_scan_cached(x, dt, A_log, Bm, Cm, D, dt_bias, self.states.ssm, p.query_start, p.lengths, max_new=self.step.max_new)


@dataclass
class Generated:
    tokens: List[List[int]]              # without the prompt, with the end token where it came
    logprobs: List[List[float]]
    entropies: List[List[float]]
    alternatives: Optional[List[List[List[Tuple[int, float]]]]] = None


@torch.no_grad()
def generate(model: CausalLMBase, prompts: Sequence[Sequence[int]], max_new_tokens: int, cache: Optional[PagedCache] = None,
             temperature: float = 0.0, top_k: int = 1, end_token: Optional[int] = None, alternatives: bool = False,
             generator: Optional[torch.Generator] = None) -> Generated:
    """Continues every prompt by up to ``max_new_tokens`` tokens: the likeliest one at temperature 0, else one of the ``top_k`` likeliest in
    proportion to p^(1 / temperature).  Log probabilities are the model's, without the temperature; ``alternatives`` returns the ``top_k`` tokens too."""
    if not prompts or any(len(p) == 0 for p in prompts):
        raise ValueError("every request needs a prompt of one token at least")
    if max_new_tokens < 1 or temperature < 0 or top_k < 1:
        raise ValueError("max_new_tokens and top_k have to be positive, temperature not negative")
    device, B = next(model.parameters()).device, len(prompts)
    if cache is None:
        cache = PagedCache(model, B, sum(len(p) + max_new_tokens for p in prompts))
    if cache.requests < B:
        raise ValueError(f"the cache holds {cache.requests} requests, {B} were given")
    if any(cache.held[:B]):
        raise ValueError(f"the cache's first {B} requests have to be empty: they hold {cache.held[:B]} tokens")

    def there(numbers):                                      # a list on the device, without waiting for it
        return torch.tensor(numbers).to(device, non_blocking=True)

    rows = list(range(B))                                    # requests that go on
    live = there(rows)
    new = [len(p) for p in prompts] + [0] * (cache.requests - B)
    tokens = there([t for p in prompts for t in p])
    chosen, kept = [], []
    none = torch.full((cache.requests,), -100, dtype=torch.long, device=device)
    try:
        for n in range(max_new_tokens):
            step = cache.step(new)
            h = model(tokens.unsqueeze(0), past_key_values=step, return_hidden=True)[0]
            r = ops.token_logprobs(ops.linear(h[0, step.last_rows()], model.output_weight()), none, top_k)
            if temperature > 0 and top_k > 1:
                pick = torch.multinomial(torch.softmax(r.top_logprob / temperature, -1), 1, generator=generator)
            else:
                pick = torch.zeros(cache.requests, 1, dtype=torch.long, device=device)
            tok, lp = r.top_index.gather(1, pick)[:, 0], r.top_logprob.gather(1, pick)[:, 0]
            chosen.append((tok, lp, r.entropy))
            kept.append((rows, r.top_index, r.top_logprob))
            if end_token is not None:
                ended = (tok == end_token).tolist()          # the one thing that the host waits for
                cache.release([b in rows and ended[b] for b in range(cache.requests)])
                rows = [b for b in rows if not ended[b]]
                if not rows:
                    break
                live = there(rows)
            new = [1 if b in rows else 0 for b in range(cache.requests)]
            tokens = tok[live] if len(rows) < cache.requests else tok
    finally:                                                 # also where a step was refused or interrupted
        if rows:
            cache.release([b in rows for b in range(cache.requests)])
    out = Generated([[] for _ in range(B)], [[] for _ in range(B)], [[] for _ in range(B)], [[] for _ in range(B)] if alternatives else None)
    for (tok, lp, h), (alive, index, top) in zip(chosen, kept):
        tok, lp, h = tok.tolist(), lp.tolist(), h.tolist()
        for b in alive:
            out.tokens[b].append(tok[b])
            out.logprobs[b].append(lp[b])
            out.entropies[b].append(h[b])
        if alternatives:
            index, top = index.tolist(), top.tolist()
            for b in alive:
                out.alternatives[b].append(list(zip(index[b], top[b])))
    return out


@torch.no_grad()
def score(model, input_ids: Tensor, top_k: int = 0, pad_token: Optional[int] = None, chunk: int = 4096) -> ops.TokenLogprobs:
    """Log probability, entropy and likeliest tokens at every position of (B, T) texts but the last: entry t is about token t + 1 (0 where that is
    ``pad_token``).  Works with every model of the framework; the logits of ``chunk`` positions are in memory at a time."""
    if input_ids.dim() != 2 or input_ids.shape[1] < 2:
        raise ValueError("texts have to be (B, T), T at least 2")
    B, T = input_ids.shape
    h = model(input_ids, return_hidden=True)[0][:, :-1].flatten(0, 1)
    target = input_ids[:, 1:].flatten()
    if pad_token is not None:
        target = target.masked_fill(target == pad_token, -100)
    parts = [ops.token_logprobs(ops.linear(x, model.output_weight()), t, top_k) for x, t in zip(h.split(chunk), target.split(chunk))]
    return ops.TokenLogprobs(*(torch.cat(p).view(B, T - 1, *p[0].shape[1:]) for p in zip(*parts)))


def main(argv=None) -> None:
    from .config import TrainingConfig, get_model_config_for_size
    from .models.configs import get_hybrid_config
    from .models.hybrid import create_hybrid_model
    from .models.transformer import create_model
    ap = argparse.ArgumentParser(description="Generates from a randomly initialised model and reports the rate.")
    ap.add_argument("--model_size", default="0.6B")
    ap.add_argument("--block_pattern", default=None, help="a hybrid of M (Mamba-2) and A (dense attention) blocks instead of a transformer, such as MMA")
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prompt_length", type=int, default=512)
    ap.add_argument("--max_new_tokens", type=int, default=64)
    ap.add_argument("--top_k", type=int, default=8)
    ap.add_argument("--temperature", type=float, default=0.8)
    a = ap.parse_args(argv)
    device = "cuda" if torch.cuda.is_available() else "cpu"
    if a.block_pattern:
        config = get_hybrid_config(TrainingConfig(model_size=a.model_size), a.block_pattern, -1, verbose=False)
        model = create_hybrid_model(config)
    else:
        config = get_model_config_for_size(a.model_size)
        model = create_model(config)
    model = model.to(device, torch.bfloat16 if device == "cuda" else torch.float32).eval()
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, config.vocab_size, (max(1, a.prompt_length - 7 * i),), generator=g).tolist() for i in range(a.requests)]
    for _ in range(2):                                       # the first pass builds tables and loads kernels
        t = time.perf_counter()
        out = generate(model, prompts, a.max_new_tokens, temperature=a.temperature, top_k=a.top_k)
        if device == "cuda":
            torch.cuda.synchronize()
        t = time.perf_counter() - t
    made = sum(map(len, out.tokens))
    print(f"{a.requests} requests, {sum(map(len, prompts))} prompt tokens, {made} generated in {t:.3f} s ({made / t:.0f} tokens/s), "
          f"mean log probability {sum(map(sum, out.logprobs)) / made:.3f}, mean entropy {sum(map(sum, out.entropies)) / made:.3f}")


if __name__ == "__main__":
    main()
