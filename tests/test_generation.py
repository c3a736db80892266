"""Generation and scoring through the paged 8-bit cache: on the CPU in fp32, on a GPU in bf16."""
import pytest
import torch

from nsa_optim_b200 import ops
from nsa_optim_b200.config import ModelConfig
from nsa_optim_b200.generation import PagedCache, generate, score
from nsa_optim_b200.models.hybrid import HybridConfig, create_hybrid_model
from nsa_optim_b200.models.transformer import create_model


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    yield request.param
    if request.param == "cuda":
        ops.native_module().check_status()


def small(dev, attention="dense", heads=4, kv=2, head_dim=64, layers=2, vocab=512):
    torch.manual_seed(3)
    config = ModelConfig(name="small", hidden_size=256, intermediate_size=512, num_hidden_layers=layers, num_attention_heads=heads, num_key_value_heads=kv,
                         head_dim=head_dim, vocab_size=vocab, max_position_embeddings=256, attention_type=attention)
    model = create_model(config)
    for p in model.parameters():
        if p.dim() == 2:
            torch.nn.init.normal_(p, std=0.06)
    return model.to(dev, torch.bfloat16 if dev == "cuda" else torch.float32).eval()


def texts(lengths, vocab=512):
    g = torch.Generator().manual_seed(7)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def whole(model, ids, dev):
    """Logits of a text by the ordinary forward."""
    with torch.no_grad():
        return model(torch.tensor([ids], device=dev))[0][0].float()


def off(got, want):
    return float((got.float() - want).norm() / want.norm())


@pytest.mark.parametrize("head_dim,heads,kv", [(64, 4, 2), (128, 8, 1)])
def test_steps_agree_with_the_whole_text(dev, head_dim, heads, kv):
    """Prompts, pieces and single tokens of requests of different lengths against the forward over the whole text.  Codes are off by up to half a step, a
    step at most 2/127 of the page's largest number, about 3.5 times a typical one: 0.03 / sqrt(3) = 1.6 % of a key or a value, twice that of an
    attention output with its probabilities, which the residual stream dilutes; 0.1 leaves a factor of three."""
    model = small(dev, heads=heads, kv=kv, head_dim=head_dim)
    ids = texts([90, 33, 70])
    cache = PagedCache(model, requests=4, tokens=400, page_size=16)
    at = [0, 0, 0, 0]
    for new in ([40, 33, 0, 0], [1, 0, 17, 0], [1, 0, 1, 0], [0, 0, 30, 0], [48, 0, 22, 0]):
        packed = [t for b in range(3) for t in ids[b][at[b]:at[b] + new[b]]]
        step = cache.step(new)
        with torch.no_grad():
            logits = model(torch.tensor([packed], device=dev), past_key_values=step)[0][0]
        row = 0
        for b in range(3):
            if new[b]:
                assert off(logits[row:row + new[b]], whole(model, ids[b], dev)[at[b]:at[b] + new[b]]) < 0.1
            row += new[b]
            at[b] += new[b]
        assert cache.lengths.tolist() == at and int(step.plan.shortfall) == 0
    used = sum(-(-n // 16) for n in at)
    assert int(cache.free_count) == cache.free.numel() - used
    cache.release([True, False, True, False])
    assert cache.lengths.tolist() == [0, 33, 0, 0] and int(cache.free_count) == cache.free.numel() - 3


def test_greedy_tokens_are_the_likeliest(dev):
    model = small(dev)
    prompts = texts([5, 40, 1])
    out = generate(model, prompts, 12, top_k=3, alternatives=True)
    assert [len(t) for t in out.tokens] == [12] * 3
    for b, p in enumerate(prompts):
        logp = torch.log_softmax(whole(model, p + out.tokens[b], dev), -1)
        for i, tok in enumerate(out.tokens[b]):
            row = logp[len(p) + i - 1]
            alts = out.alternatives[b][i]
            assert alts[0] == (tok, out.logprobs[b][i]) and alts[0][1] >= alts[1][1] >= alts[2][1]
            spread = float(row.max() - row.mean())
            assert row[tok] >= row.max() - 0.1 * spread and abs(row[tok] - out.logprobs[b][i]) < 0.1 * spread
            assert abs(out.entropies[b][i] + float((row.exp() * row).sum())) < 0.1 * spread


def test_requests_do_not_see_one_another(dev):
    """The same tokens whether a request runs alone or beside others that end earlier."""
    model = small(dev)
    prompts = texts([21, 64, 7, 30])
    together = generate(model, prompts, 20)
    end = together.tokens[1][4]
    cut = generate(model, prompts, 20, end_token=end)
    for b, p in enumerate(prompts):
        alone = generate(model, [p], 20)
        same = [x == y for x, y in zip(alone.tokens[0], together.tokens[b])]
        first = same.index(False) if False in same else 20
        if first < 20:                                       # products of other shapes round differently: only a near tie may fall otherwise
            assert abs(alone.logprobs[0][first] - together.logprobs[b][first]) < 0.05
        stop = together.tokens[b].index(end) + 1 if end in together.tokens[b] else 20
        if first >= stop:
            assert cut.tokens[b][:1] == together.tokens[b][:1] and (end not in cut.tokens[b][:-1])
    assert len(cut.tokens[1]) <= 5 and cut.tokens[1][-1] == end


def test_a_cache_is_used_again(dev):
    model = small(dev)
    cache = PagedCache(model, requests=3, tokens=120, page_size=32)
    prompts = texts([30, 25])
    first = generate(model, prompts, 6, cache=cache)
    assert cache.lengths.tolist() == [0, 0, 0] and int(cache.free_count) == cache.free.numel()
    assert sorted(cache.free.tolist()) == list(range(cache.free.numel()))
    again = generate(model, prompts, 6, cache=cache)
    assert first.tokens == again.tokens and first.logprobs == again.logprobs


def test_sampling(dev):
    model = small(dev)
    prompts = texts([9, 12])
    g = torch.Generator(device=dev).manual_seed(1)
    out = generate(model, prompts, 30, temperature=1.0, top_k=5, alternatives=True, generator=g)
    picks = [[t for t, _ in alts].index(tok) for b in range(2) for tok, alts in zip(out.tokens[b], out.alternatives[b])]
    assert len(set(picks)) > 1 and max(picks) < 5
    for b in range(2):
        for tok, lp, alts in zip(out.tokens[b], out.logprobs[b], out.alternatives[b]):
            assert dict(alts)[tok] == lp


@pytest.mark.parametrize("kind", ["dense", "nsa", "hybrid"])
def test_scores(dev, kind):
    if kind == "hybrid":
        torch.manual_seed(0)
        model = create_hybrid_model(HybridConfig(d_model=256, vocab_size=512, block_pattern="MDA", block_repeats=1, num_attention_heads=4,
                                                 num_key_value_heads=2, deltanet_head_dim=128, deltanet_num_heads=2, intermediate_size=512))
        model = model.to(dev, torch.bfloat16 if dev == "cuda" else torch.float32).eval()
    else:
        model = small(dev, attention=kind)
    ids = torch.tensor(texts([70, 70]), device=dev)
    ids[1, 50:] = 0
    r = score(model, ids, top_k=3, pad_token=0, chunk=33)
    logits = model(ids)[0].detach().float()[:, :-1]
    logp = torch.log_softmax(logits, -1)
    want = logp.gather(-1, ids[:, 1:, None])[..., 0].masked_fill(ids[:, 1:] == 0, 0.0)
    # the logits of other chunks of rows are rounded the same: only the log probability's own error, 2^-20 of numbers below 2^5, and in bf16 a last bit of
    # the logits where a product is cut otherwise
    tol = 2.0 ** -15 if dev == "cpu" else 2.0 ** -4
    assert r.logprob.shape == (2, 69) and (r.logprob - want).abs().max() < tol
    assert (r.entropy + (logp.exp() * logp).sum(-1)).abs().max() < tol
    assert r.top_index.shape == (2, 69, 3) and (r.top_logprob - logp.topk(3).values).abs().max() < tol


def test_refusals(dev):
    model = small(dev, layers=1)
    for bad in ([], [[]], [[1], []]):
        with pytest.raises(ValueError):
            generate(model, bad, 3)
    for kw in (dict(max_new_tokens=0), dict(max_new_tokens=2, temperature=-1.0), dict(max_new_tokens=2, top_k=0)):
        with pytest.raises(ValueError):
            generate(model, [[1]], **kw)
    cache = PagedCache(model, requests=1, tokens=64)
    with pytest.raises(ValueError):
        generate(model, [[1], [2]], 2, cache=cache)
    for new in ([1, 1], [-1]):
        with pytest.raises(ValueError):
            cache.step(new)
    with pytest.raises(ValueError):
        model(torch.zeros(2, 3, dtype=torch.long, device=dev), past_key_values=cache.step([6]))
    with pytest.raises(ValueError):
        model(torch.zeros(1, 3, dtype=torch.long, device=dev), past_key_values=cache.step([3]), use_cache=True)
    with pytest.raises(ValueError):
        PagedCache(small(dev, attention="nsa", layers=1), requests=1, tokens=64)
    with pytest.raises(ValueError):
        score(model, torch.zeros(4, dtype=torch.long, device=dev))


@pytest.mark.gpu
def test_a_step_is_native(native):
    """No part of a step runs on the PyTorch implementation, and nothing waits for the device."""
    model = small("cuda")
    cache = PagedCache(model, requests=2, tokens=200)
    ids = torch.tensor([texts([50])[0]], device="cuda")
    rows = torch.tensor([0], device="cuda")
    for new in ([30, 20], [1, 1]):
        native.fallback_counts(reset=True)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            with torch.no_grad():
                h = model(ids[:, :sum(new)], past_key_values=cache.step(new), return_hidden=True)[0]
                ops.token_logprobs(ops.linear(h[0, rows], model.output_weight()), rows, 4)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert native.fallback_counts() == {}


def state_of(cache):
    return cache.held, cache.lengths.tolist(), int(cache.free_count), sorted(cache.free.tolist()), cache.table.tolist()


def test_a_step_beyond_the_cache_is_refused(dev):
    """A step that needs more pages than there are changes nothing; one that needs them all goes through."""
    model = small(dev, layers=1)
    cache = PagedCache(model, requests=3, tokens=32, page_size=16)            # five pages
    cache.step([17, 0, 16])
    before = state_of(cache)
    for new in ([0, 33, 0], [16, 0, 17], [0, 1, 17], [49, 0, 0]):
        with pytest.raises(ValueError):
            cache.step(new)
        assert state_of(cache) == before
    assert int(cache.step([15, 1, 16]).plan.shortfall) == 0 and int(cache.free_count) == 0
    cache.release([False, True, False])
    cache.step([1, 0, 0])
    assert int(cache.free_count) == 0


def test_a_cache_too_small_for_the_prompts_is_refused(dev):
    model = small(dev)
    prompts = texts([60, 55])
    with pytest.raises(ValueError):
        generate(model, prompts, 8, cache=PagedCache(model, requests=2, tokens=48, page_size=16))
    cache = PagedCache(model, requests=2, tokens=112, page_size=16)            # nine pages: 63 and 60 tokens are eight
    assert generate(model, prompts, 8, cache=cache).tokens == generate(model, prompts, 8).tokens


def test_a_cache_in_use_is_refused(dev):
    """generate takes the first requests of a cache: they have to be empty, others may be under way."""
    model = small(dev)
    prompts = texts([21, 9])
    want = generate(model, prompts, 5).tokens
    cache = PagedCache(model, requests=3, tokens=200, page_size=16)
    cache.step([0, 0, 20])
    assert generate(model, prompts, 5, cache=cache).tokens == want and cache.held == [0, 0, 20]
    cache.step([0, 3, 0])
    before = state_of(cache)
    with pytest.raises(ValueError):
        generate(model, prompts, 5, cache=cache)
    assert state_of(cache) == before


@pytest.mark.parametrize("call", [1, 4])
def test_an_interrupted_generation_leaves_its_cache_empty(dev, call, monkeypatch):
    model = small(dev)
    prompts = texts([21, 9])
    cache = PagedCache(model, requests=3, tokens=200, page_size=16)
    cache.step([0, 0, 20])
    want = generate(model, prompts, 6, cache=cache).tokens
    real, calls = ops.token_logprobs, []

    def interrupted(*args):
        calls.append(1)
        if len(calls) == call:
            raise KeyboardInterrupt
        return real(*args)
    monkeypatch.setattr(ops, "token_logprobs", interrupted)
    with pytest.raises(KeyboardInterrupt):
        generate(model, prompts, 6, cache=cache)
    monkeypatch.undo()
    assert cache.held == cache.lengths.tolist() == [0, 0, 20] and int(cache.free_count) == cache.free.numel() - 2
    assert generate(model, prompts, 6, cache=cache).tokens == want


def test_rows_without_a_given_token_are_ignored_ones(dev, monkeypatch):
    """A debug build records tokens that are neither ignored nor in the vocabulary."""
    model = small(dev, layers=1)
    real, given = ops.token_logprobs, []

    def watched(logits, tokens, top_k=0, ignore_index=-100):
        given.append((tokens.tolist(), ignore_index))
        return real(logits, tokens, top_k, ignore_index)
    monkeypatch.setattr(ops, "token_logprobs", watched)
    generate(model, texts([3, 5]), 3)
    assert len(given) == 3 and all(t == ignored for tokens, ignored in given for t in tokens)


def test_rotary_tables_grow_seldom(dev, monkeypatch):
    """Requests beyond the configured length: the table doubles instead of being built again for every token, and keeps its values."""
    from nsa_optim_b200.models.kernels import RotaryEmbedding
    emb, built = RotaryEmbedding(64, 16), []
    real = RotaryEmbedding._set_cos_sin_cache
    monkeypatch.setattr(RotaryEmbedding, "_set_cos_sin_cache", lambda self, n, device=None: (built.append(n), real(self, n, device=device)))
    want = ops.oracle.rope_tables(64, 300, emb.base, device=dev)
    for n in list(range(1, 65)) + [300]:
        cos, sin = emb.rows(torch.arange(n, device=dev), n)
        assert torch.equal(cos, want[0][:n]) and torch.equal(sin, want[1][:n])
    assert len(built) <= 4 and max(built) <= 600


@pytest.mark.gpu
@pytest.mark.parametrize("sampled", [False, True])
def test_generation_does_not_wait(native, sampled, monkeypatch):
    """Without an end token nothing makes the host wait before the results are read, also in a cache with more requests than prompts."""
    model = small("cuda")
    cache = PagedCache(model, requests=5, tokens=300)
    prompts = texts([30, 7, 50])
    kw = dict(cache=cache, temperature=0.8, top_k=4) if sampled else dict(cache=cache)
    generate(model, prompts, 4, **kw)
    real, read = PagedCache.release, []

    def release(self, finished):                                # the last thing before results are read
        real(self, finished)
        read.append(1)
        torch.cuda.set_sync_debug_mode("default")
    monkeypatch.setattr(PagedCache, "release", release)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        generate(model, prompts, 4, **kw)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert len(read) == 1


def test_requests_go_on_when_others_end(dev):
    """What is generated behind another request's end: the same tokens as without an end, up to the request's own, exactly on the CPU, on a GPU up to a near tie (products
    of other shapes round differently)."""
    model = small(dev)
    prompts = texts([21, 64, 7, 30])
    cache = PagedCache(model, requests=6, tokens=600, page_size=16)
    together = generate(model, prompts, 20, cache=cache)
    end = together.tokens[1][4]
    cut = generate(model, prompts, 20, cache=cache, end_token=end)
    assert cache.held == [0] * 6 and int(cache.free_count) == cache.free.numel()
    stops = [t.index(end) + 1 if end in t else 20 for t in together.tokens]
    assert min(stops) < max(stops) - 3                          # of these inputs: some go on
    for b, stop in enumerate(stops):
        want, got = together.tokens[b][:stop], cut.tokens[b]
        n = min(len(want), len(got))
        differs = next((i for i in range(n) if want[i] != got[i]), None)
        if differs is None:
            assert len(want) == len(got)
            assert max(abs(x - y) for x, y in zip(together.logprobs[b], cut.logprobs[b])) < (1e-4 if dev == "cpu" else 0.05)
        else:
            assert dev == "cuda" and abs(together.logprobs[b][differs] - cut.logprobs[b][differs]) < 0.05


def test_drafts_are_taken_back(dev):
    """Tokens that are verified and rejected leave the cache with their pages; none is lost, and what follows agrees with the whole text (the bound of
    test_steps_agree_with_the_whole_text: codes may have been rounded once more where a rejected token raised a page's scale)."""
    model = small(dev)
    ids = texts([100, 60, 80])
    cache = PagedCache(model, requests=3, tokens=260, page_size=16)
    at, gen = [0, 0, 0], torch.Generator().manual_seed(5)
    for turn, (right, drafted) in enumerate((([30, 16, 1], [0, 0, 0]), ([1, 1, 15], [17, 15, 1]), ([1, 0, 16], [3, 0, 33]), ([0, 31, 1], [0, 16, 0]),
                                             ([1, 1, 1], [40, 0, 0]), ([20, 1, 20], [5, 5, 5]))):
        packed = []
        for b in range(3):
            packed += ids[b][at[b]:at[b] + right[b]] + torch.randint(0, 512, (drafted[b],), generator=gen).tolist()
        new = [r + d for r, d in zip(right, drafted)]
        with torch.no_grad():
            logits = model(torch.tensor([packed], device=dev), past_key_values=cache.step(new))[0][0]
        row = 0
        for b in range(3):
            if right[b]:
                assert off(logits[row:row + right[b]], whole(model, ids[b], dev)[at[b]:at[b] + right[b]]) < 0.1
            row += new[b]
            at[b] += right[b]
        cache.take_back(drafted)
        assert cache.held == cache.lengths.tolist() == at
        held = [-(-n // 16) for n in at]
        table = cache.table.tolist()
        assert all(p == -1 for b in range(3) for p in table[b][held[b]:])
        pages = [p for b in range(3) for p in table[b][:held[b]]] + cache.free[:int(cache.free_count)].tolist()
        assert sorted(pages) == list(range(cache.free.numel()))
    cache.take_back(at)
    assert cache.held == [0, 0, 0] and int(cache.free_count) == cache.free.numel()


def test_refused_drafts(dev):
    cache = PagedCache(small(dev, layers=1), requests=2, tokens=64)
    cache.step([5, 0])
    before = state_of(cache)
    for counts in ([6, 0], [0, 1], [-1, 0], [1], [1, 0, 0]):
        with pytest.raises(ValueError):
            cache.take_back(counts)
    assert state_of(cache) == before


@pytest.mark.gpu
def test_taking_drafts_back_does_not_wait(native):
    cache = PagedCache(small("cuda", layers=1), requests=2, tokens=640)
    cache.step([100, 70])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        cache.take_back([50, 0])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert cache.lengths.tolist() == [50, 70]


def test_a_step_knows_its_positions(dev):
    """A step whose requests have left the cache when it runs: its tokens are stored nowhere, and no row behind the rotary tables is asked for."""
    model = small(dev, layers=1)
    cache = PagedCache(model, requests=2, tokens=400)
    step = cache.step([300, 0])                                # the model's tables have 256 rows
    cache.release([True, False])
    with torch.no_grad():
        h = model(torch.tensor(texts([300]), device=dev), past_key_values=step, return_hidden=True)[0]
    assert h.isfinite().all()
