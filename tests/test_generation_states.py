"""Generation with Mamba-2 models and hybrids, and with scaled, partial and interleaved rotary positions: on the CPU in fp32, on a GPU in bf16."""
import math

import pytest
import torch

from nsa_optim_b200 import generation, ops
from nsa_optim_b200.config import ModelConfig
from nsa_optim_b200.generation import PagedCache, generate, score
from nsa_optim_b200.models.hybrid import HybridConfig, create_hybrid_model
from nsa_optim_b200.models.kernels import RotaryEmbedding, apply_rotary_pos_emb
from nsa_optim_b200.models.mamba import Mamba2Config, create_mamba2
from nsa_optim_b200.models.transformer import create_model


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    yield request.param
    if request.param == "cuda":
        ops.native_module().check_status()


def placed(model, dev):
    g = torch.Generator().manual_seed(5)
    for p in model.parameters():
        if p.dim() == 2:
            p.data.normal_(std=0.06, generator=g)
    return model.to(dev, torch.bfloat16 if dev == "cuda" else torch.float32).eval()


def small(dev, pattern, repeats=1, vocab=512, **kw):
    """A hybrid of the pattern, or for None a Mamba-2 model; the widths that the kernels serve."""
    torch.manual_seed(4)
    if pattern is None:
        return placed(create_mamba2(Mamba2Config(d_model=256, n_layers=2, vocab_size=vocab)), dev)
    return placed(create_hybrid_model(HybridConfig(d_model=256, vocab_size=vocab, block_pattern=pattern, block_repeats=repeats, num_attention_heads=4,
                                                   num_key_value_heads=2, head_dim=64, max_position_embeddings=256, intermediate_size=256, rope_theta=1e4, **kw)), dev)


def texts(lengths, vocab=512):
    g = torch.Generator().manual_seed(9)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def whole(model, ids, dev):
    with torch.no_grad():
        return model(torch.tensor([ids], device=dev))[0][0].float()


def off(got, want):
    return float((got.float() - want).norm() / want.norm())


def steps(model, ids, cache, plans, dev):
    """(request, logits, first position) of every step's requests."""
    at = [0] * cache.requests
    for new in plans:
        packed = [t for b in range(len(ids)) for t in ids[b][at[b]:at[b] + new[b]]]
        with torch.no_grad():
            logits = model(torch.tensor([packed], device=dev), past_key_values=cache.step(new))[0][0]
        row = 0
        for b in range(len(ids)):
            if new[b]:
                yield b, logits[row:row + new[b]], at[b]
            row += new[b]
            at[b] += new[b]


@pytest.mark.parametrize("pattern", [None, "M", "MA", "AMM"])
def test_steps_agree_with_the_whole_text(dev, pattern):
    """Prompts, pieces and single tokens of requests of different lengths against the forward over the whole text.  Without attention nothing but the order of
    sums and roundings of activations differs: fp32 of some thousand operations on the CPU, about twenty roundings of 2^-8 a layer on a GPU, random and so 2^-8
    sqrt(60) = 0.03 at most of what they are of.  With attention the cache's 8 bits: 0.1, as in the transformer's test."""
    model = small(dev, pattern)
    ids = texts([190, 33, 70])
    cache = PagedCache(model, requests=4, tokens=600, page_size=16)
    limit = 0.1 if pattern and "A" in pattern else 0.03 if dev == "cuda" else 2e-4
    plans = [[140, 33, 0, 0], [1, 0, 17, 0], [1, 0, 1, 0], [0, 0, 30, 0], [48, 0, 22, 0]]
    want = [whole(model, t, dev) for t in ids]
    for b, got, at in steps(model, ids, cache, plans, dev):
        assert off(got, want[b][at:at + got.shape[0]]) < limit
    assert cache.lengths.tolist() == [190, 33, 70, 0]


@pytest.mark.parametrize("pattern", [None, "MA"])
def test_greedy_tokens_are_the_likeliest(dev, pattern):
    model = small(dev, pattern)
    prompts = texts([5, 140, 1])
    out = generate(model, prompts, 10)
    for b, p in enumerate(prompts):
        logp = torch.log_softmax(whole(model, p + out.tokens[b], dev), -1)
        for i, tok in enumerate(out.tokens[b]):
            row = logp[len(p) + i - 1]
            spread = float(row.max() - row.mean())
            assert row[tok] >= row.max() - 0.1 * spread and abs(row[tok] - out.logprobs[b][i]) < 0.1 * spread


@pytest.mark.parametrize("pattern", [None, "MA"])
def test_a_cache_is_used_again(dev, pattern):
    """A finished request's states are not those of the next one in its place."""
    model = small(dev, pattern)
    cache = PagedCache(model, requests=3, tokens=200, page_size=32)
    prompts = texts([30, 25])
    first = generate(model, prompts, 6, cache=cache)
    generate(model, texts([60, 3, 9]), 4, cache=cache)
    again = generate(model, prompts, 6, cache=cache)
    assert first.tokens == again.tokens and first.logprobs == again.logprobs and cache.held == [0] * 3


def test_requests_end_by_themselves(dev):
    model = small(dev, "MA")
    prompts = texts([21, 64, 7])
    together = generate(model, prompts, 12)
    end = together.tokens[1][3]
    cut = generate(model, prompts, 12, end_token=end)
    assert cut.tokens[1][-1] == end and len(cut.tokens[1]) <= 4
    assert all(c[:1] == t[:1] for c, t in zip(cut.tokens, together.tokens))


def test_models_of_mixers_alone_have_no_limit(dev):
    """No pages, and so no length at which they end."""
    model = small(dev, None)
    cache = PagedCache(model, requests=1, tokens=0)
    ids = texts([90])
    want = whole(model, ids[0], dev)
    for _, got, at in steps(model, ids, cache, [[60], [30]], dev):
        assert off(got, want[at:at + got.shape[0]]) < (0.03 if dev == "cuda" else 2e-4)
    cache.release([True])
    assert cache.held == [0] and cache.lengths.tolist() == [0]


def test_refusals(dev):
    model = small(dev, "MA")
    cache = PagedCache(model, requests=2, tokens=64)
    step = cache.step([3, 0])
    with pytest.raises(ValueError):
        cache.take_back([1, 0])
    assert cache.held == [3, 0]
    with pytest.raises(ValueError):
        model(torch.zeros(3, 1, dtype=torch.long, device=dev), past_key_values=step)
    with pytest.raises(ValueError):
        model(torch.zeros(1, 3, dtype=torch.long, device=dev), labels=torch.zeros(1, 3, dtype=torch.long, device=dev), past_key_values=step)
    with pytest.raises(ValueError):
        model(torch.zeros(1, 3, dtype=torch.long, device=dev), past_key_values=[(None, None)])
    for pattern, kw in (("MD", {}), ("MA", dict(attention_type="nsa"))):
        with pytest.raises(ValueError):
            PagedCache(small(dev, pattern, **kw), requests=1, tokens=64)


def test_scores_of_a_mixer_model(dev):
    model = small(dev, None)
    ids = torch.tensor(texts([40, 40]), device=dev)
    lp = score(model, ids)
    for b in range(2):
        want = torch.log_softmax(whole(model, ids[b].tolist(), dev), -1)[:-1].gather(1, ids[b, 1:, None])[:, 0]
        assert off(lp.logprob[b], want) < 0.02


def test_the_command(capsys):
    generation.main(["--block_pattern", "MA", "--model_size", "1M", "--requests", "2", "--prompt_length", "9", "--max_new_tokens", "2"])
    assert "4 generated" in capsys.readouterr().out


@pytest.mark.gpu
@pytest.mark.parametrize("pattern", [None, "MA"])
def test_a_step_is_native_and_does_not_wait(native, pattern):
    model = small("cuda", pattern)
    cache = PagedCache(model, requests=2, tokens=400)
    ids = torch.tensor([texts([200])[0]], device="cuda")
    with torch.no_grad():
        model(ids[:, :2], past_key_values=cache.step([1, 1]))
    for new in ([130, 20], [1, 1], [5, 0]):
        native.fallback_counts(reset=True)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            with torch.no_grad():
                model(ids[:, :sum(new)], past_key_values=cache.step(new), return_hidden=True)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert native.fallback_counts() == {}


@pytest.mark.gpu
def test_a_captured_step():
    """A step of single tokens as a graph, replayed: the states go on as they do without one."""
    model = small("cuda", "M")
    ids = texts([30])[0]
    tables = []
    for captured in (False, True):
        cache = PagedCache(model, requests=1, tokens=64)
        with torch.no_grad():
            model(torch.tensor([ids[:10]], device="cuda"), past_key_values=cache.step([10]))
            step = cache.step([1])
            tok = torch.tensor([[ids[10]]], device="cuda")
            if captured:
                kept = [t.clone() for s in cache.layers for t in s]
                model(tok, past_key_values=step)
                for t, k in zip([t for s in cache.layers for t in s], kept):
                    t.copy_(k)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = model(tok, past_key_values=step)[0]
            rows = []
            for i in range(10, 20):
                tok.fill_(ids[i])
                if captured:
                    graph.replay()
                else:
                    out = model(tok, past_key_values=step)[0]      # the same step again: a mixer looks at its state alone
                rows.append(out.clone())
        tables.append(torch.stack(rows))
    assert torch.equal(*tables)


# ------------------------------------------------------------------------------------------------ rotary positions
def test_scaled_tables():
    """Against the formulas pair by pair, in Python's numbers; fp32 keeps 2^-24 of a cosine, 2^-22 is left for the angle's."""
    D, theta, L, f, original = 32, 1e4, 40, 4.0, 16.0
    pos = list(range(L))

    def rate(i, kind):
        r = theta ** (-2 * i / D)
        if kind == "linear":
            return r / f
        if kind == "ntk":
            return (theta * f ** (D / (D - 2))) ** (-2 * i / D)
        turns = original * r / (2 * math.pi)
        keep = min(max((turns - 1) / 31, 0.0), 1.0)
        return r * keep + r / f * (1 - keep)
    for spec, kind, size in (("linear:4", "linear", 1), ("ntk:4", "ntk", 1), ("yarn:4:16", "yarn", 1 + 0.1 * math.log(4))):
        cos, sin = ops.rope_tables(D, L, theta, spec)
        assert cos.dtype == torch.float32 and cos.shape == sin.shape == (L, D // 2)
        want = torch.tensor([[p * rate(i, kind) for i in range(D // 2)] for p in pos], dtype=torch.double)
        assert float((cos.double() - size * want.cos()).abs().max()) < 2.0 ** -22 and float((sin.double() - size * want.sin()).abs().max()) < 2.0 ** -22
    assert rate(0, "ntk") == 1.0 and abs(rate(D // 2 - 1, "ntk") * f / theta ** (-(D - 2) / D) - 1) < 1e-12      # the fastest pair as it was, the slowest slowed by f
    plain = ops.rope_tables(D, L, theta)
    assert all(torch.equal(a, b) for a, b in zip(plain, ops.oracle.rope_tables(D, L, theta)))
    far = ops.rope_tables(64, 131072, 5e5, "linear:1")
    a = 131071 * 5e5 ** (-2 / 64)
    assert abs(float(far[0][-1, 1]) - math.cos(a)) < 1e-6 and abs(float(far[1][-1, 1]) - math.sin(a)) < 1e-6


def test_specifications():
    for bad in ("linear", "linear:0.5", "yarn:4", "yarn:4:0", "ntk:x", "cubic:2", "linear:2:3", "linear:inf", "yarn:4:nan"):
        with pytest.raises(ValueError):
            ops.rope_tables(32, 4, 1e4, bad)
        with pytest.raises(ValueError):
            RotaryEmbedding(32, scaling=bad)
    for dim in (0, 1, 7):
        with pytest.raises(ValueError):
            RotaryEmbedding(dim)
    with pytest.raises(ValueError):
        ops.rope_tables(2, 4, 1e4, "ntk:2")
    with pytest.raises(ValueError):
        ModelConfig(name="x", hidden_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2, intermediate_size=64, rotary_dim=33)
    with pytest.raises(ValueError):
        HybridConfig(d_model=64, num_attention_heads=2, rotary_dim=64)


def test_interleaved_is_halves_of_other_columns(dev):
    """The same turn with the columns in another order."""
    dtype = torch.bfloat16 if dev == "cuda" else torch.float32
    emb = RotaryEmbedding(32, 64, 1e4, interleaved=True)
    q, k = torch.randn(2, 9, 3, 48, device=dev).to(dtype), torch.randn(2, 9, 1, 48, device=dev).to(dtype)
    cos, sin = emb(q)
    order = torch.cat([torch.arange(0, 32, 2), torch.arange(1, 32, 2), torch.arange(32, 48)]).to(dev)
    for a, b in zip(apply_rotary_pos_emb(q, k, cos, sin, True), apply_rotary_pos_emb(q[..., order], k[..., order], cos, sin)):
        assert torch.equal(a[..., order], b)


@pytest.mark.parametrize("options", [dict(rotary_dim=32), dict(rope_interleaved=True), dict(rotary_dim=16, rope_interleaved=True, rope_scaling="yarn:4:64"),
                                     dict(rope_scaling="ntk:8"), dict(rope_scaling="linear:2")])
def test_options_reach_the_model(dev, options):
    """Trained, evaluated and generated with the same positions: the loss has gradients, and steps over the cache agree with the whole text."""
    torch.manual_seed(6)
    config = ModelConfig(name="small", hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                         vocab_size=256, max_position_embeddings=64, **options)
    model = placed(create_model(config), dev)
    ids = texts([100, 41], 256)
    want = [whole(model, t, dev) for t in ids]
    plain = placed(create_model(ModelConfig(**{**vars(config), **{k: v for k, v in dict(rope_scaling=None, rotary_dim=None, rope_interleaved=False).items()}})), dev)
    plain.load_state_dict(model.state_dict())
    assert off(whole(plain, ids[0], dev), want[0]) > 0.01
    cache = PagedCache(model, requests=2, tokens=200, page_size=16)
    for b, got, at in steps(model, ids, cache, [[60, 40], [39, 1], [1, 0]], dev):
        assert off(got, want[b][at:at + got.shape[0]]) < 0.1
    model.train()
    t = torch.tensor([ids[0]], device=dev)
    model(t, labels=t)[1].backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())


def test_options_of_the_command_line():
    from nsa_optim_b200.train import build_model, build_training_config, parse_args
    for extra in ([], ["--block_pattern", "MA", "--block_repeats", "1"]):
        args = parse_args(["--model_size", "1M", "--context_length", "64", "--synthetic_data", "--head_dim", "64", "--num_heads", "2", "--num_kv_heads", "1", "--mamba_type", "none",
                           "--rope_scaling", "yarn:4:16", "--rotary_dim", "32", "--rope_interleaved", *extra])
        model = build_model(build_training_config(args), args, verbose=False)[0]
        emb = [m for m in model.modules() if isinstance(m, RotaryEmbedding)]
        assert emb and all((m.dim, m.scaling, m.interleaved) == (32, "yarn:4:16", True) for m in emb)


def test_rotary_calls_of_one_side_at_a_time(dev):
    """Queries and keys that one launch cannot take together are turned as each of them alone, and rows that do not fit the tokens are refused, not passed over."""
    emb = RotaryEmbedding(64, 64, 1e4)
    q, k = torch.randn(2, 9, 3, 64, device=dev).to(torch.bfloat16), torch.randn(2, 9, 1, 64, device=dev).to(torch.bfloat16)
    cos, sin = emb(q)
    for a, b, c, s in ((q, k, cos, sin), (q, k[:1], cos, sin), (q, k.float(), cos, sin), (q, k, cos[3:4], sin[3:4]), (q[:, :1], k, cos[:1], sin[:1])):
        for got, x in zip(apply_rotary_pos_emb(a, b, c, s), (a, b)):
            assert got.dtype == x.dtype and torch.equal(got, ops.rope(x, c, s))
    for c, s, interleaved in ((cos[:5], sin[:5], False), (emb.cos_cached, emb.sin_cached, False), (cos[:5], sin[:5], True), (cos[:5, :8], sin[:5, :8], False)):
        with pytest.raises((ValueError, RuntimeError)):
            apply_rotary_pos_emb(q, k, c, s, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_of_each_sequence(dev, interleaved):
    """Ids (B, T) turn each sequence by its own, as one call for each of them does; ids (1, T) and (T) turn all alike."""
    dtype = torch.bfloat16 if dev == "cuda" else torch.float32
    emb = RotaryEmbedding(32, 64, 1e4, interleaved=interleaved)
    q, k = torch.randn(3, 9, 4, 64, device=dev).to(dtype), torch.randn(3, 9, 2, 64, device=dev).to(dtype)
    ids = torch.stack([torch.arange(9), torch.arange(40, 49), torch.randint(0, 70, (9,))]).to(dev)
    got = apply_rotary_pos_emb(q, k, *emb(q, ids), interleaved)
    for b in range(3):
        alone = apply_rotary_pos_emb(q[b:b + 1], k[b:b + 1], *emb(q[b:b + 1], ids[b]), interleaved)
        assert all(torch.equal(x[b:b + 1], y) for x, y in zip(got, alone))
    for same in (ids[1:2], ids[1], ids[1:2].expand(3, -1)):
        for x, y in zip(apply_rotary_pos_emb(q, k, *emb(q, same), interleaved), apply_rotary_pos_emb(q, k, *emb(q, ids[1]), interleaved)):
            assert torch.equal(x, y)
    for bad in (ids[:2], ids[None]):
        with pytest.raises(ValueError):
            emb(q, bad)


@pytest.mark.parametrize("hybrid", [False, True])
def test_models_turn_each_sequence_by_its_own_positions(dev, hybrid):
    """A batch whose second sequence begins at another position is two batches of one."""
    if hybrid:
        model = small(dev, "A")
    else:
        model = placed(create_model(ModelConfig(name="small", hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=4,
                                                num_key_value_heads=2, head_dim=64, vocab_size=256, max_position_embeddings=64)), dev)
    tokens = torch.tensor([t[:24] for t in texts([24, 24], 256)], device=dev)
    ids = torch.stack([torch.arange(24), 3 * torch.arange(24) + 5]).to(dev)       # steps of three: attention sees other distances
    with torch.no_grad():
        both = model(tokens, position_ids=ids)[0]
        each = torch.cat([model(tokens[b:b + 1], position_ids=ids[b])[0] for b in range(2)])
        other = model(tokens, position_ids=ids[0])[0]
    assert off(both[1], other[1].float()) > 0.01
    # the same sums in products of other shapes: fp32 of some hundred operations, or a few roundings of 2^-8 of activations and logits
    assert off(both, each.float()) < (0.02 if dev == "cuda" else 1e-5)


@pytest.mark.parametrize("options", [{}, dict(scaling="linear:2"), dict(interleaved=True)])
def test_layers_that_turn_by_themselves(dev, options):
    """Rows of the step's positions, looked up by the step, and attention over what comes turned: the same as turning on the way in."""
    model = small(dev, "A")
    dtype = next(model.parameters()).dtype
    emb = RotaryEmbedding(64, 64, 1e4, **options)
    outs = []
    for inside in (True, False):
        torch.manual_seed(3)
        cache = PagedCache(model, requests=2, tokens=100, page_size=16)
        for new in ([20, 7], [1, 1]):
            step = cache.step(new)
            q, k, v = (torch.randn(1, sum(new), h, 64, device=dev).to(dtype) for h in (4, 2, 2))
            if inside:
                outs.append(step[0].attend(q, k, v, emb))
            else:
                cos, sin = step[0].rotary(emb)
                assert torch.equal(cos, step.rotary(RotaryEmbedding(64, 64, 1e4, **options))[0]) and cos.shape == (sum(new), 32)
                outs.append(step[0].attend(*apply_rotary_pos_emb(q, k, cos, sin, emb.interleaved), v))
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    cache = PagedCache(model, requests=2, tokens=100, page_size=16)
    step = cache.step([2, 2])
    assert not torch.equal(step.rotary(RotaryEmbedding(64, 64, 1e4))[1], step.rotary(RotaryEmbedding(64, 64, 1e4, "linear:2"))[1])


@pytest.mark.parametrize("hybrid", [False, True])
def test_layers_share_the_rotary_tables(dev, hybrid):
    """Generation builds the tables of one layer, not as many as there are layers."""
    if hybrid:
        model = small(dev, "AMA")
    else:
        model = placed(create_model(ModelConfig(name="small", hidden_size=128, intermediate_size=256, num_hidden_layers=3, num_attention_heads=4,
                                                num_key_value_heads=2, head_dim=64, vocab_size=512, max_position_embeddings=32)), dev)
    generate(model, texts([40, 3]), 30)
    tables = [m for m in model.modules() if isinstance(m, RotaryEmbedding)]
    assert len(tables) > 1 and [m.max_seq_len_cached >= 70 for m in tables] == [True] + [False] * (len(tables) - 1)
