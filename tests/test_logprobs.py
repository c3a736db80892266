"""Log probabilities of given tokens, entropies and the likeliest tokens against 64 bits: on the CPU the PyTorch implementation, on a GPU the
kernels."""
import math

import pytest
import torch

from nsa_optim_b200 import ops

BF, F32, INF = torch.bfloat16, torch.float32, math.inf


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    yield request.param
    if request.param == "cuda":
        ops.native_module().check_status()


def oracle(x, tokens, k, ignore=-100):
    """(logprob, entropy, top logprob, top index, log p, p) of a matrix in 64 bits."""
    x = x.double().cpu()
    N, V = x.shape
    m = x.amax(-1, keepdim=True)
    empty = m == -INF
    e = torch.exp(x - m.masked_fill(empty, 0.0))
    logS = e.sum(-1, keepdim=True).masked_fill(empty, 1.0).log()
    logp = torch.where(empty, x, x - m - logS)
    p = torch.where(empty, 0.0, logp.exp())
    H = -(p * logp.masked_fill(logp == -INF, 0.0)).sum(-1)
    tok = tokens.cpu()
    ok = (tok != ignore) & (tok >= 0) & (tok < V)
    chosen = torch.where(ok, logp.gather(1, tok.where(ok, 0)[:, None])[:, 0], 0.0)
    index = torch.empty(N, k, dtype=torch.long)
    for i, row in enumerate(x.tolist()):
        index[i] = torch.tensor(sorted(range(V), key=lambda j: (not math.isnan(row[j]), -row[j] if row[j] == row[j] else 0, j))[:k], dtype=torch.long)
    return chosen, H, logp.gather(1, index), index, logp, p, ok


def sums_error(V):
    """Relative error of a row's sums in 32 bits: 1/256 of the row added one by one, a few levels above, 2 units of 2^-22 for each exponential."""
    return (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -21


def near(got, want, tol):
    got = got.double().cpu()
    assert got.shape == want.shape
    fin = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~fin].nan_to_num(nan=5.0), want[~fin].nan_to_num(nan=5.0))
    bad = (got - want).abs()[fin] > tol[fin]
    assert not bad.any(), (got[fin][bad][:4], want[fin][bad][:4])


def check(x, tokens, k, ignore=-100, grads=None):
    """One call, and with `grads` its gradient, against 64 bits; x is (N, V)."""
    N, V = x.shape
    x = x.detach().requires_grad_(grads is not None)
    r = ops.token_logprobs(x, tokens, k, ignore)
    chosen, H, top, index, logp, p, ok = oracle(x.detach(), tokens, k, ignore)
    assert [t.dtype for t in r] == [F32, F32, F32, torch.int64] and torch.equal(r.top_index.cpu(), index)
    s = sums_error(V)
    near(r.logprob.detach(), chosen, s + 2.0 ** -22 * chosen.abs())
    near(r.top_logprob.detach(), top, s + 2.0 ** -22 * top.abs())
    near(r.entropy.detach(), H, s * (1 + 2 * H) + 2.0 ** -22 * H)
    if grads is None:
        return r
    g, gH, gt = grads
    outs = [(r.logprob, g), (r.entropy, gH), (r.top_logprob, gt)]
    outs = [(o, d) for o, d in outs if d is not None]
    dx, = torch.autograd.grad([o for o, _ in outs], x, [d for _, d in outs])
    want = torch.zeros(N, V, dtype=torch.double)
    size = torch.zeros(N, dtype=torch.double)
    some = ~(x.detach().cpu() == -INF).all(-1)
    if g is not None:
        want[torch.arange(N), tokens.cpu().where(ok, 0)] += torch.where(ok & some, g.double().cpu(), 0.0)
    if gt is not None:
        want.scatter_add_(1, index, torch.where(some[:, None], gt.double().cpu(), 0.0))
    direct = want.abs()
    G = want.sum(-1, keepdim=True)
    want = want - p * G
    size = p * (direct.sum(-1, keepdim=True) + G.abs())
    if gH is not None:
        lp = logp.masked_fill(logp == -INF, 0.0)
        want = want - torch.where(p > 0, gH.double().cpu()[:, None] * p * (lp + H[:, None]), 0.0)
        size = size + gH.double().cpu().abs()[:, None] * p * (lp.abs() + H[:, None] + 1)
    # a probability's relative error is that of the sums and of its exponent, |log p| * 2^-23 and the exponential's own
    rel = s + 2.0 ** -21 + 2.0 ** -22 * logp.abs().clamp(max=200)
    tol = size * (rel + 2.0 ** -22) + direct * 2.0 ** -22 * (k + 2) + want.abs() * (2.0 ** -8 if x.dtype == BF else 2.0 ** -23) + 1e-37
    assert dx.dtype == x.dtype
    near(dx, want, tol)
    return r


def logits(gen, N, V, dtype, dev, size=3.0, pitch=0):
    x = (torch.randn(N, V + pitch, generator=gen) * size).to(dtype).to(dev)
    return x[:, :V]


def tokens_of(gen, N, V, dev):
    t = torch.randint(0, V, (N,), generator=gen)
    t[::5] = -100
    return t.to(dev)


def grads_of(gen, N, k, dev):
    return tuple(torch.randn(s, generator=gen).to(dev) for s in ((N,), (N,), (N, k)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (7, 31, 5), (5, 257, 20), (2, 1000, 32), (4, 4099, 7), (2, 5000, 40), (1, 32000, 20),
                                   (3, 50257, 1), (2, 151936, 8)])
@pytest.mark.parametrize("pitch", [0, 3])
def test_sizes(dev, dtype, N, V, k, pitch):
    gen = torch.Generator().manual_seed(N * V + k)
    check(logits(gen, N, V, dtype, dev, pitch=pitch), tokens_of(gen, N, V, dev), k, grads=grads_of(gen, N, k, dev))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(148, 2049), (149, 300), (600, 1111), (1500, 128), (37, 9000)])
def test_many_rows(native, dtype, N, V):
    gen = torch.Generator().manual_seed(N)
    check(logits(gen, N, V, dtype, "cuda"), tokens_of(gen, N, V, "cuda"), 4, grads=grads_of(gen, N, 4, "cuda"))


@pytest.mark.parametrize("which", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)])
def test_each_gradient_alone(dev, which):
    gen = torch.Generator().manual_seed(1)
    g = grads_of(gen, 6, 3, dev)
    check(logits(gen, 6, 777, F32, dev), tokens_of(gen, 6, 777, dev), 3, grads=tuple(t if w else None for t, w in zip(g, which)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_equal_logits_come_in_order(dev, dtype):
    """Whole rows of one value, few values, zeros of both signs, the largest at the ends."""
    gen = torch.Generator().manual_seed(2)
    V = 3001
    x = torch.randint(-2, 3, (6, V), generator=gen).to(dtype)
    x[0] = 1.5
    x[1] = -0.0
    x[1, 5::2] = 0.0
    x[2, -1] = x[2, 0] = 7
    x[3] = torch.arange(V) / 16                                     # ascending: every logit is the best so far
    x[4] = -torch.arange(V) / 16
    check(x.to(dev), tokens_of(gen, 6, V, dev), 20, grads=grads_of(gen, 6, 20, dev))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_tokens_that_may_not_follow(dev, dtype):
    """-inf almost everywhere, everywhere, at the given token, and where fewer are left than are asked for; logits of the type's lowest value."""
    gen = torch.Generator().manual_seed(3)
    N, V = 8, 1031
    x = logits(gen, N, V, dtype, "cpu")
    x[0, 1:] = -INF
    x[1] = -INF
    x[2, 3:] = -INF
    x[3, ::2] = -INF
    low = torch.finfo(dtype).min
    x[4, 5:] = low
    x[5] = low
    x[6, :] = -INF
    x[6, 700] = low
    x[7, 100:] = -INF
    tok = torch.tensor([0, 4, 9, 2, 7, 3, 700, 50])
    check(x.to(dev), tok.to(dev), 6, grads=grads_of(gen, N, 6, dev))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_narrow_and_wide_distributions(dev, dtype):
    gen = torch.Generator().manual_seed(4)
    N, V = 7, 2000
    x = logits(gen, N, V, dtype, "cpu")
    x[0] *= 30
    x[1, 17] = 100.0
    x[2] = 0
    x[3] += 1e4
    x[4] -= 1e4
    x[5] *= 1e-3
    x[6, 3] = 30.0
    check(x.to(dev), tokens_of(gen, N, V, dev), 5, grads=grads_of(gen, N, 5, dev))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logits_that_are_not_finite(dev, dtype):
    gen = torch.Generator().manual_seed(5)
    x = logits(gen, 4, 600, dtype, "cpu")
    x[0, 77] = x[0, 99] = math.nan
    x[1, 500] = INF
    x[2, 3] = INF
    x[2, 300] = math.nan
    r = ops.token_logprobs(x.to(dev).requires_grad_(), torch.tensor([1, 500, 300, 4], device=dev), 3)
    assert r.logprob.isnan().tolist() == [True, True, True, False] == r.entropy.isnan().tolist()
    assert r.top_index[0, :2].tolist() == [77, 99] and r.top_index[1, 0] == 500 and r.top_index[2, :2].tolist() == [300, 3]
    dx, = torch.autograd.grad(r.logprob.sum(), r.logprob.grad_fn.next_functions[0][0].variable) if dev == "cuda" else (None,)
    if dx is not None:
        assert dx[:3].isnan().all() and not dx[3].isnan().any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,k", [(20011, 1), (20011, 20), (70001, 32)])
def test_few_long_rows(dev, dtype, V, k):
    """Rows that several blocks share: their likeliest tokens equal, in one part or spread over all, fewer than asked for, or not numbers."""
    gen = torch.Generator().manual_seed(8)
    x = logits(gen, 7, V, dtype, "cpu")
    x[0] = -0.0
    x[0, 3::7] = 0.0
    x[1, V - 40:] = 20.0
    x[2, ::V // 37] = 19.0
    x[3] = -INF
    x[4] = -INF
    x[4, [5, V // 2, V - 1]] = torch.tensor([1.0, 3.0, 2.0]).to(dtype)
    x[5, V // 3:] = torch.finfo(dtype).min
    x[6, :] = torch.arange(V) / 1024
    check(x.to(dev), tokens_of(gen, 7, V, dev), k, grads=grads_of(gen, 7, k, dev))
    x = logits(gen, 2, V, dtype, "cpu")
    x[0, [V - 2, 9]] = math.nan
    x[1, V // 2] = INF
    r = ops.token_logprobs(x.to(dev), torch.tensor([4, 4], device=dev), k)
    assert r.logprob.isnan().all() and r.entropy.isnan().all() and r.top_index[0, 0] == 9 and r.top_index[1, 0] == V // 2
    assert k == 1 or r.top_index[0, 1] == V - 2


def test_tokens_that_do_not_count(dev):
    gen = torch.Generator().manual_seed(6)
    x = logits(gen, 5, 100, F32, dev)
    r = check(x, torch.tensor([3, 7, 5, 7, 0], device=dev), 2, ignore=7, grads=grads_of(gen, 5, 2, dev))
    assert not r.logprob[[1, 3]].any()
    r = check(x, torch.tensor([-1, 100, 1 << 40, -(1 << 40), 99], device=dev), 2, grads=grads_of(gen, 5, 2, dev))
    assert not r.logprob[:4].any() and r.logprob[4] != 0
    if dev == "cuda":
        ops.native_module().read_status()                               # a debug build records such tokens


def test_shapes_and_strides(dev):
    gen = torch.Generator().manual_seed(7)
    x = logits(gen, 24, 130, F32, dev)
    tok = tokens_of(gen, 24, 130, dev)
    want = ops.token_logprobs(x, tok, 3)
    for a, b in ((x.view(2, 3, 4, 130), tok.view(2, 3, 4)), (x.t().contiguous().t(), tok), (x.repeat_interleave(2, 0)[::2], tok),
                 (x, torch.stack([tok, tok], 1)[:, 0])):
        got = ops.token_logprobs(a, b, 3)
        for g, w in zip(got, want):
            assert torch.allclose(g.reshape(w.shape), w, rtol=1e-6, atol=1e-6)
    one = ops.token_logprobs(x[3], tok[3], 2)
    assert one.logprob.shape == () and one.top_index.shape == (2,) and torch.allclose(one.logprob, want.logprob[3], rtol=1e-6)
    none = ops.token_logprobs(x[:0], tok[:0], 2)
    assert none.logprob.shape == (0,) and none.top_logprob.shape == (0, 2)
    leaf = x.view(2, 12, 130).transpose(0, 1).detach().requires_grad_()
    ops.token_logprobs(leaf, tok.view(2, 12).t(), 0).logprob.sum().backward()
    flat = x.detach().requires_grad_()
    ops.token_logprobs(flat, tok, 0).logprob.sum().backward()
    assert torch.allclose(leaf.grad.transpose(0, 1).reshape(24, 130), flat.grad, atol=1e-7)


def test_gradient_against_differences(dev):
    """Central differences along random directions: h = 2^-6, an error of h^2 times third derivatives (of the order of the sum of the outputs' weights)
    and of 2^-22 * 20 / h for each of 18 fp32 results."""
    gen = torch.Generator().manual_seed(8)
    N, V, k, h = 3, 60, 4, 2.0 ** -6
    x, tok = logits(gen, N, V, F32, dev, size=1.0), torch.tensor([5, -100, 59], device=dev)
    g, gH, gt = grads_of(gen, N, k, dev)
    leaf = x.detach().requires_grad_()

    def f(y):
        r = ops.token_logprobs(y, tok, k)
        return r, (r.logprob.double() * g).sum() + (r.entropy.double() * gH).sum() + (r.top_logprob.double() * gt).sum()

    r, loss = f(leaf)
    grad, = torch.autograd.grad(loss, leaf)
    for _ in range(5):
        u = torch.randn(N, V, generator=gen).to(dev) / 8
        (ra, a), (rb, b) = f(x + h * u), f(x - h * u)
        if not (torch.equal(ra.top_index, r.top_index) and torch.equal(rb.top_index, r.top_index)):
            u[r.top_index.new_tensor(range(N))[:, None], r.top_index] = 0
            (ra, a), (rb, b) = f(x + h * u * 0.01), f(x - h * u * 0.01)
            a, b = a, b
            slope, tol = (a - b) / (0.02 * h), 1.0
        else:
            slope, tol = (a - b) / (2 * h), 18 * 20 * 2.0 ** -22 / h + 20 * h * h
        assert abs(float(slope - (grad.double() * u).sum())) <= tol


def test_saved_logits_may_be_moved(dev):
    """Hooks that keep saved tensors elsewhere return them dense, whatever their pitch was."""
    gen = torch.Generator().manual_seed(9)
    x, tok = logits(gen, 5, 90, F32, dev, pitch=7), tokens_of(gen, 5, 90, dev)
    a, b = x.detach().requires_grad_(), x.detach().requires_grad_()
    ops.token_logprobs(a, tok, 2).logprob.sum().backward()
    with torch.autograd.graph.save_on_cpu():
        loss = ops.token_logprobs(b, tok, 2).logprob.sum()
    loss.backward()
    assert torch.equal(a.grad, b.grad)


@pytest.mark.gpu
def test_large_offsets(native):
    """More than 2^31 logits."""
    N, V = 14200, 151936
    x = torch.zeros(N, V, dtype=BF, device="cuda")
    tok = torch.full((N,), V - 1, device="cuda")
    x[-1, 7] = 3.0
    x[-1, V - 1] = 2.0
    r = ops.token_logprobs(x, tok, 2)
    assert r.top_index[-1].tolist() == [7, V - 1] and r.top_index[0].tolist() == [0, 1]
    S = math.exp(3) + math.exp(2) + V - 2
    assert abs(float(r.logprob[-1]) - (2 - math.log(S))) < 1e-4 and abs(float(r.logprob[5]) + math.log(V)) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(3, 151936), (700, 3001)])
def test_the_same_bits_again(native, N, V):
    gen = torch.Generator().manual_seed(10)
    x, tok = logits(gen, N, V, BF, "cuda"), tokens_of(gen, N, V, "cuda")
    first = ops.token_logprobs(x, tok, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        with torch.cuda.stream(side):
            other = ops.token_logprobs(x, tok, 8)
        again = ops.token_logprobs(x, tok, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, other, again))


@pytest.mark.parametrize("change", [dict(tokens=lambda x, t: t.int()), dict(tokens=lambda x, t: t[:2]), dict(tokens=lambda x, t: t[:, None]), dict(k=-1), dict(k=11),
                                    dict(logits=lambda x, t: x[:, :0]), dict(logits=lambda x, t: x[0, 0])])
def test_refusals(dev, change):
    x, tok = torch.zeros(3, 10, device=dev), torch.zeros(3, dtype=torch.long, device=dev)
    k = change.get("k", 2)
    a = change["logits"](x, tok) if "logits" in change else x
    t = change["tokens"](x, tok) if "tokens" in change else tok
    with pytest.raises(ValueError):
        ops.token_logprobs(a, t, k)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_entropy_gradient_beside_masked_logits(dev, dtype):
    """A token of probability 0 has no part in the gradient, however large the entropy's is: its log probability times that may be infinite."""
    gen = torch.Generator().manual_seed(12)
    x = logits(gen, 4, 300, dtype, "cpu")
    x[:, 100:] = torch.finfo(dtype).min
    g = grads_of(gen, 4, 3, dev)
    check(x.to(dev), tokens_of(gen, 4, 300, dev), 3, grads=(g[0], torch.tensor([1.5, -40.0, 1e3, 2.0], device=dev), g[2]))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", [1e7, 1e8, 1e9, 1e10, 7e12, 1e20, 1e30, 3e38])
@pytest.mark.parametrize("V", [5003, 40009])
def test_logits_far_from_zero(dev, dtype, size, V):
    """Masks of any size in whole stretches of the columns, single logits as large, rows that lie far from zero as a whole."""
    gen = torch.Generator().manual_seed(11)
    x = logits(gen, 8, V, dtype, "cpu")
    x[0, :V // 2] = -size
    x[1, V // 2:] = -size
    x[2, 700:] = -size
    x[2, :700] = -size / 2
    x[3, 4000] = size
    x[4, [3, V - 3]] = size
    x[5] = size
    x[6] = -size
    x[7] = -size
    x[7, V // 3] = 5.0
    tok = torch.tensor([V - 2, 5, 3, 4000, V - 3, 17, 18, V // 3])
    check(x.to(dev), tok.to(dev), 6, grads=grads_of(gen, 8, 6, dev))
