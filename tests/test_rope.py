"""Rotary positions of queries and keys against complex numbers in 64 bits: on the CPU the PyTorch implementation, on a GPU the kernel."""
import pytest
import torch

from nsa_optim_b200 import ops

BF = torch.bfloat16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    yield request.param
    if request.param == "cuda":
        ops.native_module().check_status()


def tables(R, L, dev, theta=1e4):
    a = torch.arange(L, dtype=torch.double)[:, None] * theta ** (-torch.arange(0, R, 2, dtype=torch.double) / R)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def turned(x, cos, sin, interleaved):
    """x (B, T, H, D) in 64 bits times unit numbers, rows (T, R/2) or (B, T, R/2), and the size of what is summed."""
    x, R = x.double(), 2 * cos.shape[-1]
    z = torch.complex(cos.double(), sin.double())
    z = (z[None] if z.dim() == 2 else z)[:, :, None]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    w = torch.complex(a, b) * z
    y, size = x.clone(), x.abs()
    parts = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., parts[0]], y[..., parts[1]] = w.real, w.imag
    size[..., parts[0]] = size[..., parts[1]] = a.abs() + b.abs()
    return y, size


def near(got, want, size):
    """A rounding to the type, half a step, and two products and a sum in fp32: three half steps of their size, and as much for the tables' product."""
    assert got.shape == want.shape
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() * 1.001 + 4 * 2.0 ** -24 * size
    assert bool(((got.double() - want).abs() <= tol).all())


SHAPES = [  # B, T, Hq, Hk, D, R
    (1, 1, 1, 1, 64, 64), (2, 7, 4, 2, 64, 32), (1, 33, 3, 1, 128, 128), (3, 5, 2, 2, 128, 32), (1, 9, 2, 1, 256, 192), (2, 3, 5, 1, 24, 8),
    (1, 4, 2, 2, 7, 6), (1, 6, 1, 3, 80, 2), (2, 300, 16, 8, 64, 64), (1, 513, 32, 2, 128, 128), (1, 2, 1, 1, 2, 2), (2, 5, 3, 3, 32, 16),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both_directions(dev, shape, dtype, interleaved):
    B, T, Hq, Hk, D, R = shape
    cos, sin = tables(R, T + 3, dev)
    q, k, dq, dk = (torch.randn(B, T, h, D, device=dev).to(dtype) for h in (Hq, Hk, Hq, Hk))
    q.requires_grad_(), k.requires_grad_()
    yq, yk = ops.rope_qk(q, k, cos, sin, interleaved=interleaved)
    for y, x in ((yq, q), (yk, k)):
        assert y.dtype == dtype and y.is_contiguous()
        near(y.detach(), *turned(x.detach(), cos[:T], sin[:T], interleaved))
        assert torch.equal(y.detach()[..., R:], x.detach()[..., R:])
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for g, d in ((gq, dq), (gk, dk)):
        near(g, *turned(d, cos[:T], -sin[:T], interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,Hq,Hk", [(601, 600, 2, 1), (1300, 1280, 1, 2), (4800, 16, 1, 1), (16, 16, 300, 40), (3, 2, 500, 100)])
def test_wide_heads_and_many(dev, D, R, Hq, Hk, interleaved):
    """A token that is more than one block's work, in both directions, with gradients that are one number repeated."""
    cos, sin = tables(R, 9, dev)
    for dtype in (BF, torch.float32):
        q, k = (torch.randn(2, 5, h, D, device=dev).to(dtype).requires_grad_() for h in (Hq, Hk))
        yq, yk = ops.rope_qk(q, k, cos, sin, interleaved=interleaved)
        one = torch.randn(1, 1, 1, D, device=dev).to(dtype)
        gq, gk = torch.autograd.grad((yq, yk), (q, k), (one.expand_as(q), one.expand_as(k)))
        for y, g, x in ((yq, gq, q), (yk, gk, k)):
            near(y.detach(), *turned(x.detach(), cos[:5], sin[:5], interleaved))
            near(g, *turned(one.expand_as(x), cos[:5], -sin[:5], interleaved))


@pytest.mark.parametrize("D,R", [(64, 64), (128, 32), (10, 4)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("each", [False, True])
def test_positions(dev, D, R, itype, each):
    B, T, L = 3, 11, 50
    cos, sin = tables(R, L, dev)
    at = torch.randint(0, L, (B, T) if each else (T,), device=dev).to(itype)
    q, k = torch.randn(B, T, 4, D, device=dev).to(BF), torch.randn(B, T, 1, D, device=dev).to(BF)
    for y, x in zip(ops.rope_qk(q, k, cos, sin, at), (q, k)):
        near(y, *turned(x, cos[at.long()], sin[at.long()], False))


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_outside_the_tables(dev, interleaved):
    cos, sin = tables(32, 8, dev)
    q, k = torch.randn(1, 5, 2, 64, device=dev).to(BF), torch.randn(1, 5, 2, 64, device=dev).to(BF)
    at = torch.tensor([7, 8, -1, 2 ** 31 - 1, 0], device=dev)
    out = torch.tensor([False, True, True, True, False], device=dev)
    for y, x in zip(ops.rope_qk(q, k, cos, sin, at, interleaved), (q, k)):
        assert bool(y[:, out, :, :32].isnan().all()) and not bool(y[:, ~out].isnan().any()) and torch.equal(y[..., 32:], x[..., 32:])
    for y in ops.rope_qk(q, k, cos[:0], sin[:0], interleaved=interleaved):
        assert bool(y[..., :32].isnan().all())
    y = ops.rope_qk(q, k, cos[:3], sin[:3], interleaved=interleaved)[0]              # without positions token t takes row t
    assert bool(y[:, 3:, :, :32].isnan().all()) and not bool(y[:, :3].isnan().any())


def test_strides_and_places(dev):
    """Slices of a fused projection, heads in front of tokens, an odd first column, one head for all: views are read where they are."""
    cos, sin = tables(64, 20, dev)
    both = torch.randn(2, 20, 8, 64, device=dev).to(BF)
    views = [(both[:, :, :4], both[:, :, 4:6]), (both.transpose(1, 2).contiguous().transpose(1, 2), both[:, :, ::2]),
             (torch.randn(2, 20, 3, 65, device=dev).to(BF)[..., 1:], torch.randn(2, 40, 3, 66, device=dev).to(BF)[:, ::2, :, 1:65]),
             (both[:, :, :1].expand(-1, -1, 6, -1), both[:1].expand(2, -1, -1, -1)), (both.flip(0), both[..., :1].expand(-1, -1, -1, 64))]
    for q, k in views:
        for y, x in zip(ops.rope_qk(q, k, cos, sin), (q, k)):
            near(y, *turned(x, cos, sin, False))


def test_empty(dev):
    cos, sin = tables(64, 20, dev)
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64), (2, 5, 0, 64)):
        q = torch.randn(shape, device=dev).to(BF)
        k = torch.randn(*shape[:2], 1, 64, device=dev).to(BF)
        yq, yk = ops.rope_qk(q, k, cos, sin)
        assert yq.shape == q.shape and yk.shape == k.shape
        near(yk, *turned(k, cos[:shape[1]], sin[:shape[1]], False))


@pytest.mark.parametrize("D", [64, 128])
def test_whole_heads_are_the_same_as_rope(dev, D):
    cos, sin = tables(D, 70, dev)
    q, k = torch.randn(2, 70, 6, D, device=dev).to(BF), torch.randn(2, 70, 2, D, device=dev).to(BF)
    yq, yk = ops.rope_qk(q, k, cos, sin)
    assert torch.equal(yq, ops.rope(q, cos, sin)) and torch.equal(yk, ops.rope(k, cos, sin))


def test_gradient_is_the_transpose(dev):
    """The turn is linear: its change along v, seen by g, is the gradient's along v.  Sums of 2 x 9 x 3 x 32 products of numbers about 1, each off by half a
    step of fp32 at most three times over on either side, size 2 with both of a pair: 4 * 2^-24 * sum |g| (|v_a| + |v_b|)."""
    cos, sin = tables(16, 9, dev)
    q = torch.randn(2, 9, 3, 32, device=dev, requires_grad=True)
    k = torch.randn(2, 9, 1, 32, device=dev, requires_grad=True)
    for interleaved in (False, True):
        v, g = torch.randn_like(q), torch.randn_like(q)
        y, _ = ops.rope_qk(q, k, cos, sin, interleaved=interleaved)
        dq, dk = torch.autograd.grad(y, (q, k), g, allow_unused=True)
        assert dk is None or not bool(dk.any())                                  # only the queries were used
        with torch.no_grad():
            along = (ops.rope_qk(v, k, cos, sin, interleaved=interleaved)[0].double() * g).sum()
        size = float((turned(v, cos, sin, interleaved)[1] * g.abs()).sum())
        assert abs(float(along - (dq.double() * v).sum())) <= 8 * 2.0 ** -24 * size


def test_gradient_by_differences():
    cos, sin = tables(6, 4, "cpu")
    q = torch.randn(1, 4, 2, 8, dtype=torch.double, requires_grad=True)
    k = torch.randn(1, 4, 1, 8, dtype=torch.double, requires_grad=True)
    # fp32 inside: steps of 1/64 leave 2^-24 * 64 of a difference's rounding
    for interleaved in (False, True):
        assert torch.autograd.gradcheck(lambda a, b: ops.rope_qk(a, b, cos, sin, None, interleaved), (q, k), eps=2.0 ** -6, atol=1e-4)


def test_refusals(dev):
    cos, sin = tables(64, 20, dev)
    q, k = torch.randn(2, 5, 4, 64, device=dev).to(BF), torch.randn(2, 5, 2, 64, device=dev).to(BF)
    for bad in (lambda: ops.rope_qk(q[0], k[0], cos, sin), lambda: ops.rope_qk(q, k[:, :4], cos, sin), lambda: ops.rope_qk(q, k[..., :32], cos, sin),
                lambda: ops.rope_qk(q, k.float(), cos, sin), lambda: ops.rope_qk(q[..., :32], k[..., :32], cos, sin),
                lambda: ops.rope_qk(q, k, cos[:, :0], sin[:, :0]), lambda: ops.rope_qk(q, k, cos, sin[:, :8]), lambda: ops.rope_qk(q, k, cos[0], sin[0]),
                lambda: ops.rope_qk(q, k, cos.long(), sin.long()), lambda: ops.rope_qk(q, k, cos, sin, torch.zeros(4, dtype=torch.long, device=dev)),
                lambda: ops.rope_qk(q, k, cos, sin, torch.zeros(5, device=dev)), lambda: ops.rope_qk(q, k, cos, sin, torch.zeros(5, 2, dtype=torch.long, device=dev))):
        with pytest.raises(ValueError):
            bad()


def test_refusals_with_gradients_of_the_tables(dev):
    """The same calls are refused where the tables want a gradient."""
    cos, sin = (t.requires_grad_() for t in tables(64, 20, dev))
    q, k = torch.randn(2, 5, 4, 64, device=dev).to(BF), torch.randn(2, 5, 2, 64, device=dev).to(BF)
    for bad in (dict(positions=torch.zeros(5, device=dev)), dict(positions=torch.zeros(1, dtype=torch.long, device=dev)), dict(k=k.float()), dict(k=k[:1]),
                dict(q=q[..., :32], k=k[..., :32]), dict(positions=torch.zeros(5, dtype=torch.bool, device=dev))):
        with pytest.raises(ValueError):
            ops.rope_qk(**{**dict(q=q, k=k, cos=cos, sin=sin), **bad})
    ops.rope_qk(q, k, cos, sin)[0].float().sum().backward()
    assert bool(torch.isfinite(cos.grad[:5]).all()) and not bool(cos.grad[5:].any())


@pytest.mark.gpu
def test_many_tokens():
    """More tokens than one pass of the grid has threads for: each CTA takes several turns."""
    cos, sin = tables(128, 40000, "cuda")
    q, k = torch.randn(1, 40000, 17, 128, device="cuda").to(BF), torch.randn(1, 40000, 2, 128, device="cuda").to(BF)
    for interleaved in (False, True):
        for y, x in zip(ops.rope_qk(q, k, cos, sin, interleaved=interleaved), (q, k)):
            near(y, *turned(x, cos, sin, interleaved))


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    cos, sin = tables(64, 20, "cuda")
    q, k = torch.randn(2, 20, 4, 64, device="cuda").to(BF), torch.randn(2, 20, 2, 64, device="cuda").to(BF)
    want = ops.rope_qk(q, k, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rope_qk(q, k, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rope_qk(q, k, cos, sin)
    q.copy_(torch.randn_like(q))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, ops.rope_qk(q, k, cos, sin)))
