"""The paged 8-bit key / value cache against its definition in 64 bits: on the CPU the PyTorch implementation, on a GPU the kernels."""
import math

import pytest
import torch

from nsa_optim_b200 import ops

BF = torch.bfloat16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    yield request.param
    if request.param == "cuda":
        ops.native_module().check_status()


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------------------------ plan and release
def plan_oracle(lengths, new, table, free, count, N, P):
    """Token by token, on lists."""
    table, left, lack, start, slots, pos = [list(r) for r in table], min(max(count, 0), len(free)), 0, [0], [], []
    total = []
    for b, n in enumerate(new):
        at = max(lengths[b], 0)
        for _ in range(max(n, 0)):
            if len(slots) == N:
                break
            j, off = divmod(at, P)
            if off == 0:
                page = -1
                if j < len(table[b]) and left:
                    left -= 1
                    page = free[left]
                lack += page < 0
                if j < len(table[b]):
                    table[b][j] = page
            page = table[b][j] if j < len(table[b]) else -1
            slots.append(page * P + off if page >= 0 else -1)
            pos.append(at)
            at += 1
        start.append(len(slots))
        total.append(at)
    pad = N - len(slots)
    return start, total, slots + [-1] * pad, pos + [0] * pad, [left], [lack], table


def make_tables(lengths, W, P, gen, spare):
    """Pages in a random order: (table, free)."""
    held = [min(-(-max(n, 0) // P), W) for n in lengths]
    ids = torch.randperm(sum(held) + spare, generator=gen).tolist()
    table = []
    for n in held:
        table.append([ids.pop() for _ in range(n)] + [-1] * (W - n))
    return table, ids


PLANS = [
    ([0], [1], 1, 4, 16, 3), ([16], [0], 0, 4, 16, 3), ([15], [1], 1, 4, 16, 0), ([16], [1], 1, 4, 16, 0),     # a full page, no page left
    ([0, 5, 31], [70, 0, 2], 72, 8, 32, 9), ([3, 3, 3], [200, 1, 1], 202, 3, 16, 40),                           # a table too narrow
    ([7, 9], [5, 6], 8, 4, 16, 5), ([7, 9], [5, 6], 20, 4, 16, 5), ([-3, 4], [2, -5], 2, 4, 16, 5),              # fewer and more places than tokens
    ([100, 200, 300], [1, 400, 1], 402, 64, 256, 1), ([0] * 40, [64] * 40, 2560, 2, 64, 17),
]


@pytest.mark.parametrize("case", PLANS, ids=range(len(PLANS)))
@pytest.mark.parametrize("more", [0, 5])
def test_plan(dev, case, more):
    lengths, new, N, W, P, spare = case
    gen = torch.Generator().manual_seed(W + P)
    table, free = make_tables(lengths, W, P, gen, spare)
    count = len(free) + more                                    # a height above the stack's size is its size
    want = plan_oracle(lengths, new, table, free, count, N, P)
    t = i32(table, dev)
    got = ops.cache_plan(i32(lengths, dev), i32(new, dev), t, i32(free, dev), i32([count], dev), N, P)
    for g, w in zip((*got, t), (want[0], want[1], want[2], want[3], want[4], want[5], want[6])):
        assert g.tolist() == w
    assert got.slots.dtype == got.positions.dtype == torch.int64 and got.lengths.dtype == torch.int32


@pytest.mark.parametrize("B", [1, 33, 1024, 1025, 3000])
def test_plan_of_many_requests(dev, B):
    gen = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, 200, (B,), generator=gen).tolist()
    new = (torch.randint(0, 40, (B,), generator=gen) * (torch.rand(B, generator=gen) < 0.5)).tolist()
    table, free = make_tables(lengths, 16, 16, gen, B)
    want = plan_oracle(lengths, new, table, free, len(free), sum(new), 16)
    t = i32(table, dev)
    got = ops.cache_plan(i32(lengths, dev), i32(new, dev), t, i32(free, dev), i32([len(free)], dev), sum(new), 16)
    for g, w in zip((*got, t), want):
        assert g.tolist() == w


@pytest.mark.parametrize("B,W", [(1, 1), (5, 40), (1030, 3)])
@pytest.mark.parametrize("room", [1000000, 7])
def test_release(dev, B, W, room):
    gen = torch.Generator().manual_seed(B)
    P = 16
    lengths = torch.randint(0, 17 * W, (B,), generator=gen).tolist()
    table, free = make_tables(lengths, W, P, gen, 3)
    table[0][0] = -1                                            # a page that was never given
    done = (torch.rand(B, generator=gen) < 0.6).tolist()
    done[0] = True
    stack, want_table = free[:], [list(r) for r in table]
    for b in range(B):
        if done[b]:
            stack += [p for p in table[b][:min(W, -(-lengths[b] // P))] if p >= 0]
            want_table[b] = [-1] * W
    size = min(room, len(stack) + 4)
    f = i32((free + [-7] * len(stack))[:size], dev)
    t = i32(table, dev)
    got_len, got_count = ops.cache_release(torch.tensor(done, device=dev), i32(lengths, dev), t, f, i32([min(len(free), size)], dev), P)
    stack = stack[:size]
    assert got_len.tolist() == [0 if d else n for d, n in zip(done, lengths)] and got_count.tolist() == [len(stack)]
    assert f.tolist()[:len(stack)] == stack and t.tolist() == want_table


# ------------------------------------------------------------------------------------------------ append and values
def step_oracle(amax):
    """The smallest 2^e >= amax / 127, e in -60..60; NaN where there is none."""
    if not amax < math.inf:
        return math.nan
    e = -60
    while 127 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e if e <= 60 else math.nan


class Cache:
    """The definition: values of every page in 64 bits, and the kernels' tensors beside them."""

    def __init__(self, dev, pages, H, D, P):
        self.t = ops.cache_pages(pages, H, D, P, device=dev)
        self.v = torch.zeros(2, pages, P, H, D, dtype=torch.double)
        self.s = torch.full((pages, H, 2), 2.0 ** -60, dtype=torch.double)
        self.held = torch.zeros(pages, dtype=torch.long)          # tokens of each page: places behind them mean nothing
        self.P, self.H, self.D, self.n, self.dev = P, H, D, pages, dev

    def append(self, k, v, table, start, lengths):
        ops.cache_append(self.t, k, v, i32(table, self.dev), i32(start, self.dev), i32(lengths, self.dev))
        P = self.P
        for b in range(len(lengths)):
            lo, hi = start[b], start[b + 1]
            pos = lengths[b] - (hi - lo)
            while lo < hi:
                off = pos % P
                m = min(hi - lo, P - off)
                page = table[b][pos // P] if pos // P < len(table[b]) else -1
                if 0 <= page < self.n:
                    self.held[page] = off + m
                    for i, x in enumerate((k, v)):
                        part = x[lo:lo + m].double().cpu()
                        for h in range(self.H):
                            y = part[:, h]
                            a = math.inf if bool(y.isnan().any()) else float(y.abs().max())
                            old, step = float(self.s[page, h, i]), step_oracle(a)
                            if off:
                                step = math.nan if math.isnan(old) or math.isnan(step) else max(step, old)
                            if off and not math.isnan(step):
                                self.v[i, page, :off, h] = (self.v[i, page, :off, h] / step).round() * step
                            self.s[page, h, i] = step
                            self.v[i, page, off:off + m, h] = 0.0 if math.isnan(step) else (y / step).round() * step
                lo, pos = lo + m, pos + m

    def values(self):
        """What the pages hold: NaN where their scale is."""
        s = self.s.permute(2, 0, 1)[:, :, None, :, None]
        return torch.where(s.isnan(), torch.nan, self.v)

    def check(self):
        assert torch.equal(self.t.scale.double().cpu().nan_to_num(nan=-1.0), self.s.nan_to_num(nan=-1.0))
        ids = torch.randperm(self.n)
        got = ops.cache_values(self.t, i32(ids.tolist(), self.dev))
        want = self.values()[:, ids]
        held = torch.arange(self.P) < self.held[ids][:, None]
        for g, w in zip(got, want):
            assert g.dtype == BF and g.shape == w.shape
            assert torch.equal(g.double().cpu().nan_to_num(nan=77.0)[held], w.nan_to_num(nan=77.0)[held])


def some(gen, n, H, D, dev, wide=False, size=1.0):
    """(n, H, D) bf16, in a wider matrix where asked."""
    x = torch.randn(n, 3 * H * D + 8 if wide else H * D, generator=gen) * size
    x = x.to(BF).to(dev)
    return x[:, H * D:2 * H * D].unflatten(1, (H, D)) if wide else x.view(n, H, D)


@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("H,D", [(1, 64), (3, 128), (2, 192)])
def test_append_in_steps(dev, P, H, D):
    """Prompts, single tokens and idle requests in turn; later tokens larger and smaller than the page's; pages used again."""
    gen = torch.Generator().manual_seed(P + H)
    lengths, W = [0, 0, 0, 0], 600 // P + 3
    ids = torch.randperm(4 * W, generator=gen).tolist()
    table = [ids[i * W:(i + 1) * W] for i in range(4)]
    c = Cache(dev, 4 * W, H, D, P)
    for turn, new in enumerate([[P + 3, 0, 1, 2 * P], [1, 1, 1, 1], [1, 0, 1, 1], [P, 37, 15, 1], [0, 0, 0, 3], [1, 1, 1, 1]]):
        lengths = [a + b for a, b in zip(lengths, new)]
        start = [sum(new[:i]) for i in range(5)]
        size = [1.0, 3.7, 0.01, 130.0, 1e-20, 2.0][turn]
        c.append(some(gen, start[4], H, D, dev, turn % 2 == 0, size), some(gen, start[4], H, D, dev, turn % 2 == 1, 1 / size), table, start, lengths)
        c.check()
    c.append(some(gen, 5, H, D, dev, size=1e-3), some(gen, 5, H, D, dev), [table[0]], [0, 5], [5])          # the first request's pages again
    c.check()


def test_append_of_many_tokens(dev):
    """More tokens than are looked at one by one: several requests in a window, pages that begin inside one."""
    gen = torch.Generator().manual_seed(5)
    new = [700, 1, 0, 3, 64, 1300, 5, 1, 63, 900, 2]
    past = [10, 63, 9, 64, 0, 1, 127, 128, 1, 0, 62]
    P, H, D = 64, 2, 64
    table, _ = make_tables([a + b for a, b in zip(past, new)], 24, P, gen, 0)
    pages = 1 + max(max(r) for r in table)
    c = Cache(dev, pages, H, D, P)
    start = [sum(past[:i]) for i in range(len(past) + 1)]
    c.append(some(gen, start[-1], H, D, dev), some(gen, start[-1], H, D, dev), table, start, past)
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    c.append(some(gen, start[-1], H, D, dev, True, 2.0), some(gen, start[-1], H, D, dev), table, start, [a + b for a, b in zip(past, new)])
    c.check()


@pytest.mark.parametrize("value", [0.0, -0.0, 127.0, 127.5, 254.0, 255.0, 2.0 ** -60, 1e-38, 2.0 ** 66, 1.27 * 2.0 ** 66, 3e38, math.inf, -math.inf, math.nan])
def test_append_of_special_values(dev, value):
    P, H, D = 16, 2, 64
    c = Cache(dev, 3, H, D, P)
    gen = torch.Generator().manual_seed(3)
    x, y = some(gen, 20, H, D, dev), some(gen, 20, H, D, dev)
    x[3, 1, 7] = value
    y[18, 0, 60] = value
    c.append(x, y, [[2, 0]], [0, 20], [20])
    c.check()
    c.append(torch.zeros_like(x[:1]), torch.full_like(y[:1], value), [[2, 0]], [0, 1], [21])
    c.check()
    c.append(x[:1], y[:1], [[0, 2]], [0, 1], [1])                    # the page begins anew
    c.check()


def test_tokens_without_a_page_are_left_out(dev):
    P, H, D = 16, 1, 64
    gen = torch.Generator().manual_seed(4)
    c = Cache(dev, 4, H, D, P)
    c.append(some(gen, 60, H, D, dev), some(gen, 60, H, D, dev), [[1, -1, 3], [7, 0, 2]], [0, 50, 60], [50, 20])    # page 7 is none, a table of 48 tokens
    c.check()


def test_values_of_no_page_are_zero(dev):
    p = ops.cache_pages(2, 1, 64, 16, device=dev)
    p.k.fill_(200)
    k, v = ops.cache_values(p, i32([-1, 0, 2, 1 << 30], dev))
    assert k.shape == (4, 16, 1, 64) and not k[[0, 2, 3]].any() and k[1].all() and not v.any()


def test_nothing_to_append(dev):
    p = ops.cache_pages(2, 1, 64, 16, device=dev)
    before = [t.clone() for t in p]
    e = torch.empty(0, 1, 64, dtype=BF, device=dev)
    ops.cache_append(p, e, e, i32([[0], [1]], dev), i32([0, 0, 0], dev), i32([3, 0], dev))
    assert all(torch.equal(a, b) for a, b in zip(before, p))
    assert ops.cache_values(p, i32([], dev))[0].shape == (0, 16, 1, 64)
    assert ops.cache_attention(e, p, i32([[0], [1]], dev), i32([0, 0, 0], dev), i32([3, 0], dev)).shape == (0, 1, 64)


# ------------------------------------------------------------------------------------------------ attention
def attention_oracle(q, c, table, start, lengths, window, scale):
    """(output, largest |v| that each output's row sees) in 64 bits."""
    N, Hq, D = q.shape
    G = Hq // c.H
    vals = c.values()
    out, big = torch.zeros(N, Hq, D, dtype=torch.double), torch.zeros(N, Hq, D, dtype=torch.double)
    for b in range(len(lengths)):
        new = start[b + 1] - start[b]
        for i in range(start[b], start[b + 1]):
            pos = lengths[b] - new + i - start[b]
            keys = [(table[b][j // c.P], j % c.P) for j in range(max(0, pos - window + 1 if window else 0), pos + 1) if j // c.P < len(table[b])]
            keys = [(p, o) for p, o in keys if 0 <= p < c.n]
            if not keys:
                continue
            pg, of = (torch.tensor(x) for x in zip(*keys))
            k, v = vals[0][pg, of], vals[1][pg, of]                                         # (L, H, D)
            for h in range(Hq):
                p = torch.softmax(k[:, h // G] @ q[i, h].double().cpu() * scale, 0)
                out[i, h] = p @ v[:, h // G]
                big[i, h] = v[:, h // G].abs().amax(0)
    return out, big


def close(got, want, big):
    """bf16 results of probabilities rounded to 11 bits: half a step of the result's rounding (8 significant bits: 2^-8 of it), 2^-11 of the largest value that
    a probability multiplies, and as much again for sums and exponentials in 32 bits."""
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    bad = (got - want).abs() > want.abs() * 2.0 ** -8 + big * 2.0 ** -10 + 1e-37
    assert not bad.any(), (got[bad][:4], want[bad][:4], int(bad.sum()))


def filled(dev, gen, lengths, H, D, P, W=None, sizes=(1.0,)):
    """A cache with requests of some lengths, their tokens of different sizes in turn."""
    W = W or max(1, -(-max(lengths) // P))
    table, _ = make_tables(lengths, W, P, gen, 0)
    c = Cache(dev, max(1, 1 + max(max(r) for r in table)), H, D, P)
    start = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    k, v = (some(gen, start[-1], H, D, dev) * torch.tensor(sizes, device=dev, dtype=BF).repeat(start[-1] // len(sizes) + 1)[:start[-1], None, None]
            for _ in "kv")
    c.append(k, v, table, start, lengths)
    return c, table


def attend(c, q, table, new, lengths, window=0, scale=None, max_new=None):
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    got = ops.cache_attention(q, c.t, i32(table, c.dev), i32(start, c.dev), i32(lengths, c.dev), window=window, scale=scale,
                              max_new=max_new or max(new))
    want, big = attention_oracle(q, c, table, start, lengths, window, c.D ** -0.5 if scale is None else scale)
    close(got, want, big)
    return got


@pytest.mark.parametrize("Hq,H,D", [(1, 1, 64), (4, 2, 128), (16, 1, 128), (6, 2, 64), (40, 2, 64), (3, 3, 128)])
@pytest.mark.parametrize("P", [16, 64, 128])
def test_attention_of_single_tokens(dev, Hq, H, D, P):
    gen = torch.Generator().manual_seed(Hq + P)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 517]
    c, table = filled(dev, gen, lengths, H, D, P, sizes=(1.0, 0.2, 3.0))
    attend(c, some(gen, len(lengths), Hq, D, dev, wide=P == 64, size=2.0), table, [1] * len(lengths), lengths)


@pytest.mark.parametrize("new", [[1, 0, 3, 8], [2, 2, 2, 2], [33, 1, 0, 100], [5, 17, 64, 1]])
@pytest.mark.parametrize("window", [0, 1, 20, 64, 1000])
def test_attention_of_several_tokens(dev, new, window):
    gen = torch.Generator().manual_seed(window + sum(new))
    past, H, G, D, P = [0, 5, 200, 64], 2, 4, 64, 32
    lengths = [a + b for a, b in zip(past, new)]
    c, table = filled(dev, gen, lengths, H, D, P)
    q = some(gen, sum(new), H * G, D, dev, size=2.0)
    a = attend(c, q, table, new, lengths, window)
    b = attend(c, q, table, new, lengths, window, max_new=1)           # the hint does not matter
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * a.float().abs().max()


@pytest.mark.parametrize("L", [4096, 5001])
def test_attention_over_a_long_context(dev, L):
    gen = torch.Generator().manual_seed(L)
    c, table = filled(dev, gen, [L, 70], 1, 128, 64, sizes=(1.0, 4.0, 0.5))
    attend(c, some(gen, 2, 8, 128, dev, size=3.0), table, [1, 1], [L, 70])
    attend(c, some(gen, 7, 8, 128, dev, size=3.0), table, [4, 3], [L, 70], window=700)


def test_requests_that_see_nothing(dev):
    """No tokens at all, no page behind a table's entry, a table too narrow: zeros, or attention over what is there."""
    gen = torch.Generator().manual_seed(1)
    c, table = filled(dev, gen, [40, 40, 40], 1, 64, 16)
    table[1] = [-1, -1, -1]
    table[2] = [table[2][0], -1, 99]
    got = attend(c, some(gen, 3, 2, 64, dev), table, [1, 1, 1], [40, 40, 40])
    assert not got[1].any() and got[0].any() and got[2].any()
    assert not attend(c, some(gen, 2, 2, 64, dev), table[1:], [1, 1], [40, 0])[0].any()
    attend(c, some(gen, 2, 2, 64, dev), [r[:2] for r in table[:2]], [1, 1], [40, 33])
    got = attend(c, some(gen, 5, 2, 64, dev), [[-1, table[0][1], -1]], [5], [20], max_new=1)         # the first queries see nothing
    assert not got[0].any() and got[4].any()
    assert not attend(c, some(gen, 1, 2, 64, dev), [[-1, table[0][1], table[0][2]]], [1], [40], window=8).isnan().any()


def test_values_that_are_not_finite(dev):
    """A page without a scale reaches the queries that see it, and no others, whatever lies behind a request's length."""
    gen = torch.Generator().manual_seed(2)
    lengths = [50, 50, 50]
    table, _ = make_tables(lengths, 4, 16, gen, 0)
    for side in (0, 1):
        c = Cache(dev, 12, 2, 64, 16)
        x = [some(gen, 150, 2, 64, dev), some(gen, 150, 2, 64, dev)]
        x[side][60, 1, 5] = math.inf                                                              # request 1, page 0, head 1
        x[side][149, 0, 5] = math.nan                                                             # request 2, the last page, head 0
        c.append(*x, table, [0, 50, 100, 150], lengths)
        got = attend(c, some(gen, 3, 4, 64, dev), table, [1, 1, 1], lengths)
        assert [bool(got[b, h].isnan().any()) for b in range(3) for h in (0, 2)] == [False, False, False, True, True, False]
        attend(c, some(gen, 3, 4, 64, dev), table, [1, 1, 1], [50, 50, 40])                        # behind the length
        attend(c, some(gen, 3, 4, 64, dev), table, [1, 1, 1], lengths, window=10)                  # before the window


def test_queries_of_every_size(dev):
    """Zero, tiny, huge and non-finite queries; keys of which one dominates."""
    gen = torch.Generator().manual_seed(6)
    c, table = filled(dev, gen, [90] * 6, 1, 64, 32, sizes=(1.0, 1.0, 1.0, 30.0))
    q = some(gen, 6, 2, 64, dev)
    q[0] = 0
    q[1] *= 1e-30
    q[2] *= 300.0
    q[3, 0, 3], q[4, 1, 9] = math.nan, math.inf
    q[5, 0] = 0
    q[5, 0, :2] = torch.tensor([1e30, 1.0], dtype=BF)
    attend(c, q[:3], table[:3], [1] * 3, [90] * 3)
    got = ops.cache_attention(q, c.t, i32(table, dev), i32(list(range(7)), dev), i32([90] * 6, dev))
    nan = got.isnan().flatten(2)
    assert nan[3, 0].all() and nan[4, 1].all() and not nan[3, 1].any() and not nan[4, 0].any() and not nan[5].any()


def test_pages_of_very_different_scale(dev):
    """The page that counts may have values far smaller than those of a page that does not."""
    D, P = 64, 16
    c = Cache(dev, 3, 1, D, P)
    gen = torch.Generator().manual_seed(7)
    k, v = some(gen, 48, 1, D, dev, size=0.1), some(gen, 48, 1, D, dev)
    k[5, 0, 0] = 12.0
    v[:16] *= 1e-7
    v[16:32] = 0
    c.append(k, v, [[0, 1, 2]], [0, 48], [48])
    q = torch.zeros(1, 1, D, dtype=BF, device=dev)
    q[0, 0, 0] = 60.0                                                        # e^-90 for all tokens but the fifth
    got = ops.cache_attention(q, c.t, i32([[0, 1, 2]], dev), i32([0, 1], dev), i32([48], dev))
    want, _ = attention_oracle(q, c, [[0, 1, 2]], [0, 1], [48], 0, D ** -0.5)
    assert ((got.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + c.values()[1, 0].abs().max() * 2.0 ** -10).all()


@pytest.mark.parametrize("scale", [0.0, 0.3, -0.2])
def test_a_scale_of_ones_own(dev, scale):
    gen = torch.Generator().manual_seed(8)
    c, table = filled(dev, gen, [33, 100], 2, 64, 16)
    attend(c, some(gen, 2, 4, 64, dev), table, [1, 1], [33, 100], scale=scale)


def test_head_dim_of_192(dev):
    gen = torch.Generator().manual_seed(9)
    c, table = filled(dev, gen, [33, 100], 2, 192, 16)
    attend(c, some(gen, 3, 4, 192, dev), table, [1, 2], [33, 100])


@pytest.mark.gpu
def test_many_requests_of_one_call(native):
    gen = torch.Generator().manual_seed(10)
    lengths = torch.randint(1, 90, (700,), generator=gen).tolist()
    c, table = filled("cuda", gen, lengths, 2, 64, 16)
    attend(c, some(gen, 700, 8, 64, "cuda"), table, [1] * 700, lengths)


@pytest.mark.gpu
def test_the_same_bits_again_and_on_another_stream(native):
    gen = torch.Generator().manual_seed(11)
    lengths = [3000, 17, 900]
    c, table = filled("cuda", gen, lengths, 2, 128, 64)
    q = some(gen, 3, 32, 128, "cuda")
    args = (q, c.t, i32(table, "cuda"), i32([0, 1, 2, 3], "cuda"), i32(lengths, "cuda"))
    first = ops.cache_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(side):
            other = ops.cache_attention(*args)
        again = ops.cache_attention(*args)                             # both streams at once
        torch.cuda.synchronize()
        assert torch.equal(first, other) and torch.equal(first, again)


@pytest.mark.gpu
def test_a_captured_step(native):
    """A step in a CUDA graph: the same results when it is replayed, also with other lengths in the same tensors."""
    gen = torch.Generator().manual_seed(12)
    lengths = [2000, 130]
    c, table = filled("cuda", gen, [2100, 200], 2, 128, 64)
    q, t, start, n = some(gen, 2, 8, 128, "cuda"), i32(table, "cuda"), i32([0, 1, 2], "cuda"), i32(lengths, "cuda")
    ops.cache_attention(q, c.t, t, start, n)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.cache_attention(q, c.t, t, start, n)
    for lengths in ([2000, 130], [2100, 3], [65, 200]):
        n.copy_(i32(lengths, "cuda"))
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            want = ops.cache_attention(q, c.t, t, start, n)
            assert torch.equal(o, want)


def test_the_framework_records_no_gradient(dev):
    gen = torch.Generator().manual_seed(13)
    c, table = filled(dev, gen, [20], 1, 64, 16)
    q = some(gen, 1, 2, 64, dev).requires_grad_()
    assert not ops.cache_attention(q, c.t, i32(table, dev), i32([0, 1], dev), i32([20], dev)).requires_grad


# ------------------------------------------------------------------------------------------------ refusals
def _good(dev):
    p = ops.cache_pages(4, 2, 64, 16, device=dev)
    x = torch.zeros(3, 2, 64, dtype=BF, device=dev)
    return dict(p=p, k=x, v=x, q=torch.zeros(3, 4, 64, dtype=BF, device=dev), table=i32([[0, 1], [2, 3]], dev), start=i32([0, 1, 3], dev),
                lengths=i32([5, 6], dev), new=i32([1, 2], dev), free=i32([1], dev), count=i32([1], dev), N=3, P=16, ids=i32([0], dev), window=0,
                done=torch.tensor([True, False], device=dev))


BAD = [
    dict(table=lambda g: g["table"].long()), dict(table=lambda g: g["table"][0]), dict(table=lambda g: g["table"][:1]),
    dict(start=lambda g: g["start"][:2]), dict(start=lambda g: g["start"].long()), dict(lengths=lambda g: g["lengths"].float()),
    dict(lengths=lambda g: g["lengths"][:1]),
    dict(p=lambda g: ops.KVPages(g["p"].k, g["p"].v[:2], g["p"].scale)), dict(p=lambda g: ops.KVPages(g["p"].v, g["p"].k, g["p"].scale)),
    dict(p=lambda g: ops.KVPages(g["p"].k, g["p"].v, g["p"].scale.double())), dict(p=lambda g: ops.KVPages(g["p"].k.int(), g["p"].v, g["p"].scale)),
    dict(p=lambda g: ops.KVPages(g["p"].k, g["p"].v.transpose(3, 4).contiguous().transpose(3, 4), g["p"].scale)),
    dict(k=lambda g: g["k"][:, :1]), dict(k=lambda g: g["k"][:2]), dict(v=lambda g: g["v"].float()), dict(k=lambda g: g["k"][0], v=lambda g: g["v"][0]),
    dict(q=lambda g: g["q"][:, :3]), dict(q=lambda g: g["q"][:, :0]), dict(q=lambda g: g["q"][0]), dict(q=lambda g: g["q"][..., :32]), dict(window=lambda g: -1),
    dict(new=lambda g: g["new"].long()), dict(new=lambda g: g["new"][:1]), dict(free=lambda g: g["free"].float()), dict(count=lambda g: i32([1, 2], g["count"].device)),
    dict(N=lambda g: -1), dict(P=lambda g: 24), dict(P=lambda g: 8), dict(P=lambda g: 512), dict(ids=lambda g: g["ids"].long()), dict(ids=lambda g: g["ids"][None]),
    dict(done=lambda g: g["done"].int()), dict(done=lambda g: g["done"][:1]), dict(table=lambda g: g["table"].t()),
]
CALLS = {
    "plan": (lambda g: ops.cache_plan(g["lengths"], g["new"], g["table"], g["free"], g["count"], g["N"], g["P"]), {"lengths", "new", "table", "free", "count", "N", "P"}),
    "release": (lambda g: ops.cache_release(g["done"], g["lengths"], g["table"], g["free"], g["count"], g["P"]), {"done", "lengths", "table", "free", "count", "P"}),
    "append": (lambda g: ops.cache_append(g["p"], g["k"], g["v"], g["table"], g["start"], g["lengths"]), {"p", "k", "v", "table", "start", "lengths"}),
    "values": (lambda g: ops.cache_values(g["p"], g["ids"]), {"p", "ids"}),
    "attention": (lambda g: ops.cache_attention(g["q"], g["p"], g["table"], g["start"], g["lengths"], g["window"]), {"q", "p", "table", "start", "lengths", "window"}),
}


REFUSED = [(call, i) for call, (_, takes) in CALLS.items() for i, bad in enumerate(BAD) if set(bad) <= takes]


@pytest.mark.parametrize("call,i", REFUSED, ids=[f"{c}-{i}-{'-'.join(BAD[i])}" for c, i in REFUSED])
def test_refusals(dev, call, i):
    f, bad = CALLS[call][0], BAD[i]
    g = _good(dev)
    f(g)
    g = _good(dev)
    for name, make in bad.items():
        g[name] = make(g)
    if set(bad) == {"table"} and not g["table"].is_contiguous() and call in ("append", "attention"):
        return f(g)                                                    # read, not written: any order
    before = [t.clone() for t in g["p"]]
    with pytest.raises(ValueError):
        f(g)
    assert all(torch.equal(a, b) for a, b in zip(before, g["p"]))


@pytest.mark.parametrize("args", [(0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 32, 16), (1, 1, 100, 16), (1, 1, 64, 17), (1, 1, 64, 512)])
def test_refused_caches(dev, args):
    with pytest.raises(ValueError):
        ops.cache_pages(*args, device=dev)


@pytest.mark.gpu
def test_tensors_on_two_devices_are_refused(native):
    g = _good("cuda")
    for name in ("table", "start", "lengths"):
        with pytest.raises(ValueError):
            ops.cache_attention(g["q"], g["p"], *(t.cpu() if n == name else t for n, t in (("table", g["table"]), ("start", g["start"]), ("lengths", g["lengths"]))))
    with pytest.raises(ValueError):
        ops.cache_append(ops.KVPages(*(t.cpu() for t in g["p"])), g["k"], g["v"], g["table"], g["start"], g["lengths"])
    with pytest.raises(ValueError):
        ops.cache_plan(g["lengths"], g["new"].cpu(), g["table"], g["free"], g["count"], 3, 16)


# ------------------------------------------------------------------------------------------------ rows of no request
def poisoned(like):
    """Leaves NaN in the memory that the allocator hands out next."""
    if like.is_cuda:
        for _ in range(2):
            some = [torch.full_like(like, math.nan) for _ in range(16)]
            del some


@pytest.mark.parametrize("Hq,D", [(4, 64), (16, 128), (2, 192)])
@pytest.mark.parametrize("start", [[0, 2, 3], [5, 7, 10], [3, 3, 3]])
def test_queries_of_no_request_get_zeros(dev, Hq, D, start):
    """More places than tokens, as in a step of a fixed size, and requests out of the middle of a packed step."""
    gen = torch.Generator().manual_seed(14)
    lengths = [40, 70]
    c, table = filled(dev, gen, lengths, 1, D, 16)
    q = some(gen, 12, Hq, D, dev)
    args = (c.t, i32(table, dev), i32(start, dev), i32(lengths, dev))
    poisoned(q)
    got = ops.cache_attention(q, *args)
    close(got, *attention_oracle(q, c, table, start, lengths, 0, D ** -0.5))
    assert not got[:start[0]].any() and not got[start[2]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [768, 769, 1600])
def test_requests_of_several_launches(native, B):
    """More requests than one launch takes, of one to three new tokens or none, with places of nobody before and behind them."""
    gen = torch.Generator().manual_seed(B)
    new = torch.randint(0, 4, (B,), generator=gen).tolist()
    lengths = [n + p for n, p in zip(new, torch.randint(0, 60, (B,), generator=gen).tolist())]
    c, table = filled("cuda", gen, [max(n, 1) for n in lengths], 1, 64, 16)
    start = [3 + sum(new[:i]) for i in range(B + 1)]
    q = some(gen, start[-1] + 4, 2, 64, "cuda")
    args = (c.t, i32(table, "cuda"), i32(start, "cuda"), i32(lengths, "cuda"))
    poisoned(q)
    got = ops.cache_attention(q, *args, max_new=3)
    close(got, *attention_oracle(q, c, table, start, lengths, 0, 0.125))
    assert not got[:3].any() and not got[start[-1]:].any()


@pytest.mark.parametrize("before", [1, 5, 40, 2100])
def test_tokens_of_no_request_are_left_out(dev, before):
    """Requests out of the middle of a packed step: rows before the first one's and behind the last one's are not theirs."""
    gen = torch.Generator().manual_seed(before)
    past, new, P = [40, 0, 20], [3, 0, 40], 16
    total = [a + b for a, b in zip(past, new)]
    table, _ = make_tables(total, 5, P, gen, 0)
    c = Cache(dev, 1 + max(max(r) for r in table), 2, 64, P)
    at = [0, 40, 40, 60]
    c.append(some(gen, 60, 2, 64, dev), some(gen, 60, 2, 64, dev), table, at, past)
    start = [before, before + 3, before + 3, before + 43]
    rows = start[-1] + 7
    c.append(some(gen, rows, 2, 64, dev, size=2.0), some(gen, rows, 2, 64, dev, size=0.5), table, start, total)
    c.check()


# ------------------------------------------------------------------------------------------------ probabilities and scores of any size
@pytest.mark.parametrize("size", [1e4, 1e6, 1e7, 1e8, 1e9, 1e20, 1e30])
@pytest.mark.parametrize("sign", [1, -1, 0])
def test_scores_far_from_zero(dev, size, sign):
    """Finite scores of any size, all positive, all negative or both.  Queries are drawn until the largest score stands out by more than fp32 can lose: it takes
    all of the probability."""
    gen = torch.Generator().manual_seed(15)
    lengths, D, P = [90, 33, 5], 64, 16
    table, _ = make_tables(lengths, 6, P, gen, 0)
    c = Cache(dev, 1 + max(max(r) for r in table), 1, D, P)
    k, v = some(gen, 128, 1, D, dev), some(gen, 128, 1, D, dev)
    c.append(k.abs() if sign else k, v, table, [0, 90, 123, 128], lengths)
    q = torch.empty(5, 4, D, dtype=BF)
    for i, (b, keys) in enumerate(((0, 90), (1, 31), (1, 32), (1, 33), (2, 5))):
        pages = torch.tensor([table[b][j // P] for j in range(keys)])
        seen = c.values()[0][pages, torch.arange(keys) % P, 0]
        for h in range(4):
            stands_out = False
            while not stands_out:
                q[i, h] = (torch.randn(D, generator=gen).abs() * sign if sign else torch.randn(D, generator=gen)) * size
                x = seen @ q[i, h].double()
                gap = -x.topk(2).values.diff().item()
                stands_out = gap > x.abs().max() * 2.0 ** -10 and gap / 8 > 50
    for most in (1, 3):
        attend(c, q.to(dev), table, [1, 3, 1], lengths, max_new=most)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq", [8, 16])
def test_a_token_that_takes_nearly_all(native, Hq):
    """65536 keys; the first takes 99.7 % of the probability and has the value 0, so that the output is the sum of what is left, 2^-24 of the largest each.  As many
    row tiles as the kernel has workers (8 per SM), so that one of them walks a whole context.  The other values are all 1: errors are relative, 2^-8
    of the result's rounding, 2^-11 of the probabilities', as much again for sums and exponentials."""
    P, D, L = 64, 64, 65536
    n = 8 * torch.cuda.get_device_properties(0).multi_processor_count
    k, v = torch.zeros(L, 1, D, dtype=BF, device="cuda"), torch.ones(L, 1, D, dtype=BF, device="cuda")
    k[0, 0, 0], v[0] = 8.0, 0.0
    t, table = ops.cache_pages(L // P, 1, D, P, device="cuda"), torch.arange(L // P, dtype=torch.int32, device="cuda")[None]
    ops.cache_append(t, k, v, table, i32([0, L], "cuda"), i32([L], "cuda"))
    q = torch.zeros(n, Hq, D, dtype=BF, device="cuda")
    q[:, :, 0] = 16.875                                                # e^16.875 with the first key, 1 with the others
    got = ops.cache_attention(q, t, table, i32([0, n], "cuda"), i32([L], "cuda")).double().cpu()
    others = torch.arange(L - n, L, dtype=torch.double)
    want = (others / (others + math.exp(16.875)))[:, None, None]
    assert ((got - want).abs() <= want * (2.0 ** -8 + 2.0 ** -10)).all(), (got[0, 0, 0], want[0], got[-1, -1, -1], want[-1])


@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 40, 2 ** 31 - 1, 2 ** 40])
def test_windows_that_hold_everything(dev, window):
    """The largest windows, also where a request is given more queries than it has tokens: the first of them see nothing."""
    gen = torch.Generator().manual_seed(16)
    lengths, new = [5, 70, 20], [9, 3, 30]
    c, table = filled(dev, gen, lengths, 2, 64, 16)
    got = attend(c, some(gen, 42, 8, 64, dev), table, new, lengths, window)
    assert not got[:4].any() and got[4:12].flatten(1).any(1).all() and not got[12:22].any() and got[22:].flatten(1).any(1).all()
