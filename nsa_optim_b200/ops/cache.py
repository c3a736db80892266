"""A paged key / value cache in 8 bits: its layout, and its ops in PyTorch (any device).

The pages of a layer are three tensors (:class:`KVPages`).  A page holds P tokens (a power of two, 16 to 256) of every KV head:

  * ``k`` uint8 (pages, Hkv, P/2, D/64, 2, 64): token 2i+e, columns 64j .. 64j+63 at [page, head, i, j, e];
  * ``v`` uint8 (pages, Hkv, P/16, D, 16): 16 tokens of a column side by side;
  * ``scale`` fp32 (pages, Hkv, 2): steps of the keys and of the values.

A code u stands for (u - 128) * scale.  The scale of a page, head and side is the smallest power of two 2^e, e in -60 .. 60, of which no
value in the page needs more than 127; it never falls while the page is in use.  A power of two makes every code's value a bf16
number, and lets a later, larger token raise the scale without a second rounding error of its own kind: the codes that are there
are shifted (half to even).  Values that are not finite, or larger than 127 * 2^60, make the page's scale NaN, and so the attention of the
queries that see it, instead of being clipped silently.  The orders of ``k`` and ``v`` are those in which a warp of the attention kernel feeds its
matrix instructions, so that a lane's 16 bytes are one load and nothing is transposed on the way.

Requests share the pages: ``table`` (B, W) int32 lists the pages of each request in order, ``free`` int32 and ``free_count`` (1) are a stack
of the pages that nobody holds.  The new tokens of a step are packed one request after another, N in all; ``query_start`` (B + 1) int32 says
where each begins, ``lengths`` (B) int32 how many tokens it has in the cache with them.

A request holds the pages of its first ceil(lengths / P) entries of ``table``; entries behind them count as empty, whatever is in them.  So who lowers a length
(drafted tokens that were rejected) gives the pages behind it back first, as ``generation.PagedCache.take_back`` does.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

MIN_EXP, MAX_EXP = -60, 60


class KVPages(NamedTuple):
    """Keys and values of one layer (see the module)."""
    k: Tensor
    v: Tensor
    scale: Tensor

    @property
    def page_size(self) -> int:
        return 2 * self.k.shape[2]


class CachePlan(NamedTuple):
    """Where the tokens of a step go: ``slots`` (N) int64 are page * P + offset (-1: no page), ``positions`` (N) int64 their places in the request
    (0 behind the last token), ``free_count`` the stack's new height, ``shortfall`` (1) how many pages were needed and not there."""
    query_start: Tensor
    lengths: Tensor
    slots: Tensor
    positions: Tensor
    free_count: Tensor
    shortfall: Tensor


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def new_pages(pages: int, heads: int, head_dim: int, page_size: int, device=None) -> KVPages:
    """Empty pages of one layer."""
    _need(pages > 0 and heads > 0, "a cache needs pages and heads")
    _need(head_dim > 0 and head_dim % 64 == 0, "a cache needs a head_dim that is a multiple of 64")
    _check_page_size(page_size)
    return KVPages(torch.full((pages, heads, page_size // 2, head_dim // 64, 2, 64), 128, dtype=torch.uint8, device=device),
                   torch.full((pages, heads, page_size // 16, head_dim, 16), 128, dtype=torch.uint8, device=device),
                   torch.full((pages, heads, 2), 2.0 ** MIN_EXP, device=device))


def _check_page_size(P: int) -> None:
    _need(16 <= P <= 256 and P & (P - 1) == 0, f"a page holds a power of two of 16 to 256 tokens, got {P}")


def _check_pages(p: KVPages) -> Tuple[int, int, int, int]:
    _need(p.k.dim() == 6 and p.v.dim() == 5 and p.scale.dim() == 3, "expected the three tensors of a KVPages")
    n, H, P2, J = p.k.shape[:4]
    P, D = 2 * P2, 64 * J
    _check_page_size(P)
    _need(tuple(p.k.shape[4:]) == (2, 64) and tuple(p.v.shape) == (n, H, P // 16, D, 16) and tuple(p.scale.shape) == (n, H, 2),
          "the shapes of a KVPages do not belong together")
    _need(p.k.dtype == torch.uint8 and p.v.dtype == torch.uint8 and p.scale.dtype == torch.float32, "a KVPages is uint8, uint8 and float32")
    _need(p.k.is_contiguous() and p.v.is_contiguous() and p.scale.is_contiguous(), "the tensors of a KVPages have to be contiguous")
    return n, H, P, D


def _check_i32(t: Tensor, dims: int, what: str) -> None:
    _need(t.dim() == dims and t.dtype == torch.int32, f"{what} has to be an int32 tensor of {dims} dimension(s)")


def _check_step(table: Tensor, query_start: Tensor, lengths: Tensor) -> int:
    _check_i32(table, 2, "table")
    _check_i32(query_start, 1, "query_start")
    _check_i32(lengths, 1, "lengths")
    B = lengths.shape[0]
    _need(B > 0 and table.shape[0] == B and query_start.shape[0] == B + 1, "table, query_start and lengths have to be of the same requests")
    return B


# ------------------------------------------------------------------ pages and slots of a step
def plan(lengths: Tensor, new: Tensor, table: Tensor, free: Tensor, free_count: Tensor, num_tokens: int, page_size: int) -> CachePlan:
    for t, d, what in ((lengths, 1, "lengths"), (new, 1, "new"), (table, 2, "table"), (free, 1, "free"), (free_count, 1, "free_count")):
        _check_i32(t, d, what)
    _check_page_size(page_size)
    B, W = table.shape
    _need(B > 0 and W > 0 and lengths.shape[0] == B and new.shape[0] == B, "lengths, new and table have to be of the same requests")
    _need(free_count.shape[0] == 1 and num_tokens >= 0, "free_count has one element, num_tokens is not negative")
    _need(table.is_contiguous(), "table has to be contiguous: it is changed in place")
    dev, P = lengths.device, page_size
    ends = new.clamp(min=0).cumsum(0).clamp(max=num_tokens)
    start = torch.nn.functional.pad(ends, (1, 0)).to(torch.int32)
    past = lengths.clamp(min=0)
    total = past + (start[1:] - start[:-1])
    held, need = (past + P - 1) // P, (total + P - 1) // P
    take = need.clamp(max=W) - held.clamp(max=W)
    first = torch.nn.functional.pad(take.cumsum(0), (1, 0))
    at = torch.arange(W, device=dev)
    fresh = (at >= held[:, None]) & (at < need[:, None])
    order = (first[:-1, None] + at - held[:, None])[fresh]
    count = free_count.clamp(0, free.shape[0])
    if free.shape[0]:
        table[fresh] = torch.where(order < count, free[(count - 1 - order).clamp(min=0)], -1).to(torch.int32)
    else:
        table[fresh] = -1
    i = torch.arange(num_tokens, device=dev)
    b = torch.searchsorted(start[1:].contiguous(), i.to(torch.int32), right=True)
    there = b < B
    b = b.clamp(max=B - 1)
    pos = torch.where(there, past[b].long() + i - start[b], 0)
    page = torch.where(there & (pos // P < W), table[b, (pos // P).clamp(max=W - 1)], -1)
    slots = torch.where(page >= 0, page.long() * P + pos % P, -1)
    got = torch.minimum(first[-1:], count)
    lacking = (need - held).sum().view(1) - got
    return CachePlan(start, total.to(torch.int32), slots, pos, (count - got).to(torch.int32), lacking.to(torch.int32))


def release(finished: Tensor, lengths: Tensor, table: Tensor, free: Tensor, free_count: Tensor, page_size: int) -> Tuple[Tensor, Tensor]:
    for t, d, what in ((lengths, 1, "lengths"), (table, 2, "table"), (free, 1, "free"), (free_count, 1, "free_count")):
        _check_i32(t, d, what)
    _check_page_size(page_size)
    B, W = table.shape
    _need(finished.dtype == torch.bool and tuple(finished.shape) == (B,) and lengths.shape[0] == B and free_count.shape[0] == 1,
          "finished is a truth value for each request, free_count has one element")
    _need(table.is_contiguous() and free.is_contiguous(), "table and free have to be contiguous: they are changed in place")
    at = torch.arange(W, device=lengths.device)
    mine = finished[:, None] & (at < ((lengths + page_size - 1) // page_size)[:, None]) & (table >= 0)
    pages = table[mine]
    count = free_count.clamp(0, free.shape[0])
    place = count + torch.arange(pages.numel(), device=lengths.device)
    ok = place < free.shape[0]
    free[place[ok]] = pages[ok]
    table[finished] = -1
    return torch.where(finished, 0, lengths), (count + ok.sum()).to(torch.int32)


# ------------------------------------------------------------------ values in and out
def _codes(p: KVPages, ids: Tensor) -> Tuple[Tensor, Tensor]:
    """(n, P, Hkv, D) codes of the keys and of the values of some pages, as fp32 whole numbers."""
    n, H, P, D = ids.numel(), p.k.shape[1], p.page_size, p.v.shape[3]
    k = p.k[ids].permute(0, 2, 4, 1, 3, 5).reshape(n, P, H, D)
    v = p.v[ids].permute(0, 2, 4, 1, 3).reshape(n, P, H, D)
    return k.float() - 128, v.float() - 128


def _store(p: KVPages, ids: Tensor, k: Tensor, v: Tensor) -> None:
    n, P, H, D = k.shape
    p.k[ids] = (k + 128).to(torch.uint8).view(n, P // 2, 2, H, D // 64, 64).permute(0, 3, 1, 4, 2, 5)
    p.v[ids] = (v + 128).to(torch.uint8).view(n, P // 16, 16, H, D).permute(0, 3, 1, 4, 2)


def step_of(amax: Tensor) -> Tensor:
    """The scale for values up to ``amax`` (not negative), NaN where there is none."""
    m, e = torch.frexp(amax.float())
    e = torch.where(m > 127 / 128, e - 6, e - 7)
    step = torch.ldexp(torch.ones_like(m), e.clamp(MIN_EXP, MAX_EXP))
    step = torch.where(amax > 0, step, 2.0 ** MIN_EXP)
    return torch.where(torch.isfinite(amax) & ((e <= MAX_EXP) | (amax == 0)), step, float("nan"))


def _check_new(p: KVPages, k: Tensor, v: Tensor) -> Tuple[int, int, int, int]:
    n, H, P, D = _check_pages(p)
    _need(k.dim() == 3 and k.shape == v.shape and tuple(k.shape[1:]) == (H, D) and k.dtype == v.dtype,
          f"keys and values have to be (tokens, {H}, {D}) and of one type, got {tuple(k.shape)} and {tuple(v.shape)}")
    return n, H, P, D


def append(p: KVPages, k: Tensor, v: Tensor, table: Tensor, query_start: Tensor, lengths: Tensor) -> None:
    n, H, P, D = _check_new(p, k, v)
    B = _check_step(table, query_start, lengths)
    start, total, W = query_start.tolist(), lengths.tolist(), table.shape[1]
    for b in range(B):
        lo, hi = min(start[b], k.shape[0]), min(start[b + 1], k.shape[0])
        pos = total[b] - (start[b + 1] - start[b])
        while lo < hi:
            off = pos % P
            m = min(hi - lo, P - off)
            page = int(table[b, pos // P]) if 0 <= pos // P < W else -1
            if 0 <= page < n:
                ids = torch.tensor([page], device=k.device)
                codes, scale = list(_codes(p, ids)), p.scale[page].clone()
                for i, x in enumerate((k, v)):
                    part = x[lo:lo + m].float()
                    step = step_of(torch.where(torch.isnan(part), float("inf"), part.abs()).amax((0, 2)))
                    if off:
                        step = torch.where(torch.isnan(scale[:, i]), scale[:, i], torch.where(step < scale[:, i], scale[:, i], step))
                        ratio = scale[:, i] / step
                        old = codes[i][0, :off]
                        codes[i][0, :off] = torch.where(torch.isnan(ratio)[:, None], old, (old * ratio[:, None]).round())
                    codes[i][0, off:off + m] = torch.where(torch.isnan(step)[:, None], 0.0, (part / step[:, None]).round())
                    p.scale[page, :, i] = step
                _store(p, ids, *codes)
            lo, pos = lo + m, pos + m


def values(p: KVPages, ids: Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
    n = _check_pages(p)[0]
    _check_i32(ids, 1, "ids")
    inside = (ids >= 0) & (ids < n)
    at = torch.where(inside, ids, 0).long()
    out = []
    for i, c in enumerate(_codes(p, at)):
        x = c * p.scale[at, :, i][:, None, :, None]
        out.append(torch.where(inside[:, None, None, None], x, 0.0).to(dtype))
    return out[0], out[1]


# ------------------------------------------------------------------ attention
def _check_queries(q: Tensor, p: KVPages, table: Tensor, query_start: Tensor, lengths: Tensor, window: int) -> Tuple[int, int, int, int]:
    n, H, P, D = _check_pages(p)
    _check_step(table, query_start, lengths)
    _need(q.dim() == 3 and q.shape[2] == D and q.shape[1] > 0 and q.shape[1] % H == 0,
          f"queries have to be (tokens, a multiple of {H} heads, {D}), got {tuple(q.shape)}")
    _need(window >= 0, "window has to be 0 (none) or more")
    return n, H, P, D


def attention(q: Tensor, p: KVPages, table: Tensor, query_start: Tensor, lengths: Tensor, window: int = 0,
              scale: Optional[float] = None) -> Tensor:
    n, H, P, D = _check_queries(q, p, table, query_start, lengths, window)
    N, Hq = q.shape[:2]
    G, scale = Hq // H, D ** -0.5 if scale is None else scale
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    start, total, W = query_start.tolist(), lengths.tolist(), table.shape[1]
    for b in range(len(total)):
        lo, hi, L = min(start[b], N), min(start[b + 1], N), total[b]
        if hi <= lo or L <= 0:
            continue
        ids = table[b, :min(W, -(-L // P))]
        k, v = (x.flatten(0, 1)[:L] for x in values(p, ids, torch.float32))
        at = torch.arange(k.shape[0], device=q.device)
        own = L - (start[b + 1] - start[b]) + torch.arange(hi - lo, device=q.device)
        seen = (at <= own[:, None]) & ((ids >= 0) & (ids < n)).repeat_interleave(P)[:k.shape[0]]
        if window:
            seen &= at > own[:, None] - window
        x = torch.einsum("thgd,lhd->htgl", q[lo:hi].float().view(hi - lo, H, G, D), k) * scale
        x = x.masked_fill(~seen[None, :, None], float("-inf"))
        pr = torch.softmax(x, -1).masked_fill(~seen[None, :, None], 0.0)
        v = v.masked_fill(~seen.any(0)[:, None, None], 0.0)
        out[lo:hi] = torch.einsum("htgl,lhd->thgd", pr, v).reshape(hi - lo, Hq, D).to(q.dtype)
    return out
