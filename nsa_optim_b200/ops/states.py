"""States of the Mamba-2 mixer between steps of generation: their layout, and the ops that continue them in PyTorch (any device).

A layer's states are two tensors (:class:`ScanStates`), a row for each of B requests:

  * ``conv`` (B, W - 1, C), of the activations' type: the last W - 1 inputs of the short causal convolution, the oldest first;
  * ``ssm`` fp32 (B, H, P, S): the scan's state of each head, P columns of the head by S states.

The new tokens of a step are packed one request after another, as for the paged cache (:mod:`nsa_optim_b200.ops.cache`): ``query_start`` (B + 1) int32 says where
each request begins, ``lengths`` (B) int32 how many tokens it has with them.  A request all of whose tokens are new begins from zeros, whatever its row
holds, so that a finished request's row needs no clearing; a request without new tokens keeps its row.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F
from torch import Tensor


class ScanStates(NamedTuple):
    """States of one layer (see the module)."""
    conv: Tensor
    ssm: Tensor


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def new_states(requests: int, heads: int, head_dim: int, d_state: int, channels: int, width: int, device=None, dtype=torch.bfloat16) -> ScanStates:
    _need(min(requests, heads, head_dim, d_state, channels) > 0 and width > 1, "states need requests, heads, columns, channels, and a convolution of 2 taps at least")
    return ScanStates(torch.zeros(requests, width - 1, channels, dtype=dtype, device=device),
                      torch.zeros(requests, heads, head_dim, d_state, device=device))


def check_step(query_start: Tensor, lengths: Tensor, state: Tensor) -> None:
    for t, what in ((query_start, "query_start"), (lengths, "lengths")):
        _need(t.dim() == 1 and t.dtype == torch.int32, f"{what} has to be an int32 tensor of 1 dimension(s)")
        _need(t.device == state.device, f"{what} is on another device")
    B = lengths.shape[0]
    _need(B > 0 and query_start.shape[0] == B + 1 and state.shape[0] == B, "query_start, lengths and the state have to be of the same requests")
    _need(state.is_contiguous(), "the state has to be contiguous: it is changed in place")


def check_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Tensor, query_start: Tensor, lengths: Tensor) -> None:
    _need(x.dim() == 2 and weight.dim() == 2 and weight.shape[0] == x.shape[1] and weight.shape[1] > 1,
          f"expected inputs (tokens, channels) and a weight (channels, 2 taps or more), got {tuple(x.shape)} and {tuple(weight.shape)}")
    _need(bias is None or tuple(bias.shape) == (x.shape[1],), "bias has one number a channel")
    _need(state.dim() == 3 and tuple(state.shape[1:]) == (weight.shape[1] - 1, x.shape[1]) and state.dtype == x.dtype,
          f"the state has to be (requests, {weight.shape[1] - 1}, {x.shape[1]}) of the inputs' type, got {tuple(state.shape)}")
    _need(all(t is None or t.device == x.device for t in (weight, bias, state)), "the convolution's tensors are on different devices")
    check_step(query_start, lengths, state)


def conv1d(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Tensor, query_start: Tensor, lengths: Tensor, activation: bool = True) -> Tensor:
    check_conv(x, weight, bias, state, query_start, lengths)
    x, W, y = x.detach(), weight.shape[1], torch.zeros_like(x, memory_format=torch.contiguous_format)
    start, total = query_start.tolist(), lengths.tolist()
    for b, (lo, hi) in enumerate(zip(start, start[1:])):
        lo, hi, new = max(lo, 0), min(hi, x.shape[0]), hi - lo
        if hi <= lo:
            continue
        before = torch.zeros_like(state[b]) if total[b] <= new else state[b]
        u = torch.cat([before, x[lo:hi]])
        z = torch.zeros(hi - lo, x.shape[1], device=x.device) if bias is None else bias.detach().to(x.dtype).float().expand(hi - lo, -1)
        for j in range(W):                                   # in this order, so that the bits are the same however a text is cut
            z = z + u[j:j + hi - lo].float() * weight.detach()[:, j].to(x.dtype).float()
        y[lo:hi] = (F.silu(z) if activation else z).to(x.dtype)
        state[b] = u[u.shape[0] - (W - 1):]
    return y


def check_scan(x: Tensor, dt: Tensor, A_log: Tensor, Bm: Tensor, Cm: Tensor, D: Optional[Tensor], dt_bias: Tensor, state: Tensor, query_start: Tensor,
               lengths: Tensor) -> None:
    _need(x.dim() == 3 and Bm.dim() == 3, "expected x (tokens, heads, columns), B and C (tokens, groups, states)")
    n, H, P = x.shape
    G, S = Bm.shape[1:]
    _need(tuple(dt.shape) == (n, H) and Bm.shape[0] == n and Bm.shape == Cm.shape and G > 0 and H % G == 0,
          f"dt has to be ({n}, {H}), B and C ({n}, a divisor of {H} groups, states), got {tuple(dt.shape)}, {tuple(Bm.shape)} and {tuple(Cm.shape)}")
    _need(x.dtype == dt.dtype == Bm.dtype == Cm.dtype, "x, dt, B and C have to be of one type")
    _need(all(tuple(t.shape) == (H,) for t in (A_log, dt_bias, D) if t is not None), "A_log, dt_bias and D have one number a head")
    _need(state.dim() == 4 and tuple(state.shape[1:]) == (H, P, S) and state.dtype == torch.float32,
          f"the state has to be fp32 (requests, {H}, {P}, {S}), got {tuple(state.shape)}")
    _need(all(t is None or t.device == x.device for t in (dt, A_log, Bm, Cm, D, dt_bias, state)), "the scan's tensors are on different devices")
    check_step(query_start, lengths, state)


def scan(x: Tensor, dt: Tensor, A_log: Tensor, Bm: Tensor, Cm: Tensor, D: Optional[Tensor], dt_bias: Tensor, state: Tensor, query_start: Tensor,
         lengths: Tensor, chunk: int = 64) -> Tensor:
    """Chunked, fp32 throughout."""
    check_scan(x, dt, A_log, Bm, Cm, D, dt_bias, state, query_start, lengths)
    y = torch.zeros_like(x, memory_format=torch.contiguous_format)
    start, total, rep = query_start.tolist(), lengths.tolist(), x.shape[1] // Bm.shape[1]
    step = F.softplus(dt.detach().float() + dt_bias.detach().float())
    log_decay = (step * -torch.exp(A_log.detach().float())).clamp(min=-1000.0)       # a decay of zero either way, and sums of them that stay finite
    for b, (lo, hi) in enumerate(zip(start, start[1:])):
        lo, hi, new = max(lo, 0), min(hi, x.shape[0]), hi - lo
        if hi <= lo:
            continue
        h = torch.zeros_like(state[b]) if total[b] <= new else state[b].clone()
        for i in range(lo, hi, chunk):
            j = min(i + chunk, hi)
            xf = x.detach()[i:j].float()
            cum = log_decay[i:j].double().cumsum(0).t()                                         # (H, L)
            xd = (xf * step[i:j, :, None]).transpose(0, 1)                                      # (H, L, P)
            Bh, Ch = (m.detach()[i:j].float().repeat_interleave(rep, 1).transpose(0, 1) for m in (Bm, Cm))
            L = torch.ones(j - i, j - i, dtype=torch.bool, device=x.device).tril()
            decay = torch.exp((cum[:, :, None] - cum[:, None]).masked_fill(~L, float("-inf"))).float()
            o = ((Ch @ Bh.transpose(1, 2)).masked_fill(~L, 0.0) * decay) @ xd + (Ch @ h.transpose(1, 2)) * torch.exp(cum).float()[..., None]
            o = o.transpose(0, 1)
            y[i:j] = (o if D is None else o + D.detach().float()[:, None] * xf).to(x.dtype)
            h = h * torch.exp(cum[:, -1]).float()[:, None, None] + (xd * torch.exp(cum[:, -1:] - cum).float()[..., None]).transpose(1, 2) @ Bh
        state[b] = h
    return y
