"""The attention operators' definitions in 64 bits, on the CPU (torch): what tests compare the kernels with.

Nothing here looks at the package's code: a rotation is a product of complex numbers, an 8-bit rounding is the
nearest multiple of the step at a value's magnitude, a softmax is the ratio of two sums."""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch


def rotate(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """``x [tokens, heads, dim]``: pairs of the first ``2 len(inv_freq)`` elements turned by position * inv_freq."""
    rotary = 2 * inv_freq.numel()
    if rotary == 0 or x.numel() == 0:
        return x
    head = x[..., :rotary]
    z = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    angle = torch.outer(positions.double(), inv_freq.double())
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = torch.view_as_real(z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., rotary:]), -1)


def qk_norm_rope(x: torch.Tensor, q_weight, k_weight, positions, inv_freq, q_heads: int, k_heads: int, eps: float,
                 interleaved: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``x [tokens, columns]`` in float64 (the ranks' sum), differentiable."""
    dim = q_weight.numel()
    q, k, v = x.view(x.shape[0], -1, dim).tensor_split((q_heads, q_heads + k_heads), 1)
    out = [rotate(w * h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps), positions, inv_freq, interleaved)
           for h, w in ((q, q_weight), (k, k_weight))]
    return out[0], out[1], v


def qk_norm_rope_grad(parts: Sequence[torch.Tensor], grads, q_weight, k_weight, positions, inv_freq, eps, interleaved):
    """Gradients of <outputs, grads> with respect to the sum and the two weights."""
    x = sum(p.double() for p in parts).requires_grad_()
    w = [q_weight.double().requires_grad_(), k_weight.double().requires_grad_()]
    y = qk_norm_rope(x, *w, positions, inv_freq, grads[0].shape[1], grads[1].shape[1], eps, interleaved)
    value = sum((a * g.double()).sum() for a, g in zip(y, grads))
    got = torch.autograd.grad(value, (x, *w), allow_unused=True)
    return [torch.zeros_like(t) if g is None else g for g, t in zip(got, (x, *w))]


def stored(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values a cache of ``dtype`` holds of rows ``x [..., dim]``, in float64."""
    if dtype == torch.bfloat16:
        return x.to(torch.bfloat16).double()
    x = x.double()
    finite = torch.isfinite(x)
    largest = torch.where(finite, x.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.full_like(largest, -110.0)
    for n in range(-110, 122):                         # the least exponent that is large enough
        e = torch.where((448.0 * 2.0 ** (n - 1) < largest) & (n > -110), float(n), e)
    y = x / torch.exp2(e)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20, max=448.0))), min=-6.0) - 3)
    y = torch.round(y / step) * step
    y = torch.where(e == 120, y.clamp(-240.0, 240.0), y) * torch.exp2(e)     # 256 times 2^120 would be no finite number
    return torch.where(finite, y, math.nan)


def attention(q: torch.Tensor, keys: List[torch.Tensor], values: List[torch.Tensor], scale: Optional[float] = None):
    """``q [batch, q_heads, dim]``; ``keys[b]``, ``values[b]``: ``[tokens of b, kv_heads, dim]``.  Returns out and lse."""
    batch, q_heads, dim = q.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    outs, lses = torch.zeros(batch, q_heads, dim, dtype=torch.float64), torch.full((batch, q_heads), -math.inf, dtype=torch.float64)
    for b in range(batch):
        if keys[b].shape[0] == 0:
            continue
        group = q_heads // keys[b].shape[1]
        for h in range(q_heads):
            s = keys[b][:, h // group].double() @ q[b, h].double() * scale
            lses[b, h] = torch.logsumexp(s, 0)
            outs[b, h] = torch.softmax(s, 0) @ values[b][:, h // group].double()
    return outs, lses


def join(outs: Sequence[torch.Tensor], lses: Sequence[torch.Tensor]):
    lse = torch.stack([t.double() for t in lses])
    whole = torch.logsumexp(lse, 0)
    w = torch.where(lse == -math.inf, 0.0, torch.exp(lse - whole))
    out = torch.zeros_like(outs[0], dtype=torch.float64)
    for i, o in enumerate(outs):
        out = out + torch.where(w[i][..., None] == 0, 0.0, w[i][..., None] * o.double())
    return out, whole
