"""The operators of a decoder served with fewer bits from their definitions, on the CPU."""

from __future__ import annotations

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
POWERS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def to_fp4(x):
    """(codes [..., d / 2], scales [..., d / 32]) of rows [..., d]: by distances to the levels, in 64 bits."""
    low, high = POWERS[x.dtype]
    blocks = x.detach().cpu().double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, low)
    for i in range(low, high):
        e = torch.where(top > 7.0 * 2.0**i, i + 1.0, e)
    finite = torch.isfinite(blocks).all(-1, keepdim=True)
    e = torch.where(finite, e, 0.0)
    far = ((blocks.abs() * 2.0**-e).unsqueeze(-1) - LEVELS).abs()
    # the nearest, and of two the one with an even code
    near = far == far.min(-1, keepdim=True).values
    cost = torch.where(near, torch.arange(8) % 2, 2)
    code = cost.argmin(-1) + 8 * torch.signbit(blocks).long()
    code = torch.where(finite, code, 0).flatten(-2)
    scales = torch.where(finite, e + 127, 255.0).squeeze(-1)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scales.to(torch.uint8)


def from_fp4(codes, scales):
    """The values in 64 bits."""
    codes, scales = codes.cpu().long(), scales.cpu()
    code = torch.stack([codes % 16, codes // 16], -1).flatten(-2)
    size = LEVELS[code % 8] * torch.where(code >= 8, -1.0, 1.0).double()
    power = torch.where(scales == 255, float("nan"), 2.0 ** (scales.double() - 127))
    return size * power.repeat_interleave(32, -1)


def weights64(logits, temperature):
    """exp((l - max) / T) in 64 bits; 0 for -inf and NaN."""
    x = logits.detach().cpu().double()
    x = torch.where(torch.isnan(x), -float("inf"), x)
    if x.max() == float("inf"):
        return (x == float("inf")).double()
    return torch.exp((x - x.max()) / temperature)


def staying(logits, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(weights, whether a token stays) of one row."""
    w = weights64(logits, temperature)
    x = logits.detach().cpu().double()
    order = torch.sort(torch.where(torch.isnan(x), -float("inf"), x), descending=True, stable=True).indices
    down = w[order]
    if top_k is not None:
        down[top_k:] = 0.0
    stay = down > 0
    if top_p is not None and top_p < 1:
        stay &= (down.cumsum(0) - down) < top_p * down.sum()
    if min_p is not None:
        stay &= down >= min_p
    stay[0] = True
    out = torch.zeros_like(stay)
    out[order] = stay
    return w, out


def int8_rows(x):
    """(q, scale) by the definition's 32-bit operations, which IEEE rounds alike everywhere."""
    x = x.detach().cpu().float()
    finite = torch.isfinite(x).all(-1, keepdim=True)
    top = x.abs().amax(-1, keepdim=True).clamp(min=2.0**-100)
    q = torch.where(finite, torch.round(x * (torch.full_like(top, 127.0) / top)), 0.0)
    return q.to(torch.int8), torch.where(finite, top / torch.full_like(top, 127.0), float("nan")).squeeze(-1)
