"""The decoder operators from their definitions in 64 bits, with bounds for the kernels' outputs.

An attention output is o = sum_j w_j v_j, w_j = e_j / sum e, e_j = exp(s_j - m).  The kernels' o differs by
  * the weights' rounding to the type of the product, at most ``weight`` relative to each (half a step;
    0 where they stay in 32 bits) plus ``tiny`` absolute to each e_j (half of the smallest fp16 step);
  * the scores: 32-bit products and sums of D terms, (D + 2) 2^-24 scale sum |q||k| each.  The error of a
    score moves its weight and, through the sum, all of them: twice its relative size;
  * exponential, its argument and the partial sums' rescales: 2^-20 relative is more than they have;
  * sums of n terms in 32 bits, numerator and denominator: 2 n 2^-24 relative to sum w |v|;
  * the output's rounding, half a step.
"""

from __future__ import annotations

import math

import torch

HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def attend64(q, k, v, visible, scale):
    """q [lq, d], k [lk, d], v [lk, dv] in any type, visible [lq, lk]: (o, magnitude, score error, sum |v| / l)
    in 64 bits on the CPU.  What is not visible does not count, whatever it holds."""
    q, k, v = q.detach().cpu().double(), k.detach().cpu().double(), v.detach().cpu().double()
    visible = visible.cpu()
    lq, dv = q.shape[0], v.shape[1]
    o = torch.zeros(lq, dv, dtype=torch.float64)
    mag, tail, err = torch.zeros_like(o), torch.zeros_like(o), torch.zeros(lq, 1, dtype=torch.float64)
    for r in range(lq):
        seen = visible[r].nonzero().flatten()
        if seen.numel() == 0:
            continue
        ks, vs = k[seen], v[seen]
        s = (ks @ q[r]) * scale
        e = torch.exp(s - s.max())
        w = e / e.sum()
        o[r] = w @ vs
        mag[r] = w @ vs.abs()
        tail[r] = vs.abs().sum(0) / e.sum()
        err[r] = (q.shape[1] + 2) * 2.0**-24 * abs(scale) * (ks.abs() @ q[r].abs()).max()
    return o, mag, err, tail


def attention_bound(dtype, o, mag, err, tail, keys, weight, tiny):
    relative = weight + 2 * err + 2.0**-20 + 2 * (keys + 8) * 2.0**-24
    return HALF[dtype] * o.abs() + (1 + HALF[dtype]) * (relative * mag + tiny * tail) + 1e-30


def prompt_rounding(dtype):
    """(weight, tiny) of the prompt kernel: weights in the type."""
    return {torch.float32: (0.0, 0.0), torch.float16: (2.0**-11, 2.0**-25), torch.bfloat16: (2.0**-8, 0.0)}[dtype]


def token_rounding(dtype):
    """(weight, tiny) of the single-token kernel: weights in two parts of the type."""
    return {torch.float32: (0.0, 0.0), torch.float16: (2.0**-22, 2.0**-25), torch.bfloat16: (2.0**-16, 0.0)}[dtype]


def assert_within(actual, expected, bound, what=""):
    a = actual.detach().cpu().double()
    nan = torch.isnan(expected)
    assert torch.equal(torch.isnan(a), nan), f"{what}: NaN where none is due, or none where one is"
    inf = torch.isinf(expected)
    assert torch.equal(a[inf], expected[inf]), f"{what}: infinities differ"
    fine = ~nan & ~inf
    off = torch.where(fine, (a - expected).abs() - bound, torch.full_like(bound, -1.0))
    if off.numel():
        worst = int(off.flatten().argmax())
        assert float(off.max()) <= 0, (
            f"{what}: {int((off > 0).sum())} of {off.numel()} outside; {float(a.flatten()[worst]):.6g} for "
            f"{float(expected.flatten()[worst]):.6g} +- {float(bound.flatten()[worst]):.3g} at {worst}")


def window_visible(lq, lk, window, sinks):
    p = torch.arange(lq).view(-1, 1) + (lk - lq)
    j = torch.arange(lk).view(1, -1)
    near = (p - j < window) if window is not None else torch.ones(lq, lk, dtype=torch.bool)
    return (j <= p) & (near | (j < sinks))


def check_window(out, q, k, v, window, sinks, scale=None, what=""):
    """out, q [hq, lq, d], k, v [hkv, lk, d] of one sequence."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    visible = window_visible(q.shape[1], k.shape[1], window, sinks)
    group = q.shape[0] // k.shape[0]
    for h in range(q.shape[0]):
        parts = attend64(q[h], k[h // group], v[h // group], visible, scale)
        keys = int(visible.sum(1).max()) if visible.numel() else 0
        assert_within(out[h], parts[0], attention_bound(out.dtype, *parts, keys, *prompt_rounding(out.dtype)),
                      f"{what} head {h}")


def rows_of(cache, table, length, page):
    """Keys or values [length, heads, dim] of one sequence."""
    j = torch.arange(length, device=cache.device)
    return cache[table.to(torch.int64)[j // page], j % page]


def check_token(out, q, kc, vc, table, length, window=None, sinks=0, scale=None, what=""):
    """out [hq, dv], q [hq, d], one sequence's table row."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    visible = window_visible(1, length, window, sinks) if length else torch.zeros(1, 0, dtype=torch.bool)
    safe = torch.where((table >= 0) & (table < kc.shape[0]), table, 0)
    k, v = (rows_of(c, safe, length, kc.shape[1]).cpu() for c in (kc, vc))
    group = q.shape[0] // kc.shape[2]
    for h in range(q.shape[0]):
        parts = attend64(q[h:h + 1], k[:, h // group], v[:, h // group], visible, scale)
        assert_within(out[h:h + 1], parts[0],
                      attention_bound(out.dtype, *parts, int(visible.sum()), *token_rounding(out.dtype)),
                      f"{what} head {h}")


def rotate64(x, positions, sections, base=10000.0, inv_freq=None, interleaved_axes=False, interleaved_pairs=False,
             inverse=False):
    """(rotated x, bound without the output's rounding) in 64 bits; x [..., heads, d], positions [axes, ...].

    Sine and cosine: the reduced angle (at most pi) rounded to 32 bits, pi 2^-24, and the function's own
    error, at most 4 2^-24; two products and a sum, 2 2^-24 more: 10 2^-24 (|x0| + |x1|).  The angle t itself
    is formed in 64 bits on both sides, half a step 2^-53 |t| for each rounding: here the product; there 2 pi,
    the division by it, the product and its reduction: 6 2^-53 |t| (1e-4 at t = 2^40, nothing at 2^20)."""
    n = sum(sections)
    order, left = [], list(sections)
    while any(left):
        for a in range(len(left)):
            take = 1 if interleaved_axes else left[a]
            take = min(take, left[a])
            order += [a] * take
            left[a] -= take
    freq = inv_freq or [base ** (-i / n) for i in range(n)]
    y = x.detach().cpu().double().clone()
    bound = torch.zeros_like(y)
    pos = positions.detach().cpu().double()
    for i in range(n):
        t = (pos[order[i]] * freq[i]).unsqueeze(-1) * (-1.0 if inverse else 1.0)
        a, b = (2 * i, 2 * i + 1) if interleaved_pairs else (i, i + n)
        x0, x1 = y[..., a].clone(), y[..., b].clone()
        y[..., a] = x0 * t.cos() - x1 * t.sin()
        y[..., b] = x1 * t.cos() + x0 * t.sin()
        bound[..., a] = bound[..., b] = (10 * 2.0**-24 + 6 * 2.0**-53 * t.abs()) * (x0.abs() + x1.abs())
    return y, bound


def check_rotated(out, x, positions, sections, what="", **kw):
    y, bound = rotate64(x, positions, sections, **kw)
    h = HALF[out.dtype]
    # the smallest fp16 numbers have a step of their own
    assert_within(out, y, bound * (1 + h) + h * y.abs() + (2.0**-25 if out.dtype == torch.float16 else 1e-40), what)
