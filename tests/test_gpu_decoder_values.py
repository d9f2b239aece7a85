"""Attention over pages and under a window at the ends of the number range, against the 64-bit definition."""

from __future__ import annotations

import math

import pytest
import torch

from batch_invariant_ops import (check_cache_indices, paged_attention_batch_invariant,
                                 sliding_window_attention_batch_invariant as window_attention,
                                 varlen_sliding_window_attention_batch_invariant as packed_attention)

from _decoder import HALF, assert_within, attend64, attention_bound, prompt_rounding, token_rounding, window_visible

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


def randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def paged(k, v, page=16):
    """k [keys, heads, d], v [keys, heads, dv] as caches with their pages backwards, and the table."""
    n = k.shape[0]
    count = max(1, -(-n // page))
    caches = []
    for x in (k, v):
        c = torch.full((count, page, *x.shape[1:]), float("nan"), dtype=x.dtype)
        c.flatten(0, 1)[:n] = x
        caches.append(c.flip(0).contiguous().cuda())
    return *caches, torch.arange(count - 1, -1, -1, dtype=torch.int32).view(1, count).cuda()


def token(q, k, v, **kw):
    """q [hq, d] against k [keys, hkv, d], v [keys, hkv, dv] (on the CPU)."""
    kc, vc, table = paged(k, v)
    lengths = torch.tensor([k.shape[0]], dtype=torch.int32).cuda()
    return paged_attention_batch_invariant(q.unsqueeze(0).cuda(), kc, vc, table, lengths, **kw)[0]


def exact_scores(out, q, k, v, visible, scale, rounding, what):
    """As the definition for scores that are exact in 32 bits: they add nothing to the bound.  out, q [rows, d], k, v
    [keys, d] of one head."""
    o, mag, err, tail = attend64(q, k, v, visible, scale)
    assert_within(out, o, attention_bound(out.dtype, o, mag, torch.zeros_like(err), tail, int(visible.sum(1).max()), *rounding), what)


# An element of the queries, one of the keys, the head size, the type.  All keys of a kind have the same score to the bit,
# and those of the other kind one so far away that its weight is 0 in 64 bits too.
HUGE = [
    (19968.0, 19968.0, 128, BF16), (20096.0, 18944.0, 128, BF16), (-20096.0, 18944.0, 128, BF16), (5736.0, 5736.0, 128, F16),
    (6832.0, 6832.0, 64, F16), (-6832.0, 6832.0, 64, F16), (2.0**40, 1.5 * 2.0**40, 64, BF16), (3.0 * 2.0**50, 5.0 * 2.0**40, 72, F32),
    (20001.0, 20001.0, 64, F32), (2.0**60, 2.0**60, 128, F32),
]


@pytest.mark.parametrize("x, y, d, dtype", HUGE)
@pytest.mark.parametrize("n", [1, 40, 700, 2500])
def test_token_attention_of_huge_scores(x, y, d, dtype, n):
    """Every third key has the largest score, all others far smaller ones: the mean of those values."""
    q = torch.full((2, d), x, dtype=dtype)
    k = torch.full((n, 1, d), y, dtype=dtype)
    other = torch.arange(n) % 3 != 0 if x > 0 else torch.arange(n) % 3 == 0
    k[other] = k[other] / 2
    v = randn(n, 1, 64, seed=n, dtype=dtype)
    out = token(q, k, v)
    for h in range(2):
        exact_scores(out[h:h + 1], q[h:h + 1], k[:, 0], v[:, 0], torch.ones(1, n, dtype=torch.bool), d**-0.5, token_rounding(dtype),
                     f"head {h}")


def steps(n, dtype, seed, sign=1.0):
    """Scores 4096 a + 16 b + j, exact in 32 bits, j random in -60 .. 60 and the rest near 2^20 / log2 e: arguments of 2^x on
    both sides of 2^20.  (q [1, 8 or 16 bytes of elements], k.)"""
    g = torch.Generator().manual_seed(seed)
    j = torch.randint(-60, 61, (n,), generator=g)
    d = 8
    q, k = torch.zeros(1, d), torch.zeros(n, 1, d)
    q[0, :3] = torch.tensor([4096.0, 16.0, 1.0])
    k[:, 0, 0], k[:, 0, 1], k[:, 0, 2] = 177.0 * sign, 114.0 * sign, j.float()
    return q.to(dtype), k.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, sign", [(50, 1.0), (3000, 1.0), (700, -1.0)])
def test_token_attention_of_large_scores_close_together(dtype, n, sign):
    q, k = steps(n, dtype, n, sign)
    v = randn(n, 1, 64, seed=n + 1, dtype=dtype)
    exact_scores(token(q, k, v, scale=1.0), q, k[:, 0], v[:, 0], torch.ones(1, n, dtype=torch.bool), 1.0, token_rounding(dtype), "")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e12, -1e12, 1e37, 3e38])
def test_token_attention_with_a_huge_scale(dtype, scale):
    """The value of the one key with the largest product."""
    n, d = 300, 64
    q, k, v = randn(2, d, seed=1, dtype=dtype), randn(n, 1, d, seed=2, dtype=dtype), randn(n, 1, d, seed=3, dtype=dtype)
    out = token(q, k, v, scale=scale)
    s = (k[:, 0].double() @ q.double().T) * math.copysign(1.0, scale)
    top = s.topk(2, dim=0).values
    assert float((top[0] - top[1]).min()) > 1e-3  # far more than the 32-bit sums' error
    want = v[s.argmax(0), 0].double()
    assert_within(out, want, HALF[dtype] * want.abs() + 2.0**-22 * want.abs())


# Rows and keys of the kinds of tiles: few rows, few before keys in ranges, many.
TILES = [(1, 1), (7, 40), (4, 3000), (130, 200)]


def prompt(q, k, v, window=None, sinks=0, **kw):
    """q [rows, hq, d], k and v [keys, hkv, ...] on the CPU: dense output [rows, hq, dv]; the packed one has to agree where it
    takes the same tiles, and has to hold by itself where it does not."""
    dense = window_attention(*(x.transpose(0, 1).unsqueeze(0).cuda() for x in (q, k, v)), window, sinks, enable_gqa=True, **kw)
    offsets = [torch.tensor([0, x.shape[0]], dtype=torch.int32).cuda() for x in (q, k)]
    packed = packed_attention(*(x.unsqueeze(0).cuda() for x in (q, k, v)), *offsets, window, sinks, **kw)
    return dense[0].transpose(0, 1), packed[0]


@pytest.mark.parametrize("x, y, d, dtype", HUGE)
@pytest.mark.parametrize("lq, lk", TILES)
def test_prompts_of_huge_scores(x, y, d, dtype, lq, lk):
    q = torch.full((lq, 2, d), x, dtype=dtype)
    k = torch.full((lk, 1, d), y, dtype=dtype)
    k[torch.arange(lk) % 3 != 0 if x > 0 else torch.arange(lk) % 3 == 0] /= 2
    v = randn(lk, 1, 64, seed=lk, dtype=dtype)
    for window, sinks in ((None, 0), (9, 1)):
        visible = window_visible(lq, lk, window, sinks)
        for out in prompt(q, k, v, window, sinks):
            for h in range(2):
                exact_scores(out[:, h], q[:, h], k[:, 0], v[:, 0], visible, d**-0.5, prompt_rounding(dtype), f"head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq, lk, sign", [(5, 60, 1.0), (6, 3000, 1.0), (5, 700, -1.0), (140, 300, 1.0)])
def test_prompts_of_large_scores_close_together(dtype, lq, lk, sign):
    q, k = steps(lk, dtype, lk, sign)
    q, v = q.unsqueeze(0).expand(lq, 1, -1).contiguous(), randn(lk, 1, 64, seed=lk + 1, dtype=dtype)
    visible = window_visible(lq, lk, None, 0)
    for out in prompt(q, k, v, scale=1.0):
        exact_scores(out[:, 0], q[:, 0], k[:, 0], v[:, 0], visible, 1.0, prompt_rounding(dtype), "")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e12, -1e12, 1e37, 3e38])
@pytest.mark.parametrize("lq", [3, 90])
def test_prompts_with_a_huge_scale(dtype, scale, lq):
    n, d = 300, 64
    q = randn(1, 2, d, seed=1, dtype=dtype).expand(lq, 2, d).contiguous()
    k, v = randn(n, 1, d, seed=2, dtype=dtype), randn(n, 1, d, seed=3, dtype=dtype)
    s = (k[:, 0].double() @ q[0].double().T) * math.copysign(1.0, scale)
    for out in prompt(q, k, v, scale=scale):
        for r in range(lq):
            seen = n - lq + r + 1
            top = s[:seen].topk(2, dim=0).values
            assert float((top[0] - top[1]).min()) > 1e-3  # far more than the 32-bit sums' error
            want = v[s[:seen].argmax(0), 0].double()
            assert_within(out[r], want, HALF[dtype] * want.abs() + 2.0**-22 * want.abs(), f"row {r}")


# Products of queries and keys reach 1e36 and more, where any scale but 0 counts.
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-45, 1e-39, -3e-37, 2e-36])
@pytest.mark.parametrize("lq", [3, 90])
def test_tiny_scales(dtype, scale, lq):
    n, d = 300, 64
    q, k = (1e18 * randn(x, 2, d, seed=x, dtype=F32) for x in (lq, n))
    q, k, v = q.to(dtype), k.to(dtype), randn(n, 2, d, seed=9, dtype=dtype)
    held = float(torch.tensor(scale, dtype=F32))  # as the kernels hold it
    outs = [(o, window_visible(lq, n, None, 0), prompt_rounding(dtype)) for o in prompt(q, k, v, scale=scale)]
    outs.append((token(q[-1], k, v, scale=scale).unsqueeze(0), window_visible(1, n, None, 0), token_rounding(dtype)))
    for out, visible, rounding in outs:
        for h in range(2):
            parts = attend64(q[-len(out):, h], k[:, h], v[:, h], visible, held)
            assert_within(out[:, h], parts[0], attention_bound(dtype, *parts, n, *rounding), f"head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_scale_of_zero_and_infinities(dtype):
    """0 times a product that is not finite is NaN."""
    q, k, v = (randn(x, 1, 64, seed=x, dtype=dtype) for x in (5, 70, 71))
    v = v[:70]
    q[2, 0, 9], q[3, 0, 1] = float("nan"), float("inf")
    for bad in (None, 3):
        if bad is not None:
            k[68, 0, 0] = float("-inf")
        visible = window_visible(5, 70, 20, 0)
        for out in prompt(q, k, v, 20, scale=0.0):
            parts = attend64(q[:, 0], k[:, 0], v[:, 0], visible, 0.0)
            assert_within(out[:, 0], parts[0], torch.nan_to_num(attention_bound(dtype, *parts, 20, *prompt_rounding(dtype)), 0.0))
        for r in (0, 2, 3):
            assert bool(torch.isnan(token(q[r], k, v, scale=0.0)).all()) == (r > 0 or bad is not None)


@pytest.mark.parametrize("dtype, down", [(BF16, 117), (F32, 117), (F16, 6)])
@pytest.mark.parametrize("n", [1, 40, 700, 2500])
def test_token_attention_of_small_values(dtype, down, n):
    """Equal weights: the mean of values near the type's smallest normal numbers, down to its own rounding.  (Without the
    1e-30 that the general bound adds.  Sums of n products in 32 bits, their mean and the shares of its parts: 2 (n + 8) 2^-24
    of the mean magnitude; products below 2^-126 lose 2^-149 each.)"""
    q = torch.zeros(3, 64, dtype=dtype)
    k, v = randn(n, 1, 64, seed=n, dtype=dtype), randn(n, 1, 64, seed=n + 1, dtype=F32)
    v = ((v + v.sign() / 16) * 2.0**-down).to(dtype)
    o = v[:, 0].double().mean(0)
    bound = HALF[dtype] * o.abs() + 2 * (n + 8) * 2.0**-24 * v[:, 0].double().abs().mean(0) + 2.0**-149
    assert_within(token(q, k, v), o.expand(3, 64), bound.expand(3, 64))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [40, 700, 2500, 40000])
def test_token_attention_of_the_largest_and_the_smallest_values(dtype, n):
    """Columns whose sums pass the range, in some chunks and not in others, beside columns of small values; each query by itself,
    one of which hardly sees the large values (weights below 2^-400).  Sums that pass the range are of weights 2^-9 times their
    size at most (256 keys of a wavefront): products that lose 2^-150 leave 2^-141 in the means."""
    d = 64
    q, k = torch.zeros(2, d, dtype=dtype), torch.zeros(n, 1, d, dtype=dtype)
    small = float(torch.tensor(1.2345 * 2.0**-117, dtype=dtype))
    v = torch.full((n, 1, d), small, dtype=dtype)
    large = torch.arange(n) < max(20, n // 3)
    v[large, 0, ::2] = 0.96 * torch.finfo(dtype).max
    k[large, 0, 0] = -300.0
    q[1, 0] = 8.0  # scores of -300 at the large values
    out = token(q, k, v).double().cpu()
    o = v[:, 0].double().mean(0)
    relative = HALF[dtype] + 2 * (n + 8) * 2.0**-24
    assert_within(out[:1], o.unsqueeze(0), (relative * o.abs() + 2.0**-141).unsqueeze(0))
    want = torch.full((1, d), small, dtype=torch.float64)
    assert_within(out[1:], want, relative * want + 2.0**-141)


@pytest.mark.parametrize("dtype, n, top", [(BF16, 600000, 17.375), (F16, 100000, 17.40625)])
def test_prompts_of_many_small_weights(dtype, n, top):
    """Keys of weight 2^-25.1 beside one of 1, which make 2^-6 (600000 keys) or 2^-8 (100000) of the output together.  Values are
    positive, so that a sum's error is 2^-24 for each of the additions on a value's way: one for each block of 64 keys and 64 in a
    block, in the numerator and the denominator.  The many weights are rounded once to the type: all alike, the other one is 1.  (fp16's
    smallest step is 2^-24, half of it 2^-25, and weights are 2^7 times their size in it: 2^-32 each.)"""
    lq, d = 65, 8
    q, k = torch.zeros(lq, 1, d, dtype=dtype), torch.zeros(n, 1, d, dtype=dtype)
    q[:, 0, 0] = 8.0
    k[50, 0, 0] = top
    v = randn(n, 1, d, seed=78, dtype=dtype).abs() + 1
    v[50] = 1.0
    rows = [0, 40, 64]
    visible = window_visible(1, n, None, 0).expand(3, n).clone()
    for i, r in enumerate(rows):
        visible[i, n - lq + r + 1:] = False
    o, mag, err, tail = attend64(q[rows, 0], k[:, 0], v[:, 0], visible, 0.125)
    share = (o - 1).abs()  # of the many, at least: their values are over 1
    relative = 2.0**-20 + 2 * err + 2 * (n / 64 + 64) * 2.0**-24
    bound = HALF[dtype] * o.abs() + (1 + HALF[dtype]) * (relative * mag + HALF[dtype] * 4 * share + (2.0**-32 if dtype == F16 else 0.0) * tail)
    for out in prompt(q, k, v, scale=0.125):
        assert_within(out[rows, 0], o, bound)
