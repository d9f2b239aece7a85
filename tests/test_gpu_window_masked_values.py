"""Windowed attention where values or keys are not finite: what a row does not see changes none of its bits, and what it sees
reaches it column by column."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import (check_cache_indices, sliding_window_attention_batch_invariant as window_attention,
                                 varlen_sliding_window_attention_batch_invariant as packed_attention)

from _decoder import window_visible
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


def randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# heads, key heads, head size, rows, keys, window, sinks: every kind of tile (16-bit: four wavefronts for rows or heads of a
# group; two and key turns; ranges of keys; float32: two and key turns)
SHAPES = [
    (4, 1, 64, 200, 200, 37, 2), (2, 2, 64, 150, 260, 37, 2), (4, 4, 128, 140, 140, 50, 0), (4, 2, 128, 130, 200, 70, 5),
    (8, 2, 72, 100, 100, 20, 3), (2, 1, 64, 40, 300, 37, 2), (3, 3, 128, 5, 90, 20, 1), (4, 1, 64, 20, 3000, 2500, 3),
    (2, 2, 128, 7, 1500, 1400, 0), (4, 1, 256, 70, 130, 33, 2), (2, 1, 200, 16, 2000, 1900, 2), (1, 1, 64, 3, 3, 1, 1),
]


def columns(out, want, visible, spoilt):
    """``want`` with the spoilt values {(key, column): value} that each row sees."""
    want = want.clone()
    for r in range(visible.shape[0]):
        for col in {c for _, c in spoilt}:
            seen = [x for (j, c), x in spoilt.items() if c == col and bool(visible[r, j])]
            if not seen:
                continue
            x = sum(seen)  # inf - inf is NaN
            want[:, :, r, col] = x
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(out), nan)
    assert_bitwise(torch.where(nan, 0, out), torch.where(nan, 0, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, hkv, d, lq, lk, window, sinks", SHAPES)
def test_values_that_are_not_finite(dtype, hq, hkv, d, lq, lk, window, sinks):
    if dtype == F32 and d > 128:
        pytest.skip("float32 heads go up to 128")
    q, k, v = (randn(2, h, n, d, seed=h + n, dtype=dtype) for h, n in ((hq, lq), (hkv, lk), (hkv, lk)))
    clean = window_attention(q, k, v, window, sinks, enable_gqa=True)
    visible = window_visible(lq, lk, window, sinks)
    mid = lk - max(1, lq // 2)
    for spoilt in ({(mid, 5): NAN}, {(mid, 5): INF, (mid, d - 1): -INF}, {(0, 0): -INF, (lk - 1, 3): INF, (mid, 0): INF, (mid, 7): NAN},
                   {(j, c): INF for j in range(mid, lk) for c in (1, d // 2 + 1)}):
        bad = v.clone()
        for (j, c), x in spoilt.items():
            bad[:, :, j, c] = x
        columns(window_attention(q, k, bad, window, sinks, enable_gqa=True), clean, visible, spoilt)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, hkv, d, lq, lk, window, sinks", SHAPES)
def test_what_stands_behind_a_row(dtype, hq, hkv, d, lq, lk, window, sinks):
    """Keys and values behind a row, and those that its window has passed, hold NaN and infinities."""
    if dtype == F32 and d > 128:
        pytest.skip("float32 heads go up to 128")
    q, k, v = (randn(1, h, n, d, seed=h + n + 1, dtype=dtype) for h, n in ((hq, lq), (hkv, lk), (hkv, lk)))
    clean = window_attention(q, k, v, window, sinks, enable_gqa=True)
    visible = window_visible(lq, lk, window, sinks)
    for r in {0, lq // 2, lq - 1}:
        hidden = (~visible[r]).nonzero().flatten().cuda()
        for x in (NAN, INF, -INF):
            kb, vb = k.clone(), v.clone()
            kb[:, :, hidden] = x
            vb[:, :, hidden] = x
            out = window_attention(q, kb, vb, window, sinks, enable_gqa=True)
            same = ~(visible & ~visible[r]).any(1)  # rows that see nothing else than row r does
            assert bool(same[r])
            assert_bitwise(out[:, :, same.cuda()], clean[:, :, same.cuda()], f"as row {r} with {x}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq, hkv, d, lq, lk, window, sinks", SHAPES[:8])
def test_sums_past_the_range_beside_values_that_are_not_finite(dtype, hq, hkv, d, lq, lk, window, sinks):
    q, k = (randn(1, h, n, d, seed=h + n + 2, dtype=dtype) for h, n in ((hq, lq), (hkv, lk)))
    v = torch.full((1, hkv, lk, d), 0.97 * torch.finfo(dtype).max, dtype=dtype).cuda()
    v[..., ::2] *= -0.5
    clean = window_attention(q * 0.1, k, v, window, sinks, enable_gqa=True)
    assert bool(torch.isfinite(clean).all())
    mean = v[0, 0, 0].double()
    assert float(((clean.double() - mean) / mean).abs().max()) <= 2.0**-6
    mid = lk - max(1, lq // 2)
    bad = v.clone()
    bad[:, :, mid, 4], bad[:, :, mid, 9] = NAN, -INF
    columns(window_attention(q * 0.1, k, bad, window, sinks, enable_gqa=True), clean, window_visible(lq, lk, window, sinks),
            {(mid, 4): NAN, (mid, 9): -INF})


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_neighbours(dtype):
    """Sequences of one tile and of several; one holds NaN and infinities, the others keep their bits."""
    lengths = [40, 130, 20, 300, 1]
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32).cuda()
    total = sum(lengths) + 30
    q, k, v = (randn(1, total, h, 64, seed=h, dtype=dtype) for h in (4, 2, 2))
    clean = packed_attention(q, k, v, cu, cu, 50, 3)
    for s in range(5):
        a, b = int(cu[s]), int(cu[s + 1])
        kb, vb = k.clone(), v.clone()
        kb[:, (a + b) // 2], vb[:, a] = NAN, INF
        vb[:, int(cu[-1]):] = NAN
        out = packed_attention(q, kb, vb, cu, cu, 50, 3)
        assert_bitwise(out[:, :a], clean[:, :a])
        assert_bitwise(out[:, b:], clean[:, b:])
        assert not bool(torch.isfinite(out[:, a]).any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_replays(dtype):
    """A captured call meets finite values, then others, then finite ones again."""
    q, k, v = (randn(1, h, 150, 64, seed=h + 7, dtype=dtype) for h in (4, 2, 2))
    window_attention(q, k, v, 30, 2, enable_gqa=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = window_attention(q, k, v, 30, 2, enable_gqa=True)
    for i, x in enumerate((None, NAN, None, INF)):
        v.copy_(randn(1, 2, 150, 64, seed=20 + i, dtype=dtype))
        if x is not None:
            v[:, :, 60, 3] = x
        graph.replay()
        got = held.clone()
        torch.cuda.synchronize()
        want = window_attention(q, k, v, 30, 2, enable_gqa=True)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(want).any()) == (x is not None and x != x)
        assert_bitwise(torch.nan_to_num(got, 0.0), torch.nan_to_num(want, 0.0))
