"""Rows and linear layers of 8-bit integers against their definitions.

Sums of products are exact integers.  The kernel rounds them to 32-bit floats, multiplies with the row's step, and adds the
channel's multiple and the bias in one operation: three roundings of 2^-24 relative to |sum s t| (and one to the
result's size), then the output's half step."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import linear_int8_batch_invariant, quantize_tokens_int8

from _decoder import HALF
from _served import int8_rows
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
I8, F32 = torch.int8, torch.float32


def ints(*shape, seed, low=-127):
    return torch.randint(low, 128, shape, generator=torch.Generator().manual_seed(seed)).to(I8)


def check(out, x, xs, w, ws, bias, what=""):
    sums = (x.cpu().double() @ w.cpu().double().t()) * xs.cpu().double().unsqueeze(-1) * ws.cpu().double()
    want = sums if bias is None else sums + bias.cpu().double()
    half = HALF[out.dtype]
    bound = (1 + half) * 2.0**-24 * (3 * sums.abs() + want.abs()) + half * want.abs() + (2.0**-25 if out.dtype == torch.float16 else 1e-40)
    off = (out.cpu().double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} of {off.numel()} outside, the worst by {float(off.max()):.3g}"


def case(m, n, k, dtype, seed=1, bias=True, low=-127):
    g = torch.Generator().manual_seed(seed + 50)
    xs, ws = (torch.rand(m, generator=g) + 0.5) * 0.02, (torch.rand(n, generator=g) + 0.5) * 0.01
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    return [t if t is None else t.cuda() for t in (ints(m, k, seed=seed, low=low), xs, ints(n, k, seed=seed + 1, low=low), ws, b)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 5, 16, 17, 32, 33, 64, 65, 130, 300, 1024])
@pytest.mark.parametrize("n, k", [(1, 1), (16, 128), (100, 63), (130, 2050), (520, 384), (2048, 5120)])
def test_product(dtype, m, n, k):
    args = case(m, n, k, dtype, bias=(m + n) % 2 == 0)
    check(linear_int8_batch_invariant(*args, dtype=dtype), *args, f"{m} x {n} x {k}")


@pytest.mark.parametrize("m, n, k", [(4096, 2048, 256), (2048, 1024, 1024), (1000, 3000, 128), (700, 600, 640), (257, 513, 2048)])
def test_large_products(m, n, k):
    args = case(m, n, k, torch.bfloat16)
    check(linear_int8_batch_invariant(*args), *args)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_the_longest_sums(m):
    """All products at their largest: 2^14 each, sums just below 2^31."""
    k = 131071
    x, w = torch.full((m, k), -128, dtype=I8).cuda(), torch.full((20, k), -128, dtype=I8).cuda()
    w[3] = 127
    ones = torch.ones(m, device="cuda"), torch.ones(20, device="cuda")
    out = linear_int8_batch_invariant(x, ones[0], w, ones[1], dtype=F32).cpu().double()
    want = torch.full((m, 20), 16384.0 * k, dtype=torch.float64)
    want[:, 3] = -128.0 * 127 * k
    assert torch.equal(out, want.float().double())


@pytest.mark.parametrize("m", [4, 64, 100, 513])
@pytest.mark.parametrize("k", [256, 200])
def test_a_row_alone_has_the_same_bits(m, k):
    x, xs, w, ws, b = case(m, 300, k, torch.bfloat16, seed=5)
    out = linear_int8_batch_invariant(x, xs, w, ws, b)
    for at in (slice(0, 1), slice(m - 2, m), slice(0, m // 2)):
        assert_bitwise(linear_int8_batch_invariant(x[at], xs[at], w, ws, b), out[at])


@pytest.mark.parametrize("m", [7, 100])
@pytest.mark.parametrize("k", [256, 130])
def test_layouts(m, k):
    """Rows and scales by strides, rows off 16 bytes, leading dimensions, a weight whose rows are columns."""
    x, xs, w, ws, b = case(m, 90, k, torch.float16, seed=7)
    want = linear_int8_batch_invariant(x, xs, w, ws, b, dtype=torch.float16)
    wide = torch.zeros(m, k + 33, dtype=I8, device="cuda")
    wide[:, 5:5 + k] = x
    tall = torch.zeros(90, k + 16, dtype=I8, device="cuda")
    tall[:, :k] = w
    strided = torch.stack([xs, xs], 1)[:, 1], torch.stack([ws, ws], 1)[:, 1], torch.stack([b, b], 1)[:, 1]
    for xx, ww in ((wide[:, 5:5 + k], tall[:, :k]), (x.t().contiguous().t(), w.t().contiguous().t()), (x, tall[:, :k])):
        assert_bitwise(linear_int8_batch_invariant(xx, strided[0], ww, strided[1], strided[2], dtype=torch.float16), want)
    got = linear_int8_batch_invariant(x.view(1, m, k), xs.view(1, m), w, ws, b, dtype=torch.float16)
    assert got.shape == (1, m, 90)
    assert_bitwise(got[0], want)
    assert_bitwise(linear_int8_batch_invariant(x[0], xs[0], w, ws, b, dtype=torch.float16), want[0])
    assert linear_int8_batch_invariant(x[:0], xs[:0], w, ws, b, dtype=torch.float16).shape == (0, 90)
    assert linear_int8_batch_invariant(x, xs, w[:0], ws[:0], b[:0], dtype=torch.float16).shape == (m, 0)


def test_broadcast_rows():
    x, xs, w, ws, b = case(1, 70, 256, torch.bfloat16, seed=9)
    many = linear_int8_batch_invariant(x.expand(100, 256), xs.expand(100), w, ws, b)
    assert_bitwise(many, linear_int8_batch_invariant(x, xs, w, ws, b).expand(100, 70))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, k", [(1, 1), (3, 7), (5, 64), (9, 511), (4, 1024), (3, 1025), (7, 2048), (2, 8192), (2, 8201), (2, 40003)])
def test_quantised_rows(dtype, rows, k):
    x = (torch.randn(rows, k, generator=torch.Generator().manual_seed(k)) * torch.logspace(-3, 2, rows).view(-1, 1)).to(dtype)
    q, scale = quantize_tokens_int8(x.cuda())
    want_q, want_scale = int8_rows(x)
    assert torch.equal(q.cpu(), want_q)
    assert_bitwise(scale.cpu(), want_scale)
    # off by half a step, and the roundings of x 127 / m
    off = (q.cpu().double() * scale.cpu().double().unsqueeze(-1) - x.double()).abs()
    assert bool((off <= (0.5 + 127 * 4 * 2.0**-24) * scale.cpu().double().unsqueeze(-1)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_the_ends(dtype):
    big, small, inf, nan = float(torch.finfo(dtype).max), float(torch.finfo(dtype).tiny), float("inf"), float("nan")
    x = torch.zeros(9, 40)
    x[1, 3] = big
    x[2] = -big
    x[3, 5] = small
    x[4, 7], x[5, 8], x[6, 9] = inf, -inf, nan
    x[7] = torch.arange(40) - 20.0
    x[8, 39] = 2.0**-120 if dtype != torch.float16 else 2.0**-24
    x = x.to(dtype)
    q, scale = quantize_tokens_int8(x.cuda())
    want_q, want_scale = int8_rows(x)
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(torch.isnan(scale.cpu()), torch.isnan(want_scale)) and int(torch.isnan(want_scale).sum()) == 3
    fine = ~torch.isnan(want_scale)
    assert_bitwise(scale.cpu()[fine], want_scale[fine])
    w = ints(6, 40, seed=3).cuda()
    out = linear_int8_batch_invariant(q, scale, w, torch.ones(6).cuda(), dtype=F32)
    assert torch.equal(torch.isnan(out.cpu()).all(1), torch.isnan(want_scale)) and torch.equal(torch.isnan(out.cpu()).any(1), torch.isnan(want_scale))


def test_quantised_layouts():
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    q, scale = quantize_tokens_int8(x)
    wide = torch.zeros(6, 401, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:301] = x
    for other in (wide[:, 1:301], x.t().contiguous().t()):
        q2, s2 = quantize_tokens_int8(other)
        assert torch.equal(q2, q) and torch.equal(s2, scale) and q2.is_contiguous()
    q3, s3 = quantize_tokens_int8(x.view(2, 3, 300))
    assert q3.shape == (2, 3, 300) and s3.shape == (2, 3) and torch.equal(q3.view(6, 300), q) and torch.equal(s3.view(6), scale)
    q4, s4 = quantize_tokens_int8(x[2])
    assert torch.equal(q4, q[2]) and s4.shape == () and torch.equal(s4, scale[2])
    assert quantize_tokens_int8(x[:0])[0].shape == (0, 300)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_linear_layer(dtype):
    """Quantised and multiplied, near the layer in full: each factor is off by at most half a step."""
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(20, 512, generator=g).to(dtype), torch.randn(70, 512, generator=g) * 0.05
    qw, ws = quantize_tokens_int8(w.cuda())
    q, s = quantize_tokens_int8(x.cuda())
    out = linear_int8_batch_invariant(q, s, qw, ws, dtype=dtype)
    check(out, q, s, qw, ws, None)
    full = x.double() @ w.double().t()
    dx, dw = 0.501 * s.cpu().double().view(-1, 1), 0.501 * ws.cpu().double().view(1, -1)
    bound = dx * w.double().abs().sum(1) + dw * x.double().abs().sum(1, keepdim=True) + 512 * dx * dw
    assert bool(((out.cpu().double() - full).abs() <= bound + HALF[dtype] * full.abs() + HALF[dtype] * bound).all())


@pytest.mark.parametrize("m, k, step", [(3, 200, 3 << 30), (40, 256, (1 << 27) + 16), (40, 200, (1 << 27) + 1)])
def test_far_rows(m, k, step):
    """Offsets past 32 bits, in each kernel."""
    args = case(m, 48, k, torch.bfloat16)
    x = torch.empty((m - 1) * step + k, dtype=I8, device="cuda").as_strided((m, k), (step, 1))
    x.copy_(args[0])
    want = linear_int8_batch_invariant(*args)
    assert_bitwise(linear_int8_batch_invariant(x, *args[1:]), want)
    q, steps = quantize_tokens_int8(args[0].to(torch.bfloat16))
    del x
    rows = torch.empty((m - 1) * (step // 2) + k, dtype=torch.bfloat16, device="cuda").as_strided((m, k), (step // 2, 1))
    rows.copy_(args[0])
    far = quantize_tokens_int8(rows)
    assert torch.equal(far[0], q) and torch.equal(far[1], steps)


@pytest.mark.parametrize("k", [128, 100])
def test_outputs_past_32_bits(k):
    m, n = 70000, 32768
    x, xs, w, ws, b = case(m, n, k, torch.bfloat16)
    out = linear_int8_batch_invariant(x, xs, w, ws, b)
    for rows in (slice(0, 3), slice(65530, 65540), slice(m - 2, m)):
        assert_bitwise(out[rows], linear_int8_batch_invariant(x[rows], xs[rows], w, ws, b))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, n, k", [(4, 40, 64), (24, 40, 128), (100, 130, 128), (100, 130, 130), (512, 2048, 256), (2100, 4100, 128)])
def test_large_rows_and_small_channels(dtype, m, n, k):
    """Products whose sum times the row's step is past 32-bit floats, and the result is not: steps as rows at the end of bfloat16 have."""
    x, xs, w, ws, b = case(m, n, k, dtype, seed=11)
    g = torch.Generator().manual_seed(12)
    xs = xs * torch.tensor([2.0**124, 2.0**123, 1.0, -(2.0**124)])[torch.randint(0, 4, (m,), generator=g)].cuda()  # (0.01 to 0.03 of them)
    ws = ws * torch.tensor([2.0**-118, 2.0**-117])[torch.randint(0, 2, (n,), generator=g)].cuda()
    x[1] = 0
    assert float(((x.double() @ w.double().t()).abs() * xs.double().abs().view(-1, 1)).max()) > 2.0**128
    out = linear_int8_batch_invariant(x, xs, w, ws, b, dtype=dtype)
    assert bool(torch.isfinite(out).all())
    check(out, x, xs, w, ws, b)
    assert_bitwise(linear_int8_batch_invariant(x[:3], xs[:3], w, ws, b, dtype=dtype), out[:3])
    # sums of 0 times what two large factors make; infinite and undefined steps and channels as before
    ws[0], ws[1], ws[2], xs[1] = 2.0**100, float("nan"), float("inf"), 2.0**126
    out = linear_int8_batch_invariant(x, xs, w, ws, b, dtype=dtype)
    assert bool((out[1, 0] == b[0]) & torch.isnan(out[1, 1]) & torch.isnan(out[1, 2]))
    assert_bitwise(out[1, 3:], b[3:])
    xs[1], xs[3] = float("inf"), float("nan")
    out = linear_int8_batch_invariant(x, xs, w, ws, b, dtype=dtype)
    assert bool(torch.isnan(out[1]).all() & torch.isnan(out[3]).all())
