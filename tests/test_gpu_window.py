"""Sliding-window attention with sinks against the 64-bit definition: dense, packed, masks, values, layouts."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import (check_cache_indices, sliding_window_attention_batch_invariant as window_attention,
                                 varlen_sliding_window_attention_batch_invariant as packed_attention)

from _decoder import assert_within, attend64, attention_bound, check_window, prompt_rounding, window_visible
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


def randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def check(batch, hq, hkv, lq, lk, d, dv, window, sinks, seed, dtype=BF16, scale=None):
    q, k, v = (randn(batch, h, n, x, seed=seed + i, dtype=dtype)
               for i, (h, n, x) in enumerate(((hq, lq, d), (hkv, lk, d), (hkv, lk, dv))))
    out = window_attention(q, k, v, window, sinks, scale=scale, enable_gqa=hq != hkv)
    assert out.shape == (batch, hq, lq, dv) and out.dtype == dtype
    for b in range(batch):
        check_window(out[b], q[b], k[b], v[b], window, sinks, scale, f"sample {b}")
    return q, k, v, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, dv", [(128, 128), (64, 64), (72, 72), (8, 8), (128, 64), (40, 104)])
@pytest.mark.parametrize("lq, lk, window, sinks", [
    (1, 1, 1, 0), (5, 5, 2, 1), (130, 130, 50, 4), (257, 257, 64, 0), (200, 333, 100, 3), (33, 33, None, 0), (1, 300, 70, 2),
    (140, 20, 8, 1),
])
def test_dense(dtype, d, dv, lq, lk, window, sinks):
    check(2, 2, 1, lq, lk, d, dv, window, sinks, 1, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (1, 64), (63, 1), (64, 64), (65, 0), (127, 5), (128, 128), (129, 0), (300, 2),
                                           (299, 400), (2**40, 0), (None, 7)])
def test_windows_and_sinks(dtype, window, sinks):
    check(1, 2, 2, 300, 300, 64, 64, window, sinks, 10, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d, dv", [(256, 256), (192, 128), (64, 136)])
def test_wide_heads(dtype, d, dv):
    check(1, 2, 1, 150, 170, d, dv, 60, 3, 20, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 2, 3, 4, 6, 8])
@pytest.mark.parametrize("d", [64, 88, 128, 256])
@pytest.mark.parametrize("lq", [50, 64, 65, 130])
def test_heads_of_a_group(dtype, group, d, lq):
    """Query heads that share a workgroup, with few rows and many."""
    if dtype == torch.float32 and d > 128:
        pytest.skip("float32 heads go up to 128")
    check(1, 2 * group, 2, lq, 170, d, d, 60, 3, 25, dtype)
    if d == 64 and group < 4:
        check(1, 2 * group, 2, lq, 170, d, d, None, 0, 26, dtype)  # a longer window takes another tile


@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("d", [72, 128])
def test_long_float32_prompts(group, d):
    q, k, v = (randn(1, h, 2050, d, seed=27 + h, dtype=torch.float32) for h in (group, 1, 1))
    out = window_attention(q, k, v, 100, 4, enable_gqa=True)
    for a in (0, 1000, 1900):  # a part of the rows, with the keys up to its last
        rows = slice(a, a + 150)
        check = out[0, :, rows], q[0, :, rows], k[0, :, :a + 150], v[0, :, :a + 150]
        check_window(*check, 100, 4, what=f"rows from {a}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group, lq", [(4, 200), (4, 40), (2, 200), (1, 200)])
def test_masked_values_with_heads_of_a_group(dtype, group, lq):
    q, k, v = (randn(1, h, n, 64, seed=28 + h, dtype=dtype) for h, n in ((2 * group, lq), (2, 200), (2, 200)))
    for at, bad in ((170, float("nan")), (190, float("inf")), (20, float("nan"))):
        k[:, :, at] = bad
        v[:, :, at + 1] = bad
    out = window_attention(q, k, v, 7, 2, enable_gqa=True)
    seen = torch.isnan(out[0]).any(-1)
    assert bool(seen.any()) and not bool(seen.all())
    first = 200 - lq
    for r in range(lq):  # a row is touched if and only if it sees one of the six
        p = first + r
        touched = any(0 <= p - x < 7 for at in (170, 190, 20) for x in (at, at + 1))
        if not touched:
            assert not bool(torch.isnan(out[0, :, r]).any()) and not bool(torch.isinf(out[0, :, r]).any()), f"row {r}"
    fine = torch.tensor([not any(0 <= first + r - x < 7 for at in (170, 190, 20) for x in (at, at + 1)) for r in range(lq)])
    clean = [torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (k, v)]
    for h in range(2 * group):
        parts = attend64(q[0, h], clean[0][0, h // group], clean[1][0, h // group], window_visible(lq, 200, 7, 2), 0.125)
        bound = attention_bound(dtype, *parts, 9, *prompt_rounding(dtype))
        assert_within(out[0, h][fine.cuda()], parts[0][fine], bound[fine], f"head {h}")


def test_longer_than_the_window_many_times():
    check(1, 4, 2, 2000, 2000, 64, 64, 130, 4, 30)


@pytest.mark.parametrize("scale", [0.0, -0.25, 3.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(scale, dtype):
    check(1, 1, 1, 70, 90, 64, 64, 40, 2, 40, dtype, scale=scale)


def pack(lengths_q, lengths_k, hq, hkv, d, dv, seed, dtype=BF16, tail_q=0, tail_k=0, index=torch.int32):
    tq, tk = sum(lengths_q) + tail_q, sum(lengths_k) + tail_k
    q, k, v = randn(1, tq, hq, d, seed=seed, dtype=dtype), randn(1, tk, hkv, d, seed=seed + 1, dtype=dtype), randn(
        1, tk, hkv, dv, seed=seed + 2, dtype=dtype)
    cu = [torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=index).cuda() for x in (lengths_q, lengths_k)]
    return q, k, v, *cu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_packed(dtype, index):
    """Sequences of no, one and many tokens; more and fewer keys than queries; rows behind the last one."""
    lq, lk = [5, 0, 129, 1, 200, 17, 0, 3], [5, 4, 129, 90, 260, 0, 0, 1]
    q, k, v, cu_q, cu_k = pack(lq, lk, 4, 2, 64, 72, 50, dtype, tail_q=140, tail_k=9, index=index)
    out = packed_attention(q, k, v, cu_q, cu_k, 60, 3)
    assert out.shape == (1, sum(lq) + 140, 4, 72)
    for s in range(len(lq)):
        a, b = sum(lq[:s]), sum(lk[:s])
        check_window(out[0, a:a + lq[s]].transpose(0, 1), q[0, a:a + lq[s]].transpose(0, 1), k[0, b:b + lk[s]].transpose(0, 1),
                     v[0, b:b + lk[s]].transpose(0, 1), 60, 3, what=f"sequence {s}")
    assert float(out[0, sum(lq):].abs().max()) == 0.0


def test_many_sequences():
    """More sequences than a wavefront looks through at a time."""
    lengths = [(7 * i) % 23 for i in range(150)]
    lengths[70] = 500
    q, k, v, cu, _ = pack(lengths, lengths, 2, 1, 64, 64, 60)
    out = packed_attention(q, k, v, cu, cu, 9, 1)
    for s in (0, 1, 62, 63, 64, 70, 127, 128, 149):
        a, b = sum(lengths[:s]), sum(lengths[:s + 1])
        check_window(out[0, a:b].transpose(0, 1), *(x[0, a:b].transpose(0, 1) for x in (q, k, v)), 9, 1, what=f"sequence {s}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq, lk, window, sinks", [
    (1, 1023, None, 0), (1, 1024, None, 0), (7, 1500, None, 0), (16, 9001, None, 0), (16, 3000, 1100, 4), (5, 3000, 990, 20),
    (33, 1055, None, 0), (33, 1056, None, 0), (64, 4097, None, 0), (64, 5000, 4090, 64), (3, 2000, 1, 1500), (16, 40, None, 0),
])
def test_few_rows_before_many_keys(dtype, lq, lk, window, sinks):
    """Both sides of the sizes at which the keys are cut into ranges."""
    for hq, hkv, d, dv in ((4, 2, 64, 64), (3, 1, 128, 72)):
        check(1, hq, hkv, lq, lk, d, dv, window, sinks, 80, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_of_wide_heads_before_many_keys(dtype):
    check(2, 4, 1, 20, 2000, 256, 200, None, 0, 81, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ranges_of_keys_joined(dtype):
    """Their bits in every batch and by strides; masked and infinite keys, values at the end of the range, a graph."""
    q, k, v = (randn(3, h, n, 64, seed=82 + h, dtype=dtype) for h, n in ((4, 20), (2, 3000), (2, 3000)))
    out = window_attention(q, k, v, 2500, 3, enable_gqa=True)
    for b in range(3):
        assert_bitwise(window_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], 2500, 3, enable_gqa=True)[0], out[b])
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert_bitwise(window_attention(*turned, 2500, 3, enable_gqa=True), out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = window_attention(q, k, v, 2500, 3, enable_gqa=True)
    for seed in range(3):
        q.copy_(randn(3, 4, 20, 64, seed=90 + seed, dtype=dtype))
        graph.replay()
        assert_bitwise(held, window_attention(q, k, v, 2500, 3, enable_gqa=True))
        torch.cuda.synchronize()
    # row 10 is at 2990 and sees keys from 491 on: key 490 and value 2995 must not reach it
    big = torch.where(v > 0, 0.99, 0.9).to(dtype) * torch.finfo(dtype).max
    clean = window_attention(q, k, big, 2500, 3, enable_gqa=True)
    assert bool(torch.isfinite(clean).all())
    check_window(clean[0], q[0], k[0], big[0], 2500, 3, what="the largest values")
    k[:, :, 490] = float("nan")
    v[:, :, 490] = float("inf")
    v[:, :, 2995] = float("nan")
    out = window_attention(q, k, v, 2500, 3, enable_gqa=True)
    assert bool(torch.isnan(out[:, :, :10]).all())  # they see key 490
    assert bool(torch.isnan(out[:, :, 15:]).all()) and not bool(torch.isnan(out[:, :, 10:15]).any())
    for t in (k, v):
        t[:, :, 490] = 0.0
        t[:, :, 2995] = 0.0
    check_window(out[0][:, 10:15], q[0][:, 10:15], k[0][:, :2995], v[0][:, :2995], 2500, 3, what="between them")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group, lq", [(1, 150), (2, 150), (4, 150), (4, 50)])
def test_a_row_keeps_its_bits_whatever_follows(dtype, group, lq):
    """Other queries, keys and values behind a row, far larger ones among them, in its tile and in its blocks."""
    q, k, v = (randn(1, h, n, 64, seed=66 + h, dtype=dtype) for h, n in ((2 * group, lq), (2, 200), (2, 200)))
    want = window_attention(q, k, v, 90, 3, enable_gqa=True)
    for last in (3, 31, 32, lq // 2, lq - 2):
        p = 200 - lq + last  # the row's position
        other = [t.clone() for t in (q, k, v)]
        other[0][:, :, last + 1:] = 7.0 * randn(1, 2 * group, lq - last - 1, 64, seed=70, dtype=dtype)
        for t in other[1:]:
            t[:, :, p + 1:] = 5.0 * randn(1, 2, 199 - p, 64, seed=71, dtype=dtype)
        out = window_attention(*other, 90, 3, enable_gqa=True)
        assert_bitwise(out[:, :, :last + 1], want[:, :, :last + 1], f"rows up to {last}")


@pytest.mark.parametrize("count", [61, 62, 63, 64, 4093, 4094, 4095, 5000])
def test_the_search_for_a_sequence(count):
    """Both sides of the counts at which the search takes another round, with empty sequences among the others."""
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 5, (count,), generator=g)
    lengths[count // 2] = 150
    lengths[-1] = 40
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    total = int(cu[-1])
    q, k, v = (randn(1, total + 37, h, 64, seed=61 + h) for h in (4, 1, 1))
    out = packed_attention(q, k, v, cu.cuda(), cu.cuda(), 3, 1)
    assert float(out[:, total:].abs().max()) == 0.0
    # the same from the definition for all rows at once: three keys of the window and the first one, in 64 bits
    place = torch.cat([torch.arange(n) for n in lengths.tolist()])
    first = torch.arange(total) - place
    at = torch.stack([torch.arange(total) - 2, torch.arange(total) - 1, torch.arange(total), first], 1)
    seen = torch.stack([place >= 2, place >= 1, place >= 0, place >= 3], 1)
    kk, vv = (t[0, :total, 0].cpu().double()[at.clamp(min=0)] for t in (k, v))
    qq = q[0, :total].cpu().double()
    s = torch.einsum("thd,tjd->thj", qq, kk) * 0.125
    w = torch.softmax(s.masked_fill(~seen.unsqueeze(1), float("-inf")), -1)
    o, mag = (torch.einsum("thj,tjd->thd", w, x) for x in (vv, vv.abs()))
    err = 66 * 2.0**-24 * 0.125 * torch.einsum("thd,tjd->thj", qq.abs(), kk.abs()).amax(-1, keepdim=True)
    assert_within(out[0, :total], o, attention_bound(BF16, o, mag, err, torch.zeros_like(o), 4, *prompt_rounding(BF16)))


@pytest.mark.parametrize("at", [0, 3000, 4999])
def test_bad_offsets_among_many_are_reported(at):
    cu = torch.arange(5001, dtype=torch.int32)
    q = randn(1, 5000, 2, 64, seed=65)
    packed_attention(q, q, q, cu.cuda(), cu.cuda(), 3, 1)
    check_cache_indices()
    for which in range(2):
        bad = cu.clone()
        bad[at + (which == 0 or at == 0)] -= 2  # below the offset in front of it, or below zero
        offsets = [cu.cuda(), cu.cuda()]
        offsets[which] = bad.cuda()
        packed_attention(q, q, q, *offsets, 3, 1)
        with pytest.raises(RuntimeError, match="outside its tensor"):
            check_cache_indices()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bits_do_not_depend_on_the_batch(dtype):
    lengths = [300, 1, 0, 129, 700, 128]
    q, k, v, cu, _ = pack(lengths, lengths, 4, 2, 64, 64, 70, dtype)
    out = packed_attention(q, k, v, cu, cu, 100, 4)
    for s, n in enumerate(lengths):
        a = sum(lengths[:s])
        if n == 0:
            continue
        one = [x[:, a:a + n] for x in (q, k, v)]
        alone = packed_attention(*one, cu.new_tensor([0, n]), cu.new_tensor([0, n]), 100, 4)
        assert_bitwise(alone, out[:, a:a + n], f"sequence of {n} alone")
        dense = window_attention(*(x.transpose(1, 2) for x in one), 100, 4, enable_gqa=True)
        assert_bitwise(dense.transpose(1, 2), out[:, a:a + n], f"sequence of {n}, dense")
        twice = window_attention(*(x.transpose(1, 2).expand(3, -1, -1, -1) for x in one), 100, 4, enable_gqa=True)
        assert_bitwise(twice[2], dense[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_keys_and_values_never_reach_a_row(dtype, bad):
    """One key and value of each kind in the middle: rows that do not see them keep their bits, in the same
    blocks of rows and keys as those that do."""
    q, k, v = (randn(1, 2, 300, 64, seed=80 + i, dtype=dtype) for i in range(3))
    window, sinks, at = 37, 2, 150
    clean = window_attention(q, k, v, window, sinks)
    rows = torch.arange(300).cuda()
    unseen = (rows < at) | (rows >= at + window)
    for what in ("key", "value", "both"):
        k2, v2 = k.clone(), v.clone()
        if what != "value":
            k2[:, :, at] = bad
        if what != "key":
            v2[:, :, at] = bad
        out = window_attention(q, k2, v2, window, sinks)
        assert torch.isfinite(out[:, :, unseen]).all(), what
        scale = clean[:, :, unseen].double().abs().max()
        # rows that were computed again, key by key, differ by their roundings only
        assert float((out[:, :, unseen].double() - clean[:, :, unseen].double()).abs().max()) <= 2 * scale * {
            torch.float32: 1e-5, torch.float16: 2.0**-9, BF16: 2.0**-6}[dtype], what
        if what == "value" or bad != bad:
            assert not torch.isfinite(out[:, :, ~unseen]).any() if what != "key" else torch.isnan(out[:, :, ~unseen]).all()
    # a value in one column only
    v2 = v.clone()
    v2[:, :, at, 5] = bad
    out = window_attention(q, k, v2, window, sinks)
    assert not torch.isfinite(out[:, :, ~unseen, 5]).any()
    assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all() and torch.isfinite(out[:, :, unseen]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_at_the_end_of_the_range(dtype):
    """Sums of values that overflow 32 bits, where the weighted mean does not."""
    q, k = (randn(1, 1, 100, 64, seed=90 + i, dtype=dtype) for i in range(2))
    v = torch.full((1, 1, 100, 64), 3.0e38, dtype=dtype).cuda()
    out = window_attention(q * 0.01, k, v, 64, 0)
    assert torch.isfinite(out).all()
    assert float((out.double() / 3.0e38 - 1).abs().max()) <= 2.0**-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_key_far_above_many(dtype):
    n, d = 2000, 64
    q, k = torch.zeros(1, 1, 130, d, dtype=dtype).cuda(), torch.zeros(1, 1, n, d, dtype=dtype).cuda()
    q[..., 0] = 8.0
    k[0, 0, 1900, 0] = 9.6875
    v = randn(1, 1, n, d, seed=95, dtype=dtype).abs() + 1
    out = window_attention(q, k, v, 1900, 4)
    check_window(out[0], q[0], k[0], v[0], 1900, 4)


def test_scores_of_minus_infinity():
    q, k, v = (randn(1, 1, 70, 64, seed=97 + i) for i in range(3))
    q[..., 0] = 1.0
    k2 = k.clone()
    k2[:, :, 10:30, 0] = float("-inf")
    out = window_attention(q, k2, v, 8, 0)
    assert float(out[0, 0, 17:30].abs().max()) == 0.0  # these rows see only such keys
    assert torch.isfinite(out).all()


def test_layouts():
    """Heads or tokens first in memory, slices of one projection, rows off the 16 bytes."""
    qkv = randn(2, 140, (4 + 2 + 2) * 64, seed=100)
    q, k, v = (x.unflatten(-1, (-1, 64)).transpose(1, 2) for x in qkv.split([256, 128, 128], -1))
    out = window_attention(q, k, v, 50, 4, enable_gqa=True)
    want = window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 50, 4, enable_gqa=True)
    assert out.transpose(1, 2).is_contiguous() and want.is_contiguous()
    assert_bitwise(out, want)
    odd = [torch.nn.functional.pad(x, (1, 2))[..., 1:65] for x in (q, k, v)]
    assert_bitwise(window_attention(*odd, 50, 4, enable_gqa=True), want)
    spread = [torch.stack([x, x], -1)[..., 0] for x in (q, k, v)]
    assert_bitwise(window_attention(*spread, 50, 4, enable_gqa=True), want)


def test_bad_offsets_are_reported_and_stay_inside():
    lengths = [40, 130, 20]
    q, k, v, cu, _ = pack(lengths, lengths, 2, 1, 64, 64, 110)
    want = packed_attention(q, k, v, cu, cu, 30, 2)
    for bad_q, bad_k, same in (
        ([0, 40, 30, 190], [0, 40, 170, 190], 30), ([0, 40, 170, 1000], [0, 40, 170, 190], 170),
        ([5, 40, 170, 190], [0, 40, 170, 190], 0), ([0, 40, 170, 190], [0, 40, 170, 191], 170),
        ([0, 40, 170, 190], [0, 40, -3, 190], 40), ([0, -(2**31), 170, 2**31 - 1], [0, 40, 170, 190], 0),
    ):
        out = packed_attention(q, k, v, torch.tensor(bad_q, dtype=torch.int32).cuda(),
                               torch.tensor(bad_k, dtype=torch.int32).cuda(), 30, 2)
        with pytest.raises(RuntimeError, match="outside its tensor"):
            check_cache_indices()
        assert torch.isfinite(out).all()
        assert_bitwise(out[:, :same], want[:, :same])


def test_empty_calls():
    q, k, v = (randn(1, 2, n, 64, seed=120) for n in (4, 0, 0))
    assert float(window_attention(q, k, v, 3).abs().max()) == 0.0  # no keys
    assert window_attention(q[:, :, :0], q, q, 3).shape == (1, 2, 0, 64)
    assert window_attention(q[:0], k[:0], v[:0], 3).shape == (0, 2, 4, 64)
    cu = torch.zeros(1, dtype=torch.int64).cuda()
    assert float(packed_attention(q, q, q, cu, cu, 3).abs().max()) == 0.0  # rows, and no sequence


def test_graph_replays_with_other_offsets():
    lengths = [100, 130, 20]
    q, k, v, cu, _ = pack(lengths, lengths, 2, 1, 64, 64, 130)
    packed_attention(q, k, v, cu, cu, 30, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(q, k, v, cu, cu, 30, 2)
    for i, offsets in enumerate(([0, 1, 2, 3], [0, 0, 250, 250], [0, 100, 230, 250])):
        cu.copy_(torch.tensor(offsets))
        q.copy_(randn(*q.shape, seed=140 + i))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert_bitwise(got, packed_attention(q, k, v, cu, cu, 30, 2), f"replay {i}")


def test_a_gradient_is_refused():
    q = randn(1, 1, 8, 64, seed=150).requires_grad_()
    with pytest.raises(ValueError, match="no_grad"):
        window_attention(q, q.detach(), q.detach(), 3)
    with torch.no_grad():
        assert window_attention(q, q, q, 3).shape == q.shape
