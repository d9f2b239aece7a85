"""Rows on their way into a cache in pages, rotated and in 4 bits: against the operators they join, and against the format's
definition."""

from __future__ import annotations

import importlib

import pytest
import torch

from batch_invariant_ops import (
    check_cache_indices,
    multi_axis_rotary,
    paged_attention_fp4_batch_invariant,
    paged_cache_read_fp4,
    paged_cache_write,
    paged_cache_write_fp4,
    rotary_cache_write,
)

from _served import POWERS, from_fp4, to_fp4
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALVES = (BF16, F16)


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


def randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def empty4(pages, page, heads, d, dv, seed=0):
    """Caches full of what earlier requests left."""
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (pages, page, heads, n), generator=g).to(torch.uint8).cuda() for n in (d // 2, d // 32, dv // 2, dv // 32)]


def slots_for(tokens, total, seed, repeats=True):
    g = torch.Generator().manual_seed(seed)
    slots = torch.randperm(total, generator=g)[:tokens]
    if tokens > 6:
        slots[tokens // 2] = -1 - tokens  # padding
        if repeats:
            slots[3] = slots[5]
            slots[tokens - 1] = slots[1]
    return slots


def same(a, b, what=""):
    assert torch.equal(a.cpu(), b.cpu()), f"{what}: {int((a.cpu() != b.cpu()).sum())} bytes differ"


def written4(caches, k, v, slots):
    """The four tensors after the rows' writes, one by one on the CPU."""
    kc, ks, vc, vs = (c.cpu().clone() for c in caches)
    page = kc.shape[1]
    (kq, ke), (vq, ve) = to_fp4(k), to_fp4(v)
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < kc.shape[0] * page:
            for cache, rows in ((kc, kq), (ks, ke), (vc, vq), (vs, ve)):
                cache[s // page, s % page] = rows[r]
    return kc, ks, vc, vs


# (heads, kv heads, head size, value size, sections, neighbours)
LAYOUTS = [(16, 4, 128, 128, (64,), False), (8, 2, 64, 64, (10, 11, 11), True), (4, 4, 96, 64, (20,), False), (3, 1, 32, 96, (5, 2), True),
           (5, 5, 64, 32, (3,), False), (2, 1, 160, 32, (80,), False), (0, 2, 64, 64, (32,), False)]
PLAIN_ONLY = [(16, 16, 72, 80, (18, 18), True), (7, 7, 70, 6, (35,), False), (2, 1, 9, 3, (4,), False)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", LAYOUTS + PLAIN_ONLY)
@pytest.mark.parametrize("tokens", [1, 7, 333, 1100])
def test_append_is_rotation_and_write(dtype, layout, tokens):
    hq, hk, d, dv, sections, neighbours = layout
    page, pages = 7, -(-2 * tokens // 7)
    q, k, v = randn(tokens, hq, d, seed=1, dtype=dtype), randn(tokens, hk, d, seed=2, dtype=dtype), randn(tokens, hk, dv, seed=3, dtype=dtype)
    kc, vc = randn(pages, page, hk, d, seed=4, dtype=dtype), randn(pages, page, hk, dv, seed=5, dtype=dtype)
    positions = torch.randint(0, 100000, (len(sections), tokens), generator=torch.Generator().manual_seed(6)).cuda()
    slots = slots_for(tokens, pages * page, 7).cuda()
    kw = dict(base=500000.0, interleaved_axes=neighbours, interleaved_pairs=neighbours)
    want_q, want_k = (multi_axis_rotary(x, None, positions, sections, **kw) for x in (q, k))
    want = kc.clone(), vc.clone()
    paged_cache_write(want_k, v, *want, slots)
    got = rotary_cache_write(q, k, v, kc, vc, slots, positions, sections, **kw)
    assert_bitwise(got, want_q)
    assert_bitwise(kc, want[0])
    assert_bitwise(vc, want[1])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tokens", [1, 7, 333, 1100])
def test_append_in_four_bits(dtype, layout, tokens):
    hq, hk, d, dv, sections, neighbours = layout
    page, pages = 16, -(-2 * tokens // 16)
    q, k, v = randn(tokens, hq, d, seed=1, dtype=dtype), randn(tokens, hk, d, seed=2, dtype=dtype), randn(tokens, hk, dv, seed=3, dtype=dtype)
    caches = empty4(pages, page, hk, d, dv)
    positions = torch.randint(0, 100000, (len(sections), tokens), generator=torch.Generator().manual_seed(6)).to(torch.int32).cuda()
    slots = slots_for(tokens, pages * page, 7)
    kw = dict(interleaved_axes=neighbours, interleaved_pairs=neighbours)
    want_q, want_k = (multi_axis_rotary(x, None, positions, sections, **kw) for x in (q, k))
    want = written4(caches, want_k, v, slots)
    got = rotary_cache_write(q, k, v, caches[0], caches[2], slots.cuda(), positions, sections, key_scales=caches[1], value_scales=caches[3], **kw)
    assert_bitwise(got, want_q)
    for name, a, b in zip(("keys", "key scales", "values", "value scales"), caches, want):
        same(a, b, name)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("heads, d, dv, page", [(4, 128, 128, 16), (1, 32, 64, 1), (3, 96, 32, 100), (2, 256, 512, 5)])
@pytest.mark.parametrize("tokens", [1, 9, 1031])
def test_write_and_read_back(dtype, heads, d, dv, page, tokens):
    pages = -(-2 * tokens // page)
    # rows of very different sizes
    size = torch.logspace(-6, 3, tokens).view(-1, 1, 1).to(dtype).cuda()
    k, v = randn(tokens, heads, d, seed=11, dtype=dtype) * size, randn(tokens, heads, dv, seed=12, dtype=dtype) * size
    caches = empty4(pages, page, heads, d, dv)
    slots = slots_for(tokens, pages * page, 13)
    want = written4(caches, k, v, slots)
    paged_cache_write_fp4(k, v, *caches, slots.cuda().to(torch.int32))
    for a, b in zip(caches, want):
        same(a, b)
    back = slots.clone()
    if tokens > 6:
        back[0] = -5
    rk, rv = paged_cache_read_fp4(*caches, back.cuda(), dtype=dtype)
    for got, codes, scales in ((rk, want[0], want[1]), (rv, want[2], want[3])):
        values = from_fp4(codes.flatten(0, 1)[back.clamp(min=0)], scales.flatten(0, 1)[back.clamp(min=0)])
        values[back < 0] = 0.0
        assert torch.equal(got.cpu().double(), values)


@pytest.mark.parametrize("dtype", HALVES)
def test_borders_of_the_format(dtype):
    """Ties, the largest and smallest numbers of the type, zeros of both signs, infinities and NaN."""
    low, high = POWERS[dtype]
    top = float(torch.finfo(dtype).max)
    rows = []
    for e in (low, low + 1, -3, 0, high - 1, high):
        p = 2.0**e
        rows.append([x * p for x in (6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6)] * 2)
        rows.append([x * p for x in (7 if e < high else 6, 0.26, 0.74, 1.24, 1.76, 2.49, 3.51, 5.03)] * 4)
        rows.append([x * p for x in (7.03 if e < high else 6, 0.0, -0.0, 3.0)] * 8)
    rows += [[0.0] * 32, [-0.0] * 32, [top] * 32, [-top, 1.0] * 16, [float(torch.finfo(dtype).smallest_normal)] * 32,
             [2.0**-24 if dtype == F16 else 2.0**-133, 0.0] * 16, [1.0] * 31 + [float("inf")], [float("-inf")] + [0.0] * 31,
             [1.0] * 16 + [float("nan")] + [2.0] * 15]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    k = x.view(-1, 1, 32).cuda()
    caches = empty4(len(rows), 1, 1, 32, 32)
    slots = torch.arange(len(rows)).cuda()
    paged_cache_write_fp4(k, k.clone(), *caches, slots)
    want = to_fp4(k)
    same(caches[0].flatten(0, 1), want[0])
    same(caches[1].flatten(0, 1), want[1])
    rk, rv = paged_cache_read_fp4(*caches, slots, dtype=dtype)
    assert_bitwise(rk, rv)
    values = from_fp4(*want)
    got = rk.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(values)) and int(torch.isnan(values).sum()) == 3 * 32
    fine = ~torch.isnan(values)
    assert torch.equal(got[fine], values[fine])
    # the format's promise: off by at most the block's power (which is at most the largest element / 3.5), short of its ends
    power = 2.0 ** (want[1].double() - 127)
    inside = fine & (x.view(-1, 1, 32).double().abs().amax(-1, keepdim=True) <= 7 * power.unsqueeze(-1)[..., 0])
    off = (got - k.cpu().double()).abs()
    assert bool((off <= power.unsqueeze(-1)[..., 0])[inside].all())


def test_rows_and_caches_by_strides():
    """One projection's output, two leading dimensions, codes and scales in one allocation, slots by strides."""
    d, hk = 64, 2
    qkv = randn(2, 5, 8 * d, seed=20)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv.split([4 * d, 2 * d, 2 * d], -1))
    one = torch.zeros(3, 8, hk, 2 * (d // 2 + d // 32) + 1, dtype=torch.uint8, device="cuda")
    caches = one[..., :32], one[..., 32:34], one[..., 35:67], one[..., 67:69]
    slots = torch.randperm(24, generator=torch.Generator().manual_seed(21))[:20].cuda().view(5, 4)[:, :2].t()
    positions = torch.arange(30, device="cuda").view(5, 2, 3).permute(2, 1, 0)
    want_q, want_k = multi_axis_rotary(q, k, positions, (12, 10, 10))
    want = written4(caches, want_k.reshape(10, hk, d), v.reshape(10, hk, d), slots.reshape(-1))
    got = rotary_cache_write(q, k, v, caches[0], caches[2], slots, positions, (12, 10, 10), key_scales=caches[1], value_scales=caches[3])
    assert_bitwise(got, want_q)
    for a, b in zip(caches, want):
        same(a, b)
    assert int(one[..., 34].sum()) == 0
    # one token, without leading dimensions
    single = rotary_cache_write(q[0, 0], k[0, 0], v[0, 0], caches[0], caches[2], slots[0, 0], positions[:, 0, 0], (12, 10, 10),
                                key_scales=caches[1], value_scales=caches[3])
    assert_bitwise(single, want_q[0, 0])


def test_empty_calls():
    kc, vc = randn(2, 4, 2, 64, seed=30), randn(2, 4, 2, 64, seed=31)
    before = kc.clone()
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    out = rotary_cache_write(kc.new_empty(0, 4, 64), kc.new_empty(0, 2, 64), kc.new_empty(0, 2, 64), kc, vc, none, none.view(1, 0), (32,))
    assert out.shape == (0, 4, 64)
    caches = empty4(2, 4, 2, 64, 64)
    left = [c.clone() for c in caches]
    paged_cache_write_fp4(kc.new_empty(0, 2, 64), kc.new_empty(0, 2, 64), *caches, none)
    k, v = paged_cache_read_fp4(*caches, none)
    assert k.shape == v.shape == (0, 2, 64)
    # a cache without pages: queries are rotated all the same
    q, rows = randn(3, 4, 64, seed=32), randn(3, 2, 64, seed=33)
    minus, p = torch.full((3,), -1, device="cuda"), torch.arange(3, device="cuda").view(1, 3)
    got = rotary_cache_write(q, rows, rows.clone(), kc[:0].clone(), vc[:0].clone(), minus, p, (32,))
    assert_bitwise(got, multi_axis_rotary(q, None, p, (32,)))
    assert_bitwise(kc, before)
    for a, b in zip(caches, left):
        same(a, b)


@pytest.mark.parametrize("tokens", [64, 1025, 20001, 70001])
def test_of_rows_for_one_slot_the_last_stays(tokens):
    """Inside a workgroup's rows, across workgroups and across launches."""
    slots = torch.randint(0, 40, (tokens,), generator=torch.Generator().manual_seed(40))
    slots[:8] = 3
    k, v = randn(tokens, 1, 32, seed=41), randn(tokens, 1, 32, seed=42)
    q, p = randn(tokens, 1, 32, seed=43), torch.arange(tokens, device="cuda").view(1, -1)
    rq, rk = multi_axis_rotary(q, k, p, (16,))
    caches = empty4(5, 8, 1, 32, 32)
    want = written4(caches, rk, v, slots)
    for _ in range(3):
        got = rotary_cache_write(q, k, v, caches[0], caches[2], slots.cuda(), p, (16,), key_scales=caches[1], value_scales=caches[3])
        assert_bitwise(got, rq)
        for a, b in zip(caches, want):
            same(a, b)


@pytest.mark.parametrize("tokens", [1500, 66000])
def test_far_apart_rows_for_one_slot(tokens):
    """Pages in any order, one repeated slot for each distance between its rows, padding and slots past the cache."""
    g = torch.Generator().manual_seed(44)
    pages = -(-tokens // 8) + 3
    slots = (torch.randperm(pages, generator=g).view(-1, 1) * 8 + torch.arange(8)).view(-1)[:tokens]
    for i, far in enumerate((1, 3, 4, 15, 16, 255, 256, 257, 1023, 1400)):
        slots[i * 5 + far] = slots[i * 5]
    slots[-1] = slots[7]
    slots[700:720] = -1
    slots[725] = pages * 8
    k, v = randn(tokens, 1, 32, seed=45), randn(tokens, 1, 32, seed=46)
    q, p = randn(tokens, 2, 32, seed=47), torch.arange(tokens, device="cuda").view(1, -1)
    rq, rk = multi_axis_rotary(q, k, p, (16,))
    kc, vc = randn(pages, 8, 1, 32, seed=48), randn(pages, 8, 1, 32, seed=49)
    want = kc.clone(), vc.clone()
    paged_cache_write(rk, v, *want, slots.cuda())
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    got = rotary_cache_write(q, k, v, kc, vc, slots.cuda().to(torch.int32), p, (16,))
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    assert_bitwise(got, rq)
    assert_bitwise(kc, want[0])
    assert_bitwise(vc, want[1])


def test_slots_past_the_cache_are_left_out_and_reported():
    caches = empty4(2, 4, 2, 32, 32)
    want = written4(caches, k := randn(3, 2, 32, seed=50), k, torch.tensor([8, 2**40, 5]))
    paged_cache_write_fp4(k, k.clone(), *caches, torch.tensor([8, 2**40, 5]).cuda())
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    check_cache_indices()
    for a, b in zip(caches, want):
        same(a, b)
    rk, rv = paged_cache_read_fp4(*caches, torch.tensor([5, 8, -1]).cuda())
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    assert int((rk[1:] != 0).sum()) == int((rv[1:] != 0).sum()) == 0
    assert torch.equal(rk[0].cpu().double(), from_fp4(*to_fp4(k))[2])


def test_autograd_knows_of_a_write():
    kc, vc = randn(2, 4, 2, 64, seed=60), randn(2, 4, 2, 64, seed=61)
    k = randn(3, 2, 64, seed=62)
    before = kc._version, vc._version
    args = torch.arange(3).cuda(), torch.arange(3).cuda().view(1, 3), (32,)
    rotary_cache_write(k.clone(), k, k.clone(), kc, vc, *args)
    assert (kc._version, vc._version) == (before[0] + 1, before[1] + 1)
    caches = empty4(2, 4, 2, 64, 64)
    before = [c._version for c in caches]
    paged_cache_write_fp4(k, k.clone(), *caches, args[0])
    assert [c._version for c in caches] == [x + 1 for x in before]
    needs = k.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        rotary_cache_write(k.clone(), needs, k, kc, vc, *args)
    with torch.no_grad():
        rotary_cache_write(k.clone(), needs, k, kc, vc, *args)


def test_rows_inside_the_caches_are_refused():
    kc, vc = randn(2, 4, 2, 64, seed=70), randn(2, 4, 2, 64, seed=71)
    args = torch.arange(4).cuda(), torch.arange(4).cuda().view(1, 4), (32,)
    with pytest.raises(ValueError, match="memory of the caches"):
        rotary_cache_write(kc[0].clone(), kc[0], vc[0].clone(), kc, vc, *args)
    with pytest.raises(ValueError, match="must not share"):
        rotary_cache_write(kc[0].clone(), kc[0].clone(), vc[0].clone(), kc, kc, *args)


def test_far_offsets():
    """A slot whose byte offset is past 32 bits (in 4 bits past 2^31), and its scales."""
    page, heads, d = 64, 2, 256
    pages = (1 << 31) // (page * heads * d // 2) + 3
    kc, vc = (torch.zeros(pages, page, heads, d // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, page, heads, d // 32, dtype=torch.uint8, device="cuda") for _ in range(2))
    k, v = randn(4, heads, d, seed=80), randn(4, heads, d, seed=81)
    slots = torch.tensor([0, pages * page - 1, pages * page - 70, 5], device="cuda")
    p = torch.arange(4, device="cuda").view(1, 4)
    rotary_cache_write(k.clone(), k, v, kc, vc, slots, p, (0,), key_scales=ks, value_scales=vs)
    for rows, codes, scales in ((k, kc, ks), (v, vc, vs)):
        want = to_fp4(rows)
        same(codes.flatten(0, 1)[slots], want[0])
        same(scales.flatten(0, 1)[slots], want[1])
    rk, rv = paged_cache_read_fp4(kc, ks, vc, vs, slots)
    assert torch.equal(rk.cpu().double(), from_fp4(*to_fp4(k))) and torch.equal(rv.cpu().double(), from_fp4(*to_fp4(v)))


def far(t, step):
    """A copy of t whose first dimension has a stride of `step` elements."""
    inner = torch.empty(t.shape[1:]).stride()
    size = (t.shape[0] - 1) * step + t[0].numel()
    return torch.empty(size, dtype=t.dtype, device="cuda").as_strided(t.shape, (step, *inner)).copy_(t)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("without_module", [False, True])
def test_far_rows_and_pages(four, without_module, request):
    """Offsets past 32 bits of new rows and of pages; with and without the host module."""
    if without_module:
        served = importlib.import_module("batch_invariant_ops.served")
        kept = served.decoder._tensor_module
        request.addfinalizer(lambda: setattr(served.decoder, "_tensor_module", kept))
        served.decoder._tensor_module = False
    q, k, v = (randn(3, 2, 64, seed=90 + i) for i in range(3))
    slots = torch.tensor([8, 1, 5], device="cuda")
    p = torch.tensor([[4, 0, 9]], device="cuda")
    if four:
        near = empty4(3, 3, 2, 64, 64)
    else:
        near = [randn(3, 3, 2, 64, seed=95 + i) for i in range(2)]
    away = [far(c, (5 << 30) // (2 * c.element_size())) for c in near]

    def write(q, k, v, caches):
        scales = dict(key_scales=caches[1], value_scales=caches[3]) if four else {}
        kc, vc = (caches[0], caches[2]) if four else caches
        return rotary_cache_write(q, k, v, kc, vc, slots, p, (32,), **scales)

    want = write(q, k, v, near)
    got = write(far(q, 5 << 29), far(k, 5 << 29), far(v, 5 << 29), away)
    assert_bitwise(got, want)
    for a, b in zip(away, near):
        assert torch.equal(a, b)
    if four:
        for a, b in zip(paged_cache_read_fp4(*away, slots), paged_cache_read_fp4(*near, slots)):
            assert_bitwise(a, b)
        table = torch.tensor([[2, 0, 1]], device="cuda")
        length = torch.tensor([9], device="cuda")
        assert_bitwise(paged_attention_fp4_batch_invariant(q[:1], *away, table, length), paged_attention_fp4_batch_invariant(q[:1], *near, table, length))
