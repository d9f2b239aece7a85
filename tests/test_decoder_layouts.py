"""Layouts that the decoder operators take: strides of dimensions with one element mean nothing."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _native as nat
from batch_invariant_ops import decoder

from _tol import assert_bitwise

BF16 = torch.bfloat16


def test_host_check_of_strides_that_are_not_used():
    """The entry point's layout check (status 2) comes before that of the pointers (status 1, for a null query)."""
    L, p = nat.load(require_gpu=False), 256

    def win(nseq=2, lk=5, hkv=2, k=(320, 128, 64), v=(320, 128, 64), at=p, cu=None):
        return L.biops_window_attention(2, nseq, 4, hkv, 5, lk, 64, 64, None, 640, 256, 64, at, *k, p, *v, p, 640, 256, 64, cu, 0, 1, cu,
                                        0, 1, 4, 0, 1.0, p, None, 0, None)

    assert win() == 1
    assert win(k=(324, 128, 64)) == 2 and win(nseq=1, k=(324, 128, 64)) == 1
    assert win(v=(320, 129, 64)) == 2 and win(lk=1, v=(320, 129, 64)) == 1 and win(lk=1, k=(320, 1 << 40, 64)) == 1
    assert win(k=(320, 128, 68)) == 2 and win(hkv=1, k=(320, 128, 68)) == 1
    assert win(k=(3, 128, 64), cu=p) == 1  # packed rows have no batch
    assert win(nseq=1, lk=1, hkv=1, k=(1, 1, 1), v=(3, 5, 7)) == 1 and win(nseq=1, lk=1, hkv=1, at=p + 4) == 2


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


def odd(t, dim):
    """The same values of a size-1 dimension with a stride of its own."""
    strides = list(t.stride())
    strides[dim] = 515
    return t.as_strided(t.shape, strides)


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_dimensions_of_one_element(python, monkeypatch):
    if python:
        monkeypatch.setattr(decoder, "_tensor_module", False)
        monkeypatch.setattr(decoder, "_direct", lambda: False)
    flat = randn(3, 515, seed=1)
    rows = flat[:, :512].view(3, 4, 2, 64).transpose(1, 2)  # samples 515 elements apart
    q = randn(3, 2, 6, 64, seed=2)
    want = bio.sliding_window_attention_batch_invariant(q, rows, rows, 3)
    assert_bitwise(want, bio.sliding_window_attention_batch_invariant(q, rows.contiguous(), rows.contiguous(), 3))
    assert_bitwise(bio.sliding_window_attention_batch_invariant(q[:1], rows[:1], rows[:1], 3), want[:1])
    for heads, keys, dim in ((2, 4, 0), (1, 4, 1), (2, 1, 2), (1, 1, 1), (1, 1, 2)):  # one sample, one head, one key
        k, v = randn(1, heads, keys, 64, seed=3), randn(1, heads, keys, 64, seed=4)
        want = bio.sliding_window_attention_batch_invariant(q[:1], k, v, 3, enable_gqa=True)
        got = bio.sliding_window_attention_batch_invariant(odd(q[:1], 0), odd(k, dim), odd(v, dim), 3, enable_gqa=True)
        assert_bitwise(got, want)
        if dim != 0:
            continue
        cu = [torch.tensor([0, n], dtype=torch.int32).cuda() for n in (6, keys)]
        k, v, one = (x.transpose(1, 2) for x in (k, v, q[:1]))
        want = bio.varlen_sliding_window_attention_batch_invariant(one, k, v, *cu, 3)
        assert_bitwise(bio.varlen_sliding_window_attention_batch_invariant(odd(one, 0), odd(k, 0), odd(v, 0), *cu, 3), want)


@pytest.mark.gpu
def test_one_page_one_head_one_row():
    """The same for the caches' operators and the rotation."""
    q, kc, vc = randn(1, 1, 64, seed=5), randn(1, 1, 1, 64, seed=6), randn(1, 1, 1, 64, seed=7)
    table, lengths = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([[0]], [1]))
    want = bio.paged_attention_batch_invariant(q, kc, vc, table, lengths)
    k2, v2 = odd(odd(kc, 0), 2), odd(odd(vc, 1), 2)
    assert_bitwise(bio.paged_attention_batch_invariant(odd(q, 1), k2, v2, odd(table, 1), odd(lengths, 0)), want)
    new = randn(1, 1, 64, seed=8)
    bio.paged_cache_write(odd(new, 0), odd(new, 1), k2, v2, odd(torch.tensor([0]).cuda(), 0))
    assert_bitwise(kc.view(-1), new.view(-1))
    assert_bitwise(vc.view(-1), new.view(-1))
    p = torch.tensor([[3]]).cuda()
    want = bio.multi_axis_rotary(new, new, p, (32,))
    for a, b in zip(bio.multi_axis_rotary(odd(new, 0), odd(new, 1), odd(p, 1), (32,)), want):
        assert_bitwise(a, b)
    bio.check_cache_indices()


def brute(a, b):
    def places(t):
        at = torch.full((1,), t.storage_offset())
        for n, s in zip(t.shape, t.stride()):
            at = (at.view(-1, 1) + torch.arange(n) * s).flatten()
        return set(at.tolist())

    return bool(places(a) & places(b))


def pairs():
    """Views of one allocation, with whether they are fit for keys and values."""
    base = torch.zeros(4000)

    def at(offset, shape, strides):
        return base.as_strided(shape, strides, offset)

    kv = base[:1536].view(2, 3, 4, 4, 16)
    yield kv[0], kv[1], True
    yield kv[1], kv[0], True
    yield kv[0], kv[0], False
    for dim in range(1, 5):
        two = base[:1536].view(*[(3, 4, 4, 16)[i] for i in range(dim - 1)], 2, *[(3, 4, 4, 16)[i] for i in range(dim - 1, 4)])
        yield two.select(dim - 1, 0), two.select(dim - 1, 1), True
        yield two.select(dim - 1, 1), two.select(dim - 1, 0), True
    fused = base[:3 * 4 * 2 * 40].view(3, 4, 2, 40)
    yield fused[..., :16], fused[..., 16:], True
    yield fused[..., :24], fused[..., 24:], True
    yield fused[..., :24], fused[..., 16:], False
    yield fused[..., 8:16], fused[..., :16], False
    heads = base[:3 * 4 * 6 * 16].view(3, 4, 6, 16)
    yield heads[:, :, :3], heads[:, :, 3:], True
    yield heads[:, :, :4], heads[:, :, 2:], False
    yield heads[:, :, 0::2], heads[:, :, 1::2], True
    pages = base[:3 * 4 * 2 * 16].view(3, 4, 2, 16)
    yield pages[:2], pages[1:], False
    yield pages[:1], pages[2:], True
    yield pages[:, :2], pages[:, 2:], True
    yield pages[:1, :, :1], pages[:1, :, 1:], True
    turned = base[:768].view(2, 3, 2, 4, 16).transpose(2, 3)
    yield turned[0], turned[1], True
    yield at(0, (2, 2, 2, 8), (64, 16, 8, 1)), at(40, (2, 2, 2, 8), (64, 16, 8, 1)), False
    yield at(0, (2, 2, 2, 8), (64, 16, 8, 1)), at(32, (2, 2, 2, 8), (64, 16, 8, 1)), True


def test_caches_that_share_memory_are_recognised():
    for i, (a, b, fit) in enumerate(pairs()):
        assert decoder._share(a, b) is not fit, i
        if fit:
            assert not brute(a, b), i  # what is taken never overlaps
    assert not decoder._share(torch.zeros(2, 2, 2, 8), torch.zeros(2, 2, 2, 8))
    assert not decoder._share(torch.zeros(0, 2, 2, 8), torch.zeros(0, 2, 2, 8))


@pytest.mark.gpu
def test_shared_caches_are_refused_and_interleaved_ones_written():
    slots = torch.tensor([5, 0, 11]).cuda()
    for i, (a, b, fit) in enumerate(pairs()):
        if a.shape[2] != b.shape[2] or a.shape[:3] != b.shape[:3]:
            continue
        base = torch.zeros(4000, dtype=BF16).cuda()
        kc, vc = (base.as_strided(t.shape, t.stride(), t.storage_offset()) for t in (a, b))
        k, v = (randn(3, t.shape[2], t.shape[3], seed=i + j) for j, t in enumerate((a, b)))
        at = slots % (kc.shape[0] * kc.shape[1])
        if not fit:
            with pytest.raises(ValueError, match="share memory"):
                bio.paged_cache_write(k, v, kc, vc, at)
            continue
        bio.paged_cache_write(k, v, kc, vc, at)
        for r, s in enumerate(at.tolist()):
            if s in at.tolist()[r + 1:]:
                continue
            assert_bitwise(kc[s // kc.shape[1], s % kc.shape[1]], k[r])
            assert_bitwise(vc[s // kc.shape[1], s % kc.shape[1]], v[r])
    bio.check_cache_indices()


@pytest.mark.gpu
def test_values_that_are_a_part_of_the_keys():
    """The same elements of the same rows: one cache for both."""
    slots = torch.tensor([5, 0, 11]).cuda()
    for part in (slice(0, 64), slice(0, 48), slice(16, 64), slice(8, 56)):
        kc, k = torch.zeros(3, 4, 2, 64, dtype=BF16).cuda(), randn(3, 2, 64, seed=30 + part.stop)
        bio.paged_cache_write(k, k[..., part], kc, kc[..., part], slots)
        assert_bitwise(kc.flatten(0, 1)[slots], k)
        assert int((kc != 0).any(-1).any(-1).sum()) == 3
        bio.paged_cache_write(k[..., part], k, kc[..., part], kc, slots.flip(0))
        assert_bitwise(kc.flatten(0, 1)[slots.flip(0)], k)
        for other in (k.clone()[..., part], k[..., slice(part.start + 8, part.stop + 8)] if part.stop <= 56 else k.flip(0)[..., part]):
            with pytest.raises(ValueError, match="share memory"):
                bio.paged_cache_write(k, other, kc, kc[..., part], slots)
    bio.check_cache_indices()
