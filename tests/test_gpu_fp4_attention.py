"""Attention of one new token over a cache in 4 bits, against the 64-bit definition on the values that the bits stand for."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import check_cache_indices, paged_attention_fp4_batch_invariant

from _decoder import assert_within, attend64, attention_bound, check_token
from _served import from_fp4, to_fp4
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
HALVES = (BF16, F16)


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


class Batch:
    """Sequences of their own lengths in pages of their own, and the values of the cache."""

    def __init__(self, lengths, hq, hkv, d, dv, page, dtype=BF16, seed=1, size=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.dtype = list(lengths), dtype
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + 2
        order = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(lengths), max(counts) + 1), -(1 << 20), dtype=torch.int32)
        for b, n in enumerate(counts):
            self.table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        k = (torch.randn(pages, page, hkv, d, generator=g) * size).to(dtype)
        v = torch.randn(pages, page, hkv, dv, generator=g).to(dtype)
        self.q = torch.randn(len(lengths), hq, d, generator=g).to(dtype).cuda()
        caches = [*to_fp4(k), *to_fp4(v)]
        self.values = [from_fp4(*caches[:2]), from_fp4(*caches[2:])]
        self.caches = [c.cuda() for c in caches]
        self.table, self.lens = self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda()

    def run(self, **kw):
        return paged_attention_fp4_batch_invariant(self.q, *self.caches, self.table, self.lens, **kw)

    def check(self, out, window=None, sinks=0, scale=None, only=None):
        for b in range(len(self.lengths)) if only is None else only:
            check_token(out[b], self.q[b], *self.values, self.table[b].cpu(), self.lengths[b], window, sinks, scale, f"sequence {b}")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("hq, hkv, d, dv, page", [
    (16, 4, 128, 128, 16), (8, 2, 64, 64, 64), (4, 4, 32, 32, 1), (6, 2, 96, 64, 7), (7, 1, 64, 128, 100), (3, 3, 160, 96, 16),
    (40, 2, 128, 64, 32), (4, 2, 256, 256, 16), (2, 1, 32, 256, 5), (2, 2, 224, 32, 16), (5, 1, 128, 192, 33)])
def test_lengths(dtype, hq, hkv, d, dv, page):
    """From nothing to several chunks, tiles and pages that end anywhere; empty sequences among others."""
    batch = Batch([1, 0, 31, 32, 33, 127, 128, 129, 300, 513, 0, 2, 64], hq, hkv, d, dv, page, dtype)
    out = batch.run()
    batch.check(out)
    assert int((out[[1, 10]] != 0).sum()) == 0


@pytest.mark.parametrize("lengths", [[2047], [2048, 2049, 4096], [4097, 5000, 1]])
def test_long_sequences(lengths):
    batch = Batch(lengths, 4, 2, 128, 128, 16)
    batch.check(batch.run())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 4), (37, 0), (100, 3), (600, 64), (1 << 40, 5)])
@pytest.mark.parametrize("d", [64, 128])
def test_windows(dtype, window, sinks, d):
    batch = Batch([1, 40, 700, 3, 1300], 8, 2, d, d, 16, dtype, seed=2)
    batch.check(batch.run(window=window, sinks=sinks), window, sinks)


def test_pages_without_a_visible_key_are_not_read():
    batch = Batch([500, 700], 4, 2, 64, 64, 16, seed=3)
    out = batch.run(window=40, sinks=4)
    batch.table[:, 1:25] = -1
    assert_bitwise(batch.run(window=40, sinks=4), out)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 3.0])
def test_scales(scale):
    batch = Batch([5, 200, 33], 4, 2, 64, 64, 16, seed=4)
    batch.check(batch.run(scale=scale), scale=scale)


def test_large_scores():
    """A softmax of one key, however large the scores."""
    batch = Batch([50, 300], 4, 2, 128, 128, 16, seed=5, size=3e4)
    batch.check(batch.run())


def test_values_at_the_end_of_the_range():
    """Sums of the largest values leave the range of 32 bits, means do not."""
    batch = Batch([200, 1000], 2, 1, 64, 64, 16, seed=6)
    batch.caches[3].fill_(252)  # 2^125
    batch.values[1] = from_fp4(batch.caches[2], batch.caches[3])
    batch.check(batch.run())


def test_a_block_that_is_not_finite():
    """NaN reaches the rows that see it, and no others: behind the end, outside of the window, on no page of the sequence."""
    batch = Batch([100, 70, 130], 4, 2, 64, 64, 16, seed=7)
    clean = batch.run(window=40, sinks=2)
    at = lambda b, j: (int(batch.table[b, j // 16]), j % 16)  # noqa: E731
    batch.caches[3][at(0, 20)] = 255  # (out of sight)
    batch.caches[1][at(0, 20)] = 255
    batch.caches[1][at(0, 105)] = 255  # behind the end
    batch.caches[3][at(0, 105)] = 255
    batch.caches[3][at(1, 69)] = 255  # seen: in all values
    batch.caches[1][at(2, 1)][0, 0] = 255  # seen: the first head's keys
    out = batch.run(window=40, sinks=2)
    assert_bitwise(out[0], clean[0])
    assert bool(torch.isnan(out[1]).all())
    assert bool(torch.isnan(out[2, :2]).all())
    assert_bitwise(out[2, 2:], clean[2, 2:])


def test_what_lies_behind_a_sequence_does_not_matter():
    batch = Batch([33, 100, 7], 4, 2, 128, 64, 16, seed=8)
    want = batch.run()
    for b, n in enumerate(batch.lengths):
        for j in range(n, -(-n // 16) * 16):
            for c in batch.caches:
                c[int(batch.table[b, j // 16]), j % 16] = 255
    assert_bitwise(batch.run(), want)


@pytest.mark.parametrize("count", [1, 5, 130, 200])
def test_a_sequence_alone_has_the_same_bits(count):
    lengths = [(37 * i) % 400 for i in range(count)]
    lengths[count // 2] = 2500
    batch = Batch(lengths, 8, 2, 64, 64, 16, seed=9)
    out = batch.run()
    for b in {0, count // 2, count - 1, count // 3}:
        alone = paged_attention_fp4_batch_invariant(batch.q[b:b + 1], *batch.caches, batch.table[b:b + 1], batch.lens[b:b + 1])
        assert_bitwise(alone[0], out[b], f"sequence {b}")
    batch.check(out, only={count // 2, 0})


def test_bound_of_the_lengths():
    batch = Batch([40, 100, 3], 4, 2, 64, 64, 16, seed=10)
    want = batch.run()
    assert_bitwise(batch.run(max_length=100), want)
    out = batch.run(max_length=99)
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    assert int((out[1] != 0).sum()) == 0
    assert_bitwise(out[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("lengths", [[40, 100, 3], [3000, 1000, 2100]])
def test_bad_pages_and_lengths(lengths):
    batch = Batch(lengths, 4, 2, 64, 64, 16, seed=11)
    want = batch.run()
    batch.table[1, 0] = batch.caches[0].shape[0]
    batch.lens[2] = -1
    out = batch.run()
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    check_cache_indices()
    assert int((out[1:] != 0).sum()) == 0
    assert_bitwise(out[0], want[0])


def test_layouts():
    """Heads before slots in memory, rows off 16 bytes, codes and scales in one allocation, wide queries, 64-bit tables."""
    batch = Batch([33, 0, 270], 6, 3, 96, 64, 16, seed=12)
    want = batch.run()
    caches = []
    for c in batch.caches:
        wide = torch.zeros(c.shape[0], c.shape[2], c.shape[1], c.shape[3] + 3, dtype=torch.uint8, device="cuda")
        part = wide[..., 1:1 + c.shape[3]].transpose(1, 2)
        part.copy_(c)
        caches.append(part)
    q = torch.zeros(3, 6, 200, dtype=BF16, device="cuda")[..., 7:103]
    q.copy_(batch.q)
    table = torch.zeros(3, 2 * batch.table.shape[1], dtype=torch.int64, device="cuda")[:, ::2]
    table.copy_(batch.table)
    assert_bitwise(paged_attention_fp4_batch_invariant(q, *caches, table, batch.lens.long()), want)


def test_empty_batches():
    batch = Batch([5], 4, 2, 64, 64, 16)
    out = paged_attention_fp4_batch_invariant(batch.q[:0], *batch.caches, batch.table[:0], batch.lens[:0])
    assert out.shape == (0, 4, 64)
    out = paged_attention_fp4_batch_invariant(batch.q, *batch.caches, batch.table[:, :0], batch.lens * 0)
    assert int((out != 0).sum()) == 0


def test_it_is_the_attention_of_the_values():
    """Near what the attention over 16-bit pages gives for the values that are read back."""
    batch = Batch([500, 20], 8, 2, 128, 128, 16, seed=13)
    slots = torch.arange(batch.caches[0].shape[0] * 16, device="cuda")
    k, v = (x.view(-1, 16, 2, 128) for x in bio.paged_cache_read_fp4(*batch.caches, slots))
    other = bio.paged_attention_batch_invariant(batch.q, k, v, batch.table, batch.lens)
    batch.check(other)
    batch.check(batch.run())


def test_far_offsets():
    """Pages whose byte offsets are past 31 bits."""
    page, heads, d = 64, 2, 256
    pages = (1 << 31) // (page * heads * d // 2) + 3
    g = torch.Generator().manual_seed(14)
    rows = [torch.randn(2, page, heads, d, generator=g).to(BF16) for _ in range(2)]
    small = [*to_fp4(rows[0]), *to_fp4(rows[1])]
    caches = []
    for c in small:
        big = torch.zeros(pages, *c.shape[1:], dtype=torch.uint8, device="cuda")
        big[[pages - 1, 0]] = c.cuda()
        caches.append(big)
    q = torch.randn(1, 4, d, generator=g).to(BF16).cuda()
    out = paged_attention_fp4_batch_invariant(q, *caches, torch.tensor([[pages - 1, 0]], device="cuda"), torch.tensor([100], device="cuda"))
    check_token(out[0], q[0], from_fp4(*small[:2]), from_fp4(*small[2:]), torch.tensor([0, 1]), 100)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("hq, hkv", [(16, 1), (17, 1), (32, 2), (33, 1)])
@pytest.mark.parametrize("d, dv", [(32, 256), (256, 160), (256, 256), (96, 192)])
def test_many_query_heads_and_wide_values(dtype, hq, hkv, d, dv):
    """Workgroups with 16 query heads of the widest outputs, alone and in chunks that are joined."""
    batch = Batch([1, 0, 130, 700], hq, hkv, d, dv, 16, dtype, seed=15)
    batch.check(batch.run())
    only = Batch([40], hq, hkv, d, dv, 16, dtype, seed=16)
    only.check(only.run())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n, far", [(3000, 4.0), (40000, 9.0), (40000, 15.0), (200000, 16.0)])
def test_one_key_far_above_many(dtype, n, far):
    """The others' small weights are most of what its small value leaves."""
    page, d = 64, 64
    pages = -(-n // page)
    k, v = torch.zeros(pages, page, 1, d), torch.full((pages, page, 1, d), 2.0)
    k[0, 3, 0, 0], v[0, 3, 0] = 4.0, 0.5
    caches = [*to_fp4(k.to(dtype)), *to_fp4(v.to(dtype))]
    q = torch.zeros(1, 2, d, dtype=dtype)
    q[0, :, 0] = torch.tensor([far / 4, far / 8])
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    out = paged_attention_fp4_batch_invariant(q.cuda(), *(c.cuda() for c in caches), table.cuda(), torch.tensor([n]).cuda(), scale=1.0)
    check_token(out[0], q[0], from_fp4(*caches[:2]), from_fp4(*caches[2:]), table[0], n, scale=1.0)


@pytest.mark.parametrize("n", [40, 128, 900, 5000])
@pytest.mark.parametrize("far", [11.0, 14.0, 15.0, 16.5, 18.0])
def test_small_weights_of_fp16_count(n, far):
    """One key far above many, with values of 0: the output is what the others' weights of e^-far say.  They are held times 2^7 in
    two parts of fp16: to 2^-22 of themselves, or to half of its smallest step over 2^7, 2^-32 of the largest."""
    page, d = 16, 64
    pages = -(-n // page)
    k, v = torch.zeros(pages, page, 1, d), torch.full((pages, page, 1, d), 1536.0)
    k[0, 3, 0, 0], v[0, 3, 0] = 4.0, 0.0
    caches = [*to_fp4(k.to(F16)), *to_fp4(v.to(F16))]
    q = torch.zeros(1, 2, d, dtype=F16)
    q[0, :, 0] = torch.tensor([far / 4, far / 4 - 0.0625])
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    out = paged_attention_fp4_batch_invariant(q.cuda(), *(c.cuda() for c in caches), table.cuda(), torch.tensor([n]).cuda(), scale=1.0)
    keys, values = (from_fp4(*caches[i:i + 2]).flatten(0, 1)[:n, 0] for i in (0, 2))
    for h in range(2):
        parts = attend64(q[:, h], keys, values, torch.ones(1, n, dtype=torch.bool), 1.0)
        assert_within(out[:, h], parts[0], attention_bound(F16, *parts, n, 2.0**-22, 2.0**-32), f"head {h}")
