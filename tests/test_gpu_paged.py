"""The cache in pages: writes, and attention of one new token per sequence against the 64-bit definition."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import check_cache_indices, paged_attention_batch_invariant, paged_cache_write

from _decoder import assert_within, attend64, attention_bound, check_token
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


def randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# -------------------------------------------------------------------------------- writes ----
def written(cache, rows, slots):
    """The cache after the rows' writes, one by one on the CPU."""
    out = cache.cpu().clone()
    page = out.shape[1]
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < out.shape[0] * page:
            out[s // page, s % page] = rows[r].cpu()
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, dv, page, heads", [(128, 128, 16, 4), (64, 64, 64, 2), (72, 80, 100, 3), (8, 24, 1, 1), (70, 6, 7, 5),
                                                (1, 3, 3, 2), (192, 128, 16, 1)])
@pytest.mark.parametrize("tokens", [1, 7, 8, 9, 300])
def test_write(dtype, d, dv, page, heads, tokens):
    pages = -(-2 * tokens // page)
    k, v = randn(tokens, heads, d, seed=1, dtype=dtype), randn(tokens, heads, dv, seed=2, dtype=dtype)
    kc, vc = randn(pages, page, heads, d, seed=3, dtype=dtype), randn(pages, page, heads, dv, seed=4, dtype=dtype)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[:tokens]
    slots[tokens // 2] = -1 - tokens  # padding
    want_k, want_v = written(kc, k, slots), written(vc, v, slots)
    paged_cache_write(k, v, kc, vc, slots.cuda().to(torch.int32 if tokens % 2 else torch.int64))
    assert_bitwise(kc.cpu(), want_k)
    assert_bitwise(vc.cpu(), want_v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, dv, page, heads", [(128, 128, 16, 4), (72, 80, 100, 3), (70, 6, 7, 5), (1, 3, 3, 2), (256, 300, 64, 9),
                                                (8, 0, 4, 1), (512, 512, 8, 3)])
@pytest.mark.parametrize("tokens", [1024, 1031])
def test_write_of_many_rows(dtype, d, dv, page, heads, tokens):
    """Several rows of a workgroup, rows shorter and longer than its threads, slots that repeat, scattered and padding."""
    pages = -(-2 * tokens // page)
    k, v = randn(tokens, heads, d, seed=21, dtype=dtype), randn(tokens, heads, dv, seed=22, dtype=dtype)
    kc, vc = randn(pages, page, heads, d, seed=23, dtype=dtype), randn(pages, page, heads, dv, seed=24, dtype=dtype)
    g = torch.Generator().manual_seed(25)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[100:400] = torch.arange(300) + 11  # a prompt
    slots[torch.randint(0, tokens, (64,), generator=g)] = -1
    slots[::97] = slots[torch.randint(0, tokens, (len(slots[::97]),), generator=g)]
    slots[40:44] = 5  # neighbours, and the rest of their workgroup padding
    slots[44:48] = -1
    want_k, want_v = written(kc, k, slots), written(vc, v, slots)
    paged_cache_write(k, v, kc, vc, slots.cuda())
    assert_bitwise(kc.cpu(), want_k)
    assert_bitwise(vc.cpu(), want_v)


def test_write_from_and_into_views():
    """Rows from one projection's output, caches as halves of one allocation, slots by strides."""
    qkv = randn(2, 5, 8 * 64, seed=6)
    k, v = qkv[..., 256:384].view(2, 5, 2, 64), qkv[..., 384:].view(2, 5, 2, 64)
    both = randn(6, 2, 4, 2, 64, seed=7)
    slots = torch.randperm(24, generator=torch.Generator().manual_seed(8))[:20].cuda().view(5, 4)[:, :2].t()
    want_k = written(both[:, 0], k.reshape(10, 2, 64), slots.reshape(-1))
    want_v = written(both[:, 1], v.reshape(10, 2, 64), slots.reshape(-1))
    paged_cache_write(k, v, both[:, 0], both[:, 1], slots)
    assert_bitwise(both[:, 0].cpu(), want_k)
    assert_bitwise(both[:, 1].cpu(), want_v)


@pytest.mark.parametrize("tokens", [64, 20001])
def test_of_rows_for_one_slot_the_last_stays(tokens):
    """Inside a workgroup's rows, across workgroups and across launches."""
    g = torch.Generator().manual_seed(9)
    slots = torch.randint(0, 40, (tokens,), generator=g)
    slots[:8] = 3
    k, v = randn(tokens, 1, 32, seed=10), randn(tokens, 1, 32, seed=11)
    kc, vc = randn(5, 8, 1, 32, seed=12), randn(5, 8, 1, 32, seed=13)
    want = [written(c, x, slots) for c, x in ((kc, k), (vc, v))]
    for _ in range(3):
        paged_cache_write(k, v, kc, vc, slots.cuda())
        assert_bitwise(kc.cpu(), want[0])
        assert_bitwise(vc.cpu(), want[1])


def test_empty_writes():
    kc = randn(2, 4, 2, 8, seed=14)
    before = kc.clone()
    paged_cache_write(kc.new_empty(0, 2, 8), kc.new_empty(0, 2, 8), kc, kc.clone(), torch.empty(0, dtype=torch.int64).cuda())
    empty = kc.new_empty(0, 4, 2, 8)
    paged_cache_write(randn(3, 2, 8, seed=15), randn(3, 2, 8, seed=16), empty, empty.clone(), torch.full((3,), -1).cuda())
    assert_bitwise(kc, before)


def test_slots_past_the_cache_are_left_out_and_reported():
    kc = randn(2, 4, 2, 8, seed=17)
    before = kc.clone()
    k = randn(3, 2, 8, seed=18)
    paged_cache_write(k, k, kc, kc.clone(), torch.tensor([8, 2**40, 5]).cuda())
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    check_cache_indices()
    assert_bitwise(kc[1, 1], k[2])
    kc[1, 1] = before[1, 1]
    assert_bitwise(kc, before)


@pytest.mark.parametrize("heads_in_front", [False, True])
def test_autograd_knows_of_a_write(heads_in_front):
    """By both host paths: a cache that a graph has saved cannot change unnoticed."""
    kc = randn(2, 4, 2, 8, seed=31)
    vc = randn(2, 4, 2, 8, seed=32)
    k = randn(1, 3, 2, 8, seed=33) if heads_in_front else randn(3, 2, 8, seed=33)  # (four dimensions: in Python)
    w = torch.ones_like(kc, requires_grad=True)
    loss = (kc * w).sum()
    before = kc._version, vc._version
    paged_cache_write(k, k, kc, vc, torch.arange(3).cuda().view(k.shape[:-2]))
    assert (kc._version, vc._version) == (before[0] + 1, before[1] + 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        kc = torch.zeros(2, 4, 2, 8, dtype=BF16, device="cuda")
        paged_cache_write(k, k, kc, kc.clone(), torch.arange(3).cuda().view(k.shape[:-2]))
        assert_bitwise(kc[0, :3], k.view(3, 2, 8))


def test_a_page_is_copied():
    kc, vc = randn(4, 4, 2, 8, seed=34), randn(4, 4, 2, 16, seed=35)
    want = kc[1].clone(), vc[1].clone()
    paged_cache_write(kc[1], vc[1], kc, vc, torch.arange(8, 12).cuda())
    assert_bitwise(kc[2], want[0])
    assert_bitwise(vc[2], want[1])
    assert_bitwise(kc[1], want[0])


def test_a_gradient_is_refused():
    kc = randn(2, 4, 2, 8, seed=19)
    k = randn(3, 2, 8, seed=20).requires_grad_()
    with pytest.raises(ValueError, match="no_grad"):
        paged_cache_write(k, k.detach(), kc, kc.clone(), torch.arange(3).cuda())
    with torch.no_grad():
        paged_cache_write(k, k.detach(), kc, kc.clone(), torch.arange(3).cuda())
    assert_bitwise(kc[0, :3], k.detach())


# ----------------------------------------------------------------------------- attention ----
def batch(lengths, hkv, d, dv, page, seed, dtype=BF16, spare=3, index=torch.int32):
    """Caches whose unused slots and pages hold NaN, a table whose unused entries point nowhere."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), max(counts + [1])), -(2**31) if index == torch.int32 else 2**40, dtype=index)
    kc = torch.full((pages, page, hkv, d), float("nan"), dtype=dtype)
    vc = torch.full((pages, page, hkv, dv), float("nan"), dtype=dtype)
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            table[b, i] = order.pop()
            m = min(page, n - i * page)
            kc[table[b, i], :m] = torch.randn(m, hkv, d, generator=g).to(dtype)
            vc[table[b, i], :m] = torch.randn(m, hkv, dv, generator=g).to(dtype)
    return kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lengths, dtype=index).cuda()


def check(lengths, hq, hkv, d, dv, page, seed, dtype=BF16, index=torch.int32, **kw):
    kc, vc, table, lens = batch(lengths, hkv, d, dv, page, seed, dtype, index=index)
    q = randn(len(lengths), hq, d, seed=seed + 1, dtype=dtype)
    out = paged_attention_batch_invariant(q, kc, vc, table, lens, **kw)
    assert out.shape == (len(lengths), hq, dv) and out.dtype == dtype
    kw.pop("max_length", None)
    for b, n in enumerate(lengths):
        check_token(out[b], q[b], kc, vc, table[b], n, what=f"sequence {b} of {n}", **kw)
    return q, kc, vc, table, lens, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, hkv, d, dv, page", [
    (16, 4, 128, 128, 16), (4, 4, 64, 64, 64), (16, 16, 72, 72, 32), (8, 1, 128, 64, 7), (17, 1, 80, 128, 16),
    (35, 1, 8, 8, 1), (4, 2, 256, 256, 128), (2, 1, 192, 128, 16), (2, 2, 64, 256, 100), (7, 1, 256, 16, 33),
])
def test_token_attention(dtype, hq, hkv, d, dv, page):
    check([0, 1, 31, 32, 33, 64, 127, 128, 129, 257, 700], hq, hkv, d, dv, page, 100, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 4), (32, 0), (100, 1), (128, 4), (124, 4), (129, 64), (600, 700), (5000, 3)])
def test_token_attention_with_a_window(dtype, window, sinks):
    check([0, 1, 5, 32, 33, 101, 128, 200, 333, 1000], 8, 2, 64, 64, 16, 200, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_long_sequences(index):
    """Both sides of the lengths at which chunks grow, and of the most chunks."""
    check([1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8192, 20000, 32767, 32768, 32769, 70001, 3], 4, 1, 64, 64, 16, 300, index=index)


@pytest.mark.parametrize("count", [2, 3, 64, 65, 127, 128, 129, 150])
def test_batches_of_many_sequences(count):
    """Both sides of the batches whose chunks are listed."""
    lengths = [(37 * i) % 300 for i in range(count)]
    lengths[count - 2] = 1500
    lengths[count // 2] = 0
    q, kc, vc, table, lens, out = check(lengths, 2, 1, 64, 64, 16, 360)
    for b in {0, 1, count - 2, count - 1}:
        assert_bitwise(paged_attention_batch_invariant(q[b:b + 1], kc, vc, table[b:b + 1], lens[b:b + 1])[0], out[b])
    if count < 10:
        return
    bad = lens.clone()
    bad[count - 3] = -1
    again = paged_attention_batch_invariant(q, kc, vc, table, bad)
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()
    assert float(again[count - 3].abs().max()) == 0.0
    assert_bitwise(again[:count - 3], out[:count - 3])


def test_tables_of_every_width():
    """The most chunks that a table allows, at the widths where it changes; the lengths are the same."""
    lengths = [128, 1, 77]
    kc, vc, table, lens = batch(lengths, 2, 64, 64, 16, 350)
    q = randn(3, 4, 64, seed=351)
    want = paged_attention_batch_invariant(q, kc, vc, table, lens)
    for width in (8, 9, 64, 65, 256, 257, 512, 2048, 2049, 5000):
        wide = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
        wide[:, :8] = table[:, :8]
        assert_bitwise(paged_attention_batch_invariant(q, kc, vc, wide, lens), want, f"{width} pages")


def test_pages_behind_the_window_are_not_read():
    lengths = [500, 90, 64]
    kc, vc, table, lens = batch(lengths, 2, 64, 64, 16, 400)
    q = randn(3, 4, 64, seed=401)
    want = paged_attention_batch_invariant(q, kc, vc, table, lens, window=50, sinks=3)
    free = table.clone()
    free[0, 1:(500 - 50) // 16] = -1  # only the sinks' page and the window's stay
    free[1, 1:(90 - 50) // 16] = 2**30
    assert_bitwise(paged_attention_batch_invariant(q, kc, vc, free, lens, window=50, sinks=3), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bits_do_not_depend_on_the_batch(dtype):
    lengths = [300, 1, 9000, 0, 2500, 129, 128]
    kc, vc, table, lens = batch(lengths, 2, 128, 128, 16, 500, dtype)
    q = randn(len(lengths), 8, 128, seed=501, dtype=dtype)
    out = paged_attention_batch_invariant(q, kc, vc, table, lens)
    for b, n in enumerate(lengths):
        width = max(1, -(-n // 16))
        alone = paged_attention_batch_invariant(q[b:b + 1], kc, vc, table[b:b + 1, :width].contiguous(), lens[b:b + 1])
        assert_bitwise(alone[0], out[b], f"sequence of {n}")
        assert_bitwise(paged_attention_batch_invariant(q[b:b + 1], kc, vc, table[b:b + 1], lens[b:b + 1], max_length=n)[0], out[b])
    # nor on what pages hold it, or how large they are
    again = batch(lengths, 2, 128, 128, 48, 500, dtype)
    j = [torch.arange(n).cuda() for n in lengths]
    kc2, vc2, table2, _ = again
    for b, n in enumerate(lengths):
        kc2[table2[b].long()[j[b] // 48], j[b] % 48] = kc[table[b].long()[j[b] // 16], j[b] % 16]
        vc2[table2[b].long()[j[b] // 48], j[b] % 48] = vc[table[b].long()[j[b] // 16], j[b] % 16]
    assert_bitwise(paged_attention_batch_invariant(q, kc2, vc2, table2, lens), out)
    for _ in range(3):
        assert_bitwise(paged_attention_batch_invariant(q, kc, vc, table, lens), out)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0, 1e-30])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(scale, dtype):
    check([0, 1, 40, 300], 4, 2, 64, 64, 16, 600, dtype, scale=scale, window=250, sinks=2)


def test_layouts():
    """Queries of one projection, caches that share an allocation or have heads in front, tables by strides."""
    lengths = [70, 200, 5]
    kc, vc, table, lens = batch(lengths, 2, 64, 64, 16, 700)
    q = randn(3, 4, 64, seed=701)
    want = paged_attention_batch_invariant(q, kc, vc, table, lens)
    wide = randn(3, 8 * 64, seed=702)
    wide[:, 64:320] = q.view(3, 256)
    both = torch.stack([kc, vc], 1)
    turned = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc)]
    padded = [torch.nn.functional.pad(c, (1, 6))[..., 1:65] for c in (kc, vc)]  # rows off the 16 bytes
    wide_table = torch.stack([table, table + 1], 2)[..., 0]
    for caches in ((both[:, 0], both[:, 1]), turned, padded):
        assert_bitwise(paged_attention_batch_invariant(wide[:, 64:320].view(3, 4, 64), *caches, wide_table,
                                                       torch.stack([lens, lens], 1)[:, 0]), want)
    assert_bitwise(paged_attention_batch_invariant(q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, table, lens), want)


def test_offsets_past_32_bits():
    """The last pages of caches of 5 GiB each (2.6e9 elements)."""
    pages, page, hkv, d = 40000, 64, 8, 128
    kc = torch.zeros(pages, page, hkv, d, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    lengths = [150, 64]
    table = torch.tensor([[pages - 1, 0, pages - 3], [pages - 2, -1, -1]], dtype=torch.int32).cuda()
    rows = [(randn(150, hkv, d, seed=801), randn(150, hkv, d, seed=802)), (randn(64, hkv, d, seed=803), randn(64, hkv, d, seed=804))]
    for b, n in enumerate(lengths):
        j = torch.arange(n).cuda()
        paged_cache_write(*rows[b], kc, vc, table[b].long()[j // page] * page + j % page)
    q = randn(2, 16, d, seed=805)
    out = paged_attention_batch_invariant(q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32).cuda())
    small_k, small_v, small, lens = batch(lengths, hkv, d, d, page, 806)
    for b, n in enumerate(lengths):
        j = torch.arange(n).cuda()
        paged_cache_write(*rows[b], small_k, small_v, small[b].long()[j // page] * page + j % page)
    assert_bitwise(out, paged_attention_batch_invariant(q, small_k, small_v, small, lens))
    check_token(out[0], q[0], small_k, small_v, small[0], 150)


def test_bad_lengths_and_pages_give_zeros_and_are_reported():
    lengths = [70, 200, 5, 33]
    kc, vc, table, lens = batch(lengths, 2, 64, 64, 16, 900)
    q = randn(4, 4, 64, seed=901)
    want = paged_attention_batch_invariant(q, kc, vc, table, lens)

    def report(rows, table=table, lens=lens, **kw):
        out = paged_attention_batch_invariant(q, kc, vc, table, lens, **kw)
        with pytest.raises(RuntimeError, match="outside its tensor"):
            check_cache_indices()
        for b in range(4):
            if b in rows:
                assert float(out[b].abs().max()) == 0.0
            else:
                assert_bitwise(out[b], want[b])

    for value in (-1, kc.shape[0], 2**31 - 1, -(2**31)):
        bad = table.clone()
        bad[1, 5] = value
        report([1], table=bad)
        bad[2, 0] = value
        report([1, 2], table=bad)
    for value in (-1, table.shape[1] * 16 + 1, 2**31 - 1, -(2**31)):
        bad = lens.clone()
        bad[0] = value
        report([0], lens=bad)
    report([1], max_length=100)
    report([1, 0], max_length=64)  # one chunk
    bad = lens.to(torch.int64)
    bad[3] = 2**40 + 33
    report([3], lens=bad)
    none = paged_attention_batch_invariant(q, kc, vc, table[:, :0], torch.zeros_like(lens))
    assert float(none.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_end_of_the_range(dtype):
    """Their mean is in the range where their sum is not."""
    lengths = [2, 40, 700, 3000]
    kc, vc, table, lens = batch(lengths, 1, 64, 64, 16, 1100, dtype)
    vc.copy_(torch.where(torch.isnan(vc), vc, torch.where(vc > 0, 0.99, 0.9) * torch.finfo(dtype).max))
    q = randn(4, 2, 64, seed=1101, dtype=dtype)
    out = paged_attention_batch_invariant(q, kc, vc, table, lens)
    assert bool(torch.isfinite(out).all())
    for b, n in enumerate(lengths):
        check_token(out[b], q[b], kc, vc, table[b], n, what=f"sequence of {n}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dtype):
    """A score of -inf has weight 0; one of +inf or NaN makes its own row NaN and no other."""
    kc, vc, table, lens = batch([40, 200, 300], 1, 64, 64, 16, 1000, dtype)
    q = randn(3, 2, 64, seed=1001, dtype=dtype)
    q[:, :, 0] = 1.0
    clean = paged_attention_batch_invariant(q, kc, vc, table, lens)
    page, at = int(table[1, 150 // 16]), 150 % 16
    kc[page, at, 0, 0] = float("nan")
    out = paged_attention_batch_invariant(q, kc, vc, table, lens)
    assert torch.isnan(out[1]).all()
    assert_bitwise(out[0], clean[0])
    assert_bitwise(out[2], clean[2])
    kc[page, at, 0, 0] = float("-inf")  # the query's element is 1: a score of -inf
    vc[page, at] = 0.0
    check_token(paged_attention_batch_invariant(q, kc, vc, table, lens)[1], q[1], kc, vc, table[1], 200)
    kc[:, :, 0, 0] = float("-inf")  # every score of every row
    assert float(paged_attention_batch_invariant(q, kc, vc, table, lens).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_key_far_above_many(dtype):
    """4096 keys of weight near 2^-14 beside one of weight 1: the tail counts, however small each part is."""
    d, n = 64, 4097
    kc, vc, table, lens = batch([n], 1, d, d, 16, 1100, dtype)
    q = torch.zeros(1, 1, d, dtype=dtype, device="cuda")
    q[0, 0, 0] = 8.0
    j = torch.arange(n, device="cuda")
    kc.zero_()
    kc[int(table[0, 5]), 3, 0, 0] = 9.7 if dtype != BF16 else 9.6875
    vc[table[0].long()[j // 16], j % 16] = vc[table[0].long()[j // 16], j % 16].abs() + 1
    out = paged_attention_batch_invariant(q, kc, vc, table, lens)
    check_token(out[0], q[0], kc, vc, table[0], n)


def test_graphs_share_nothing():
    """Two captured calls, replayed in turn with new inputs, give the eager results."""
    sets = []
    for i, lengths in enumerate(([400, 3, 90], [700, 64, 1])):
        kc, vc, table, lens = batch(lengths, 2, 64, 64, 16, 1200 + i)
        q = randn(3, 8, 64, seed=1210 + i)
        paged_attention_batch_invariant(q, kc, vc, table, lens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention_batch_invariant(q, kc, vc, table, lens)
        sets.append((graph, q, kc, vc, table, lens, out))
    for i in range(4):
        for graph, q, *_ in sets:
            q.copy_(randn(3, 8, 64, seed=1220 + i))
            graph.replay()
        for _, q, kc, vc, table, lens, out in sets:
            got = out.clone()
            assert_bitwise(got, paged_attention_batch_invariant(q, kc, vc, table, lens), f"replay {i}")
        torch.cuda.synchronize()


def test_other_streams():
    lengths = [900, 30]
    kc, vc, table, lens = batch(lengths, 2, 64, 64, 16, 1300)
    q = randn(2, 4, 64, seed=1301)
    want = paged_attention_batch_invariant(q, kc, vc, table, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(paged_attention_batch_invariant(q, kc, vc, table, lens))
    torch.cuda.synchronize()
    for out in outs:
        assert_bitwise(out, want)


def test_empty_batches():
    kc, vc, table, lens = batch([5], 2, 64, 64, 16, 1400)
    assert paged_attention_batch_invariant(kc.new_empty(0, 4, 64), kc, vc, table[:0], lens[:0]).shape == (0, 4, 64)
    assert paged_attention_batch_invariant(kc.new_empty(1, 0, 64), kc, vc, table, lens).shape == (1, 0, 64)


def test_many_sequences():
    """More rows than a launch has workgroups in a wave, most of them short."""
    n = 3000
    lengths = [(i * 7) % 40 for i in range(n)]
    lengths[17] = 400
    kc, vc, table, lens = batch(lengths, 1, 16, 16, 8, 1500)
    q = randn(n, 3, 16, seed=1501)
    out = paged_attention_batch_invariant(q, kc, vc, table, lens)
    for b in (0, 1, 2, 17, 1499, 2998, 2999):
        check_token(out[b], q[b], kc, vc, table[b], lengths[b], what=f"sequence {b}")
    assert bio.paged_attention_batch_invariant is paged_attention_batch_invariant


@pytest.mark.parametrize("n", [40, 128, 900, 5000])
@pytest.mark.parametrize("far", [11.0, 14.0, 15.0, 16.5, 18.0])
def test_small_weights_of_fp16_count(n, far):
    """One key far above many, with values of 0: the output is what the others' weights of e^-far say.  They are held times 2^7 in
    two parts of fp16: to 2^-22 of themselves, or to half of its smallest step over 2^7, 2^-32 of the largest."""
    page, d = 16, 64
    pages = -(-n // page)
    k, v = torch.zeros(pages, page, 1, d, dtype=F16), torch.full((pages, page, 1, d), 1536.0, dtype=F16)
    k[0, 3, 0, 0], v[0, 3, 0] = 4.0, 0.0
    q = torch.zeros(1, 2, d, dtype=F16)
    q[0, :, 0] = torch.tensor([far / 4, far / 4 - 0.0625])
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    out = paged_attention_batch_invariant(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor([n]).cuda(), scale=1.0)
    for h in range(2):
        parts = attend64(q[:, h], k.flatten(0, 1)[:n, 0], v.flatten(0, 1)[:n, 0], torch.ones(1, n, dtype=torch.bool), 1.0)
        assert_within(out[:, h], parts[0], attention_bound(F16, *parts, n, 2.0**-22, 2.0**-32), f"head {h}")
