"""The next token from given random numbers, against the filters' definition in 64 bits.

A random number in the middle of a token's interval of the running sum has to give that token.  Intervals that are tested are at
least 1e-5 of the whole: a 32-bit random number is off by 2^-25, the sums of at most 2^20 weights rounded to 2^-43 by
2^-24 at the very most.  Borders of top-p are put into the middle of a token's weight in the same way."""

from __future__ import annotations

import math

import pytest
import torch

from batch_invariant_ops import sample_tokens_batch_invariant

from _served import staying

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def logits_of(vocab, seed, dtype=F32, spread=2.5, rows=1):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def middle(w, stay, p):
    """A top-p whose border is in the middle of a token's weight, at about p."""
    down = torch.sort(torch.where(stay, w, 0.0), descending=True).values
    upto = down.cumsum(0) / down.sum()
    i = int((upto < p).sum().clamp(max=len(upto) - 1))
    return float(upto[i] - 0.5 * down[i] / down.sum())


def check_row(row, temperature=1.0, top_k=None, top_p=None, min_p=None, count=40, seed=0, kw=None, least=1e-5):
    """Random numbers in the middle of the tokens' intervals, one call for all of them."""
    w, stay = staying(row, temperature, top_k, top_p, min_p)
    kept = torch.where(stay, w, 0.0)
    upto = kept.cumsum(0)
    total = upto[-1]
    large = (kept / total > least).nonzero().flatten()
    pick = large[torch.randperm(len(large), generator=torch.Generator().manual_seed(seed))[:count]]
    pick = torch.cat([pick, large[[0, -1]], kept.argmax().view(1)])
    u = ((upto[pick] - 0.5 * kept[pick]) / total).float()
    rows = row.expand(len(pick), -1).cuda()
    got = sample_tokens_batch_invariant(rows, u.cuda(), **(kw if kw is not None else dict(
        temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)))
    assert torch.equal(got.cpu(), pick), f"{int((got.cpu() != pick).sum())} of {len(pick)} tokens differ"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 511, 513, 2049, 32000, 131072])
def test_plain(dtype, vocab):
    check_row(logits_of(vocab, 1, dtype)[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [5, 1000, 40001])
@pytest.mark.parametrize("top_k", [1, 2, 40, 997, 5000, 10**9])
def test_top_k(dtype, vocab, top_k):
    check_row(logits_of(vocab, 2, dtype)[0], top_k=top_k)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("vocab", [5, 1000, 40001, 200000])
@pytest.mark.parametrize("p", [1e-6, 0.3, 0.9, 0.999, 1.0])
@pytest.mark.parametrize("temperature", [0.3, 1.0, 4.0])
def test_top_p(dtype, vocab, p, temperature):
    row = logits_of(vocab, 3, dtype)[0]
    w, stay = staying(row, temperature)
    check_row(row, temperature, top_p=middle(w, stay, p) if p < 1 else 1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top_k, p", [(3, 0.5), (50, 0.9), (900, 0.97), (20000, 0.5), (20000, 0.99), (39000, 0.999)])
def test_top_k_then_top_p(dtype, top_k, p):
    row = logits_of(40001, 4, dtype)[0]
    w, stay = staying(row, 1.3, top_k)
    check_row(row, 1.3, top_k, middle(w, stay, p))


@pytest.mark.parametrize("top_k, p", [(None, None), (30, None), (None, 0.8), (500, 0.9)])
@pytest.mark.parametrize("min_p", [0.0, 1e-3, 0.05, 0.6, 1.0])
def test_min_p(top_k, p, min_p):
    row = logits_of(5003, 5)[0]
    if p is not None:
        w, stay = staying(row, 0.8, top_k)
        p = middle(w, stay, p)
    check_row(row, 0.8, top_k, p, min_p)


@pytest.mark.parametrize("vocab, top_k, m", [(100, 37, None), (40000, 12345, None), (40000, None, 777), (40000, 30000, 20001), (131072, 1, None),
                                             (5000, 4999, 4999)])
def test_equal_logits(vocab, top_k, m):
    """All the same: the first of them by their index.  (m: top-p with its border in the middle of token m.)"""
    row = torch.full((vocab,), -3.25)
    check_row(row, 0.7, top_k, None if m is None else (m - 0.5) / (top_k or vocab))


@pytest.mark.parametrize("levels", [2, 3, 17])
@pytest.mark.parametrize("top_k, share", [(2000, None), (None, 0.6), (9000, 0.5)])
def test_few_different_logits(levels, top_k, share):
    """Thousands of equal logits, more than the list of a border holds: the cut is inside of one level."""
    row = torch.randint(0, levels, (30000,), generator=torch.Generator().manual_seed(6)).float() * 0.5
    p = None
    if share is not None:
        w, stay = staying(row, 1.0, top_k)
        p = middle(w, stay, share)
    check_row(row, 1.0, top_k, p)


@pytest.mark.parametrize("vocab", [150, 600, 1100, 2048, 9000])
@pytest.mark.parametrize("levels", [1, 2, 400])
@pytest.mark.parametrize("top_k, share", [(None, 0.7), (101, None), (149, 0.6)])
def test_borders_of_many_tokens(vocab, levels, top_k, share):
    """Borders' lists of a hundred to two thousand tokens, of few or of many different weights, alone and among far smaller ones."""
    g = torch.Generator().manual_seed(vocab + levels)
    row = torch.full((vocab,), -30.0)
    some = torch.randperm(vocab, generator=g)[:min(vocab, 2000)]
    row[some] = torch.randint(0, levels, (len(some),), generator=g).float() * 1e-3
    p = None
    if share is not None:
        w, stay = staying(row, 1.0, top_k)
        p = middle(w, stay, share)
    check_row(row, 1.0, top_k, p)


@pytest.mark.parametrize("spread", [1e-6, 1e-3, 30.0, 1e4])
@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 1.0, 1e6])
def test_narrow_and_wide_distributions(spread, temperature):
    row = logits_of(3001, 7, spread=spread)[0]
    check_row(row, temperature, 100)
    w, stay = staying(row, temperature)
    check_row(row, temperature, top_p=middle(w, stay, 0.7))


def test_the_most_likely_token():
    x = logits_of(5000, 8, rows=4)
    x[1, 4000] = x[1, 30] = 50.0
    x[2] = 0.0
    u = torch.tensor([0.0, 0.5, 0.99, 0.3])
    want = torch.tensor([int(x[0].argmax()), 30, 0, int(x[3].argmax())])
    for kw in (dict(temperature=0), dict(temperature=0.0, top_k=5, top_p=0.5, min_p=0.1), dict(top_k=1), dict(temperature=torch.zeros(4).cuda()),
               dict(temperature=torch.full((4,), -1.0).cuda()), dict(temperature=torch.full((4,), float("nan")).cuda()),
               dict(top_p=torch.zeros(4).cuda()), dict(top_p=torch.full((4,), -1.0).cuda())):
        assert torch.equal(sample_tokens_batch_invariant(x.cuda(), u.cuda(), **kw).cpu(), want), kw
    # a min-p above 1 in a tensor leaves the largest logits
    got = sample_tokens_batch_invariant(x.cuda(), u.cuda(), min_p=torch.full((4,), 3.0).cuda()).cpu()
    assert got.tolist() == [int(x[0].argmax()), 4000, 4950, int(x[3].argmax())]


def test_infinities_and_nan():
    inf, nan = float("inf"), float("nan")
    x = torch.full((9, 700), -inf)
    x[1, 650] = -5.0
    x[2, 3], x[2, 600] = inf, inf
    x[3] = nan
    x[4, 5], x[4, 6] = nan, 2.0
    x[5] = 0.0
    x[5, :350] = -inf
    x[6] = 1.0
    x[6, ::2] = nan
    x[7] = -3.4e38
    x[8] = inf
    u = torch.tensor([0.5, 0.5, 0.75, 0.5, 0.9, 0.0, 0.0, 0.5, 0.5])
    want = [-1, 650, 600, -1, 6, 350, 1, 350, 350]
    for kw in ({}, dict(top_k=10**6), dict(top_p=1.0), dict(min_p=0.5)):
        assert sample_tokens_batch_invariant(x.cuda(), u.cuda(), **kw).tolist() == want, kw
    assert sample_tokens_batch_invariant(x.cuda(), u.cuda(), top_k=1).tolist() == [-1, 650, 3, -1, 6, 350, 1, 0, 0]
    assert sample_tokens_batch_invariant(x.cuda(), u.cuda(), temperature=0.0).tolist() == [-1, 650, 3, -1, 6, 350, 1, 0, 0]


def test_random_numbers_outside_of_their_range():
    x = logits_of(1000, 9, rows=5).cuda()
    x[:, 0], x[:, 999] = 9.0, 9.0
    u = torch.tensor([-0.5, 1.0, 7.0, float("nan"), 0.99999994]).cuda()
    assert sample_tokens_batch_invariant(x, u).tolist() == [0, 999, 999, 0, 999]


def test_settings_of_each_row():
    rows, vocab = 12, 3001
    x = logits_of(vocab, 10, rows=rows)
    temperature = torch.linspace(0.4, 1.8, rows)
    top_k = torch.tensor([0, -3, 1, 5, 40, 200, 3000, 3001, 9999, 60, 7, 1500])
    min_p = torch.linspace(0.0, 0.03, rows)
    top_p = torch.empty(rows)
    u, want = torch.empty(rows), torch.empty(rows, dtype=torch.int64)
    for r in range(rows):
        k = int(top_k[r]) if 0 < int(top_k[r]) else None
        t = float(temperature[r].double())
        top_p[r] = middle(*staying(x[r], t, k), 0.2 + 0.06 * r)
        w, stay = staying(x[r], t, k, float(top_p[r].double()), float(min_p[r].double()))
        kept = torch.where(stay, w, 0.0)
        upto = kept.cumsum(0)
        large = (kept > 1e-4 * upto[-1]).nonzero().flatten()
        want[r] = large[r % len(large)]
        u[r] = (upto[want[r]] - 0.5 * kept[want[r]]) / upto[-1]
    for index in (torch.int32, torch.int64):
        wide = [torch.stack([a, a + 1], 1).cuda()[:, 0] for a in (u, temperature, top_p, min_p)]  # (by strides)
        got = sample_tokens_batch_invariant(x.cuda(), wide[0], temperature=wide[1], top_k=top_k.to(index).cuda(), top_p=wide[2], min_p=wide[3])
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_alone_has_the_same_token(dtype):
    x = logits_of(50257, 11, dtype, rows=300).cuda()
    u = torch.rand(300, generator=torch.Generator().manual_seed(12)).cuda()
    kw = dict(temperature=1.1, top_k=2000, top_p=0.95, min_p=1e-4)
    got = sample_tokens_batch_invariant(x, u, **kw)
    for at in (slice(0, 1), slice(7, 9), slice(100, 164)):
        assert torch.equal(sample_tokens_batch_invariant(x[at], u[at], **kw), got[at])
    for _ in range(3):
        assert torch.equal(sample_tokens_batch_invariant(x, u, **kw), got)


def test_shapes_and_strides():
    x = logits_of(1000, 13, rows=6).cuda()
    u = torch.rand(6, generator=torch.Generator().manual_seed(14)).cuda()
    want = sample_tokens_batch_invariant(x, u, top_k=50)
    got = sample_tokens_batch_invariant(x.view(2, 3, 1000), u.view(2, 3), top_k=50)
    assert got.shape == (2, 3) and torch.equal(got.view(-1), want)
    assert torch.equal(sample_tokens_batch_invariant(x[4], u[4], top_k=50), want[4])
    wide = torch.zeros(6, 2007, device="cuda")
    wide[:, 3:1003] = x
    assert torch.equal(sample_tokens_batch_invariant(wide[:, 3:1003], u, top_k=50), want)
    assert torch.equal(sample_tokens_batch_invariant(x.t().contiguous().t(), u, top_k=50), want)
    odd = torch.zeros(6, 1001, dtype=BF16, device="cuda")
    odd[:, 1:] = x
    assert torch.equal(sample_tokens_batch_invariant(odd[:, 1:], u), sample_tokens_batch_invariant(odd[:, 1:].contiguous(), u))
    assert sample_tokens_batch_invariant(x[:0], u[:0]).shape == (0,)


def test_the_largest_vocabulary():
    row = logits_of(1 << 20, 15)[0]
    w, stay = staying(row, 1.0, 700000)
    check_row(row, 1.0, 700000, middle(w, stay, 0.97))
    check_row(torch.zeros(1 << 20), 1.0, 999999, least=5e-7)  # (sums of equal weights are exact)


@pytest.mark.parametrize("top_p", [None, 0.8])
@pytest.mark.parametrize("vocab", [1000, 10000])
def test_far_rows(vocab, top_p):
    """Offsets past 32 bits."""
    x = logits_of(vocab, 16, BF16, rows=3).cuda()
    u = torch.rand(3, generator=torch.Generator().manual_seed(17)).cuda()
    far = torch.empty(2 * (1 << 31) + vocab, dtype=BF16, device="cuda").as_strided((3, vocab), (1 << 31, 1))
    far.copy_(x)
    assert torch.equal(sample_tokens_batch_invariant(far, u, top_p=top_p), sample_tokens_batch_invariant(x, u, top_p=top_p))


def test_a_tangent_of_a_setting_is_refused():
    x, u = torch.zeros(2, 5, device="cuda"), torch.zeros(2, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(torch.ones(2, device="cuda"), torch.ones(2, device="cuda"))
        with pytest.raises(ValueError, match="forward-mode"):
            sample_tokens_batch_invariant(x, u, temperature=t)


def test_needs_no_gradient():
    x = torch.zeros(2, 5, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        sample_tokens_batch_invariant(x, torch.zeros(2, device="cuda"))
    with torch.no_grad():
        assert sample_tokens_batch_invariant(x, torch.zeros(2, device="cuda")).tolist() == [0, 0]


@pytest.mark.parametrize("step", [1, (1 << 29) + 1, (1 << 30) - 1])
def test_a_weight_is_off_by_less_than_a_part_in_2_33(step):
    """Two logits 1 apart at temperatures that put the second one's octaves y = log2(e) / T next to the borders of each of the 1024
    parts of an octave (and into the middle).  Its weight w is within 2^-33 w of the definition, and then rounded to a multiple of
    2^-43 (2^-41 w at most, w being above 2^-3), y to one of 2^-40 (2^-41 w).  So with a top-p of 1 / (1 + w (1 - d)), d = 2^-33 + 2^-39,
    more than that has gone before it only if it were too small: it stays; with 1 / (1 + w (1 + d)) it goes.  (top-p as a number is
    one of 64 bits: 2^-53 / w.)"""
    x, u = torch.tensor([[0.0, -1.0]]).cuda(), torch.tensor([0.99999994]).cuda()
    d, got = 2.0**-33 + 2.0**-39, []
    for i in range(1024):
        t = 1.4426950408889634 / ((i % 2) + (i + step * 2.0**-30) / 1024)
        w = math.exp(-1.0 / t)
        for off in (-d, d):
            got.append(sample_tokens_batch_invariant(x, u, temperature=t, top_p=1.0 / (1.0 + w * (1.0 + off))))
    got = torch.cat(got).view(-1, 2).cpu()
    assert int((got[:, 0] != 1).sum()) == 0, "weights that are too small"
    assert int((got[:, 1] != 0).sum()) == 0, "weights that are too large"


def test_settings_that_are_not_numbers():
    """NaN in a tensor: a temperature of 0, and no filter elsewhere."""
    x = logits_of(5000, 18, rows=40).cuda()
    u = torch.rand(40, generator=torch.Generator().manual_seed(19)).cuda()
    nan = torch.full((40,), float("nan")).cuda()
    plain = sample_tokens_batch_invariant(x, u)
    assert int((plain != x.argmax(1)).sum()) > 20
    assert torch.equal(sample_tokens_batch_invariant(x, u, temperature=nan), x.argmax(1))
    assert torch.equal(sample_tokens_batch_invariant(x, u, top_p=nan), plain)
    assert torch.equal(sample_tokens_batch_invariant(x, u, min_p=nan), plain)
    kept = sample_tokens_batch_invariant(x, u, top_k=30, top_p=0.9)
    assert torch.equal(sample_tokens_batch_invariant(x, u, top_k=30, top_p=0.9, min_p=nan), kept)


@pytest.mark.parametrize("rows, vocab, each", [(50000, 100, True), (50000, 30, False), (9000, 40001, True)])
def test_more_rows_than_a_workspace_holds(rows, vocab, each):
    """The same tokens as in calls of few rows, with settings by strides."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 2).to(BF16)
    wide = torch.rand(rows, 8, generator=g, device="cuda")
    kw = dict(top_k=11, top_p=0.9)
    if each:
        kw = dict(temperature=wide[:, 1] + 0.2, top_k=(wide[:, 2:4] * vocab).long()[:, 1], top_p=wide[:, 4], min_p=wide[:, 5] * 0.1)
    got = sample_tokens_batch_invariant(x, wide[:, 0], **kw)
    for at in range(0, rows, 3000):
        part = slice(at, at + 3000)
        few = {k: t[part] if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
        assert torch.equal(sample_tokens_batch_invariant(x[part], wide[part, 0], **few), got[part])
    last = {k: t[-1:] if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
    assert torch.equal(sample_tokens_batch_invariant(x[-1:], wide[-1:, 0], **last), got[-1:])
