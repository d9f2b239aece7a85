"""What the decoder operators refuse, and the host checks of their entry points: no GPU needed."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _native as nat

BF16 = torch.bfloat16


def lib():
    return nat.load(require_gpu=False)


def zeros(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def test_public_names():
    from batch_invariant_ops import decoder

    for name in decoder.__all__:
        assert getattr(bio, name) is getattr(decoder, name)


def rotary(q=None, k=None, p=None, sections=(8, 8), **kw):
    q = zeros(1, 5, 4, 64) if q is None else q
    p = torch.zeros(len(sections), *q.shape[:-2], dtype=torch.int64) if p is None else p
    return bio.multi_axis_rotary(q, k, p, sections, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: rotary(q=zeros(64)), "shape"),
    (lambda: rotary(q=zeros(1, 5, 4, 64, dtype=torch.float64)), "dtype"),
    (lambda: rotary(k=zeros(1, 5, 2, 64, dtype=torch.float16)), "must share"),
    (lambda: rotary(k=zeros(1, 6, 2, 64)), "must share"),
    (lambda: rotary(k=zeros(1, 5, 2, 32)), "must share"),
    (lambda: rotary(sections=(20, 20)), "do not fit"),
    (lambda: rotary(sections=(-1, 4)), "sections"),
    (lambda: rotary(sections=(), p=torch.zeros(0, 1, 5)), "sections"),
    (lambda: rotary(q=zeros(1, 5, 1, 512), sections=(129,)), "at most 128"),
    (lambda: rotary(inv_freq=[1.0] * 15), "inv_freq"),
    (lambda: rotary(base=0.0), "base"),
    (lambda: rotary(base=float("nan")), "base"),
    (lambda: rotary(p=torch.zeros(3, 1, 5, dtype=torch.int64)), "positions must have shape"),
    (lambda: rotary(p=torch.zeros(2, 5, dtype=torch.int64)), "positions must have shape"),
    (lambda: rotary(p=torch.zeros(2, 1, 5, dtype=torch.float64)), "int32, int64 or float32"),
    (lambda: rotary(), "ROCm GPU"),
])
def test_rotary_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def write(k=None, v=None, kc=None, vc=None, slots=None):
    k = zeros(3, 2, 64) if k is None else k
    v = zeros(3, 2, 64) if v is None else v
    kc = zeros(4, 16, 2, 64) if kc is None else kc
    vc = zeros(4, 16, 2, 64) if vc is None else vc
    return bio.paged_cache_write(k, v, kc, vc, torch.zeros(3, dtype=torch.int64) if slots is None else slots)


@pytest.mark.parametrize("call, message", [
    (lambda: write(kc=zeros(4, 16, 128)), "caches must have shape"),
    (lambda: write(vc=zeros(5, 16, 2, 64)), "must share pages"),
    (lambda: write(vc=zeros(4, 16, 2, 64, dtype=torch.float16)), "cache dtypes"),
    (lambda: write(kc=zeros(4, 16, 2, 64, dtype=torch.int16), vc=zeros(4, 16, 2, 64, dtype=torch.int16)), "cache dtypes"),
    (lambda: write(kc=zeros(4, 16, 64, 2).transpose(2, 3)), "unit stride"),
    (lambda: write(kc=zeros(1, 1, 1, 1).expand(1 << 20, 1 << 11, 2, 64), vc=zeros(1, 1, 1, 1).expand(1 << 20, 1 << 11, 2, 64)),
     "unit stride|2\\*\\*31"),
    (lambda: write(v=zeros(2, 2, 64)), "same leading"),
    (lambda: write(k=zeros(3, 2, 64, dtype=torch.float32)), "same dtype"),
    (lambda: write(k=zeros(3, 1, 64), v=zeros(3, 1, 64)), "heads and head dimensions"),
    (lambda: write(slots=torch.zeros(4, dtype=torch.int64)), "slots"),
    (lambda: write(slots=torch.zeros(3)), "slots"),
    (lambda: write(), "ROCm GPU"),
])
def test_write_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_overlapping_caches_are_recognised():
    from batch_invariant_ops.decoder import _overlaps

    assert not _overlaps(zeros(4, 16, 2, 64)) and not _overlaps(zeros(4, 2, 16, 64).transpose(1, 2))
    assert not _overlaps(zeros(4, 2, 16, 2, 64)[:, 0]) and not _overlaps(zeros(4, 16, 2, 80)[..., :64])
    assert _overlaps(zeros(1, 16, 2, 64).expand(4, 16, 2, 64)) and _overlaps(zeros(4096).as_strided((4, 4, 1, 64), (64, 32, 32, 1)))


def token(q=None, kc=None, vc=None, table=None, lengths=None, **kw):
    q = zeros(3, 4, 64) if q is None else q
    kc = zeros(4, 16, 2, 64) if kc is None else kc
    vc = zeros(4, 16, 2, 64) if vc is None else vc
    table = torch.zeros(3, 2, dtype=torch.int32) if table is None else table
    lengths = torch.ones(3, dtype=torch.int32) if lengths is None else lengths
    return bio.paged_attention_batch_invariant(q, kc, vc, table, lengths, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: token(q=zeros(3, 4, 1, 64)), "query must have shape"),
    (lambda: token(q=zeros(3, 4, 64, dtype=torch.float16)), "same dtype"),
    (lambda: token(q=zeros(3, 4, 32)), "head dimensions must match"),
    (lambda: token(q=zeros(3, 5, 64)), "divisible"),
    (lambda: token(q=zeros(3, 4, 12), kc=zeros(4, 16, 2, 12)), "multiples of 8"),
    (lambda: token(vc=zeros(4, 16, 2, 264)), "multiples of 8 up to 256"),
    (lambda: token(q=zeros(3, 4, 6, dtype=torch.float32), kc=zeros(4, 16, 2, 6, dtype=torch.float32),
                   vc=zeros(4, 16, 2, 64, dtype=torch.float32)), "multiples of 4"),
    (lambda: token(kc=zeros(0, 16, 2, 64), vc=zeros(0, 16, 2, 64)), "no pages"),
    (lambda: token(table=torch.zeros(2, 2, dtype=torch.int32)), "block_table"),
    (lambda: token(table=torch.zeros(3, 2)), "block_table"),
    (lambda: token(lengths=torch.ones(2, dtype=torch.int32)), "lengths"),
    (lambda: token(lengths=torch.ones(3)), "lengths"),
    (lambda: token(window=0), "window"),
    (lambda: token(sinks=-1), "sinks"),
    (lambda: token(max_length=-1), "max_length"),
    (lambda: token(scale=float("inf")), "scale"),
    (lambda: token(), "ROCm GPU"),
])
def test_token_attention_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def window(q=None, k=None, v=None, window=4, sinks=0, **kw):
    q = zeros(1, 4, 5, 64) if q is None else q
    k = zeros(1, 4, 5, 64) if k is None else k
    return bio.sliding_window_attention_batch_invariant(q, k, zeros(*k.shape, dtype=k.dtype) if v is None else v, window, sinks, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: window(q=zeros(4, 5, 64)), "rank-4"),
    (lambda: window(q=zeros(1, 4, 5, 64, dtype=torch.float16)), "same dtype"),
    (lambda: window(q=zeros(1, 4, 5, 64, dtype=torch.float64), k=zeros(1, 4, 5, 64, dtype=torch.float64)), "dtype"),
    (lambda: window(q=zeros(2, 4, 5, 64)), "leading"),
    (lambda: window(v=zeros(1, 4, 6, 64)), "leading"),
    (lambda: window(q=zeros(1, 4, 5, 32)), "head dimensions must match"),
    (lambda: window(k=zeros(1, 2, 5, 64)), "enable_gqa"),
    (lambda: window(k=zeros(1, 3, 5, 64), enable_gqa=True), "enable_gqa"),
    (lambda: window(q=zeros(1, 4, 5, 20), k=zeros(1, 4, 5, 20)), "multiples of 8"),
    (lambda: window(q=zeros(1, 4, 5, 132, dtype=torch.float32), k=zeros(1, 4, 5, 132, dtype=torch.float32)), "up to 128"),
    (lambda: window(window=0), "window"),
    (lambda: window(sinks=-2), "sinks"),
    (lambda: window(scale=float("nan")), "scale"),
    (lambda: window(), "ROCm GPU"),
])
def test_window_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def packed(q=None, k=None, cu_q=None, cu_k=None, window=4):
    q = zeros(1, 5, 4, 64) if q is None else q
    k = zeros(1, 5, 2, 64) if k is None else k
    cu = torch.tensor([0, 5])
    return bio.varlen_sliding_window_attention_batch_invariant(q, k, k, cu if cu_q is None else cu_q,
                                                               cu if cu_k is None else cu_k, window)


@pytest.mark.parametrize("call, message", [
    (lambda: packed(q=zeros(5, 4, 64)), "rank-4"),
    (lambda: packed(q=zeros(2, 5, 4, 64)), "batch size 1"),
    (lambda: packed(k=zeros(1, 5, 3, 64)), "divisible"),
    (lambda: packed(k=zeros(1, 5, 2, 32)), "head dimensions must match"),
    (lambda: packed(cu_q=torch.tensor([[0, 5]])), "rank 1"),
    (lambda: packed(cu_q=torch.tensor([], dtype=torch.int64)), "at least one"),
    (lambda: packed(cu_q=torch.tensor([0.0, 5.0])), "int32 or int64"),
    (lambda: packed(cu_q=torch.tensor([0, 2, 5])), "counts must match"),
    (lambda: packed(window=0), "window"),
    (lambda: packed(), "ROCm GPU"),
])
def test_packed_window_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_host_checks_of_the_entry_points():
    """Bad sizes, types and pointers return their status before any launch."""
    L = lib()
    N = None
    p = 256  # a stand-in address: every call below ends before it is touched
    x = [p, 64, 64, 64]

    def rot(dtype=2, batch=1, tokens=1, hq=1, hk=0, d=64, pos_type=0, pairs=8, turns=p, q=p):
        return L.biops_rotary(dtype, batch, tokens, hq, hk, d, q, 64, 64, 64, *x, *x, *x, p, pos_type, 1, 1, 1, pairs, turns, p,
                              0, 0, N)

    assert rot(dtype=3) == 3 and rot(pos_type=3) == 3
    assert rot(pairs=33) == 1 and rot(d=512, pairs=129) == 1 and rot(tokens=-1) == 1 and rot(turns=N) == 1 and rot(q=N) == 1
    assert rot(hq=60000, d=2048) == 1  # more than 2^26 elements a token
    assert rot(tokens=0) == 0 and rot(batch=0) == 0 and rot(hq=0) == 0

    def put(dtype=2, rows=1, heads=1, d=64, pages=4, page=16, k=p, flag=p, kc=p):
        return L.biops_paged_write(dtype, rows, heads, d, 64, k, 64, 64, p, 64, 64, kc, 64, 64, 64, p, 64, 64, 64, pages, page, p, 1,
                                   1, flag, N)

    assert put(dtype=9) == 3 and put(rows=-1) == 1 and put(pages=1 << 20, page=1 << 12) == 1 and put(heads=1 << 20) == 1
    assert put(k=N) == 1 and put(flag=N) == 1 and put(kc=N) == 1 and put(rows=0) == 0

    def att(dtype=2, batch=1, hq=4, hkv=2, d=64, dv=64, pages=4, page=16, width=2, window=0, sinks=0, scale=1.0, ws=N, wsb=0,
            table=p, out=p):
        return L.biops_paged_attention(dtype, batch, hq, hkv, d, dv, p, 64, 64, *x, *x, pages, page, table, 0, 2, 1, width, p, 0,
                                       1, -1, window, sinks, scale, out, p, ws, wsb, N)

    assert att(dtype=3) == 3 and att(hq=3) == 1 and att(hkv=0) == 1 and att(d=60) == 1 and att(dv=264) == 1
    assert att(pages=0) == 1 and att(page=0) == 1 and att(window=-1) == 1 and att(sinks=-1) == 1
    assert att(scale=float("nan")) == 1 and att(table=N) == 1 and att(out=N) == 1
    assert att(width=64) == 5 and att(width=64, ws=p, wsb=8) == 5 and att(width=64, ws=p + 4, wsb=1 << 30) == 2
    assert att(batch=0) == 0 and att(hq=0) == 0
    size = L.biops_paged_attention_workspace_size
    assert size(3, 4, 64, 8, 16, -1, 0, 0) == 0  # 128 keys: one chunk
    assert size(3, 4, 64, 9, 16, -1, 0, 0) == 3 * 4 * 2 * 66 * 4
    assert size(3, 4, 64, 9, 16, 128, 0, 0) == 0 and size(3, 4, 64, 1 << 20, 16, -1, 100, 28) == 0
    assert size(3, 4, 64, 1 << 20, 16, -1, 0, 0) == size(3, 4, 64, 2048, 16, -1, 0, 0) == 3 * 4 * 64 * 66 * 4
    assert size(3, 4, 64, 256, 16, -1, 0, 0) == size(3, 4, 64, 260, 16, -1, 0, 0) == 3 * 4 * 16 * 66 * 4  # the most up to there
    assert size(-1, 4, 64, 8, 16, -1, 0, 0) == -1 and size(3, 4, 264, 8, 16, -1, 0, 0) == -1

    def win(dtype=2, nseq=1, hq=4, hkv=2, lq=5, lk=5, d=64, window=4, sinks=0, scale=1.0, q=p, cu_q=N, flag=p, ws=N, wsb=0):
        return L.biops_window_attention(dtype, nseq, hq, hkv, lq, lk, d, 64, q, 64, 64, 64, *x, *x, *x, cu_q, 0, 1, N, 0, 1, window,
                                        sinks, scale, flag, ws, wsb, N)

    assert win(dtype=3) == 3 and win(hq=5) == 1 and win(hkv=0) == 1 and win(d=36) == 1 and win(dtype=0, d=132) == 1
    assert win(window=0) == 1 and win(sinks=-1) == 1 and win(scale=float("inf")) == 1 and win(q=N) == 1
    assert win(cu_q=p) == 1 and win(lq=1 << 31) == 1 and win(lk=-1) == 1
    assert win(lk=2000, window=1 << 40) == 5 and win(lk=2000, window=1 << 40, ws=p, wsb=8) == 5
    assert win(lk=2000, window=1 << 40, ws=p + 4, wsb=1 << 30) == 2
    size = L.biops_window_attention_workspace_size
    assert size(3, 4, 5, 1023, 64, 1 << 40, 0) == 0 and size(3, 4, 65, 1 << 20, 64, 1 << 40, 0) == 0
    assert size(3, 4, 5, 1024, 64, 1 << 40, 0) == 3 * 4 * 5 * 2 * 66 * 4 and size(3, 4, 5, 1 << 20, 64, 1000, 18) == 0
    assert size(3, 4, 5, 1 << 20, 64, 1000, 19) == size(3, 4, 5, 1024, 64, 1 << 40, 0)
    assert size(3, 4, 50, 8192, 64, 1 << 40, 1 << 40) == 3 * 4 * 50 * 10 * 66 * 4  # 800 keys a range at least
    assert size(3, 4, 5, 1 << 30, 64, 1 << 40, 0) == 3 * 4 * 5 * 16 * 66 * 4
    assert size(-1, 4, 5, 9, 64, 1, 0) == -1 and size(1, 4, 5, 9, 64, 0, 0) == -1 and size(1 << 40, 4, 64, 1 << 20, 64, 1 << 40, 0) == -1
    assert win(lq=0) == 0 and win(nseq=0) == 0 and win(hq=0) == 0
    assert L.biops_window_attention_max_head(nat.F32) == 128 and L.biops_window_attention_max_head(nat.BF16) == 256


def test_fast_call_bindings_match():
    fast = importlib.import_module("batch_invariant_ops._biops_fast")
    L = lib()
    p, x = 256, (256, 64, 64, 64)
    args = (9, 1, 1, 1, 0, 64, *x, *x, *x, *x, p, 0, 1, 1, 1, 8, p, p, 0, 0, None)
    assert fast.rotary(*args) == L.biops_rotary(*args) == 3
    args = (9, 1, 1, 64, 64, p, 64, 64, p, 64, 64, *x, *x, 4, 16, p, 1, 1, p, None)
    assert fast.paged_write(*args) == L.biops_paged_write(*args) == 3
    args = (3, 4, 64, 9, 16, -1, 0, 0)
    assert fast.paged_attention_workspace_size(*args) == L.biops_paged_attention_workspace_size(*args) > 0
    args = (2, 1, 4, 2, 64, 64, p, 64, 64, *x, *x, 4, 16, p, 0, 2, 1, 64, p, 0, 1, -1, 0, 0, 1.0, p, p, None, 0, None)
    assert fast.paged_attention(*args) == L.biops_paged_attention(*args) == 5
    args = (2, 1, 5, 2, 5, 5, 64, 64, *x, *x, *x, *x, None, 0, 1, None, 0, 1, 4, 0, 1.0, p, None, 0, None)
    assert fast.window_attention(*args) == L.biops_window_attention(*args) == 1
    for fn in (fast.rotary, fast.paged_write, fast.paged_attention, fast.window_attention):
        with pytest.raises(TypeError):
            fn(1, 2)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            nat.fast_function("biops_rotary")


def test_frequencies_may_be_a_tensor():
    """Numbers are taken from it at the call: a change of the tensor is a change of the plan."""
    f = torch.tensor([0.5, 0.25], dtype=torch.float64)
    seen = []
    from batch_invariant_ops import decoder

    plan = decoder._rotary_plan
    for value in (0.5, 0.125):
        f[0] = value
        with pytest.raises((RuntimeError, ValueError)):  # on the CPU
            bio.multi_axis_rotary(zeros(1, 2, 4), None, torch.zeros(1, 1, dtype=torch.int64), (2,), inv_freq=f)
        seen.append(plan((2,), 10000.0, tuple(map(float, f)), False, False).turns.tolist())
    assert seen[0][0] == 4 * seen[1][0] and seen[0][1] == seen[1][1]


def test_frequencies_and_axes():
    """The host's table: turns per position and axis of every pair."""
    from batch_invariant_ops.decoder import _rotary_plan

    plan = _rotary_plan((2, 1, 3), 100.0, None, True, False)
    assert plan.axis.tolist() == [0, 1, 2, 0, 2, 2] and plan.pairs == 6
    plan = _rotary_plan((2, 1, 3), 100.0, None, False, False)
    assert plan.axis.tolist() == [0, 0, 1, 2, 2, 2]
    two_pi = 6.283185307179586
    assert plan.turns.tolist() == [100.0 ** (-i / 6) / two_pi for i in range(6)]
    assert _rotary_plan((1, 1), 10.0, (0.5, 0.25), False, True).turns.tolist() == [0.5 / two_pi, 0.25 / two_pi]
    assert (ctypes.c_double * 2).from_address(_rotary_plan((1, 1), 10.0, (0.5, 0.25), False, True).turns_at)[1] == 0.25 / two_pi
