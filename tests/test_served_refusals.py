"""What the operators of a decoder served with fewer bits refuse, and the host checks of their entry points: no GPU needed."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _native as nat

BF16, U8, I8, F32 = torch.bfloat16, torch.uint8, torch.int8, torch.float32


def zeros(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def test_public_names():
    from batch_invariant_ops import served

    for name in served.__all__:
        assert getattr(bio, name) is getattr(served, name)


def four(pages=4, page=16, heads=2, d=64, dv=64):
    return [zeros(pages, page, heads, n, dtype=U8) for n in (d // 2, d // 32, dv // 2, dv // 32)]


def append(q=None, k=None, v=None, kc=None, vc=None, slots=None, positions=None, sections=(32,), **kw):
    q, k, v = (zeros(3, n, 64) if t is None else t for t, n in ((q, 4), (k, 2), (v, 2)))
    kc, vc = (zeros(4, 16, 2, 64) if c is None else c for c in (kc, vc))
    slots = torch.zeros(3, dtype=torch.int64) if slots is None else slots
    positions = torch.zeros(1, 3, dtype=torch.int64) if positions is None else positions
    return bio.rotary_cache_write(q, k, v, kc, vc, slots, positions, sections, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: append(), "ROCm GPU"),
    (lambda: append(k=zeros(3, 2, 64, dtype=F32)), "same dtype"),
    (lambda: append(v=zeros(2, 2, 64)), "same leading"),
    (lambda: append(q=zeros(4, 4, 64)), "must share leading"),
    (lambda: append(q=zeros(3, 4, 32)), "must share leading"),
    (lambda: append(q=zeros(3, 4, 64, dtype=F32)), "rotary dtypes"),
    (lambda: append(slots=torch.zeros(4, dtype=torch.int64)), "slots"),
    (lambda: append(slots=torch.zeros(3)), "slots"),
    (lambda: append(positions=torch.zeros(2, 3, dtype=torch.int64)), "positions must have shape"),
    (lambda: append(positions=torch.zeros(1, 3, dtype=torch.float64)), "int32, int64 or float32"),
    (lambda: append(sections=(33,)), "do not fit"),
    (lambda: append(sections=(-1,)), "sections"),
    (lambda: append(kc=zeros(4, 16, 2, 64, dtype=torch.float16), vc=zeros(4, 16, 2, 64, dtype=torch.float16)), "same dtype"),
    (lambda: append(kc=zeros(4, 16, 2, 32)), "heads and head dimensions"),
    (lambda: append(vc=zeros(5, 16, 2, 64)), "must share pages"),
    (lambda: append(key_scales=zeros(4, 16, 2, 2, dtype=U8)), "given together"),
    (lambda: append(key_scales=zeros(4, 16, 2, 2, dtype=U8), value_scales=zeros(4, 16, 2, 2, dtype=U8)), "uint8"),
])
def test_append_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def write4(k=None, v=None, caches=None, slots=None):
    k, v = (zeros(3, 2, 64) if t is None else t for t in (k, v))
    return bio.paged_cache_write_fp4(k, v, *(caches or four()), torch.zeros(3, dtype=torch.int64) if slots is None else slots)


@pytest.mark.parametrize("call, message", [
    (lambda: write4(), "ROCm GPU"),
    (lambda: write4(k=zeros(3, 2, 64, dtype=F32), v=zeros(3, 2, 64, dtype=F32)), "bfloat16 or float16"),
    (lambda: write4(k=zeros(3, 1, 64), v=zeros(3, 1, 64)), "heads and head dimensions"),
    (lambda: write4(caches=four(d=128)), "heads and head dimensions"),
    (lambda: write4(caches=[*four()[:3], zeros(4, 16, 2, 1, dtype=U8)]), "a scale for each"),
    (lambda: write4(caches=[zeros(4, 16, 2, 24, dtype=U8), *four()[1:]]), "a scale for each"),
    (lambda: write4(caches=[*four()[:2], *four(pages=5)[2:]]), "must share pages"),
    (lambda: write4(caches=[four()[0].to(I8), *four()[1:]]), "uint8"),
    (lambda: write4(caches=[zeros(4, 16, 64, dtype=U8), *four()[1:]]), "shapes"),
    (lambda: write4(caches=[zeros(4, 16, 32, 2, dtype=U8).transpose(2, 3), *four()[1:]]), "unit stride"),
    (lambda: write4(slots=torch.zeros(3)), "slots"),
    (lambda: bio.paged_cache_read_fp4(*four(), torch.zeros(3)), "slots"),
    (lambda: bio.paged_cache_read_fp4(*four(), torch.zeros(3, dtype=torch.int64), dtype=F32), "bfloat16 or float16"),
    (lambda: bio.paged_cache_read_fp4(*four(), torch.zeros(3, dtype=torch.int64)), "ROCm GPU"),
])
def test_four_bit_rows_refuse(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_memory_that_is_shared():
    from batch_invariant_ops.served import _check_written

    kc, ks, vc, vs = four()
    rows = zeros(3, 2, 64)
    _check_written((kc, vc, ks, vs), (rows,))
    with pytest.raises(ValueError, match="must not share"):
        _check_written((kc, kc[..., :16], ks, vs), (rows,))
    with pytest.raises(ValueError, match="overlap themselves"):
        _check_written((kc[:1].expand(4, 16, 2, 32), vc, ks, vs), (rows,))
    with pytest.raises(ValueError, match="memory of the caches"):
        _check_written((kc, vc, ks, vs), (kc.view(BF16)[:3, 0],))
    # a row's codes and scales side by side in one allocation
    one = zeros(4, 16, 2, 72, dtype=U8)
    _check_written((one[..., :32], one[..., 34:66], one[..., 32:34], one[..., 66:68]), (rows,))
    with pytest.raises(ValueError, match="must not share"):
        _check_written((one[..., :32], one[..., 34:66], one[..., 31:33], one[..., 66:68]), (rows,))


def attend4(q=None, caches=None, table=None, lengths=None, **kw):
    return bio.paged_attention_fp4_batch_invariant(
        zeros(2, 4, 64) if q is None else q, *(caches or four()), zeros(2, 3, dtype=torch.int32) if table is None else table,
        zeros(2, dtype=torch.int32) if lengths is None else lengths, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: attend4(), "ROCm GPU"),
    (lambda: attend4(q=zeros(2, 4, 64, dtype=F32)), "bfloat16 or float16"),
    (lambda: attend4(q=zeros(2, 64)), "shape"),
    (lambda: attend4(q=zeros(2, 4, 32)), "must match"),
    (lambda: attend4(q=zeros(2, 3, 64)), "divisible"),
    (lambda: attend4(q=zeros(2, 4, 288), caches=four(d=288)), "multiples of 32"),
    (lambda: attend4(caches=four(dv=0)), "multiples of 32"),
    (lambda: attend4(caches=four(pages=0)), "no pages"),
    (lambda: attend4(table=zeros(3, 3, dtype=torch.int32)), "block_table"),
    (lambda: attend4(lengths=zeros(2)), "lengths"),
    (lambda: attend4(window=0), "window"),
    (lambda: attend4(sinks=-1), "sinks"),
    (lambda: attend4(max_length=-1), "max_length"),
    (lambda: attend4(scale=float("inf")), "scale"),
])
def test_attention_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def sample(logits=None, u=None, **kw):
    logits = zeros(2, 9, dtype=F32) if logits is None else logits
    return bio.sample_tokens_batch_invariant(logits, zeros(*logits.shape[:-1], dtype=F32) if u is None else u, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: sample(), "ROCm GPU"),
    (lambda: sample(logits=zeros(2, 9, dtype=torch.float64)), "logits"),
    (lambda: sample(logits=zeros(2, 0)), "1 to 1048576"),
    (lambda: sample(logits=torch.zeros(1).expand(2, (1 << 20) + 1)), "1 to 1048576"),
    (lambda: sample(logits=torch.zeros(1).expand(65537, 2)), "65536 rows"),
    (lambda: sample(logits=torch.zeros(1).expand(32769, 1 << 20)), "2\\*\\*35 logits"),
    (lambda: sample(u=zeros(2)), "uniforms"),
    (lambda: sample(u=zeros(3, dtype=F32)), "uniforms"),
    (lambda: sample(temperature=-0.5), "temperature"),
    (lambda: sample(temperature=float("nan")), "temperature"),
    (lambda: sample(temperature=float("inf")), "temperature"),
    (lambda: sample(temperature=zeros(3, dtype=F32)), "temperature"),
    (lambda: sample(temperature=zeros(2, dtype=torch.float64)), "temperature"),
    (lambda: sample(top_k=0), "top_k"),
    (lambda: sample(top_k=1.5), "top_k"),
    (lambda: sample(top_k=True), "top_k"),
    (lambda: sample(top_k=zeros(2, dtype=F32)), "top_k"),
    (lambda: sample(top_p=0.0), "top_p"),
    (lambda: sample(top_p=1.5), "top_p"),
    (lambda: sample(min_p=-0.1), "min_p"),
    (lambda: sample(min_p=1.1), "min_p"),
])
def test_sampling_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def linear(x=None, xs=None, w=None, ws=None, bias=None, **kw):
    x = zeros(3, 32, dtype=I8) if x is None else x
    w = zeros(5, 32, dtype=I8) if w is None else w
    return bio.linear_int8_batch_invariant(x, zeros(*x.shape[:-1], dtype=F32) if xs is None else xs, w,
                                           zeros(5, dtype=F32) if ws is None else ws, bias, **kw)


@pytest.mark.parametrize("call, message", [
    (lambda: linear(), "ROCm GPU"),
    (lambda: linear(x=zeros(3, 32)), "int8"),
    (lambda: linear(w=zeros(32, dtype=I8)), "int8 of shapes"),
    (lambda: linear(w=zeros(5, 31, dtype=I8)), "features"),
    (lambda: linear(x=zeros(3, 0, dtype=I8), w=zeros(5, 0, dtype=I8)), "1 to 131071"),
    (lambda: linear(x=zeros(1, dtype=I8).expand(1, 131072), w=zeros(1, dtype=I8).expand(5, 131072)), "1 to 131071"),
    (lambda: linear(xs=zeros(4, dtype=F32)), "x_scale"),
    (lambda: linear(ws=zeros(5)), "weight_scale"),
    (lambda: linear(dtype=torch.float64), "output dtype"),
    (lambda: linear(bias=zeros(5, dtype=F32)), "bias"),
    (lambda: linear(bias=zeros(4)), "bias"),
    (lambda: bio.quantize_tokens_int8(zeros(3, 4, dtype=torch.float64)), "rows must be"),
    (lambda: bio.quantize_tokens_int8(zeros(3, 0)), "1 to 131071"),
    (lambda: bio.quantize_tokens_int8(zeros(3, 4)), "ROCm GPU"),
])
def test_linear_refuses(call, message):
    with pytest.raises(ValueError, match=message):
        call()


@pytest.mark.parametrize("call", [
    lambda x: bio.quantize_tokens_int8(x),
    lambda x: bio.sample_tokens_batch_invariant(x, zeros(3, dtype=F32)),
    lambda x: append(q=x.view(3, 4, 64), k=zeros(3, 2, 64, dtype=F32), v=zeros(3, 2, 64, dtype=F32)),
])
def test_no_tangents_no_traces(call):
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(forward_ad.make_dual(zeros(3, 256, dtype=F32), torch.ones(3, 256)))
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, (zeros(3, 256, dtype=F32),))


# ------------------------------------------------------------------------- the C entry points ----
def entry(name):
    return getattr(nat.load(require_gpu=False), name)


P = ctypes.c_void_p(256)  # a pointer that is never followed: every call here ends in the host's checks


def refused(rc, code, message):
    assert rc == code, (rc, nat.last_error())
    assert message in nat.last_error()


def rotary_write(dtype=2, rows=1, hq=2, hk=1, d=64, dv=64, q=P, k=P, kc=P, ks=None, vs=None, pages=4, page=16, slots=P, pos=P,
                 pos_type=0, pairs=4, flag=P):
    turns, axis = (ctypes.c_double * 128)(), (ctypes.c_uint8 * 128)()
    return entry("biops_rotary_write")(
        dtype, rows, hq, hk, d, dv, q, 1, 1, q, 1, 1, k, 1, 1, k, 1, 1, kc, 1, 1, 1, ks, 1, 1, 1, kc, 1, 1, 1, vs, 1, 1, 1, pages, page,
        slots, 1, 1, pos, pos_type, 1, 1, pairs, ctypes.cast(turns, ctypes.c_void_p), ctypes.cast(axis, ctypes.c_void_p), 0, flag, None, 0, None)


@pytest.mark.parametrize("kw, code, message", [
    (dict(dtype=3), 3, "dtype"), (dict(dtype=0, ks=P, vs=P), 3, "dtype"), (dict(rows=-1), 1, "size"), (dict(d=-1), 1, "size"),
    (dict(pages=1 << 30, page=16), 1, "2^31"), (dict(hq=1 << 20, d=128), 1, "2^22"), (dict(pairs=33), 1, "pairs"),
    (dict(pairs=129, d=512), 1, "pairs"), (dict(pos_type=3), 3, "position"), (dict(ks=P, vs=P, d=48), 1, "multiples of 32"),
    (dict(q=None), 1, "null"), (dict(slots=None), 1, "null"), (dict(flag=None), 1, "null"), (dict(pos=None), 1, "null"),
    (dict(kc=None), 1, "null cache"), (dict(ks=P), 1, "null cache"), (dict(rows=1025), 5, "workspace"),
])
def test_rotary_write_entry(kw, code, message):
    refused(rotary_write(**kw), code, message)


def test_entries_with_nothing_to_do():
    assert rotary_write(rows=0) == 0
    assert entry("biops_paged_read_fp4")(2, 0, 1, 64, 64, *([P, 1, 1, 1] * 4), 4, 16, P, 1, 1, P, P, P, None) == 0
    assert entry("biops_quantize_int8")(2, 0, 8, P, 8, P, P, None) == 0
    assert entry("biops_linear_int8")(2, 0, 5, 8, P, 8, P, 1, P, 8, P, 1, None, P, None) == 0
    assert entry("biops_linear_int8")(2, 5, 0, 8, P, 8, P, 1, P, 8, P, 1, None, P, None) == 0


@pytest.mark.parametrize("change, code, message", [
    ({0: 0}, 3, "dtype"), ({1: -1}, 1, "batch"), ({3: 0}, 1, "heads"), ({2: 3, 3: 2}, 1, "heads"), ({4: 48}, 1, "multiples of 32"),
    ({5: 288}, 1, "multiples of 32"), ({25: 0}, 1, "without pages"), ({26: 0}, 1, "without pages"), ({36: -1}, 1, "window"),
    ({6: None}, 1, "null"), ({13: None}, 1, "null"), ({1: 1 << 28}, 1, "rows"), ({41: None}, 5, "workspace"),
    ({42: 16}, 5, "workspace"), ({41: ctypes.c_void_p(257)}, 4 - 2, "aligned"),
])
def test_attention_entry(change, code, message):
    args = [2, 2, 4, 2, 64, 64, P, 1, 1, *([P, 1, 1, 1] * 4), 8, 16, P, 0, 1, 1, 64, P, 0, 1, -1, 0, 0, 1.0, P, P, P, 1 << 30, None]
    for i, x in change.items():
        args[i] = x
    refused(entry("biops_paged_attention_fp4")(*args), code, message)


def test_sampling_entry():
    size = entry("biops_sample_workspace_size")
    assert size(0, 5) == 0 and size(1, 5) > 0 and size(1, 0) == size(1, (1 << 20) + 1) == size(65537, 5) == size(-1, 5) == -1
    assert size(2, 1 << 20) >= size(1, 1 << 20)

    def call(dtype=2, rows=2, vocab=9, logits=P, ws=P, bytes_=1 << 40):
        return entry("biops_sample")(dtype, rows, vocab, logits, 9, P, 1, None, 0, 1.0, None, 0, 0, 0, None, 0, 1.0, None, 0, 0.0, P, ws,
                                     bytes_, None)

    refused(call(dtype=3), 3, "dtype")
    refused(call(rows=-1), 1, "rows")
    refused(call(vocab=0), 1, "rows")
    refused(call(rows=32769, vocab=1 << 20), 1, "2^35 tokens in all")
    assert size(32768, 1 << 20) > 0 and size(32769, 1 << 20) == -1
    refused(call(logits=None), 1, "null")
    refused(call(bytes_=8), 5, "workspace")
    refused(call(ws=None), 5, "workspace")
    refused(call(ws=ctypes.c_void_p(264)), 2, "aligned")
    assert call(rows=0) == 0


def test_int8_entries():
    q, y = entry("biops_quantize_int8"), entry("biops_linear_int8")
    refused(q(3, 2, 8, P, 8, P, P, None), 3, "dtype")
    refused(q(2, 2, 0, P, 8, P, P, None), 1, "131071")
    refused(q(2, 2, 131072, P, 8, P, P, None), 1, "131071")
    refused(q(2, 2, 8, None, 8, P, P, None), 1, "null")
    refused(y(3, 2, 5, 8, P, 8, P, 1, P, 8, P, 1, None, P, None), 3, "dtype")
    refused(y(2, 2, 5, 131072, P, 8, P, 1, P, 8, P, 1, None, P, None), 1, "131071")
    refused(y(2, -2, 5, 8, P, 8, P, 1, P, 8, P, 1, None, P, None), 1, "rows")
    refused(y(2, 2, 5, 8, P, 8, None, 1, P, 8, P, 1, None, P, None), 1, "null")
    refused(y(2, 1 << 23, 1 << 22, 8, P, 8, P, 1, P, 8, P, 1, None, P, None), 5, "blocks")


def test_the_module_without_its_library(monkeypatch):
    """Nothing is loaded before the arguments are checked."""
    monkeypatch.setattr(nat, "load", lambda *a, **k: (_ for _ in ()).throw(AssertionError("loaded")))
    served = importlib.import_module("batch_invariant_ops.served")
    with pytest.raises(ValueError, match="int8"):
        served.linear_int8_batch_invariant(zeros(3, 4), zeros(3, dtype=F32), zeros(5, 4, dtype=I8), zeros(5, dtype=F32))


def test_caches_of_many_slots():
    """A write addresses slots, in 31 bits; attention addresses pages."""
    fours = [c[:1].expand(1 << 27, 16, *c.shape[2:]) for c in four()]
    plain = [zeros(1, 16, 2, 64).expand(1 << 27, 16, 2, 64)] * 2
    for call in (lambda: write4(caches=fours), lambda: bio.paged_cache_read_fp4(*fours, torch.zeros(3, dtype=torch.int64)),
                 lambda: bio.paged_cache_write(zeros(3, 2, 64), zeros(3, 2, 64), *plain, torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError, match="caches of more than 2"):
            call()
    for call in (lambda: attend4(caches=fours), lambda: bio.paged_attention_batch_invariant(
            zeros(2, 4, 64), *plain, zeros(2, 3, dtype=torch.int32), zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()
    with pytest.raises(ValueError, match="pages of more than 2"):
        attend4(caches=[c[:1, :1].expand(4, 1 << 31, *c.shape[2:]) for c in four()])


@pytest.mark.parametrize("rows, vocab", [(65536, 100), (65536, 4096), (65536, 8192), (65536, 1 << 19), (32768, 1 << 20), (4000, 131072), (500, 1 << 20)])
def test_the_workspace_of_sampling_is_bounded(rows, vocab):
    size = entry("biops_sample_workspace_size")
    assert 0 < size(rows, vocab) < (1 << 29) + 256 and size(1, vocab) <= size(rows, vocab)
