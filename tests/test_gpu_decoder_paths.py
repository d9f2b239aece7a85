"""The decoder operators' two host paths -- tensors handed to _biops_tensor as they are, and the Python checks
behind it -- give the same bits, and the first one takes the ordinary calls."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import check_cache_indices, decoder

from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


def calls():
    q, k, v = randn(2, 40, 4, 64, seed=1), randn(2, 40, 2, 64, seed=2), randn(2, 40, 2, 64, seed=3)
    p = torch.arange(240, device="cuda").view(3, 2, 40)
    kc, vc = randn(8, 16, 2, 64, seed=4), randn(8, 16, 2, 64, seed=5)
    table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
    lengths = torch.tensor([50, 7], device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 30, 40], device="cuda", dtype=torch.int32)
    slots = torch.arange(40, device="cuda")

    def write():
        a, b = kc.clone(), vc.clone()
        bio.paged_cache_write(k[0], v[0], a, b, slots)
        return a, b

    return {
        "rotary": lambda: bio.multi_axis_rotary(q, k, p, (8, 12, 12)),
        "rotary_one": lambda: (bio.multi_axis_rotary(q[0], None, p[:, 0], (8, 12, 12), interleaved_pairs=True),),
        "write": write,
        "token": lambda: (bio.paged_attention_batch_invariant(q[:, 0], kc, vc, table, lengths, window=20, sinks=2),),
        "token_all": lambda: (bio.paged_attention_batch_invariant(q[:, 0], kc, vc, table, lengths, scale=0.2, max_length=60),),
        "window": lambda: (bio.sliding_window_attention_batch_invariant(
            q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 9, 1, enable_gqa=True),),
        "window_all": lambda: (bio.sliding_window_attention_batch_invariant(
            q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), v.transpose(1, 2), None, scale=0.3, enable_gqa=True),),
        "packed": lambda: (bio.varlen_sliding_window_attention_batch_invariant(q[:1], k[:1], v[:1], cu, cu, 9, 1),),
    }


@pytest.mark.parametrize("name", ["rotary", "rotary_one", "write", "token", "token_all", "window", "window_all", "packed"])
def test_both_paths(name, monkeypatch):
    call = calls()[name]
    call()  # sets both up
    assert decoder._direct(), "the tensor module is not built"

    def refuse(*args):
        raise AssertionError("the Python path ran")

    with monkeypatch.context() as m:
        m.setattr(decoder, "_call", refuse)
        fast = call()
    with monkeypatch.context() as m:
        m.setattr(decoder, "_tensor_module", False)
        m.setattr(decoder, "_direct", lambda: False)
        slow = call()
    assert len(fast) == len(slow)
    for a, b in zip(fast, slow):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
        assert_bitwise(a, b)


def test_gradients_of_both_paths(monkeypatch):
    q, k = randn(2, 5, 4, 64, seed=9).requires_grad_(), randn(2, 5, 2, 64, seed=10).requires_grad_()
    p = torch.arange(20, device="cuda").view(2, 2, 5)
    g = [randn(2, 5, 4, 64, seed=11), randn(2, 5, 2, 64, seed=12)]

    def both():
        return torch.autograd.grad(bio.multi_axis_rotary(q, k, p, (20, 12)), (q, k), g)

    def alone():
        return torch.autograd.grad(bio.multi_axis_rotary(q, None, p, (20, 12)), q, g[0].transpose(-1, -2).contiguous().transpose(-1, -2))

    def broadcast():
        return torch.autograd.grad(bio.multi_axis_rotary(q, k, p, (20, 12))[1].sum(), k)

    for call in (both, alone, broadcast):
        with monkeypatch.context() as m:
            m.setattr(decoder._Rotary, "forward", None)  # the Python path's
            fast = call()
        with monkeypatch.context() as m:
            m.setattr(decoder, "_tensor_module", False)
            m.setattr(decoder, "_direct", lambda: False)
            slow = call()
        for a, b in zip(fast, slow):
            assert_bitwise(a, b)


def test_errors_are_the_python_ones():
    q = randn(1, 4, 5, 64, seed=6)
    with pytest.raises(ValueError, match="window"):
        bio.sliding_window_attention_batch_invariant(q, q, q, 0)
    with pytest.raises(ValueError, match="enable_gqa"):
        bio.sliding_window_attention_batch_invariant(q, q[:, :2], q[:, :2], 3)
    with pytest.raises(ValueError, match="multiples of 8"):
        bio.sliding_window_attention_batch_invariant(q[..., :20], q[..., :20], q[..., :20], 3)
    with pytest.raises(ValueError, match="negated"):
        z = torch.zeros(1, 1, 8, 64, dtype=torch.complex64, device="cuda").conj().imag
        bio.sliding_window_attention_batch_invariant(z, z, z, 3)
    with pytest.raises(ValueError, match="GPU"):
        bio.sliding_window_attention_batch_invariant(q, q.cpu(), q, 3)
    check_cache_indices()


def test_no_memory_for_the_workspace(monkeypatch):
    """A workspace that cannot be had raises torch's own error."""
    kc = randn(4, 64, 1, 64, seed=7)
    table = torch.zeros(1, 1 << 20, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([5], device="cuda", dtype=torch.int32)
    q = randn(1, 2, 64, seed=8)
    want = bio.paged_attention_batch_invariant(q, kc, kc, table, lengths, max_length=64)
    assert_bitwise(bio.paged_attention_batch_invariant(q, kc, kc, table, lengths), want)
    empty = torch.empty

    def refuse(*args, **kwargs):
        if kwargs.get("dtype") is torch.uint8:
            raise torch.OutOfMemoryError("no workspace")
        return empty(*args, **kwargs)

    monkeypatch.setattr(decoder, "_tensor_module", False)
    monkeypatch.setattr(decoder, "_direct", lambda: False)
    monkeypatch.setattr(torch, "empty", refuse)
    with pytest.raises(torch.OutOfMemoryError):
        bio.paged_attention_batch_invariant(q, kc, kc, table, lengths)
