"""What the decoder operators refuse rather than lose: tangents of forward mode, and a trace that would not hold the launch."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import batch_invariant_ops as bio
from batch_invariant_ops import decoder

DEVICES = [torch.device("cpu"), pytest.param(torch.device("cuda"), marks=pytest.mark.gpu)]


def calls(device):
    """Operator by name: (call on a tuple of float tensors, those tensors)."""
    def randn(*shape, seed):
        return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(device)

    q, k, v = randn(1, 6, 4, 64, seed=1), randn(1, 6, 2, 64, seed=2), randn(1, 6, 2, 64, seed=3)
    kc, vc = randn(2, 4, 2, 64, seed=4), randn(2, 4, 2, 64, seed=5)
    p, far = torch.arange(6).view(1, 1, 6).to(device), torch.arange(6.0).view(1, 1, 6).to(device)
    slots, cu = torch.arange(6).to(device), torch.tensor([0, 6]).to(device)
    table, lengths = torch.tensor([[0, 1]]).to(device), torch.tensor([7]).to(device)
    return {
        "rotary": (lambda q, k: bio.multi_axis_rotary(q, k, p, (32,)), (q, k)),
        "rotary_alone": (lambda q: bio.multi_axis_rotary(q, None, p, (32,)), (q,)),
        "positions": (lambda far: bio.multi_axis_rotary(q, None, far, (32,)), (far,)),
        "write": (lambda k, v, kc, vc: bio.paged_cache_write(k, v, kc, vc, slots), (k[0], v[0], kc, vc)),
        "token": (lambda q, kc, vc: bio.paged_attention_batch_invariant(q, kc, vc, table, lengths), (q[:, 0], kc, vc)),
        "window": (lambda q, k, v: bio.sliding_window_attention_batch_invariant(q, k, v, 3, enable_gqa=True),
                   tuple(x.transpose(1, 2) for x in (q, k, v))),
        "packed": (lambda q, k, v: bio.varlen_sliding_window_attention_batch_invariant(q, k, v, cu, cu, 3), (q, k, v)),
    }


NAMES = ["rotary", "rotary_alone", "positions", "write", "token", "window", "packed"]


@pytest.fixture(params=["module", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(decoder, "_tensor_module", False)
        monkeypatch.setattr(decoder, "_direct", lambda: False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(device, name, path):
    call, tensors = calls(device)[name]
    if device.type == "cuda":
        call(*tensors)  # sets both paths up
    for i in range(len(tensors)):
        with forward_ad.dual_level():
            duals = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(tensors)]
            with pytest.raises(ValueError, match="forward-mode"):
                call(*duals)
            if device.type == "cuda":  # a level without tangents, and tangents that nothing follows
                call(*tensors)
                with torch.inference_mode():
                    call(*duals)
                call(*(t.detach() for t in duals))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", [n for n in NAMES if n != "write"])
def test_traces_are_refused(device, name, path):
    call, tensors = calls(device)[name]
    if device.type == "cuda":
        call(*tensors)
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, tensors, check_trace=False)


@pytest.mark.gpu
def test_a_traced_write_is_refused(path):
    call, tensors = calls(torch.device("cuda"))["write"]

    def step(*t):
        call(*t)
        return t[2] + t[3]

    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(step, tensors, check_trace=False)
