"""The rotation in autograd: gradients as the engine hands them over, forward mode, tracing, capture."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import decoder, multi_axis_rotary

from _decoder import check_rotated
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu


def randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.fixture(params=["module", "python"])
def path(request, monkeypatch):
    """Both host paths."""
    if request.param == "python":
        monkeypatch.setattr(decoder, "_tensor_module", False)
        monkeypatch.setattr(decoder, "_direct", lambda: False)
    return request.param


def test_lazily_negated_gradients(path):
    """The engine hands over a gradient as it is: a negated view, or the imaginary part of a conjugate."""
    p = torch.randint(0, 99, (2, 5)).cuda()
    q, k = (randn(5, h, 32, seed=h).requires_grad_() for h in (4, 2))
    g = [randn(5, h, 32, seed=10 + h) for h in (4, 2)]
    for kind in (torch._neg_view, lambda x: torch.complex(torch.zeros_like(x), x).conj().imag):
        lazy = [kind(x) for x in g]
        assert all(x.is_neg() for x in lazy)
        for inputs in ((q, k), (q, None)):
            used = [x for x in inputs if x is not None]
            out = multi_axis_rotary(*inputs, p, (8, 4))
            out = out if isinstance(out, tuple) else (out,)
            for got, x in zip(torch.autograd.grad(out, used, lazy[:len(used)]), g):
                check_rotated(got, -x, p, (8, 4), inverse=True)
        held = lazy[0].detach().requires_grad_()  # a gradient that has one of its own
        (gq,) = torch.autograd.grad(multi_axis_rotary(q, None, p, (8, 4)), q, held, create_graph=True)
        check_rotated(gq, -g[0], p, (8, 4), inverse=True)
        (gg,) = torch.autograd.grad(gq, held, g[0])
        check_rotated(gg, g[0], p, (8, 4))
    (gq,) = torch.autograd.grad(torch._neg_view(multi_axis_rotary(q, None, p, (8, 4))), q, g[0])
    check_rotated(gq, -g[0], p, (8, 4), inverse=True)
