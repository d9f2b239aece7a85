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


class Plain(torch.Tensor):
    """A subclass, which the tensor module leaves to the Python function."""


def test_captures_beside_a_living_graph_on_the_python_path():
    p = torch.randint(0, 99, (1, 5)).cuda()
    q = randn(5, 2, 16, seed=1).as_subclass(Plain).requires_grad_()
    want = multi_axis_rotary(q.detach(), None, p, (8,))
    alive = q * 2.0
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            multi_axis_rotary(q, None, p, (8,))
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = multi_axis_rotary(q, None, p, (8,)).detach()
    graph.replay()
    assert_bitwise(got, want)


def test_captures_without_the_module(monkeypatch):
    """What cannot be told is refused; what has no leaf's gradient is captured."""
    monkeypatch.setattr(decoder, "_tensor_module", False)
    monkeypatch.setattr(decoder, "_direct", lambda: False)
    p = torch.randint(0, 99, (1, 5)).cuda()
    q = randn(5, 2, 16, seed=2).requires_grad_()
    want = multi_axis_rotary(q.detach(), None, p, (8,))
    for inputs in ((q, None), (q.detach(), q)):
        with pytest.raises(RuntimeError, match="tensor module"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                multi_axis_rotary(*inputs, p, (8,))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = multi_axis_rotary(q.detach(), None, p, (8,))
        with torch.no_grad():
            second = multi_axis_rotary(q, None, p, (8,))
    graph.replay()
    assert_bitwise(first, want)
    assert_bitwise(second, want)


def test_outputs_of_inputs_without_a_gradient_have_none(path):
    """Their keys can go straight into a cache, for one."""
    p = torch.randint(0, 99, (1, 5)).cuda()
    q, k = randn(5, 2, 16, seed=3), randn(5, 2, 16, seed=4)
    g = randn(5, 2, 16, seed=5)
    for which in (0, 1):
        inputs = [x.clone().requires_grad_() if i == which else x for i, x in enumerate((q, k))]
        out = multi_axis_rotary(*inputs, p, (8,))
        assert out[which].requires_grad and not out[1 - which].requires_grad and out[1 - which].grad_fn is None
        for a, b in zip(out, multi_axis_rotary(q, k, p, (8,))):
            assert_bitwise(a.detach(), b)
        (got,) = torch.autograd.grad(out[which], inputs[which], g)
        check_rotated(got, g, p, (8,), inverse=True)
        cache = torch.zeros(1, 5, 2, 16).cuda()
        bio.paged_cache_write(out[1 - which], out[1 - which], cache, cache.clone(), torch.arange(5).cuda())
        assert_bitwise(cache[0], out[1 - which])
        # a gradient of the gradient, with the other output used beside it
        held = g.clone().requires_grad_()
        (got,) = torch.autograd.grad(multi_axis_rotary(*inputs, p, (8,))[which], inputs[which], held, create_graph=True)
        (gg,) = torch.autograd.grad(got, held, g)
        check_rotated(gg, g, p, (8,))
    both = multi_axis_rotary(q.clone().requires_grad_(), k.clone().requires_grad_(), p, (8,))
    assert both[0].requires_grad and both[1].requires_grad
