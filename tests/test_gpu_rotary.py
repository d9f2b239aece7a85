"""Rotary positions with several axes against the 64-bit rotation, their gradient, and their layouts."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import multi_axis_rotary

from _decoder import check_rotated, rotate64
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def randn(*shape, seed, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def places(axes, *lead, seed, most=5000, dtype=torch.int64):
    return torch.randint(0, most, (axes, *lead), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, sections", [
    (128, (16, 24, 24)), (64, (32,)), (72, (18, 18)), (80, (3, 7, 9, 5)), (8, (4,)), (128, (0, 5)), (70, (17, 18)),
    (6, (1, 2)), (256, (64, 64)), (40, (1,)), (9, (4,)),
])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("axes", [False, True])
def test_rotation(dtype, d, sections, pairs, axes):
    q, k = randn(2, 13, 6, d, seed=1, dtype=dtype), randn(2, 13, 2, d, seed=2, dtype=dtype)
    p = places(len(sections), 2, 13, seed=3)
    kw = dict(base=10000.0, interleaved_axes=axes, interleaved_pairs=pairs)
    out_q, out_k = multi_axis_rotary(q, k, p, sections, **kw)
    check_rotated(out_q, q, p, sections, "queries", **kw)
    check_rotated(out_k, k, p, sections, "keys", **kw)
    assert_bitwise(out_q[..., 2 * sum(sections):], q[..., 2 * sum(sections):], "copied part")


@pytest.mark.parametrize("tokens", [0, 1, 3, 4095, 4096, 4099])
def test_token_counts(tokens):
    """Both sides of the rule that gives a workgroup more than one token, and an empty call."""
    q = randn(1, tokens, 2, 64, seed=4, dtype=torch.bfloat16)
    p = places(2, 1, tokens, seed=5)
    out = multi_axis_rotary(q, None, p, (12, 20))
    check_rotated(out, q, p, (12, 20))
    if tokens > 3:  # a token's bits do not depend on the others
        assert_bitwise(multi_axis_rotary(q[:, 2:3], None, p[:, :, 2:3], (12, 20)), out[:, 2:3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_and_negative_positions(dtype):
    """Far positions keep their angle: in 32 bits the product alone would be off by radians."""
    p = torch.tensor([[0, 1, -1, 123457, 10**6 + 1, 2**31 - 1, -(2**31), 2**40]], dtype=torch.int64).cuda()
    q = randn(8, 3, 64, seed=6, dtype=dtype)
    check_rotated(multi_axis_rotary(q, None, p, (32,), base=1e6), q, p, (32,), base=1e6)


def test_position_types_and_frequencies():
    q = randn(3, 5, 2, 32, seed=7, dtype=torch.float32)
    freq = [1.0, 0.3, 0.0, -0.2, 1e-3, 2.0, 0.7, 0.01]
    for dtype in (torch.int32, torch.int64, torch.float32):
        p = places(2, 3, 5, seed=8, dtype=dtype)
        if dtype == torch.float32:
            p = p + 0.375  # times between frames
        out = multi_axis_rotary(q, None, p, (3, 5), inv_freq=freq)
        check_rotated(out, q, p, (3, 5), str(dtype), inv_freq=freq)


def test_layouts():
    """Slices of one projection, transposed heads, one token, several leading dimensions, positions by strides."""
    qkv = randn(2, 7, (6 + 2 + 2) * 64, seed=9, dtype=torch.bfloat16)
    q, k = qkv[..., :384].view(2, 7, 6, 64), qkv[..., 384:512].view(2, 7, 2, 64)
    p = places(7, 2, 3, seed=10).permute(2, 1, 0)
    want = multi_axis_rotary(q.contiguous(), k.contiguous(), p.contiguous(), (8, 12, 12))
    for got in (multi_axis_rotary(q, k, p, (8, 12, 12)),
                [x.transpose(1, 2) for x in (
                    y.transpose(1, 2) for y in multi_axis_rotary(q.transpose(1, 2).contiguous().transpose(1, 2),
                                                                 k.transpose(1, 2).contiguous().transpose(1, 2), p, (8, 12, 12)))]):
        assert_bitwise(got[0], want[0])
        assert_bitwise(got[1], want[1])
    many = multi_axis_rotary(q.view(1, 2, 7, 6, 64), k.reshape(1, 2, 7, 2, 64), p.unsqueeze(1), (8, 12, 12))
    assert many[0].shape == (1, 2, 7, 6, 64)
    assert_bitwise(many[0][0], want[0])
    one = multi_axis_rotary(q[1, 3], k[1, 3], p[:, 1, 3], (8, 12, 12))
    assert_bitwise(one[0], want[0][1, 3])
    assert_bitwise(one[1], want[1][1, 3])
    # rows that start off the 16 bytes, elements that are not next to each other, one position for a whole batch
    odd = randn(2, 7, 6, 66, seed=11, dtype=torch.bfloat16)[..., 1:65]
    assert_bitwise(multi_axis_rotary(odd, None, p, (8, 12, 12)), multi_axis_rotary(odd.contiguous(), None, p, (8, 12, 12)))
    wide = randn(2, 7, 6, 128, seed=12, dtype=torch.float32)[..., ::2]
    assert_bitwise(multi_axis_rotary(wide, None, p, (8, 12, 12)), multi_axis_rotary(wide.contiguous(), None, p, (8, 12, 12)))
    same = p[:, :1].expand(3, 2, 7)
    assert_bitwise(multi_axis_rotary(q, None, same, (8, 12, 12)), multi_axis_rotary(q, None, same.contiguous(), (8, 12, 12)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", [False, True])
def test_gradient_is_the_inverse_rotation(dtype, pairs):
    q = randn(2, 9, 4, 72, seed=13, dtype=dtype).requires_grad_()
    k = randn(2, 9, 2, 72, seed=14, dtype=dtype).requires_grad_()
    p = places(2, 2, 9, seed=15)
    kw = dict(base=500.0, interleaved_pairs=pairs)
    out = multi_axis_rotary(q, k, p, (20, 10), **kw)
    g = [randn(*x.shape, seed=16 + i, dtype=dtype) for i, x in enumerate(out)]
    grads = torch.autograd.grad(out, (q, k), g)
    for got, want in zip(grads, g):
        check_rotated(got, want, p, (20, 10), "gradient", inverse=True, **kw)
    # against differences: the operator is linear, so a central difference of any step is its derivative
    if dtype == torch.float32:
        step = randn(*q.shape, seed=18, dtype=dtype)
        with torch.no_grad():
            diff = (multi_axis_rotary(q + step, None, p, (20, 10), **kw)
                    - multi_axis_rotary(q - step, None, p, (20, 10), **kw)).double() / 2
        directional = (grads[0].double() * step.double()).sum()
        scale = (g[0].double().abs() * diff.abs()).sum()
        assert abs(directional - (diff * g[0].double()).sum()) <= 1e-5 * scale


def test_gradients_of_one_tensor_and_of_gradients():
    q = randn(4, 2, 16, seed=19, dtype=torch.float32).requires_grad_()
    k = randn(4, 1, 16, seed=20, dtype=torch.float32)
    p = places(1, 4, seed=21)
    out_q, out_k = multi_axis_rotary(q, k, p, (8,))
    assert out_q.requires_grad
    (gq,) = torch.autograd.grad(out_q.sum(), q)
    check_rotated(gq, torch.ones_like(q), p, (8,), inverse=True)
    # only the keys' output is used, which the queries do not reach
    (none,) = torch.autograd.grad(multi_axis_rotary(q, k.requires_grad_(), p, (8,))[1].sum(), q, allow_unused=True)
    assert none is None or float(none.abs().max()) == 0.0
    # the gradient's own gradient is the rotation again
    g = torch.ones_like(q).requires_grad_()
    (gq,) = torch.autograd.grad(multi_axis_rotary(q, None, p, (8,)), q, g, create_graph=True)
    (gg,) = torch.autograd.grad(gq, g, k.expand(4, 2, 16))
    check_rotated(gg, k.expand(4, 2, 16), p, (8,))
    # broadcast inputs and gradients
    x = randn(1, 1, 16, seed=22, dtype=torch.float32).requires_grad_()
    (gx,) = torch.autograd.grad(multi_axis_rotary(x.expand(4, 2, 16), None, p, (8,)).sum(), x)
    want, bound = rotate64(torch.ones(4, 2, 16), p, (8,), inverse=True)
    assert (gx.cpu().double() - want.sum((0, 1), keepdim=True)).abs().max() <= 8 * (bound.max() + 8 * 2.0**-24 * 8)


def test_second_gradient_of_the_keys_alone():
    """Only the keys' output gets a gradient, and that gradient one of its own."""
    q, k = randn(4, 2, 16, seed=60, dtype=torch.float32), randn(4, 1, 16, seed=61, dtype=torch.float32).requires_grad_()
    p = places(1, 4, seed=62)
    for queries in (q, q.clone().requires_grad_()):
        out_k = multi_axis_rotary(queries, k, p, (8,))[1]
        g = torch.ones_like(k).requires_grad_()
        (gk,) = torch.autograd.grad(out_k, k, g, create_graph=True)
        check_rotated(gk, g, p, (8,), inverse=True)
        (gg,) = torch.autograd.grad(gk, g, k.detach())
        check_rotated(gg, k, p, (8,))


def test_graphs_outlive_the_frequency_table():
    """The host's table of a call may be gone (64 are kept) when its gradient runs."""
    q = randn(3, 2, 16, seed=63, dtype=torch.float32).requires_grad_()
    p = places(1, 3, seed=64)
    out = multi_axis_rotary(q, None, p, (8,), base=77.0)
    for i in range(100):
        multi_axis_rotary(q.detach(), None, p, (8,), base=100.0 + i)
    g = randn(3, 2, 16, seed=65, dtype=torch.float32)
    (gq,) = torch.autograd.grad(out, q, g)
    check_rotated(gq, g, p, (8,), base=77.0, inverse=True)


def test_no_gradient_for_positions():
    q = randn(3, 2, 16, seed=66, dtype=torch.float32)
    p = torch.rand(1, 3, device="cuda").requires_grad_()
    with pytest.raises(ValueError, match="positions"):
        multi_axis_rotary(q, None, p, (8,))
    with torch.no_grad():
        check_rotated(multi_axis_rotary(q, None, p, (8,)), q, p, (8,))


def test_graph_replays_forward_and_gradient():
    q = randn(5, 4, 64, seed=23, dtype=torch.bfloat16).requires_grad_()
    p = places(2, 5, seed=24)
    g = randn(5, 4, 64, seed=25, dtype=torch.bfloat16)

    def step():
        out = multi_axis_rotary(q, None, p, (16, 16))
        return out, *torch.autograd.grad(out, q, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [t.detach() for t in step()]
    for i in range(3):
        with torch.no_grad():
            q.copy_(randn(5, 4, 64, seed=30 + i, dtype=torch.bfloat16))
            p.copy_(places(2, 5, seed=40 + i))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(held, step()):
            assert_bitwise(got.detach(), want.detach(), f"replay {i}")


def test_capture_beside_a_living_graph_of_the_leaf_is_refused():
    q, k = (randn(5, h, 64, seed=26 + h, dtype=torch.bfloat16).requires_grad_() for h in (4, 2))
    p = places(2, 5, seed=29)
    for leaf in (q, k):
        alive = leaf * 2.0
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                multi_axis_rotary(q, k, p, (16, 16))
        del alive
    five = q.detach().view(1, 1, 5, 4, 64).requires_grad_()  # (the Python path)
    alive = five * 2.0
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            multi_axis_rotary(five, None, p.view(2, 1, 1, 5), (16, 16))
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [t.detach() for t in torch.autograd.grad(multi_axis_rotary(q, k, p, (16, 16)), (q, k), (q.detach(), k.detach()))]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(multi_axis_rotary(q, k, p, (16, 16)), (q, k), (q.detach(), k.detach()))
        for a, b in zip(got, want):
            assert_bitwise(a, b)


def test_without_pairs_and_with_special_values():
    q = randn(3, 2, 16, seed=26, dtype=torch.bfloat16)
    assert_bitwise(multi_axis_rotary(q, None, places(2, 3, seed=27), (0, 0)), q)
    q = q.float()
    q[0, 0, 0], q[1, 1, 3], q[2, 0, 15] = float("inf"), float("nan"), float("-inf")
    out = multi_axis_rotary(q, None, torch.zeros(1, 3, dtype=torch.int32).cuda(), (4,))
    # the pairs of these elements only: (0, 4) and (3, 7); the last one is copied
    bad = ~torch.isfinite(out)
    assert bad[0, 0, 0] and bad[1, 1, 3] and bad[2, 0, 15]
    assert int(bad.sum()) <= 5 and not bad[0, 1].any() and not bad[1, 0].any()
    nan = multi_axis_rotary(randn(1, 1, 8, seed=28, dtype=torch.float32), None, torch.full((1, 1), float("nan")).cuda(), (2,))
    assert torch.isnan(nan[..., :4]).all() and torch.isfinite(nan[..., 4:]).all()
