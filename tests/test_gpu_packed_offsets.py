"""Packed offsets that break their rules are reported: where they start, and in calls without query rows or heads."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import check_cache_indices, varlen_sliding_window_attention_batch_invariant as packed_attention

pytestmark = pytest.mark.gpu


def run(cu_q, cu_k, rows, keys, heads=2, dtype=torch.int32):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(1, n, h, 64, generator=g).to(torch.bfloat16).cuda() for n, h in ((rows, heads), (keys, 2)))
    out = packed_attention(q, k, k, *(torch.tensor(x, dtype=dtype).cuda() for x in (cu_q, cu_k)), 5, 1)
    assert out.shape == (1, rows, heads, 64) and bool(torch.isfinite(out).all())


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("cu_q, cu_k, rows, keys, heads", [
    ([0, 20, 50], [3, 20, 50], 50, 50, 2), ([2, 20, 50], [0, 20, 50], 50, 50, 2), ([0, 0, 0], [1, 1, 9], 4, 9, 2), ([0], [2], 4, 9, 2),
    ([2], [0], 4, 9, 2), ([0] * 300, [4] * 300, 4, 9, 2),
    # no query rows
    ([0, 0, 0], [0, 7, 5], 0, 9, 2), ([0, 0], [0, 10], 0, 9, 2), ([0, 1], [0, 9], 0, 9, 2), ([0, 0], [1, 9], 0, 9, 2),
    ([0] * 999 + [-1], [0] * 1000, 0, 9, 2), ([0], [1], 0, 9, 2), ([0, 0], [0, 1], 0, 0, 2),
    # no heads
    ([0, 5], [0, 10], 5, 9, 0), ([0, 6], [0, 9], 5, 9, 0), ([1, 5], [0, 9], 5, 9, 0),
])
def test_reported(cu_q, cu_k, rows, keys, heads, dtype):
    check_cache_indices()
    run(cu_q, cu_k, rows, keys, heads, dtype)
    with pytest.raises(RuntimeError, match="outside its tensor"):
        check_cache_indices()


@pytest.mark.parametrize("cu_q, cu_k, rows, keys, heads", [
    ([0, 20, 50], [0, 20, 50], 60, 55, 2), ([0], [0], 4, 9, 2), ([0], [0], 0, 9, 2), ([0, 0, 0], [0, 5, 9], 0, 9, 2),
    ([0] * 1000, [0] * 999 + [9], 0, 9, 2), ([0, 5], [0, 9], 5, 9, 0), ([0, 0], [0, 0], 0, 0, 2),
])
def test_not_reported(cu_q, cu_k, rows, keys, heads):
    run(cu_q, cu_k, rows, keys, heads)
    check_cache_indices()


def test_a_captured_check():
    cu_q, cu_k = torch.zeros(3, dtype=torch.int32).cuda(), torch.tensor([0, 4, 9], dtype=torch.int32).cuda()
    k = torch.zeros(1, 9, 2, 64, dtype=torch.bfloat16).cuda()
    packed_attention(k[:, :0], k, k, cu_q, cu_k, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed_attention(k[:, :0], k, k, cu_q, cu_k, 5)
    for bad in (False, True, False):
        cu_k[1] = 10 if bad else 4
        graph.replay()
        torch.cuda.synchronize()
        if bad:
            with pytest.raises(RuntimeError, match="outside its tensor"):
                check_cache_indices()
        else:
            check_cache_indices()
