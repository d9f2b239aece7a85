"""Attention over pages with many query heads to a key head and wide values: a workgroup's partial results take more than 64 KiB
of LDS from 16 heads with values wider than 128 on."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import check_cache_indices, paged_attention_batch_invariant

from _decoder import check_token

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("hq, hkv, d, dv", [(16, 1, 128, 256), (17, 1, 256, 256), (32, 2, 256, 200), (15, 1, 64, 256), (33, 1, 72, 136)])
def test_wide_groups_of_wide_values(dtype, hq, hkv, d, dv):
    lengths, page = [0, 1, 33, 128, 700, 3000], 16
    g = torch.Generator().manual_seed(hq * d + dv)

    def randn(*shape):
        return torch.randn(*shape, generator=g).to(dtype).cuda()

    counts = [-(-n // page) for n in lengths]
    kc, vc = randn(sum(counts), page, hkv, d), randn(sum(counts), page, hkv, dv)
    table = torch.zeros(len(lengths), max(counts), dtype=torch.int32)
    order = torch.randperm(sum(counts), generator=g).to(torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = order[sum(counts[:b]):sum(counts[:b + 1])]
    table, q = table.cuda(), randn(len(lengths), hq, d)
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    for kw in ({}, dict(window=50, sinks=4)):
        out = paged_attention_batch_invariant(q, kc, vc, table, lens, **kw)
        for b, n in enumerate(lengths):
            check_token(out[b], q[b], kc, vc, table[b], n, what=f"sequence of {n}", **kw)
    check_cache_indices()
