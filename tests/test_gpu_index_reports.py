"""Index errors are reported for a device however it is named."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops.moe import check_moe_indices, deterministic_token_choice_moe

pytestmark = pytest.mark.gpu
NAMES = [None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)]


@pytest.mark.parametrize("name", NAMES, ids=str)
def test_cache_indices(name):
    bio.check_cache_indices(name)
    kc = torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16).cuda()
    bio.paged_cache_write(kc[0, :1], kc[0, :1], kc, kc.clone(), torch.tensor([8]).cuda())
    with pytest.raises(RuntimeError, match="outside its tensor"):
        bio.check_cache_indices(name)
    bio.check_cache_indices(name)


@pytest.mark.parametrize("name", NAMES, ids=str)
def test_expert_indices(name):
    check_moe_indices(name)
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16).cuda(), torch.ones(2, 1, dtype=torch.bfloat16).cuda()
    up, down = (torch.zeros(2, *s, dtype=torch.bfloat16).cuda() for s in ((64, 64), (64, 64)))
    deterministic_token_choice_moe(x, w, torch.tensor([[0], [5]]).cuda(), up, up, down)
    with pytest.raises(RuntimeError, match="outside"):
        check_moe_indices(name)
    check_moe_indices(name)
