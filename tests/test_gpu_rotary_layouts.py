"""Rotations of tensors that are copied before the launch, on both host paths."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import decoder, multi_axis_rotary

from _decoder import check_rotated
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("lead", [(50,), (2, 25), (5, 1, 10)])
def test_copies_live_until_the_launch(python, lead, monkeypatch):
    """Strided heads are copied: the copy of the queries must not give its memory to the keys' output."""
    if python:
        monkeypatch.setattr(decoder, "_tensor_module", False)
        monkeypatch.setattr(decoder, "_direct", lambda: False)
    p = torch.randint(0, 99, (2, *lead)).cuda()
    for heads in ((4, 4), (8, 2), (2, 8)):
        wide = [randn(*lead, h, 64, 2, seed=h + i) for i, h in enumerate(heads)]
        q, k = (x[..., 0] for x in wide)
        assert q.stride(-1) == 2
        for _ in range(3):
            out = multi_axis_rotary(q, k, p, (20, 12))
            check_rotated(out[0], q, p, (20, 12), "queries")
            check_rotated(out[1], k, p, (20, 12), "keys")
        for a, b in zip(out, multi_axis_rotary(q.contiguous(), k.contiguous(), p, (20, 12))):
            assert_bitwise(a, b)
