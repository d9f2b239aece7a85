"""The decoder operators together, as a served policy runs them: rotate, write, attend to the prompt, then token by
token out of the pages.  Every step against its definition in 64 bits on what the step before it gave."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import (
    check_cache_indices,
    multi_axis_rotary,
    paged_attention_batch_invariant,
    paged_cache_write,
    sliding_window_attention_batch_invariant,
    varlen_sliding_window_attention_batch_invariant,
)
from model_invariance import run_investigation
from model_invariance.adapters import SyntheticDecoderAdapter

from _decoder import check_rotated, check_token, check_window, rows_of
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
HQ, HKV, D, PAGE, SECTIONS = 4, 2, 64, 16, (16, 8, 8)


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


class Served:
    """Prompts of their own lengths packed one behind another, and the pages they go to."""

    def __init__(self, dtype, lengths=(37, 1, 90, 16), steps=5, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.lengths, self.steps = dtype, list(lengths), steps
        total = sum(lengths)
        self.cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0)], dtype=torch.int32).cuda()
        width = -(-(max(lengths) + steps) // PAGE)
        self.table = torch.randperm(len(lengths) * width, generator=g).view(len(lengths), width).to(torch.int32).cuda()
        shape = (len(lengths) * width, PAGE, HKV, D)
        self.kc, self.vc = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.qkv = torch.randn(total, (HQ + 2 * HKV) * D, generator=g).to(dtype).cuda()
        self.new = torch.randn(steps, len(lengths), (HQ + 2 * HKV) * D, generator=g).to(dtype).cuda()
        self.place = torch.cat([torch.arange(n) for n in lengths]).cuda()
        self.owner = torch.cat([torch.full((n,), i) for i, n in enumerate(lengths)]).cuda()
        # a picture's rows and columns in front, the same place on every axis behind it
        self.positions = torch.stack([torch.where(self.place < 9, x, self.place) for x in (
            torch.zeros_like(self.place), self.place // 3, self.place % 3)])
        self.lens = torch.tensor(lengths, dtype=torch.int32).cuda()

    def slots(self, owner, place):
        return self.table.long()[owner, place // PAGE] * PAGE + place % PAGE

    @staticmethod
    def split(x):
        return (t.unflatten(-1, (-1, D)) for t in x.split([HQ * D, HKV * D, HKV * D], -1))

    def prompt(self, window, sinks):
        q, k, v = self.split(self.qkv)
        rq, rk = multi_axis_rotary(q, k, self.positions, SECTIONS)
        paged_cache_write(rk, v, self.kc, self.vc, self.slots(self.owner, self.place))
        return rq, rk, v, varlen_sliding_window_attention_batch_invariant(rq[None], rk[None], v[None], self.cu, self.cu, window, sinks)[0]

    def token(self, step, lens, window, sinks):
        """One step for sequences that hold `lens` tokens with the new one."""
        q, k, v = self.split(step)
        at = lens.long() - 1
        rq, rk = multi_axis_rotary(q, k, at.expand(3, -1), SECTIONS)
        paged_cache_write(rk, v, self.kc, self.vc, self.slots(torch.arange(len(self.lengths), device="cuda"), at))
        return rq, paged_attention_batch_invariant(rq, self.kc, self.vc, self.table, lens, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window, sinks", [(None, 0), (20, 3)])
def test_prompts_then_tokens(dtype, window, sinks):
    s = Served(dtype)
    rq, rk, v, out = s.prompt(window, sinks)
    q, k, _ = s.split(s.qkv)
    check_rotated(rq, q, s.positions, SECTIONS)
    check_rotated(rk, k, s.positions, SECTIONS)
    for b, n in enumerate(s.lengths):
        a, e = int(s.cu[b]), int(s.cu[b + 1])
        assert_bitwise(rows_of(s.kc, s.table[b], n, PAGE), rk[a:e])
        assert_bitwise(rows_of(s.vc, s.table[b], n, PAGE), v[a:e])
        rows = [t[a:e].transpose(0, 1) for t in (out, rq, rk, v)]
        check_window(*rows, window, sinks, what=f"prompt {b}")
        # the prompt's last row by the other operator
        last = paged_attention_batch_invariant(rq[e - 1:e], s.kc, s.vc, s.table[b:b + 1], s.lens[b:b + 1], window=window, sinks=sinks)
        check_token(last[0], rq[e - 1], s.kc, s.vc, s.table[b], n, window, sinks, what=f"prompt {b}'s last row")
    lens = s.lens.clone()
    for step in range(s.steps):
        lens = lens + 1
        rq, out = s.token(s.new[step], lens, window, sinks)
        for b in range(len(s.lengths)):
            check_token(out[b], rq[b], s.kc, s.vc, s.table[b], int(lens[b]), window, sinks, what=f"step {step} sequence {b}")
    # the whole sequence as one prompt: the last row of the longest, from its rows in the pages
    n = int(lens[2])
    k, v = (rows_of(c, s.table[2], n, PAGE).transpose(0, 1) for c in (s.kc, s.vc))
    again = sliding_window_attention_batch_invariant(rq[2].view(1, HQ, 1, D), k[None], v[None], window, sinks, enable_gqa=True)
    check_window(again[0], rq[2].unsqueeze(1), k, v, window, sinks, what="as a prompt")


def test_a_captured_step_replayed():
    """One graph decodes the whole answer: lengths and slots move on inside it, new rows come in from outside."""
    window, sinks = 20, 3
    eager, s = Served(torch.bfloat16), Served(torch.bfloat16)
    eager.prompt(window, sinks)
    s.prompt(window, sinks)
    step, lens = s.new[0].clone(), s.lens.clone()

    def once():
        lens.add_(1)
        return s.token(step, lens, window, sinks)[1]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    want = eager.lens.clone()
    for again in range(2):
        lens.copy_(s.lens)
        want.copy_(eager.lens)
        for i in range(s.steps):
            step.copy_(s.new[i])
            graph.replay()
            want = want + 1
            assert_bitwise(out, eager.token(eager.new[i], want, window, sinks)[1], f"step {i}")
        torch.cuda.synchronize()
    assert_bitwise(s.kc, eager.kc)
    assert_bitwise(s.vc, eager.vc)


def test_two_streams_at_once():
    """Two batches, each with caches and a stream of its own."""
    served = [Served(torch.float16, seed=i) for i in (2, 3)]
    alone = [Served(torch.float16, seed=i) for i in (2, 3)]

    def answer(s):
        got = [s.prompt(20, 3)[3]]
        lens = s.lens.clone()
        for i in range(s.steps):
            lens = lens + 1
            got.append(s.token(s.new[i], lens, 20, 3)[1])
        return got

    want = [answer(s) for s in alone]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in served]
    got = [[], []]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(served, streams)):
            with torch.cuda.stream(stream):
                got[i] = answer(s)
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(got[i], want[i]):
            assert_bitwise(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_synthetic_decoder_is_batch_invariant_end_to_end_under_the_mode(dtype):
    report = run_investigation(SyntheticDecoderAdapter(dtype=dtype), batch_sizes=(1, 2, 3, 5, 8, 17), invariant_ops=True)
    assert report["repeatability"]["exact"]
    bad = [(name, r["batch_size"]) for name, rs in report["composition_results"].items() for r in rs if r["status"] != "PASS"]
    assert not bad, f"not batch invariant: {bad}"
    assert report["end_to_end_exact"]
