"""A decoder's step with 8-bit layers, a 4-bit cache and sampled tokens: the operators together, captured, on several streams."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import (
    check_cache_indices,
    linear_int8_batch_invariant,
    multi_axis_rotary,
    paged_attention_batch_invariant,
    paged_attention_fp4_batch_invariant,
    paged_cache_read_fp4,
    paged_cache_write_fp4,
    quantize_tokens_int8,
    rotary_cache_write,
    sample_tokens_batch_invariant,
    varlen_sliding_window_attention_batch_invariant,
)

from _decoder import check_token
from _served import from_fp4, staying, to_fp4
from _tol import assert_bitwise

pytestmark = pytest.mark.gpu
HQ, HKV, D, PAGE, VOCAB, SECTIONS = 4, 2, 64, 16, 1000, (16, 8, 8)
SETTINGS = dict(temperature=0.9, top_k=200, top_p=0.95, min_p=1e-3)


@pytest.fixture(autouse=True)
def _no_error_left():
    yield
    check_cache_indices()


class Model:
    """One layer: prompts go through the window attention over what the cache holds, tokens through the cache."""

    def __init__(self, dtype=torch.bfloat16, lengths=(37, 1, 90, 16), steps=6, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.lengths, self.steps, n = dtype, list(lengths), steps, len(lengths)

        def weight(rows, cols):
            return quantize_tokens_int8((torch.randn(rows, cols, generator=g) * cols**-0.5).cuda())

        self.embed = torch.randn(VOCAB, HQ * D, generator=g).to(dtype).cuda()
        self.qkv, self.proj, self.head = weight((HQ + 2 * HKV) * D, HQ * D), weight(HQ * D, HQ * D), weight(VOCAB, HQ * D)
        self.prompts = torch.randint(0, VOCAB, (sum(lengths),), generator=g).cuda()
        self.u = torch.rand(steps + 1, n, generator=g).cuda()
        width = -(-(max(lengths) + steps) // PAGE)
        self.table = torch.randperm(n * width, generator=g).view(n, width).to(torch.int32).cuda()
        self.caches = [torch.full((n * width, PAGE, HKV, x), 255, dtype=torch.uint8, device="cuda") for x in (D // 2, D // 32) * 2]
        self.lens = torch.tensor(lengths, dtype=torch.int32).cuda()
        self.place = torch.cat([torch.arange(x) for x in lengths]).cuda()
        self.owner = torch.cat([torch.full((x,), i) for i, x in enumerate(lengths)]).cuda()
        self.cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0)], dtype=torch.int32).cuda()

    def linear(self, x, weight):
        q, s = quantize_tokens_int8(x)
        return linear_int8_batch_invariant(q, s, *weight, dtype=self.dtype)

    def split(self, h):
        sizes = [HQ * D, HKV * D, HKV * D]
        return (t.unflatten(-1, (-1, D)) for t in self.linear(h, self.qkv).split(sizes, -1))

    def answer(self, h, att, u):
        logits = self.linear(h + self.linear(att.flatten(-2), self.proj), self.head)
        return logits, sample_tokens_batch_invariant(logits, u, **SETTINGS)

    def slots(self, owner, place):
        return self.table.long()[owner, place // PAGE] * PAGE + place % PAGE

    def prompt(self):
        h = self.embed[self.prompts]
        q, k, v = self.split(h)
        q, k = multi_axis_rotary(q, k, self.place.expand(3, -1), SECTIONS)
        slots = self.slots(self.owner, self.place)
        paged_cache_write_fp4(k, v, *self.caches, slots)
        k, v = paged_cache_read_fp4(*self.caches, slots, dtype=self.dtype)  # as later tokens will see them
        att = varlen_sliding_window_attention_batch_invariant(q[None], k[None], v[None], self.cu, self.cu, None)[0]
        last = self.cu[1:].long() - 1
        return self.answer(h[last], att[last], self.u[0])

    def token(self, tokens, lens, u):
        """One step for sequences that hold `lens` tokens with the new one."""
        h = self.embed[tokens]
        q, k, v = self.split(h)
        at = lens.long() - 1
        rq = rotary_cache_write(q, k, v, self.caches[0], self.caches[2], self.slots(torch.arange(len(self.lengths), device="cuda"), at),
                                at.expand(3, -1), SECTIONS, key_scales=self.caches[1], value_scales=self.caches[3])
        att = paged_attention_fp4_batch_invariant(rq, *self.caches, self.table, lens)
        return (q, k, v, rq, att, *self.answer(h, att, u))

    def run(self):
        logits, tokens = self.prompt()
        lens, got = self.lens.clone(), [tokens]
        for i in range(self.steps):
            lens = lens + 1
            tokens = self.token(tokens, lens, self.u[i + 1])[-1]
            got.append(tokens)
        return torch.stack(got)


def check_sampled(logits, u, tokens):
    """Every token is the one whose interval of the running sum the random number is in (or next to, by 1e-6)."""
    for row, x, t in zip(logits, u.tolist(), tokens.tolist()):
        w, stay = staying(row, SETTINGS["temperature"], SETTINGS["top_k"], SETTINGS["top_p"], SETTINGS["min_p"])
        kept = torch.where(stay, w, 0.0)
        upto = kept.cumsum(0) / kept.sum()
        assert stay[t] and float(upto[t] - kept[t] / kept.sum()) - 1e-6 <= x <= float(upto[t]) + 1e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_then_tokens(dtype):
    m = Model(dtype)
    logits, tokens = m.prompt()
    check_sampled(logits, m.u[0], tokens)
    lens = m.lens.clone()
    for i in range(m.steps):
        lens = lens + 1
        q, k, v, rq, att, logits, new = m.token(tokens, lens, m.u[i + 1])
        want_q, want_k = multi_axis_rotary(q, k, (lens.long() - 1).expand(3, -1), SECTIONS)
        assert_bitwise(rq, want_q)
        at = m.slots(torch.arange(len(m.lengths), device="cuda"), lens.long() - 1)
        for rows, codes, scales in ((want_k, *m.caches[:2]), (v, *m.caches[2:])):
            bits = to_fp4(rows)
            assert torch.equal(codes.flatten(0, 1)[at].cpu(), bits[0]) and torch.equal(scales.flatten(0, 1)[at].cpu(), bits[1])
        kc, vc = from_fp4(*m.caches[:2]), from_fp4(*m.caches[2:])
        for b in range(len(m.lengths)):
            check_token(att[b], rq[b], kc, vc, m.table[b].cpu(), int(lens[b]), what=f"step {i} sequence {b}")
        check_sampled(logits, m.u[i + 1], new)
        tokens = new


@pytest.fixture
def in_python(monkeypatch):
    """Without the tensor module: the Python functions do all."""
    from batch_invariant_ops import decoder

    monkeypatch.setattr(decoder, "_tensor_module", False)
    monkeypatch.setattr(decoder, "_direct", lambda: False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_both_host_paths(dtype, request):
    """The same answer and the same bits in the cache; rows in a cache of the model's type too."""
    def plain():
        g = torch.Generator().manual_seed(7)
        q, k, v = (torch.randn(1500, n, 64, generator=g).to(dtype).cuda() for n in (4, 2, 2))
        kc, vc = (torch.zeros(100, 16, 2, 64, dtype=dtype, device="cuda") for _ in range(2))
        slots = torch.randint(-3, 1600, (1500,), generator=g).cuda()
        return rotary_cache_write(q, k, v, kc, vc, slots, torch.arange(1500, device="cuda").view(1, -1), (32,)), kc, vc

    m = Model(dtype)
    tokens, rows = m.run(), plain()
    request.getfixturevalue("in_python")
    again = Model(dtype)
    assert torch.equal(again.run(), tokens)
    for a, b in zip(again.caches, m.caches):
        assert torch.equal(a, b)
    for a, b in zip(plain(), rows):
        assert_bitwise(a, b)
    logits = torch.randn(3, 9000, generator=torch.Generator().manual_seed(8)).cuda()
    each = dict(temperature=torch.full((3,), 0.7).cuda(), top_k=torch.tensor([5, 0, 900]).cuda(), top_p=torch.tensor([1.0, 0.9, 0.5]).cuda(),
                min_p=torch.tensor([0.0, 0.1, 0.0]).cuda())
    got = sample_tokens_batch_invariant(logits, torch.tensor([0.1, 0.5, 0.9]).cuda(), **each)
    want = [int(sample_tokens_batch_invariant(logits[i:i + 1], torch.tensor([u]).cuda(), temperature=float(each["temperature"][i]),
                                              top_k=[5, None, 900][i], top_p=float(each["top_p"][i]), min_p=float(each["min_p"][i])))
            for i, u in enumerate((0.1, 0.5, 0.9))]
    assert got.tolist() == want


def test_a_query_is_needed():
    with pytest.raises(AttributeError):
        rotary_cache_write(None, *(torch.zeros(3, 2, 64, device="cuda") for _ in range(2)),
                           *(torch.zeros(4, 16, 2, 64, device="cuda") for _ in range(2)), torch.arange(3, device="cuda"),
                           torch.zeros(1, 3, dtype=torch.int64, device="cuda"), (32,))


def test_a_sequence_alone_gives_the_same_tokens():
    whole = Model().run()
    for b, n in enumerate(Model().lengths):
        m = Model()
        a, e = int(m.cu[b]), int(m.cu[b + 1])
        m.lengths, m.prompts, m.place, m.owner = [n], m.prompts[a:e], m.place[a:e], m.owner[a:e] * 0
        m.lens, m.table, m.u, m.cu = m.lens[b:b + 1], m.table[b:b + 1], m.u[:, b:b + 1], torch.tensor([0, n], dtype=torch.int32).cuda()
        assert torch.equal(m.run()[:, 0], whole[:, b])


def test_a_captured_step_replayed():
    """One graph decodes the whole answer: tokens, lengths and slots move on inside it; eager work between the replays."""
    eager, m = Model(seed=3), Model(seed=3)
    want = eager.run()
    first = m.prompt()[1]
    tokens, lens, u, step = first.clone(), m.lens.clone(), m.u[0].clone(), torch.zeros((), dtype=torch.int64, device="cuda")

    def once():
        lens.add_(1)
        step.add_(1)
        u.copy_(m.u.index_select(0, step.view(1))[0])
        tokens.copy_(m.token(tokens, lens, u)[-1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once()
    for again in range(3):
        tokens.copy_(first)
        lens.copy_(m.lens)
        step.zero_()
        for i in range(m.steps):
            graph.replay()
            assert torch.equal(tokens, want[i + 1]), f"round {again} step {i}"
            eager.token(want[0], eager.lens + 1, eager.u[1])  # (other work on the same kernels)
        torch.cuda.synchronize()


def test_two_captured_samplings_at_once():
    """Each graph has its workspace."""
    x = [(torch.randn(8, 40000, generator=torch.Generator().manual_seed(i)) * 2).cuda() for i in (1, 2)]
    u = [torch.rand(8, generator=torch.Generator().manual_seed(i)).cuda() for i in (3, 4)]
    want = [sample_tokens_batch_invariant(a, b, **SETTINGS) for a, b in zip(x, u)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in x]
    for a, b in zip(x, u):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(sample_tokens_batch_invariant(a, b, **SETTINGS))
        graphs.append(graph)
    for _ in range(5):
        for o in outs:
            o.fill_(-7)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_two_streams_at_once():
    want = [Model(torch.float16, seed=i).run() for i in (5, 6)]
    models = [Model(torch.float16, seed=i) for i in (5, 6)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in models], [None, None]
    for _ in range(3):
        for i, (m, stream) in enumerate(zip(models, streams)):
            with torch.cuda.stream(stream):
                got[i] = m.run()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("path", ["module", "python"])
@pytest.mark.parametrize("bits", [4, 16])
def test_attention_over_more_than_31_bits_of_slots(path, bits, request):
    """Pages are counted in 64 bits, on both host paths (a page repeated by its stride)."""
    if path == "python":
        request.getfixturevalue("in_python")
    g = torch.Generator().manual_seed(9)
    rows = [torch.randn(1, PAGE, HKV, D, generator=g).to(torch.bfloat16) for _ in range(2)]
    caches = [c.cuda() for x in rows for c in (to_fp4(x) if bits == 4 else (x,))]
    many = [c.expand((1 << 31) // PAGE + 5, *c.shape[1:]) for c in caches]
    q = torch.randn(2, HQ, D, generator=g).to(torch.bfloat16).cuda()
    lens = torch.tensor([40, 9]).cuda()
    table = torch.tensor([[(1 << 31) // PAGE + 4, 0, (1 << 31) // PAGE], [1 << 27, 0, 0]]).cuda()
    attention = paged_attention_fp4_batch_invariant if bits == 4 else paged_attention_batch_invariant
    assert_bitwise(attention(q, *many, table, lens), attention(q, *caches, table * 0, lens))
