"""The work that is timed for a decoder served with 8-bit weights and a 4-bit cache: new keys and values
rotated on their way into a cache in pages, the same cache in 4 bits with its write and its attention, the
choice of the next token, and linear layers of 8-bit integers.

``listed()`` names twelve cases; ``draw`` gives further ones of the same ranges.  Head counts and sizes are
those of the repository's configurations, tests and benchmark (16 query and 4 key/value heads of 128, 8 and
2 of 64, linear layers of 2048 -> 8192 and 8192 -> 2048 over 1 to 4096 rows) or generic ones.  With ``own``
false, ``run`` computes the operators from elementary products, sums, exponentials, comparisons and
indexing, in 32 bits (angles, and the sampled distributions with their borders, in 64).

A row in 4 bits is cut into blocks of 32: 32 values of one sign, two exponent and one mantissa bit (0, 0.5, 1,
1.5, 2, 3, 4, 6), two to a byte with the first in the low half, and a power of two as a biased exponent byte.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# exponents of a block: its values (multiples of 2^(e - 1), up to 6 2^e) are normal numbers of the rows' type, or fp16's steps
_EXPONENTS = {"bf16": (-125, 125), "fp16": (-23, 13)}


def _library():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "robotics-batch-invariant-ops_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import batch_invariant_ops

    return batch_invariant_ops


def listed():
    return [
        # one new token of each of 48 sequences into a cache of the model's type: bound by its launch
        dict(name="append_decode", kind="append", dtype="bf16", tokens=48, hq=16, hkv=4, d=128, sections="16,24,24",
             pairs=False, page=16, spare=4.0, four=False),
        # a batch of prompts, two thirds of a head rotated, an odd number of tokens
        dict(name="append_prompt", kind="append", dtype="fp16", tokens=16383, hq=16, hkv=4, d=96, sections="32",
             pairs=True, page=64, spare=0.3, four=False),
        # one new token of each of 64 sequences into a cache in 4 bits, read back as values
        dict(name="append4_decode", kind="append", dtype="bf16", tokens=64, hq=16, hkv=4, d=128, sections="64",
             pairs=False, page=16, spare=4.0, four=True),
        # prompts whose rotated keys are there already, into a cache in 4 bits and back
        dict(name="write4_prompt", kind="write4", dtype="bf16", tokens=32768, hkv=4, d=128, page=16, spare=0.1),
        # one request in the middle of its answer
        dict(name="decode4_single", kind="decode4", dtype="bf16", seqs=1, shortest=2047, longest=2047, hq=16, hkv=4,
             d=128, page=16, window=0, sinks=0),
        # a serving batch with lengths from a short prompt to a long document
        dict(name="decode4_batch", kind="decode4", dtype="bf16", seqs=64, shortest=250, longest=16384, hq=16, hkv=4,
             d=128, page=16, window=0, sinks=0),
        # small heads under a window with four first tokens that stay visible, pages of an odd number
        dict(name="decode4_window", kind="decode4", dtype="fp16", seqs=100, shortest=17, longest=9001, hq=8, hkv=2,
             d=64, page=49, window=1024, sinks=4),
        # the next token of one request, the same settings for every call
        dict(name="sample_one", kind="sample", dtype="bf16", rows=1, vocab=32000, temperature=0.7, top_k=40, top_p=0.95,
             min_p=0.0, each=False),
        # a batch whose requests bring their own settings, a large vocabulary in float32
        dict(name="sample_batch", kind="sample", dtype="fp32", rows=64, vocab=131072, temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.02, each=True),
        # a linear layer of one decoding step: its weights are the traffic
        dict(name="linear8_decode", kind="linear8", dtype="bf16", rows=16, k=2048, n=8192, bias=False),
        # the layer back, for a prompt: the largest product
        dict(name="linear8_prompt", kind="linear8", dtype="bf16", rows=4096, k=8192, n=2048, bias=True),
        # sizes off every tile
        dict(name="linear8_odd", kind="linear8", dtype="fp16", rows=777, k=2050, n=1031, bias=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case: every kind equally often, sizes over the logarithm of their range, cut until it costs no more
    than the largest listed case of its kind."""
    kind = rng.choice(["append", "write4", "decode4", "decode4", "sample", "linear8"])
    dtype = rng.choice(["bf16", "fp16"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 7, 8])
    d = rng.choice([64, 96, 128, 128])
    if kind == "append":
        four = rng.random() < 0.4
        turned = rng.choice([d // 2, d // 2, d // 4])
        cuts = sorted(rng.sample(range(1, turned), rng.choice([0, 0, 2])))
        sections = [b - a for a, b in zip([0, *cuts], [*cuts, turned])]
        # (a rotation may be off in its last place: in 4 bits few enough values that none of them lies next to a border)
        case = dict(kind=kind, dtype=dtype if four else rng.choice(["bf16", "fp16", "fp32"]),
                    tokens=_log_int(rng, 1, 128 if four else 16384), hq=hq, hkv=hkv, d=d,
                    sections=",".join(map(str, sections)), pairs=rng.random() < 0.4,
                    page=rng.choice([1, 16, 32, 64, 100, 128]), spare=rng.uniform(0.0, 2.0), four=four)
        shrink = "tokens"
    elif kind == "write4":
        case = dict(kind=kind, dtype=dtype, tokens=_log_int(rng, 1, 32768), hkv=hkv, d=d,
                    page=rng.choice([1, 16, 32, 64, 100, 128]), spare=rng.uniform(0.0, 1.0))
        shrink = "tokens"
    elif kind == "decode4":
        longest = _log_int(rng, 1, 32768)
        window = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        case = dict(kind=kind, dtype=dtype, seqs=_log_int(rng, 1, 128), shortest=_log_int(rng, 1, longest),
                    longest=longest, hq=hq, hkv=hkv, d=d, page=rng.choice([8, 16, 32, 64, 100, 128]), window=window,
                    sinks=rng.choice([0, 1, 4, 64]) if window else 0)
        shrink = "seqs"
    elif kind == "sample":
        vocab = _log_int(rng, 100, 131072)
        case = dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), rows=_log_int(rng, 1, 256), vocab=vocab,
                    temperature=rng.uniform(0.3, 1.5), top_k=rng.choice([0, _log_int(rng, 1, vocab)]),
                    top_p=rng.choice([1.0, rng.uniform(0.3, 1.0)]), min_p=rng.choice([0.0, rng.uniform(0.0, 0.3)]),
                    each=rng.random() < 0.5)
        shrink = "rows"
    else:
        case = dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), rows=_log_int(rng, 1, 4096),
                    k=_log_int(rng, 64, 8192), n=_log_int(rng, 64, 8192), bias=rng.random() < 0.5)
        if rng.random() < 0.6:  # most layers have whole tiles
            case["k"], case["n"] = -(-case["k"] // 128) * 128, -(-case["n"] // 64) * 64
        shrink = "rows"
    works = [work(c) for c in listed() if c["kind"] == kind]
    most = {x: max(w[x] for w in works) for x in ("bytes", "flops")}
    while case[shrink] > 1 and not _within(case, most):
        case[shrink] = case[shrink] // 2
    while not _within(case, most):
        case["longest"] = max(1, case["longest"] * 2 // 3)
        case["shortest"] = min(case["shortest"], case["longest"])
    return case


def _within(case, most):
    w = work(case)
    if case["kind"] == "decode4":  # the plain form gathers pages of the longest sequence for each
        if case["seqs"] * case["longest"] * case["hkv"] * case["d"] > 64 * 16384 * 4 * 128:
            return False
    # plain rows are read several times over, in 64 bits
    if case["kind"] == "sample" and case["rows"] * case["vocab"] > 64 * 131072:
        return False
    return w["bytes"] <= most["bytes"] and w["flops"] <= max(most["flops"], 1)


# ------------------------------------------------------------------------------- inputs ----
def _lengths(case):
    """Lengths of a batch, evenly spread over the logarithm of their range (the same for every seed)."""
    n, low, high = case["seqs"], case["shortest"], case["longest"]
    if n == 1:
        return [high]
    return [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _make(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = _DTYPES[case["dtype"]], case["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (high - low) + low

    def integers(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")

    if kind in ("append", "write4"):
        t, hkv, d, page = (case[x] for x in ("tokens", "hkv", "d", "page"))
        pages = -(-int(t * (1.0 + case["spare"])) // page)
        if t < 256:  # new tokens of as many sequences: one slot each, anywhere in the cache
            slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
        else:  # whole prompts: page after page
            order = torch.randperm(pages, generator=g, device="cuda")[:-(-t // page)]
            slots = (order.view(-1, 1) * page + torch.arange(page, device="cuda")).view(-1)[:t].contiguous()
        s = dict(slots=slots)
        if kind == "append":
            hq = case["hq"]
            qkv = normal(t, (hq + 2 * hkv) * d)  # one projection's output
            s["q"], s["k"], s["v"] = (x.unflatten(-1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], -1))
            s["positions"] = integers(0, 30000, len(_sections(case)), t)
        else:
            s["k"], s["v"] = normal(t, hkv, d), normal(t, hkv, d)
        if kind == "write4" or case["four"]:
            # what earlier requests left there
            low = 127 + _EXPONENTS[case["dtype"]][0]
            s["kc"], s["vc"] = (integers(0, 256, pages, page, hkv, d // 2).to(torch.uint8) for _ in range(2))
            s["ks"], s["vs"] = (integers(max(low, 124), 128, pages, page, hkv, d // 32).to(torch.uint8) for _ in range(2))
            s["all"] = torch.arange(pages * page, device="cuda")
        else:
            s["kc"], s["vc"] = normal(pages, page, hkv, d), normal(pages, page, hkv, d)
        return s
    if kind == "decode4":
        n, hq, hkv, d, page = (case[x] for x in ("seqs", "hq", "hkv", "d", "page"))
        lengths = torch.tensor(_lengths(case), device="cuda")[torch.randperm(n, generator=g, device="cuda")]
        width = -(-case["longest"] // page)
        counts = -(-lengths // page)
        pages = int(counts.sum())
        order = torch.randperm(pages, generator=g, device="cuda")
        table = torch.zeros(n, width, dtype=torch.int64, device="cuda")
        table[torch.arange(width, device="cuda") < counts.view(-1, 1)] = order
        s = dict(q=normal(n, hq, d), table=table.to(torch.int32), lengths=lengths.to(torch.int32))
        s["kc"], s["ks"] = _in_four_bits(normal(pages, page, hkv, d), case["dtype"])
        s["vc"], s["vs"] = _in_four_bits(normal(pages, page, hkv, d), case["dtype"])
        return s
    if kind == "sample":
        r, v = case["rows"], case["vocab"]
        logits = torch.randn(r, v, generator=g, device="cuda") * 2.0
        likely = integers(0, v, r, 24)  # a model has a few words in mind
        logits.scatter_add_(1, likely, uniform(2.0, 12.0, r, 24))
        s = dict(logits=logits.to(dtype), u=uniform(0.0, 1.0, r))
        if case["each"]:
            s["temperature"] = case["temperature"] * uniform(0.5, 1.5, r)
            s["top_k"] = integers(1, max(2, min(v, 2 * case["top_k"] or v)), r).to(torch.int32)
            s["top_p"] = (case["top_p"] * uniform(0.8, 1.1, r)).clamp(max=1.0)
            s["min_p"] = case["min_p"] * uniform(0.0, 2.0, r)
        return s
    m, k, n = (case[x] for x in ("rows", "k", "n"))
    # rows of different sizes, as a residual stream has them
    return dict(x=(torch.randn(m, k, generator=g, device="cuda") * uniform(0.2, 5.0, m, 1)).to(dtype),
                w=integers(-127, 128, n, k).to(torch.int8), ws=uniform(0.5, 1.5, n) * (k**-0.5 / 73.0),
                bias=normal(n) if case["bias"] else None)


def prepare(case, seed):
    s = dict(case=case, **_make(case, seed))
    if case["kind"] == "append":
        s["sections"] = _sections(case)
        n = sum(s["sections"])
        axis_of = [a for a, m in enumerate(s["sections"]) for _ in range(m)]
        s["axis_of"] = torch.tensor(axis_of, device="cuda")
        s["freq"] = torch.tensor([10000.0 ** (-i / n) for i in range(n)], dtype=torch.float64, device="cuda")
    if case["kind"] in ("append", "write4", "decode4"):
        s["levels"] = torch.tensor([*_LEVELS, *(-x for x in _LEVELS)], device="cuda")
    return s


# -------------------------------------------------------------------------- plain forms ----
def _in_four_bits(x, dtype):
    """(packed bytes [..., d / 2], exponent bytes [..., d / 32]) of rows [..., d]: the block's power of two is the
    smallest 2^e with every value at most 7 2^e, values go to the nearest level (ties to the even code, past 6 to 6)."""
    low, high = _EXPONENTS[dtype]
    blocks = x.float().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    fraction, exponent = torch.frexp(top)  # top = fraction 2^exponent, fraction in [0.5, 1)
    e = torch.where(fraction <= 0.875, exponent - 3, exponent - 2)
    e = torch.where(top == 0, low, e).clamp(low, high)
    sized = blocks.abs() * torch.ldexp(torch.ones_like(top), -e).unsqueeze(-1)
    code = ((sized > 0.25).int() + (sized >= 0.75).int() + (sized > 1.25).int() + (sized >= 1.75).int()
            + (sized > 2.5).int() + (sized >= 3.5).int() + (sized > 5.0).int())
    code = (code + 8 * torch.signbit(blocks).int()).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), (e + 127).to(torch.uint8)


def _values(packed, exponents, levels):
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).long()
    power = torch.ldexp(torch.ones_like(exponents, dtype=torch.float32), exponents.int() - 127)
    return (levels[codes].unflatten(-1, (-1, 32)) * power.unsqueeze(-1)).flatten(-2)


def _turned(x, angle, pairs):
    n, dtype = angle.shape[-1], x.dtype
    x = x.float()
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([ya, yb], -1).flatten(-2) if pairs else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., 2 * n:]], -1).to(dtype)


def _plain_append(s):
    case, slots, q, k = s["case"], s["slots"], None, s["k"]
    if case["kind"] == "append":
        angle = s["positions"][s["axis_of"]].movedim(0, -1).double() * s["freq"]
        q, k = (_turned(s[x], angle, case["pairs"]) for x in "qk")
    if "ks" not in s:
        s["kc"].flatten(0, 1)[slots] = k
        s["vc"].flatten(0, 1)[slots] = s["v"]
        return q, s["kc"], s["vc"]
    for rows, data, exponents in ((k, "kc", "ks"), (s["v"], "vc", "vs")):
        packed, e = _in_four_bits(rows, case["dtype"])
        s[data].flatten(0, 1)[slots] = packed
        s[exponents].flatten(0, 1)[slots] = e
    read = [_values(s[a].flatten(0, 1)[s["all"]], s[b].flatten(0, 1)[s["all"]], s["levels"]).to(k.dtype)
            for a, b in (("kc", "ks"), ("vc", "vs"))]
    return (q, *read) if q is not None else tuple(read)


def _plain_decode4(s):
    case = s["case"]
    table, lengths = s["table"].long(), s["lengths"].long().view(-1, 1)
    k = _values(s["kc"][table], s["ks"][table], s["levels"]).flatten(1, 2).transpose(1, 2).unsqueeze(2)
    v = _values(s["vc"][table], s["vs"][table], s["levels"]).flatten(1, 2).transpose(1, 2).unsqueeze(2)
    j = torch.arange(k.shape[3], device="cuda")
    seen = j < lengths
    if case["window"]:
        seen = seen & ((j >= lengths - case["window"]) | (j < case["sinks"]))
    q = s["q"].float().unflatten(1, (case["hkv"], -1)).unsqueeze(3) / math.sqrt(case["d"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).masked_fill_(~seen.view(len(table), 1, 1, 1, -1), -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(weights, v) / weights.sum(-1, keepdim=True)
    return out.squeeze(3).flatten(1, 2).to(s["q"].dtype)


def _plain_sample(s):
    """The kept tokens are a beginning of the row sorted downwards (equal ones by their index)."""
    case = s["case"]
    column = (lambda x: s[x].double().view(-1, 1)) if case["each"] else (lambda x: case[x])  # noqa: E731
    x = s["logits"].double() / column("temperature")
    weights = (x - x.amax(-1, keepdim=True)).exp()
    down, index = torch.sort(weights, dim=-1, descending=True, stable=True)
    place = torch.arange(x.shape[1], device="cuda")
    if case["each"] or case["top_k"]:
        down = torch.where(place < column("top_k"), down, 0.0)
    before = down.cumsum(-1) - down
    kept = (before < column("top_p") * down.sum(-1, keepdim=True)) & (down >= column("min_p")) & (down > 0)
    weights = torch.zeros_like(down).scatter_(1, index, torch.where(kept, down, 0.0))
    upto = weights.cumsum(-1)
    chosen = (upto > s["u"].double().view(-1, 1) * upto[:, -1:]) & (weights > 0)
    return chosen.int().argmax(-1)


def _plain_linear8(s):
    x = s["x"].float()
    top = x.abs().amax(-1, keepdim=True).clamp(min=2.0**-100)
    q = torch.round(x * torch.div(torch.full_like(top, 127.0), top))
    scale = top / 127.0
    y = torch.matmul(q, s["w"].float().t()) * scale * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return q.to(torch.int8), scale.squeeze(-1), y.to(s["x"].dtype)


_PLAIN = {"append": _plain_append, "write4": _plain_append, "decode4": _plain_decode4, "sample": _plain_sample,
          "linear8": _plain_linear8}


# -------------------------------------------------------------------------------- calls ----
def _own(s):
    bio, case = _library(), s["case"]
    if case["kind"] == "append":
        q = bio.rotary_cache_write(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["positions"], s["sections"],
                                   key_scales=s.get("ks"), value_scales=s.get("vs"), interleaved_pairs=case["pairs"])
        if not case["four"]:
            return q, s["kc"], s["vc"]
        return q, *bio.paged_cache_read_fp4(s["kc"], s["ks"], s["vc"], s["vs"], s["all"], dtype=s["k"].dtype)
    if case["kind"] == "write4":
        bio.paged_cache_write_fp4(s["k"], s["v"], s["kc"], s["ks"], s["vc"], s["vs"], s["slots"])
        return bio.paged_cache_read_fp4(s["kc"], s["ks"], s["vc"], s["vs"], s["all"], dtype=s["k"].dtype)
    if case["kind"] == "decode4":
        return bio.paged_attention_fp4_batch_invariant(s["q"], s["kc"], s["ks"], s["vc"], s["vs"], s["table"], s["lengths"],
                                                       window=case["window"] or None, sinks=case["sinks"])
    if case["kind"] == "sample":
        if case["each"]:
            return bio.sample_tokens_batch_invariant(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                                     top_p=s["top_p"], min_p=s["min_p"])
        return bio.sample_tokens_batch_invariant(s["logits"], s["u"], temperature=case["temperature"],
                                                 top_k=case["top_k"] or None, top_p=case["top_p"], min_p=case["min_p"])
    q, scale = bio.quantize_tokens_int8(s["x"])
    return q, scale, bio.linear_int8_batch_invariant(q, scale, s["w"], s["ws"], s["bias"], dtype=s["x"].dtype)


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# ----------------------------------------------------------------------- necessary work ----
def work(case):
    kind, e = case["kind"], _BYTES[case["dtype"]]
    if kind in ("append", "write4"):
        t, d, hkv = case["tokens"], case["d"], case["hkv"]
        kept = 2 * hkv * (d // 2 + d // 32 if kind == "write4" or case["four"] else e * d)
        size, flops = t * (2 * e * hkv * d + kept) + 8 * t, 0
        if kind == "write4" or case["four"]:  # and back, every slot of the cache
            slots = -(-int(t * (1.0 + case["spare"])) // case["page"]) * case["page"]
            size += slots * (kept + 2 * e * hkv * d + 8)
        if kind == "append":
            size += 2 * e * t * case["hq"] * d + 8 * t * len(_sections(case))
            flops = 6 * t * (case["hq"] + hkv) * sum(_sections(case))
        return {"bytes": size, "flops": flops}
    if kind == "decode4":
        d, hq, hkv, seen = case["d"], case["hq"], case["hkv"], 0
        for n in _lengths(case):
            start = max(0, n - (case["window"] or n))
            seen += n - start + min(case["sinks"], start)
        return {"bytes": 2 * hkv * seen * (d // 2 + d // 32) + 2 * e * case["seqs"] * hq * d, "flops": 4 * hq * d * seen}
    if kind == "sample":
        return {"bytes": case["rows"] * (e * case["vocab"] + 12), "flops": 4 * case["rows"] * case["vocab"]}
    m, k, n = (case[x] for x in ("rows", "k", "n"))
    return {"bytes": m * k * (e + 1) + 4 * m + n * k + 4 * n + e * m * n + (e * n if case["bias"] else 0),
            "flops": 2 * m * n * k}


# ------------------------------------------------------------------------ 64-bit values ----
def _rounded_to_four(rows, dtype):
    """What rows [..., d] become in 4 bits, in 64 bits: the nearest level of each block by distances, the even code
    where two are as near."""
    low, high = _EXPONENTS[dtype]
    x = rows.double().reshape(-1, 32)
    top = x.abs().max(1, keepdim=True).values
    power = torch.full_like(top, 2.0**low)
    for e in range(low, high):
        power = torch.where(top > 7.0 * 2.0**e, 2.0 ** (e + 1), power)
    levels = torch.tensor(_LEVELS, dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for at in range(0, x.shape[0], 1 << 18):
        part = x[at:at + (1 << 18)] / power[at:at + (1 << 18)]
        far = (part.abs().unsqueeze(-1) - levels).abs()
        near = far.min(-1, keepdim=True).values
        # of two levels as near, the one with an even code
        odd = torch.tensor([0, 1, 0, 1, 0, 1, 0, 1], device=x.device)
        pick = torch.where(far == near, odd, 2).min(-1).indices
        out[at:at + (1 << 18)] = levels[pick] * part.sign() * power[at:at + (1 << 18)]
    return out.reshape(rows.shape)


def _decoded(packed, exponents):
    """The values of 4-bit rows in 64 bits, from the bits' meaning: (-1)^s 2^(x - 1) 1.m, or m / 2 where x is 0."""
    codes = torch.stack([packed.long() % 16, packed.long() // 16], -1).flatten(-2)
    sign, x, m = codes // 8, codes // 2 % 4, codes % 2
    size = torch.where(x == 0, m.double() / 2, (1 + m.double() / 2) * torch.pow(2.0, (x - 1).double()))
    return torch.where(sign == 1, -size, size) * torch.pow(2.0, exponents.double() - 127).repeat_interleave(32, -1)


def _exact_append(t, case):
    out, k = [], t["k"]
    if case["kind"] == "append":
        sections = _sections(case)
        n = sum(sections)
        axis_of = [a for a, m in enumerate(sections) for _ in range(m)]
        turned = []
        for x in (t["q"], t["k"]):
            y = x.double().clone()
            for i in range(n):
                angle = t["positions"][axis_of[i]].double().unsqueeze(-1) * 10000.0 ** (-i / n)
                a, b = (2 * i, 2 * i + 1) if case["pairs"] else (i, i + n)
                z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(angle), angle)
                y[..., a], y[..., b] = z.real, z.imag
            turned.append(y)
        out.append(turned[0])
        k = turned[1]
    for name, exponents, rows in (("kc", "ks", k), ("vc", "vs", t["v"])):
        if exponents in t:
            new = _decoded(t[name], t[exponents])
            rows = _rounded_to_four(rows.to(t["k"].dtype), case["dtype"])  # a rotated key is rounded to the rows' type
        else:
            new, rows = t[name].double(), rows.double()
        new[t["slots"] // case["page"], t["slots"] % case["page"]] = rows
        out.append(new.flatten(0, 1) if exponents in t else new)
    return out


def _exact_decode4(t, case):
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    group = case["hq"] // case["hkv"]
    for b, n in enumerate(t["lengths"].tolist()):
        pages = t["table"][b, :-(-n // case["page"])].long()
        k, v = (_decoded(t[x][pages], t[y][pages]).flatten(0, 1)[:n] for x, y in (("kc", "ks"), ("vc", "vs")))
        j = torch.arange(n, device="cuda")
        hidden = (j < n - case["window"]) & (j >= case["sinks"]) if case["window"] else j < 0
        for h in range(case["hq"]):
            scores = (k[:, h // group] @ t["q"][b, h].double()) * case["d"] ** -0.5
            out[b, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), 0) @ v[:, h // group]
    return out


def exact(case, seed):
    if case["kind"] == "sample":
        return None  # whole numbers
    t = _make(case, seed)
    if case["kind"] in ("append", "write4"):
        return _exact_append(t, case)
    if case["kind"] == "decode4":
        return _exact_decode4(t, case)
    x = t["x"].double()
    top = x.abs().max(1).values
    # the steps are 32-bit numbers by definition: a row's largest value goes to 127
    q = (x.float() * torch.div(torch.full_like(top, 127.0), top).float().unsqueeze(1)).double().round()
    y = (q @ t["w"].double().t()) * (top / 127.0).unsqueeze(1) * t["ws"].double()
    return [None, top / 127.0, y if t["bias"] is None else y + t["bias"].double()]
