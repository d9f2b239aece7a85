"""Operators of a decoder served with fewer bits and fewer launches: keys and values rotated on their way into a cache in
pages, such a cache in 4 bits with its write, its read and its attention, linear layers of 8-bit integers, and the choice of
the next token.

They stand beside the operators of ``decoder`` and keep their contract: a row's bits depend on its own sequence only, device
indices are checked by the kernels and reported later (``check_cache_indices()``), no call waits for the GPU, and all of them
may be captured into a graph (the cache operators after one call outside of a capture on that device).  None has a gradient
or a forward-mode derivative or can be recorded by ``torch.jit.trace``: all are refused.  The reference has no counterpart of
them.

A cache in 4 bits is four ``uint8`` tensors: keys ``[pages, page_size, kv_heads, head_dim / 2]`` and their scales ``[..., head_dim
/ 32]``, values and theirs.  A row is cut into blocks of 32 elements.  A block's scale byte ``x`` stands for the power of two
``2 ** (x - 127)``; an element is a sign, two exponent bits and a mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6) times that power,
two to a byte, the first in the low half.  (The OCP microscaling format MXFP4.)  The power is the smallest of which no
element of the block is more than 7, so no element is off by more than that power.  Powers lie in [2 ** -125, 2 ** 125] for
bfloat16 rows and [2 ** -23, 2 ** 13] for float16 ones, where every value is a number of the rows' type; larger elements
become the largest value.  A block with an infinity or NaN has the scale byte 255 and stands for NaN as a whole.
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch

from . import _native as nat
from . import decoder
from .decoder import (
    _INDEX_TYPES,
    _POSITION_CODE,
    _call,
    _check_caches,
    _check_scale,
    _check_slots,
    _check_tensors,
    _check_window,
    _direct,
    _direct_watch,
    _fn,
    _overlaps,
    _refuse_transforms,
    _rotary_plan,
    _share,
    _unit_last,
    _watch,
)

__all__ = [
    "rotary_cache_write",
    "paged_cache_write_fp4",
    "paged_cache_read_fp4",
    "paged_attention_fp4_batch_invariant",
    "sample_tokens_batch_invariant",
    "quantize_tokens_int8",
    "linear_int8_batch_invariant",
]

_BLOCK = 32
_HALVES = (torch.bfloat16, torch.float16)


# ---------------------------------------------------------------------------- 4-bit caches ----
def _check_fp4(key_cache, key_scales, value_cache, value_scales, by_page=False) -> tuple[int, int]:
    """Head dimensions of the keys and the values of a cache in 4 bits."""
    dims = []
    for data, scales in ((key_cache, key_scales), (value_cache, value_scales)):
        if data.dim() != 4 or scales.dim() != 4:
            raise ValueError("4-bit caches have shapes [pages, page_size, kv_heads, head_dim / 2] and [..., head_dim / 32]")
        if data.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"4-bit caches and their scales are uint8, got {data.dtype} and {scales.dtype}")
        if data.shape[:3] != key_cache.shape[:3] or scales.shape[:3] != key_cache.shape[:3]:
            raise ValueError("4-bit caches and their scales must share pages, page size and heads")
        d = 2 * data.shape[3]
        if d % _BLOCK or scales.shape[3] * _BLOCK != d:
            raise ValueError(f"a 4-bit row has a scale for each {_BLOCK} elements, got {d} elements and {scales.shape[3]} scales")
        for t in (data, scales):
            if t.stride(3) != 1 and t.shape[3] > 1:
                raise ValueError("cache rows must have a unit stride")
        dims.append(d)
    _check_slots(key_cache, by_page)
    return dims[0], dims[1]


def _touch(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory between the first and the last element of one overlaps the other's."""
    if a.numel() == 0 or b.numel() == 0 or a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False

    def ends(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))

    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a0 < b1 and b0 < a1


def _check_written(caches, rows) -> None:
    for i, cache in enumerate(caches):
        if _overlaps(cache):
            raise ValueError("caches must not overlap themselves (an expanded view?)")
        if any(_share(cache, other) for other in caches[i + 1:]):
            raise ValueError("the caches and their scales must not share memory")
        if any(_touch(cache, row) for row in rows):
            raise ValueError("new rows must not lie in the memory of the caches")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., heads, dim] as [rows, heads, dim] with a unit stride in dim."""
    return _unit_last(t if t.dim() == 3 else t.reshape(-1, *t.shape[-2:]))


def _write(what, query, key, value, caches, scales, slots, positions, plan):
    """biops_rotary_write on checked tensors; the rotated query."""
    device = key.device
    watch = _watch(device)
    q, k, v = (None if t is None else _rows(t) for t in (query, key, value))
    rows = k.shape[0]
    slots = slots.reshape(-1)
    out = None
    if q is not None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        positions = positions if positions.dim() == 2 else positions.reshape(positions.shape[0], rows)

    def at(t, first):
        return (None, *([0] * (t.dim() - 1 - first))) if t is None else (t.data_ptr(), *t.stride()[first:-1])

    need = _fn("biops_rotary_write_workspace_size")(rows)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    kc, vc = caches
    ks, vs = scales if scales is not None else (None, None)
    none4 = (None, 0, 0, 0)
    _call("biops_rotary_write", nat.dtype_code(key.dtype), rows, 0 if q is None else q.shape[1], k.shape[1], k.shape[2], v.shape[2],
          *((None, 0, 0, None, 0, 0) if q is None else (*at(q, 0), *at(out, 0))), *at(k, 0), *at(v, 0),
          *at(kc, 0), *(none4 if ks is None else at(ks, 0)), *at(vc, 0), *(none4 if vs is None else at(vs, 0)),
          kc.shape[0], kc.shape[1], slots.data_ptr(), int(slots.dtype == torch.int64), slots.stride(0),
          *((None, 0, 0, 0, 0, None, None, 0) if q is None else
            (positions.data_ptr(), _POSITION_CODE[positions.dtype], positions.stride(0), positions.stride(1), plan.pairs,
             plan.turns_at, plan.axis_at, plan.neighbours)),
          watch.flag.data_ptr(), None if ws is None else ws.data_ptr(), need, nat.stream_of(k))
    # autograd has to know of the change, as of any other in place
    torch.autograd.graph.increment_version([c for c in (*caches, *(scales or ())) if not c.is_inference()])
    watch.after_call(nat.stream_of(k))
    return None if out is None else out.view(query.shape)


def _check_rows(key, value, slots) -> None:
    if key.dim() < 2 or value.dim() != key.dim() or key.shape[:-1] != value.shape[:-1]:
        raise ValueError("key and value must have shapes [..., kv_heads, dim] with the same leading dimensions")
    if value.dtype != key.dtype:
        raise ValueError("keys and values must have the same dtype")
    if slots.dtype not in _INDEX_TYPES or slots.shape != key.shape[:-2]:
        raise ValueError(f"slots must be int32 or int64 of shape {tuple(key.shape[:-2])}")


def _check_fp4_rows(key, value, key_cache, key_scales, value_cache, value_scales) -> None:
    d, dv = _check_fp4(key_cache, key_scales, value_cache, value_scales)
    if key.dtype not in _HALVES:
        raise ValueError(f"rows of a 4-bit cache are bfloat16 or float16, got {key.dtype}")
    if key.shape[-2:] != (key_cache.shape[2], d) or value.shape[-2:] != (key_cache.shape[2], dv):
        raise ValueError("keys and values must have the heads and head dimensions of their caches")


def rotary_cache_write(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slots: torch.Tensor,
    positions: torch.Tensor,
    sections: Sequence[int],
    *,
    key_scales: torch.Tensor | None = None,
    value_scales: torch.Tensor | None = None,
    base: float = 10000.0,
    inv_freq: Sequence[float] | None = None,
    interleaved_axes: bool = False,
    interleaved_pairs: bool = False,
) -> torch.Tensor:
    """``multi_axis_rotary`` of queries and keys and ``paged_cache_write`` of the rotated keys and the values, in one launch and
    with their bits.  Returns the rotated queries, a new tensor.

    ``query`` is ``[..., heads, head_dim]``, ``key`` ``[..., kv_heads, head_dim]``, ``value`` ``[..., kv_heads, value_dim]``,
    ``slots`` has their leading shape and ``positions`` is ``[axes, ...]``; the caches, slots, positions and ``sections`` and
    the options behind them are as in those two functions.  A row whose slot is negative is rotated and not written.

    With ``key_scales`` and ``value_scales`` the caches are in 4 bits (see the module): rows are bfloat16 or float16, and a
    rotated key is rounded to its type first.  The new rows must not lie in the memory of the caches, and the caches and their
    scales share none with one another.  A row has at most 2**22 elements.
    """
    plan = _rotary_plan(tuple(sections), float(base), None if inv_freq is None else tuple(map(float, inv_freq)),
                        bool(interleaved_axes), bool(interleaved_pairs))
    module, watch = _direct_watch()
    if module and query is not None:
        out = module.rotary_write(query, key, value, key_cache, value_cache, slots, positions, key_scales, value_scales, len(sections),
                                  plan.pairs, plan.turns_at, plan.axis_at, plan.neighbours, watch.flag_at)
        if out is not None:
            watch.after_call()
            return out
    if (key_scales is None) != (value_scales is None):
        raise ValueError("key_scales and value_scales are given together, or neither")
    scales = () if key_scales is None else (key_scales, value_scales)
    _refuse_transforms("rotary_cache_write", query, key, value, key_cache, value_cache, *scales, positions)
    _check_rows(key, value, slots)
    if query.dim() != key.dim() or query.shape[:-2] != key.shape[:-2] or query.shape[-1] != key.shape[-1]:
        raise ValueError("query and key must share leading dimensions and head dimension")
    if query.dtype != key.dtype or query.dtype not in nat.DIRECT_DTYPES:
        raise ValueError(f"unsupported rotary dtypes: {query.dtype} and {key.dtype}")
    if scales:
        _check_fp4_rows(key, value, key_cache, key_scales, value_cache, value_scales)
    else:
        _check_caches(key_cache, value_cache)
        if key.dtype != key_cache.dtype:
            raise ValueError("keys, values and caches must have the same dtype")
        if key.shape[-2:] != key_cache.shape[2:] or value.shape[-2:] != value_cache.shape[2:]:
            raise ValueError("keys and values must have the heads and head dimensions of their caches")
    if 2 * plan.pairs > query.shape[-1]:
        raise ValueError(f"{plan.pairs} pairs do not fit a head of {query.shape[-1]}")
    if positions.dtype not in _POSITION_CODE:
        raise ValueError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.shape != (len(sections), *query.shape[:-2]):
        raise ValueError(f"positions must have shape {(len(sections), *query.shape[:-2])}, got {tuple(positions.shape)}")
    device = _check_tensors("rotary_cache_write", query, key, value, key_cache, value_cache, *scales, slots, positions)
    _check_written((key_cache, value_cache, *scales), (query, key, value, slots, positions))
    with torch.cuda.device(device):
        return _write("rotary_cache_write", query, key, value, (key_cache, value_cache), scales or None, slots, positions, plan)


def paged_cache_write_fp4(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_cache: torch.Tensor,
    value_scales: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """``paged_cache_write`` into a cache in 4 bits (see the module): rows of bfloat16 or float16 keys ``[..., kv_heads,
    head_dim]`` and values ``[..., kv_heads, value_dim]``, each block to its power of two and its elements to the nearest level
    (ties to the even code), in place.  Slots are as there; the rows must not lie in the memory of the caches."""
    module, watch = _direct_watch()
    if module and key_scales is not None and module.rotary_write(
            None, key, value, key_cache, value_cache, slots, None, key_scales, value_scales, 0, 0, 0, 0, 0, watch.flag_at):
        watch.after_call()
        return
    _refuse_transforms("paged_cache_write_fp4", key, value, key_cache, key_scales, value_cache, value_scales)
    _check_rows(key, value, slots)
    _check_fp4_rows(key, value, key_cache, key_scales, value_cache, value_scales)
    device = _check_tensors("paged_cache_write_fp4", key, value, key_cache, key_scales, value_cache, value_scales, slots)
    _check_written((key_cache, value_cache, key_scales, value_scales), (key, value, slots))
    with torch.cuda.device(device):
        _write("paged_cache_write_fp4", None, key, value, (key_cache, value_cache), (key_scales, value_scales), slots, None, None)


def paged_cache_read_fp4(
    key_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_cache: torch.Tensor,
    value_scales: torch.Tensor,
    slots: torch.Tensor,
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys ``[..., kv_heads, head_dim]`` and values ``[..., kv_heads, value_dim]`` of the slots ``[...]`` (int32 or int64) of a
    cache in 4 bits (see the module), as attention sees them: for the prefix of a longer prompt, for example.  Exact in the
    type of the rows that were written.  A negative slot gives zeros; one past the cache too, and is reported as an error
    later.  At most 2**36 elements."""
    module, watch = _direct_watch()
    if module and dtype in _HALVES:
        out = module.paged_read4(key_cache, key_scales, value_cache, value_scales, slots, nat.DIRECT_DTYPES[dtype], watch.flag_at)
        if out is not None:
            watch.after_call()
            return out
    _refuse_transforms("paged_cache_read_fp4", key_cache, key_scales, value_cache, value_scales)
    d, dv = _check_fp4(key_cache, key_scales, value_cache, value_scales)
    if dtype not in _HALVES:
        raise ValueError(f"rows of a 4-bit cache are bfloat16 or float16, got {dtype}")
    if slots.dtype not in _INDEX_TYPES:
        raise ValueError(f"slots must be int32 or int64, got {slots.dtype}")
    device = _check_tensors("paged_cache_read_fp4", key_cache, key_scales, value_cache, value_scales, slots)
    with torch.cuda.device(device):
        watch = _watch(device)
        heads = key_cache.shape[2]
        key, value = (torch.empty((*slots.shape, heads, n), dtype=dtype, device=device) for n in (d, dv))
        flat = slots.reshape(-1)
        stream = nat.stream_of(key)
        _call("biops_paged_read_fp4", nat.dtype_code(dtype), flat.shape[0], heads, d, dv,
              *(x for t in (key_cache, key_scales, value_cache, value_scales) for x in (t.data_ptr(), *t.stride()[:3])),
              key_cache.shape[0], key_cache.shape[1], flat.data_ptr(), int(flat.dtype == torch.int64), flat.stride(0),
              key.data_ptr(), value.data_ptr(), watch.flag.data_ptr(), stream)
        watch.after_call(stream)
    return key, value


def paged_attention_fp4_batch_invariant(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_cache: torch.Tensor,
    value_scales: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
    max_length: int | None = None,
) -> torch.Tensor:
    """``paged_attention_batch_invariant`` over a cache in 4 bits (see the module): ``query`` ``[batch, heads, head_dim]`` is
    bfloat16 or float16, head dimensions are multiples of 32 up to 256, and everything else is as there.

    The cache's values become numbers of the query's type exactly (for rows that were written in that type); scores, softmax
    and sums are in 32 bits, with one rounding to the output's type, and products take the weights as two 16-bit parts.
    Returns ``[batch, heads, value_dim]``, at most 2**24 rows.
    """
    module, watch = _direct_watch()
    if module and window != 0 and (max_length is None or max_length >= 0):
        out = module.paged_attention4(query, key_cache, key_scales, value_cache, value_scales, block_table, lengths, scale,
                                      0 if window is None else window, sinks, -1 if max_length is None else max_length, watch.flag_at)
        if out is not None:
            watch.after_call()
            return out
    _refuse_transforms("paged_attention_fp4_batch_invariant", query, key_cache, key_scales, value_cache, value_scales)
    d, dv = _check_fp4(key_cache, key_scales, value_cache, value_scales, by_page=True)
    if query.dim() != 3:
        raise ValueError(f"query must have shape [batch, heads, head_dim], got {tuple(query.shape)}")
    if query.dtype not in _HALVES:
        raise ValueError(f"queries of a 4-bit cache are bfloat16 or float16, got {query.dtype}")
    batch, heads = query.shape[:2]
    pages, page_size, kv_heads = key_cache.shape[:3]
    if query.shape[2] != d:
        raise ValueError("query and key head dimensions must match")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be divisible by key/value heads")
    for n in (d, dv):
        if n < _BLOCK or n > 256:
            raise ValueError(f"paged attention over 4 bits takes head dimensions that are multiples of {_BLOCK} up to 256, got {n}")
    if pages == 0 or page_size == 0:
        raise ValueError("the cache has no pages")
    if block_table.dim() != 2 or block_table.shape[0] != batch or block_table.dtype not in _INDEX_TYPES:
        raise ValueError(f"block_table must be int32 or int64 of shape [{batch}, pages per sequence]")
    if lengths.shape != (batch,) or lengths.dtype not in _INDEX_TYPES:
        raise ValueError(f"lengths must be int32 or int64 of shape [{batch}]")
    window_size = _check_window(window, sinks)
    if max_length is not None and max_length < 0:
        raise ValueError(f"max_length must not be negative, got {max_length}")
    _check_scale(scale)
    caches = (key_cache, key_scales, value_cache, value_scales)
    device = _check_tensors("paged_attention_fp4_batch_invariant", query, *caches, block_table, lengths)
    with torch.cuda.device(device):
        query = _unit_last(query)
        watch = _watch(device)
        out = torch.empty((batch, heads, dv), dtype=query.dtype, device=device)
        if batch and heads:
            width = block_table.shape[1]
            bound = -1 if max_length is None else min(int(max_length), 0x7FFFFFFF)
            sinks = min(int(sinks), 0x7FFFFFFF)
            need = _fn("biops_paged_attention_workspace_size")(batch, heads, dv, width, page_size, bound, window_size, sinks)
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
            stream = nat.stream_of(out)
            _call("biops_paged_attention_fp4", nat.dtype_code(query.dtype), batch, heads, kv_heads, d, dv,
                  query.data_ptr(), *query.stride()[:2], *(x for t in caches for x in (t.data_ptr(), *t.stride()[:3])),
                  pages, page_size, block_table.data_ptr(), int(block_table.dtype == torch.int64), *block_table.stride(), width,
                  lengths.data_ptr(), int(lengths.dtype == torch.int64), lengths.stride(0), bound, window_size, sinks,
                  float(1.0 / math.sqrt(d) if scale is None else scale), out.data_ptr(), watch.flag.data_ptr(),
                  None if ws is None else ws.data_ptr(), need, stream)
            watch.after_call(stream)
    return out


# -------------------------------------------------------------------------------- sampling ----
_MOST_TOKENS, _MOST_ROWS, _MOST_LOGITS = 1 << 20, 65536, 1 << 35


def _setting(name, value, lead, dtypes, default, check):
    """(tensor of a value for each row or None, the value of all rows)."""
    if isinstance(value, torch.Tensor):
        if value.dtype not in dtypes or value.shape != lead:
            raise ValueError(f"{name} must be a number, or {' or '.join(map(str, dtypes))} of shape {tuple(lead)}")
        return value, default
    if value is None:
        return None, default
    if isinstance(value, bool) or not isinstance(value, (int, float)) or not check(value):
        raise ValueError(f"{name} out of range: {value!r}")
    return None, value


def sample_tokens_batch_invariant(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor | None = None,
    top_p: float | torch.Tensor | None = None,
    min_p: float | torch.Tensor | None = None,
) -> torch.Tensor:
    """The next token (int64, ``[...]``) of each row of ``logits`` ``[..., vocab]`` (bfloat16, float16 or float32), from one random
    number of ``uniforms`` (float32, ``[...]``) in [0, 1).

    Weights are ``w_i = exp((l_i - max l) / temperature)``.  Tokens are ranked by their logits, equal ones by their index, and of
    this order stay those that every filter allows: the first ``top_k``; those before which less than ``top_p`` of the weight of
    the first ``top_k`` has gone (the most likely one always stays); those with ``w_i >= min_p``.  The token is the first index
    at which the running sum of the weights that stay, in the order of the vocabulary, exceeds ``uniforms`` times all of them.  A
    temperature of 0 is the most likely token (the first of equal ones).

    Each setting is a number for all rows, or a tensor with one for each (float32; ``top_k`` int32 or int64).  In a tensor a
    temperature that is not positive means 0, a ``top_k`` below 1 and a ``top_p`` of 1 or more mean no filter, a ``top_p`` of 0 or
    less the most likely token, and a ``min_p`` above 1 means 1.  NaN is a temperature of 0, and no filter elsewhere.  Random
    numbers outside of [0, 1) count as the nearest inside (NaN as 0).

    Logits of NaN count as -inf, which are never chosen; a row without any other gives -1.  Where logits are +inf only those
    can be chosen.  Weights are formed with a relative error below 2**-33 and rounded to multiples of 2**-43 (what is less than half
    of that is never chosen, and not counted); their sums are exact, so a token does not depend on the batch.  Up to 2**20 tokens,
    65536 rows and 2**35 logits in all; the workspace of a call is at most half a gigabyte.
    """
    module = decoder._tensor_module or _direct()
    if module:
        out = module.sample(logits, uniforms, temperature, top_k, top_p, min_p)
        if out is not None:
            return out
    settings = [x for x in (temperature, top_k, top_p, min_p) if isinstance(x, torch.Tensor)]
    _refuse_transforms("sample_tokens_batch_invariant", logits, uniforms, *settings)
    if logits.dim() < 1 or logits.dtype not in nat.DIRECT_DTYPES:
        raise ValueError(f"logits must be float32, float16 or bfloat16 of shape [..., vocab], got {logits.dtype} {tuple(logits.shape)}")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if vocab < 1 or vocab > _MOST_TOKENS:
        raise ValueError(f"rows must have 1 to {_MOST_TOKENS} logits, got {vocab}")
    if lead.numel() > _MOST_ROWS:
        raise ValueError(f"at most {_MOST_ROWS} rows, got {lead.numel()}")
    if lead.numel() * vocab > _MOST_LOGITS:
        raise ValueError(f"at most 2**35 logits, got {lead.numel()} rows of {vocab}")
    if uniforms.dtype != torch.float32 or uniforms.shape != lead:
        raise ValueError(f"uniforms must be float32 of shape {tuple(lead)}")
    floats = (torch.float32,)
    each = [_setting("temperature", temperature, lead, floats, 1.0, lambda x: 0.0 <= x < math.inf),
            _setting("top_k", top_k, lead, _INDEX_TYPES, 0, lambda x: isinstance(x, int) and x >= 1),
            _setting("top_p", top_p, lead, floats, 1.0, lambda x: 0.0 < x <= 1.0),
            _setting("min_p", min_p, lead, floats, 0.0, lambda x: 0.0 <= x <= 1.0)]
    device = _check_tensors("sample_tokens_batch_invariant", logits, uniforms, *settings)
    with torch.cuda.device(device):
        x = _unit_last(logits if logits.dim() == 2 else logits.reshape(-1, vocab))
        rows = x.shape[0]
        out = torch.empty(lead, dtype=torch.int64, device=device)
        if rows:
            u = uniforms.reshape(-1)
            (t, t0), (k, k0), (p, p0), (m, m0) = ((None if a is None else a.reshape(-1), b) for a, b in each)

            def at(a):
                return (None, 0) if a is None else (a.data_ptr(), a.stride(0))

            need = _fn("biops_sample_workspace_size")(rows, vocab)
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            _call("biops_sample", nat.dtype_code(x.dtype), rows, vocab, x.data_ptr(), x.stride(0), *at(u), *at(t), float(t0),
                  at(k)[0], int(k is not None and k.dtype == torch.int64), at(k)[1], min(int(k0), _MOST_TOKENS + 1), *at(p),
                  float(p0), *at(m), float(m0), out.data_ptr(), ws.data_ptr(), need, nat.stream_of(out))
    return out


# ---------------------------------------------------------------------------- 8-bit linear ----
_MOST_TERMS = 131071  # products of -128 and -128 whose sum a 32-bit integer holds


def quantize_tokens_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``[..., features]`` (bfloat16, float16 or float32) as 8-bit integers of the same shape with a step for each row
    (float32, ``[...]``): with ``m`` the row's largest magnitude, ``step = m / 127`` and ``q = round(x * (127 / m))``, in 32-bit
    arithmetic, ties to even.  (``m`` counts as at least 2**-100.)  A row with an infinity or NaN has a step of NaN and
    zeros.  At most 131071 features and 2**23 rows."""
    module = decoder._tensor_module or _direct()
    if module:
        out = module.quantize8(x)
        if out is not None:
            return out
    _refuse_transforms("quantize_tokens_int8", x)
    if x.dim() < 1 or x.dtype not in nat.DIRECT_DTYPES:
        raise ValueError(f"rows must be float32, float16 or bfloat16 of shape [..., features], got {x.dtype} {tuple(x.shape)}")
    k = x.shape[-1]
    if k < 1 or k > _MOST_TERMS:
        raise ValueError(f"rows must have 1 to {_MOST_TERMS} features, got {k}")
    device = _check_tensors("quantize_tokens_int8", x)
    with torch.cuda.device(device):
        rows = _unit_last(x if x.dim() == 2 else x.reshape(-1, k))
        q = torch.empty(x.shape, dtype=torch.int8, device=device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
        if rows.shape[0]:
            _call("biops_quantize_int8", nat.dtype_code(x.dtype), rows.shape[0], k, rows.data_ptr(), rows.stride(0), q.data_ptr(),
                  scale.data_ptr(), nat.stream_of(q))
    return q, scale


def linear_int8_batch_invariant(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``y = (x @ weight.T) * x_scale * weight_scale + bias`` of 8-bit integers ``x`` ``[..., in_features]`` and ``weight``
    ``[out_features, in_features]`` with float32 scales for each row ``[...]`` and each output channel ``[out_features]``; ``bias``
    ``[out_features]`` is of ``dtype`` (bfloat16, float16 or float32), the output's type.

    The integer sums are exact (32 bits; at most 131071 terms), what follows is in 32-bit floats with one rounding, so the
    bits depend neither on the other rows nor on how the work is split.  At most 2**23 rows, 2**22 output channels and 2**35 outputs
    (in blocks of 64 x 64)."""
    module = decoder._tensor_module or _direct()
    if module:
        out = module.linear8(x, x_scale, weight, weight_scale, bias, nat.DIRECT_DTYPES.get(dtype, -1))
        if out is not None:
            return out
    tensors = (x, x_scale, weight, weight_scale) if bias is None else (x, x_scale, weight, weight_scale, bias)
    _refuse_transforms("linear_int8_batch_invariant", *tensors)
    if x.dim() < 1 or weight.dim() != 2 or x.dtype != torch.int8 or weight.dtype != torch.int8:
        raise ValueError("x and weight must be int8 of shapes [..., in_features] and [out_features, in_features]")
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} features, weight {k}")
    if k < 1 or k > _MOST_TERMS:
        raise ValueError(f"rows must have 1 to {_MOST_TERMS} features, got {k}")
    if x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1]:
        raise ValueError(f"x_scale must be float32 of shape {tuple(x.shape[:-1])}")
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (n,):
        raise ValueError(f"weight_scale must be float32 of shape ({n},)")
    if dtype not in nat.DIRECT_DTYPES:
        raise ValueError(f"unsupported output dtype: {dtype}")
    if bias is not None and (bias.shape != (n,) or bias.dtype != dtype):
        raise ValueError(f"bias must be {dtype} of shape ({n},)")
    device = _check_tensors("linear_int8_batch_invariant", *tensors)
    with torch.cuda.device(device):
        rows = _unit_last(x if x.dim() == 2 else x.reshape(-1, k))
        steps = x_scale.reshape(-1)
        w = _unit_last(weight)
        b = None if bias is None else bias.contiguous()
        out = torch.empty((*x.shape[:-1], n), dtype=dtype, device=device)
        if rows.shape[0] and n:
            _call("biops_linear_int8", nat.dtype_code(dtype), rows.shape[0], n, k, rows.data_ptr(), rows.stride(0), steps.data_ptr(),
                  steps.stride(0), w.data_ptr(), w.stride(0), weight_scale.data_ptr(), weight_scale.stride(0),
                  None if b is None else b.data_ptr(), out.data_ptr(), nat.stream_of(out))
    return out
