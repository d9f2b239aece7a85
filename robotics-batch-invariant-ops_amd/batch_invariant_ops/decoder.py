"""Operators of a served decoder: rotary positions with several axes, a cache of keys and values in
pages, attention of one new token over that cache, and attention with a sliding window and a few first
tokens that stay visible (sinks).

They stand beside the package's attention functions and keep their contract: a sequence's bits do not
depend on the batch it is computed in.  The reference has no counterpart of them.

Lengths, slots, page tables and packed offsets are read on the device: no call waits for the GPU, and
all of them may be captured into a graph (after one call outside of a capture on that device, which sets up
the error flag).  An index that points outside its tensor never makes a kernel read or write out of
range: the row it belongs to is zeros (a written row is left out), and the error is reported later, as
``deterministic_token_choice_moe`` reports expert indices: a later call, or ``check_cache_indices()``,
which waits, raises ``RuntimeError``.

Only ``multi_axis_rotary`` has a gradient.  The other functions refuse tensors that require one while
grad mode is on.  None has a forward-mode derivative or can be recorded by ``torch.jit.trace``: both are
refused.
"""

from __future__ import annotations

import functools
import math
import threading
import time
from collections.abc import Sequence

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _native as nat
from .moe import _IndexWatch

__all__ = [
    "multi_axis_rotary",
    "paged_cache_write",
    "paged_attention_batch_invariant",
    "sliding_window_attention_batch_invariant",
    "varlen_sliding_window_attention_batch_invariant",
    "check_cache_indices",
]

_INDEX_TYPES = (torch.int32, torch.int64)
_MOST_PAIRS = 128


class _CacheWatch(_IndexWatch):
    """Deferred report of slots, pages, lengths and packed offsets outside their tensors."""

    MESSAGE = "a cache slot, page, length or packed offset outside its tensor"
    _by_device: dict = {}
    _lock = threading.Lock()

    def __init__(self, device: torch.device):
        super().__init__(device)
        self.flag_at = self.flag.data_ptr()

    def poll(self) -> None:
        """As the base class, but a copy in flight is asked after once per PERIOD (an event query costs as
        much as the rest of a small call's host time)."""
        if self.pending and time.monotonic() - self.last >= self.PERIOD:
            super().poll()

    def after_call(self, stream: int | None = None) -> None:
        if not self.pending and time.monotonic() - self.last >= self.PERIOD:
            super().after_call(nat.stream_of(self.flag) if stream is None else stream)


def check_cache_indices(device: torch.device | str | int | None = None) -> None:
    """Raise ``RuntimeError`` if a call of this module on ``device`` (default: the current device) met an
    index outside its tensor since the last report.  Waits for the work queued on that device's current
    stream."""
    device = _CacheWatch.device(device)
    with torch.cuda.device(device):
        _CacheWatch.of(device).check()


_tensor_module = None  # csrc/tensorfast.cpp: False without it or without a GPU
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _direct():
    """The module that takes tensors as they are, or False."""
    global _tensor_module
    if _tensor_module is None:
        if _current_device is None or not torch.cuda.is_available():
            return False
        nat.load()
        torch.cuda.current_device()  # torch's own initialisation
        try:
            from . import _biops_tensor
        except ImportError:
            _biops_tensor = False
        _tensor_module = _biops_tensor
    return _tensor_module


def _direct_watch():
    """(module, watch of the current device): a pair of None until a call has set both up."""
    module = _tensor_module or _direct()
    if module:
        watch = _CacheWatch._by_device.get(_current_device())
        if watch is not None:
            watch.poll()
            return module, watch
    return None, None


def _watch(device: torch.device) -> _CacheWatch:
    watch = _CacheWatch._by_device.get(device.index)
    if watch is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call one of the cache operators on this device before capturing a graph")
        watch = _CacheWatch.of(device)
    watch.poll()
    return watch


def _refuse_transforms(what: str, *tensors) -> None:
    """A launch is no operator that a trace records, and a tangent would be lost."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be recorded by torch.jit.trace")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no forward-mode derivative")


def _check_tensors(what: str, *tensors) -> torch.device:
    """All on one ROCm GPU, none in need of a gradient; that device."""
    nat.require_gpu_tensors(*tensors)
    device = tensors[0].device
    for t in tensors:
        if t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")
        if t.is_neg():
            raise ValueError(f"{what}: a lazily negated tensor (call resolve_neg)")
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")
    return device


_fns = {}


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = nat.fast_function(name)
    return fn


def _call(name: str, *args) -> None:
    """The library entry point ``name``.  Kernels are launched on the current device, which the public
    functions make the tensors' own."""
    rc = _fn(name)(*args)
    if rc:
        nat.check(rc, name)


def _unit_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# ------------------------------------------------------------------------------- rotary ----
class _RotaryPlan:
    """Axis and frequency (in turns per position) of every pair, as host arrays."""

    __slots__ = ("turns", "axis", "pairs", "neighbours", "turns_at", "axis_at")

    def __init__(self, sections, frequencies, interleaved_axes, neighbours):
        order, left = [], list(sections)
        if interleaved_axes:
            while any(left):
                for a, n in enumerate(left):
                    if n:
                        order.append(a)
                        left[a] -= 1
        else:
            order = [a for a, n in enumerate(sections) for _ in range(n)]
        self.turns = np.array([f / (2.0 * math.pi) for f in frequencies], dtype=np.float64)
        self.axis = np.array(order, dtype=np.uint8)
        self.pairs, self.neighbours = len(order), int(neighbours)
        self.turns_at, self.axis_at = self.turns.ctypes.data, self.axis.ctypes.data


@functools.lru_cache(maxsize=64)
def _rotary_plan(sections, base, inv_freq, interleaved_axes, neighbours) -> _RotaryPlan:
    pairs = sum(sections)
    if not sections or min(sections) < 0 or len(sections) > 255:
        raise ValueError(f"sections must be counts of pairs, one per axis, got {sections}")
    if pairs > _MOST_PAIRS:
        raise ValueError(f"at most {_MOST_PAIRS} rotated pairs, got {pairs}")
    if inv_freq is None:
        if not base > 0.0 or math.isinf(base):
            raise ValueError(f"base must be positive, got {base}")
        inv_freq = [base ** (-i / pairs) for i in range(pairs)]
    elif len(inv_freq) != pairs:
        raise ValueError(f"inv_freq must have one value per pair ({pairs}), got {len(inv_freq)}")
    return _RotaryPlan(sections, inv_freq, interleaved_axes, neighbours)


_POSITION_CODE = {torch.int64: 0, torch.int32: 1, torch.float32: 2}


def _rotate(query, key, positions, plan: _RotaryPlan, inverse: bool):
    """Rotated copies of ``query`` and ``key`` (either may be None), leading dimensions [tokens] or
    [batch, tokens]."""
    outs, args = [], []
    held = []  # copies, until the launch
    some = query if query is not None else key
    for x in (query, key):
        if x is None:
            outs.append(None)
            args += (0, (None, 0, 0, 0, None, 0, 0, 0))
            continue
        x = _unit_last(x.resolve_neg())  # (a gradient comes as the engine has it)
        held.append(x)
        y = torch.empty_like(x)
        if y.stride(-1) != 1 and y.shape[-1] > 1:
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        outs.append(y)
        three = x.dim() == 3
        xs, ys = x.stride(), y.stride()
        args += (x.shape[-2], (x.data_ptr(), 0 if three else xs[0], xs[-3], xs[-2],
                               y.data_ptr(), 0 if three else ys[0], ys[-3], ys[-2]))
    three = some.dim() == 3
    ps = positions.stride()
    _call("biops_rotary", nat.dtype_code(some.dtype), 1 if three else some.shape[0], some.shape[-3],
          args[0], args[2], some.shape[-1], *args[1], *args[3], positions.data_ptr(),
          _POSITION_CODE[positions.dtype], ps[0], 0 if three else ps[1], ps[-1], plan.pairs, plan.turns_at,
          plan.axis_at, plan.neighbours, int(inverse), nat.stream_of(some))
    return outs


class _Rotary(torch.autograd.Function):
    """The rotation with its gradient, which is the inverse rotation (and so on)."""

    @staticmethod
    def forward(ctx, query, key, positions, plan, inverse):
        ctx.save_for_backward(positions)
        ctx.plan, ctx.inverse = plan, inverse
        ctx.set_materialize_grads(False)
        outs = _rotate(query, key, positions, plan, inverse)
        # what comes of a tensor without a gradient has none
        ctx.mark_non_differentiable(*(y for y, needs in zip(outs, ctx.needs_input_grad) if y is not None and not needs))
        return tuple(outs)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        (positions,) = ctx.saved_tensors
        grad_q = grad_q if ctx.needs_input_grad[0] else None
        grad_k = grad_k if ctx.needs_input_grad[1] else None
        if grad_q is not None or grad_k is not None:
            turn = _Rotary.apply if torch.is_grad_enabled() else _rotate  # (with create_graph, or without)
            grad_q, grad_k = turn(grad_q, grad_k, positions, ctx.plan, not ctx.inverse)
        return grad_q, grad_k, None, None, None


def multi_axis_rotary(
    query: torch.Tensor,
    key: torch.Tensor | None,
    positions: torch.Tensor,
    sections: Sequence[int],
    *,
    base: float = 10000.0,
    inv_freq: Sequence[float] | None = None,
    interleaved_axes: bool = False,
    interleaved_pairs: bool = False,
):
    """Rotary positions with one or several axes (time, height, width, ...), queries and keys in one launch.

    ``query`` is ``[..., heads, head_dim]``, ``key`` the same with its own number of heads (or None),
    ``positions`` ``[axes, ...]`` (int32, int64 or float32) with the leading dimensions of ``query``.  For
    ``[batch, heads, tokens, head_dim]`` tensors pass ``x.transpose(1, 2)``: strides are read as they are.

    ``sections[a]`` is the number of pairs that turn by axis ``a``; the first ``2 * sum(sections)`` elements of
    a head are rotated, the others copied.  Pairs belong to the axes block by block, or, with
    ``interleaved_axes``, to the axes in turn (an axis drops out when its pairs are used up).  Pair ``i``
    turns by ``position * inv_freq[i]``, with ``inv_freq[i] = base ** (-i / sum(sections))`` unless it is
    given as host numbers.  Pair ``i`` is elements ``(i, i + sum(sections))``, or ``(2 i, 2 i + 1)`` with
    ``interleaved_pairs``.

    Angles are computed in 64 bits, the rotation in 32, with one rounding to the tensors' type.  Returns new
    tensors ``(query, key)``, or the rotated query alone when ``key`` is None.  Differentiable with respect
    to ``query`` and ``key`` (not to ``positions``).  A capture into a graph is refused while a leaf among them has a
    living autograd graph from another stream, whose backward pass the capture would run into (without the tensor module, which
    can tell, of every leaf that requires a gradient).
    """
    plan = _rotary_plan(tuple(sections), float(base), None if inv_freq is None else tuple(map(float, inv_freq)),
                        bool(interleaved_axes), bool(interleaved_pairs))
    module = _tensor_module or _direct()
    if module:
        out = module.rotary(query, key, positions, len(sections), plan.pairs, plan.turns_at, plan.axis_at, plan.neighbours)
        if out is not None:
            return out
    tensors = (query,) if key is None else (query, key)
    _refuse_transforms("multi_axis_rotary", *tensors, positions)
    for x in tensors:
        if x.dim() < 2:
            raise ValueError(f"rotary tensors have shape [..., heads, head_dim], got {tuple(x.shape)}")
        if x.dtype not in nat.DIRECT_DTYPES:
            raise ValueError(f"unsupported rotary dtype: {x.dtype}")
    if key is not None and (key.dtype != query.dtype or key.shape[:-2] != query.shape[:-2]
                            or key.shape[-1] != query.shape[-1]):
        raise ValueError("query and key must share dtype, leading dimensions and head dimension")
    if 2 * plan.pairs > query.shape[-1]:
        raise ValueError(f"{plan.pairs} pairs do not fit a head of {query.shape[-1]}")
    if positions.dtype not in _POSITION_CODE:
        raise ValueError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.shape != (len(sections), *query.shape[:-2]):
        raise ValueError(f"positions must have shape {(len(sections), *query.shape[:-2])}, got {tuple(positions.shape)}")
    nat.require_gpu_tensors(*tensors, positions)
    if any(x.device != query.device for x in (*tensors, positions)):
        raise ValueError("query, key and positions must be on one device")
    if positions.requires_grad and torch.is_grad_enabled():
        raise ValueError("multi_axis_rotary has no gradient for positions: detach them")
    if any(x.is_neg() for x in (*tensors, positions)):
        raise ValueError("multi_axis_rotary: a lazily negated tensor (call resolve_neg)")
    if query.device.index != torch.cuda.current_device():
        with torch.cuda.device(query.device):
            return multi_axis_rotary(query, key, positions, sections, base=base, inv_freq=inv_freq,
                                     interleaved_axes=interleaved_axes, interleaved_pairs=interleaved_pairs)

    if torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        leaves = [x for x in tensors if x.requires_grad and x.is_leaf]
        if leaves and not module:
            raise RuntimeError("multi_axis_rotary: without its tensor module a capture cannot tell whether another graph of a "
                               "leaf is alive: rotate a tensor that is not a leaf, or one without a gradient")
        if leaves and module.held(*leaves) is not False:
            raise RuntimeError("multi_axis_rotary: a graph of this leaf from outside of the capture is still alive; "
                               "delete its outputs (or capture on the stream that they were made on)")

    lead = query.shape[:-2]
    q, k, p = query, key, positions
    if len(lead) not in (1, 2):  # one token, or more leading dimensions than the kernel walks
        q = query.reshape(-1, *query.shape[-2:])
        k = None if key is None else key.reshape(-1, *key.shape[-2:])
        p = positions.reshape(len(sections), -1)
    if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
        out_q, out_k = _Rotary.apply(q, k, p, plan, False)
    else:
        out_q, out_k = _rotate(q, k, p, plan, False)
    if len(lead) not in (1, 2):
        out_q = out_q.reshape(query.shape)
        out_k = None if key is None else out_k.reshape(key.shape)
    return out_q if key is None else (out_q, out_k)


# -------------------------------------------------------------------------- paged cache ----
def _check_caches(key_cache, value_cache) -> None:
    if key_cache.dim() != 4 or value_cache.dim() != 4:
        raise ValueError("caches must have shape [pages, page_size, kv_heads, head_dim]")
    if key_cache.shape[:3] != value_cache.shape[:3]:
        raise ValueError("key and value caches must share pages, page size and heads")
    if key_cache.dtype not in nat.DIRECT_DTYPES or value_cache.dtype != key_cache.dtype:
        raise ValueError(f"unsupported cache dtypes: {key_cache.dtype} and {value_cache.dtype}")
    for cache in (key_cache, value_cache):
        if cache.stride(3) != 1 and cache.shape[3] > 1:
            raise ValueError("cache rows must have a unit stride in head_dim")
    if key_cache.shape[0] * key_cache.shape[1] > 0x7FFFFFFF:
        raise ValueError("caches of more than 2**31 - 1 slots are not supported")


def _overlaps(t: torch.Tensor) -> bool:
    """Whether two elements of ``t`` may share memory (an expanded or windowed view)."""
    if t.is_contiguous():
        return False
    reach = 0
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1:
            if stride <= reach:
                return True
            reach += stride * (size - 1)
    return False


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of the key cache may lie where one of the value cache does (two views of one allocation may be
    interleaved in any dimension, if their slots have the same strides)."""
    if a.numel() == 0 or b.numel() == 0 or a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False
    if a.storage_offset() > b.storage_offset():
        a, b = b, a
    gap = b.storage_offset() - a.storage_offset()
    if gap > sum((n - 1) * s for n, s in zip(a.shape, a.stride())):
        return False
    dims = [(s, n) for s, n in zip(a.stride()[:3], a.shape[:3]) if n > 1]
    if dims != [(s, n) for s, n in zip(b.stride()[:3], b.shape[:3]) if n > 1]:
        return True
    # both at once, as one tensor with a dimension more, whose two entries are `gap` apart
    low, high = a.shape[3] - 1, b.shape[3] - 1  # how far each reaches
    for stride, size in sorted([*dims, (gap, 0)]):
        if size == 0:
            if gap <= low:
                return True
            low = high = max(low, gap + high)
        elif stride <= max(low, high):
            return True
        else:
            low, high = low + stride * (size - 1), high + stride * (size - 1)
    return False


def _part(a: torch.Tensor, b: torch.Tensor) -> int | None:
    """The element of ``a``'s rows at which ``b``'s rows begin, where one's rows are a part of the other's."""
    at = (b.data_ptr() - a.data_ptr()) // a.element_size()
    if a.stride() != b.stride() or a.shape[:-1] != b.shape[:-1]:
        return None
    inside = 0 <= at <= a.shape[-1] - b.shape[-1] or 0 <= -at <= b.shape[-1] - a.shape[-1]
    return at if inside else None


def paged_cache_write(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """Write rows of new keys ``[..., kv_heads, head_dim]`` and values ``[..., kv_heads, value_dim]`` into
    caches ``[pages, page_size, kv_heads, head_dim]`` / ``[..., value_dim]``, in place.

    ``slots`` (int32 or int64, the leading shape of ``key``) names the slot of each row: ``page * page_size +
    place``.  A negative slot leaves its row out (padding).  A slot past the cache is left out too and reported
    as an error later (see the module).  Of several rows that name one slot the last one stays.  ``key`` and
    ``value`` may be rows of the caches themselves (a page that is copied) as long as no slot that is written is
    among them.  The caches may be interleaved views of one allocation.  They must not share
    elements, unless the new rows do in the same way (values that are a part of the keys).
    """
    module, watch = _direct_watch()
    if module and module.paged_write(key, value, key_cache, value_cache, slots, watch.flag_at):
        watch.after_call()
        return
    _refuse_transforms("paged_cache_write", key, value, key_cache, value_cache)
    _check_caches(key_cache, value_cache)
    if key.dim() < 2 or value.dim() != key.dim() or key.shape[:-1] != value.shape[:-1]:
        raise ValueError("key and value must have shapes [..., kv_heads, dim] with the same leading dimensions")
    if key.dtype != key_cache.dtype or value.dtype != key_cache.dtype:
        raise ValueError("keys, values and caches must have the same dtype")
    if key.shape[-2:] != key_cache.shape[2:] or value.shape[-2:] != value_cache.shape[2:]:
        raise ValueError("keys and values must have the heads and head dimensions of their caches")
    if slots.dtype not in _INDEX_TYPES or slots.shape != key.shape[:-2]:
        raise ValueError(f"slots must be int32 or int64 of shape {tuple(key.shape[:-2])}")
    device = _check_tensors("paged_cache_write", key, value, key_cache, value_cache, slots)
    if _overlaps(key_cache) or _overlaps(value_cache):
        raise ValueError("caches must not overlap themselves (an expanded view?)")
    if _share(key_cache, value_cache) and (
            _part(key_cache, value_cache) is None or _part(key_cache, value_cache) != _part(key, value)):
        raise ValueError("the key and the value cache must not share memory")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return paged_cache_write(key, value, key_cache, value_cache, slots)
    if key.dim() != 3:
        key, value = key.reshape(-1, *key.shape[-2:]), value.reshape(-1, *value.shape[-2:])
        slots = slots.reshape(-1)
    key, value = _unit_last(key), _unit_last(value)
    watch = _watch(device)
    stream = nat.stream_of(key_cache)
    rows, heads, d = key.shape
    ks, vs = key.stride(), value.stride()
    kcs, vcs = key_cache.stride(), value_cache.stride()
    _call("biops_paged_write", nat.dtype_code(key.dtype), rows, heads, d, value.shape[2],
          key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1],
          key_cache.data_ptr(), kcs[0], kcs[1], kcs[2], value_cache.data_ptr(), vcs[0], vcs[1], vcs[2],
          key_cache.shape[0], key_cache.shape[1], slots.data_ptr(), int(slots.dtype == torch.int64),
          slots.stride(0), watch.flag.data_ptr(), stream)
    # autograd has to know of the change, as of any other in place
    torch.autograd.graph.increment_version([c for c in (key_cache, value_cache) if not c.is_inference()])
    watch.after_call(stream)


def _check_window(window, sinks) -> int:
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    return 0 if window is None else min(int(window), 0x7FFFFFFF)


def _check_scale(scale) -> None:
    if scale is not None and not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")


def _check_head_dims(what: str, dtype, most: int, *dims) -> None:
    vec = 16 // dtype.itemsize
    for d in dims:
        if d < vec or d > most or d % vec:
            raise ValueError(f"{what} takes head dimensions that are multiples of {vec} up to {most} in {dtype}, got {d}")


def paged_attention_batch_invariant(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
    max_length: int | None = None,
) -> torch.Tensor:
    """Attention of one new token per sequence over its keys and values in pages.

    ``query`` is ``[batch, heads, head_dim]``, the caches ``[pages, page_size, kv_heads, head_dim]`` and
    ``[..., value_dim]`` (``heads`` a multiple of ``kv_heads``; query head ``h`` reads key head ``h // (heads //
    kv_heads)``).  Key ``j`` of sequence ``b`` is in page ``block_table[b, j // page_size]`` at place ``j %
    page_size``; ``lengths[b]`` counts its keys, the new token's own among them.  With ``window`` the token
    sees its last ``window`` keys (itself included) and the first ``sinks`` ones; table entries of pages
    without a visible key are not read.  Slots behind a sequence's end may hold anything.  A length of
    zero gives zeros.

    ``max_length`` bounds the lengths when the table is wider than the batch needs (a smaller workspace and
    grid).  A length outside ``[0, min(max_length, pages of the table)]`` or a page outside the cache makes
    the sequence's rows zeros and is reported as an error later (see the module).

    Scores, softmax and sums are in 32 bits, with one rounding to the output's type; 16-bit products take
    the weights as two 16-bit parts.  Returns ``[batch, heads, value_dim]``.
    """
    module, watch = _direct_watch()
    if module and window != 0 and (max_length is None or max_length >= 0):
        out = module.paged_attention(query, key_cache, value_cache, block_table, lengths, scale,
                                     0 if window is None else window, sinks, -1 if max_length is None else max_length,
                                     watch.flag_at)
        if out is not None:
            watch.after_call()
            return out
    _refuse_transforms("paged_attention_batch_invariant", query, key_cache, value_cache)
    _check_caches(key_cache, value_cache)
    if query.dim() != 3:
        raise ValueError(f"query must have shape [batch, heads, head_dim], got {tuple(query.shape)}")
    if query.dtype != key_cache.dtype:
        raise ValueError("query and caches must have the same dtype")
    batch, heads, d = query.shape
    pages, page_size, kv_heads, dk = key_cache.shape
    dv = value_cache.shape[3]
    if d != dk:
        raise ValueError("query and key head dimensions must match")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be divisible by key/value heads")
    _check_head_dims("paged attention", query.dtype, 256, d, dv)
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
    device = _check_tensors("paged_attention_batch_invariant", query, key_cache, value_cache, block_table, lengths)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return paged_attention_batch_invariant(query, key_cache, value_cache, block_table, lengths, scale=scale,
                                                   window=window, sinks=sinks, max_length=max_length)
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
        qs, kcs, vcs, ts = query.stride(), key_cache.stride(), value_cache.stride(), block_table.stride()
        _call("biops_paged_attention", nat.dtype_code(query.dtype), batch, heads, kv_heads, d, dv,
              query.data_ptr(), qs[0], qs[1], key_cache.data_ptr(), kcs[0], kcs[1], kcs[2],
              value_cache.data_ptr(), vcs[0], vcs[1], vcs[2], pages, page_size,
              block_table.data_ptr(), int(block_table.dtype == torch.int64), ts[0], ts[1], width,
              lengths.data_ptr(), int(lengths.dtype == torch.int64), lengths.stride(0), bound, window_size, sinks,
              float(1.0 / math.sqrt(d) if scale is None else scale), out.data_ptr(), watch.flag.data_ptr(),
              None if ws is None else ws.data_ptr(), need, stream)
        watch.after_call(stream)
    return out


# ---------------------------------------------------------------------- windowed attention ----
_MOST_ROW_STRIDE = 1 << 23  # elements between key rows that the kernel's 32-bit offsets inside a block take


def _fetchable(t: torch.Tensor) -> bool:
    """Whether keys or values ``[batch, tokens, heads, dim]`` go straight to LDS: rows at multiples of 16 bytes."""
    vec = 16 // t.element_size()
    return ((t.stride(1) <= _MOST_ROW_STRIDE or t.shape[1] == 1) and t.data_ptr() % 16 == 0
            and all(t.stride(i) % vec == 0 or t.shape[i] == 1 for i in range(3)))


def _windowed(q, k, v, out, nseq, lengths, window_size, sinks, scale, offsets, watch):
    """biops_window_attention on tensors of [batch, tokens, heads, dim] strides."""
    k, v = (t if _fetchable(t) else t.contiguous() for t in (k, v))
    if not (_fetchable(k) and _fetchable(v)):  # contiguous, and off the 16 bytes: a slice of a flat buffer
        k, v = k.clone(), v.clone()
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
    d = q.shape[-1]
    if offsets is None:
        cu = (None, 0, 0, None, 0, 0)
        need = _fn("biops_window_attention_workspace_size")(nseq, q.shape[2], *lengths, v.shape[-1], window_size or 0x7FFFFFFF,
                                                            min(int(sinks), 0x7FFFFFFF))
    else:
        need = 0
        cu = tuple(x for t in offsets for x in (t.data_ptr(), int(t.dtype == torch.int64), t.stride(0)))
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call("biops_window_attention", nat.dtype_code(q.dtype), nseq, q.shape[2], k.shape[2], *lengths, d,
          v.shape[-1], q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2],
          v.data_ptr(), vs[0], vs[1], vs[2], out.data_ptr(), os_[0], os_[1], os_[2], *cu,
          window_size or 0x7FFFFFFF, min(int(sinks), 0x7FFFFFFF),
          float(1.0 / math.sqrt(d) if scale is None else scale),
          None if watch is None else watch.flag.data_ptr(), None if ws is None else ws.data_ptr(), need,
          nat.stream_of(out))


def sliding_window_attention_batch_invariant(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    window: int | None,
    sinks: int = 0,
    *,
    scale: float | None = None,
    enable_gqa: bool = False,
) -> torch.Tensor:
    """Causal attention ``[batch, heads, tokens, dim]`` in which every token sees its last ``window`` tokens
    (itself included; None: all) and the first ``sinks`` ones.

    The last query is the last key's token: query ``r`` is at position ``p = key_tokens - query_tokens + r``
    (a chunk of new tokens behind a prefix) and sees keys ``j <= p`` with ``p - j < window`` or ``j < sinks``.
    Rows that see nothing (more queries than keys) are zeros.  Work and memory grow with the window, not
    with the square of the length.  ``enable_gqa`` lets groups of query heads share a key/value head.

    A key that is masked for a row changes none of its bits, whatever its key and value hold; an infinity or
    NaN in a value reaches every row that sees it, whatever its weight.  Scores and sums are in 32 bits; 16-bit
    products take weights rounded to the type.  Output rows depend on their own sequence only.
    """
    module = _tensor_module or _direct()
    if module:
        out = module.window_attention(query, key, value, 0x7FFFFFFF if window is None else window, sinks, scale, enable_gqa)
        if out is not None:
            return out
    _refuse_transforms("sliding_window_attention_batch_invariant", query, key, value)
    if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
        raise ValueError("sliding-window attention expects rank-4 query, key, and value")
    if query.dtype != key.dtype or query.dtype != value.dtype:
        raise ValueError("query, key, and value must have the same dtype")
    if query.dtype not in nat.DIRECT_DTYPES:
        raise ValueError(f"unsupported attention dtype: {query.dtype}")
    if query.shape[0] != key.shape[0] or key.shape[:3] != value.shape[:3]:
        raise ValueError("leading query, key, and value dimensions must match")
    if query.shape[3] != key.shape[3]:
        raise ValueError("query and key head dimensions must match")
    heads, kv_heads = query.shape[1], key.shape[1]
    if kv_heads == 0 or heads % kv_heads or (heads != kv_heads and not enable_gqa):
        raise ValueError("query heads must equal key/value heads, or be divisible by them with enable_gqa")
    _check_head_dims("sliding-window attention", query.dtype, 128 if query.dtype == torch.float32 else 256,
                     query.shape[3], value.shape[3])
    window_size = _check_window(window, sinks)
    _check_scale(scale)
    device = _check_tensors("sliding_window_attention_batch_invariant", query, key, value)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return sliding_window_attention_batch_invariant(query, key, value, window, sinks, scale=scale,
                                                            enable_gqa=enable_gqa)
    q, k, v = _unit_last(query), _unit_last(key), _unit_last(value)
    batch, lq, lk, dv = q.shape[0], q.shape[2], k.shape[2], v.shape[3]
    # tokens before heads in memory where the queries have them so, as a projection takes its input
    if q.stride(1) < q.stride(2):
        out = torch.empty((batch, lq, heads, dv), dtype=q.dtype, device=device).transpose(1, 2)
    else:
        out = torch.empty((batch, heads, lq, dv), dtype=q.dtype, device=device)
    _windowed(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), out.transpose(1, 2), batch, (lq, lk),
              window_size, sinks, scale, None, None)
    return out


def varlen_sliding_window_attention_batch_invariant(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cumulative_seqlen_q: torch.Tensor,
    cumulative_seqlen_kv: torch.Tensor,
    window: int | None,
    sinks: int = 0,
    *,
    scale: float | None = None,
) -> torch.Tensor:
    """``sliding_window_attention_batch_invariant`` over sequence-packed inputs ``[1, total_tokens, heads,
    head_dim]``.

    The offsets (int32 or int64, on the GPU) start at zero and do not decrease; sequence ``s`` is rows
    ``offsets[s]`` to ``offsets[s + 1]`` of queries and of keys.  They are read by the kernel, without a wait.
    Rows behind the last sequence, and sequences without keys, are zeros.  Offsets that decrease, do not
    start at zero or exceed their tensor are reported as an error later (see the module); the rows they
    concern are unspecified, and nothing outside of the tensors is read or written.
    """
    module, watch = _direct_watch()
    if module:
        out = module.window_packed(query, key, value, cumulative_seqlen_q, cumulative_seqlen_kv,
                                   0x7FFFFFFF if window is None else window, sinks, scale, watch.flag_at)
        if out is not None:
            watch.after_call()
            return out
    _refuse_transforms("varlen_sliding_window_attention_batch_invariant", query, key, value)
    if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
        raise ValueError("varlen attention expects rank-4 query, key, and value")
    if query.shape[0] != 1 or key.shape[0] != 1 or value.shape[0] != 1:
        raise ValueError("varlen attention expects sequence-packed batch size 1")
    if query.dtype != key.dtype or query.dtype != value.dtype:
        raise ValueError("query, key, and value must have the same dtype")
    if query.dtype not in nat.DIRECT_DTYPES:
        raise ValueError(f"unsupported varlen attention dtype: {query.dtype}")
    if key.shape[:3] != value.shape[:3]:
        raise ValueError("key and value token and head dimensions must match")
    if query.shape[3] != key.shape[3]:
        raise ValueError("query and key head dimensions must match")
    if key.shape[2] == 0 or query.shape[2] % key.shape[2]:
        raise ValueError("query heads must be divisible by key/value heads")
    for cu in (cumulative_seqlen_q, cumulative_seqlen_kv):
        if cu.dim() != 1 or cu.numel() == 0:
            raise ValueError("cumulative sequence lengths must be rank 1, with at least one offset")
        if cu.dtype not in _INDEX_TYPES:
            raise ValueError("cumulative sequence lengths must use int32 or int64")
    if cumulative_seqlen_q.numel() != cumulative_seqlen_kv.numel():
        raise ValueError("query and KV cumulative sequence counts must match")
    _check_head_dims("sliding-window attention", query.dtype, 128 if query.dtype == torch.float32 else 256,
                     query.shape[3], value.shape[3])
    window_size = _check_window(window, sinks)
    _check_scale(scale)
    device = _check_tensors("varlen_sliding_window_attention_batch_invariant", query, key, value,
                            cumulative_seqlen_q, cumulative_seqlen_kv)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return varlen_sliding_window_attention_batch_invariant(
                query, key, value, cumulative_seqlen_q, cumulative_seqlen_kv, window, sinks, scale=scale)
    q, k, v = _unit_last(query), _unit_last(key), _unit_last(value)
    watch = _watch(device)
    out = torch.empty((1, q.shape[1], q.shape[2], v.shape[3]), dtype=q.dtype, device=device)
    _windowed(q, k, v, out, cumulative_seqlen_q.numel() - 1, (q.shape[1], k.shape[1]), window_size, sinks, scale,
              (cumulative_seqlen_q, cumulative_seqlen_kv), watch)
    watch.after_call(nat.stream_of(out))
    return out
