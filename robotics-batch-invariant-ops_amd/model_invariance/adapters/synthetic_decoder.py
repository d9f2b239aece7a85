"""A small randomly initialised decoder as a policy serves it: the prompt (an image's patches, then text)
is run once and its rotated keys and values go into a cache in pages, then the answer is produced token by
token out of the cache.  Layers alternate between a sliding window with first tokens that stay visible and
the whole sequence.  A batch's prompts have different lengths behind the same padded shape, and where its
pages lie depends on the whole batch, so a sample's answer keeps its bits only if neither reaches it.

The model runs on the first ROCm GPU (CPU when there is none, in plain torch operations, for the harness's
own tests).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F


def _plain_rotary(x: torch.Tensor, positions: torch.Tensor, sections: tuple[int, ...]) -> torch.Tensor:
    """x [..., heads, dim], positions [axes, ...]: pairs (i, i + n) turn by their section's axis."""
    n = sum(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    turn = (positions.double()[axis].movedim(0, -1) * 10000.0 ** (-torch.arange(n).double() / n)).unsqueeze(-2)
    a, b = x[..., :n].double(), x[..., n:2 * n].double()
    return torch.cat([a * turn.cos() - b * turn.sin(), b * turn.cos() + a * turn.sin(), x[..., 2 * n:].double()], -1).to(x.dtype)


def _plain_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, place: torch.Tensor, window: int | None,
                     sinks: int) -> torch.Tensor:
    """q [heads, rows, dim], k and v [kv_heads, keys, dim], place [rows]: the rows' places among the keys."""
    k, v = (t.repeat_interleave(q.shape[0] // t.shape[0], 0).float() for t in (k, v))
    p, j = place.view(-1, 1), torch.arange(k.shape[1])
    seen = j <= p
    if window is not None:
        seen = seen & ((p - j < window) | (j < sinks))
    s = (q.float() @ k.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5
    return (torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v).to(q.dtype)


class _Decoder(torch.nn.Module):
    def __init__(self, d: int, hidden: int, heads: int, kv_heads: int, layers: int, window: int, sinks: int, page: int,
                 steps: int, actions: int, g: torch.Generator, dtype: torch.dtype):
        super().__init__()

        def w(*shape):
            return torch.nn.Parameter((torch.randn(*shape, generator=g) * shape[-1] ** -0.5).to(dtype), requires_grad=False)

        self.heads, self.kv_heads, self.page, self.steps = heads, kv_heads, page, steps
        self.hd = d // heads
        pairs = self.hd // 2  # half of them for time, the rest for the two directions of an image
        self.sections = (pairs - 2 * (pairs // 4), pairs // 4, pairs // 4)
        self.windows = [(window, sinks) if i % 2 == 0 else (None, 0) for i in range(layers)]
        self.qkv = torch.nn.ParameterList([w((heads + 2 * kv_heads) * self.hd, d) for _ in range(layers)])
        self.proj = torch.nn.ParameterList([w(d, d) for _ in range(layers)])
        self.up = torch.nn.ParameterList([w(hidden, d) for _ in range(layers)])
        self.down = torch.nn.ParameterList([w(d, hidden) for _ in range(layers)])
        self.norm_weight = torch.nn.Parameter(torch.ones(d, dtype=dtype), requires_grad=False)
        self.head = w(actions, d)
        self.embed = w(d, actions)

    def rms_norm(self, x: torch.Tensor) -> torch.Tensor:
        var = x.float().pow(2).mean(-1, keepdim=True)
        return (x.float() * torch.rsqrt(var + 1e-6)).to(x.dtype) * self.norm_weight

    def project(self, layer: int, h: torch.Tensor, positions: torch.Tensor):
        """Rotated queries and keys, and values, [..., heads, dim]."""
        from batch_invariant_ops import multi_axis_rotary

        sizes = [n * self.hd for n in (self.heads, self.kv_heads, self.kv_heads)]
        q, k, v = (t.unflatten(-1, (-1, self.hd)) for t in F.linear(self.rms_norm(h), self.qkv[layer]).split(sizes, -1))
        if h.is_cuda:
            q, k = multi_axis_rotary(q, k, positions, self.sections)
        else:
            q, k = (_plain_rotary(t, positions, self.sections) for t in (q, k))
        return q, k, v

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        from batch_invariant_ops import paged_cache_write

        if k.is_cuda:
            paged_cache_write(k, v, self.k_cache[layer], self.v_cache[layer], slots)
            return
        for cache, rows in ((self.k_cache[layer], k), (self.v_cache[layer], v)):
            cache.flatten(0, 1)[slots[slots >= 0]] = rows[slots >= 0]

    def prompt_attention(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        from batch_invariant_ops import sliding_window_attention_batch_invariant

        window, sinks = self.windows[layer]
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        if q.is_cuda:
            out = sliding_window_attention_batch_invariant(q, k, v, window, sinks, enable_gqa=True)
        else:
            place = torch.arange(q.shape[2])
            out = torch.stack([_plain_attention(*x, place, window, sinks) for x in zip(q, k, v)])
        return out.transpose(1, 2)

    def token_attention(self, layer: int, q: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        from batch_invariant_ops import paged_attention_batch_invariant

        window, sinks = self.windows[layer]
        if q.is_cuda:
            return paged_attention_batch_invariant(q, self.k_cache[layer], self.v_cache[layer], self.table, lengths,
                                                   window=window, sinks=sinks)
        out = []
        for b, n in enumerate(lengths.tolist()):
            k, v = (c[layer][self.table[b].long()].flatten(0, 1)[:n].transpose(0, 1) for c in (self.k_cache, self.v_cache))
            out.append(_plain_attention(q[b].unsqueeze(1), k, v, torch.tensor([n - 1]), window, sinks).squeeze(1))
        return torch.stack(out)

    def finish(self, layer: int, h: torch.Tensor, att: torch.Tensor) -> torch.Tensor:
        h = h + F.linear(att.flatten(-2), self.proj[layer])
        return h + F.linear(F.silu(F.linear(self.rms_norm(h), self.up[layer])), self.down[layer])

    def forward(self, x: torch.Tensor, positions: torch.Tensor, length: torch.Tensor) -> dict[str, torch.Tensor]:
        """x [B, T, D] padded at the end, positions [B, axes, T], length [B]."""
        b, t, _ = x.shape
        positions = positions.transpose(0, 1)
        width = -(-(t + self.steps) // self.page)
        pages = torch.randperm(b * width, generator=torch.Generator().manual_seed(b))
        self.table = pages.view(b, width).to(torch.int32).to(x.device)
        shape = (len(self.windows), b * width, self.page, self.kv_heads, self.hd)
        # what an earlier request left in a page must not matter either
        self.k_cache, self.v_cache = (x.new_full(shape, float("nan")) for _ in range(2))

        def slots(place: torch.Tensor) -> torch.Tensor:
            return self.table.long().gather(1, place // self.page) * self.page + place % self.page

        place = torch.arange(t, device=x.device).expand(b, t)
        where = torch.where(place < length.view(b, 1), slots(place), -1)
        h = x
        for layer in range(len(self.windows)):
            q, k, v = self.project(layer, h, positions)
            self.write(layer, k, v, where)
            h = self.finish(layer, h, self.prompt_attention(layer, q, k, v))
        last = (length - 1).long()
        h = h.gather(1, last.view(b, 1, 1).expand(b, 1, h.shape[2])).squeeze(1)
        reached = positions.gather(2, last.view(1, b, 1).expand(positions.shape[0], b, 1)).amax(0).view(b)
        actions = [F.linear(self.rms_norm(h), self.head)]
        lengths = length.clone()
        for _ in range(self.steps):
            h = F.linear(torch.tanh(actions[-1]), self.embed)
            reached = reached + 1
            lengths = lengths + 1
            at = slots(lengths.view(b, 1).long() - 1).view(b)
            for layer in range(len(self.windows)):
                q, k, v = self.project(layer, h, reached.expand(positions.shape[0], b))
                self.write(layer, k, v, at)
                h = self.finish(layer, h, self.token_attention(layer, q, lengths))
            actions.append(F.linear(self.rms_norm(h), self.head))
        return {"actions": torch.stack(actions, 1), "state": h}


# "small" for quick checks; "vla" has the attention widths of the synthetic_vla adapter's preset of that name
# (D 2048, MLP 8192, 16 query / 4 KV heads of 128).
PRESETS = {
    "small": dict(tokens=77, d=256, hidden=512, heads=4, kv_heads=2, layers=2, window=24, sinks=4, page=16, steps=6),
    "vla": dict(tokens=700, d=2048, hidden=8192, heads=16, kv_heads=4, layers=4, window=256, sinks=4, page=16, steps=16),
}


class SyntheticDecoderAdapter:
    """Harness adapter around ``_Decoder``; samples are seeded prompts [T, D] of their own length."""

    name = "synthetic_decoder"

    def __init__(self, tokens: int = 77, d: int = 256, hidden: int = 512, heads: int = 4, kv_heads: int = 2,
                 layers: int = 2, window: int = 24, sinks: int = 4, page: int = 16, steps: int = 6, actions: int = 7,
                 dtype: torch.dtype = torch.bfloat16, device: str | None = None):
        self.tokens, self.d = tokens, d
        self.cfg = (d, hidden, heads, kv_heads, layers, window, sinks, page, steps, actions)
        self.dtype = dtype
        self.device = device or ("cuda" if torch.cuda.is_available() else "cpu")

    @classmethod
    def preset(cls, name: str, **overrides) -> "SyntheticDecoderAdapter":
        return cls(**{**PRESETS[name], **overrides})

    def load_model(self) -> torch.nn.Module:
        g = torch.Generator().manual_seed(1234)
        return _Decoder(*self.cfg, g=g, dtype=self.dtype).to(self.device)

    def load_example_inputs(self, count: int) -> list[dict[str, torch.Tensor]]:
        g = torch.Generator().manual_seed(4321)
        side = max(1, int((self.tokens / 2) ** 0.5))
        at = torch.arange(self.tokens)
        text = at - side * side
        image = text < 0
        positions = torch.stack([torch.where(image, 0, side + text), torch.where(image, at // side, side + text),
                                 torch.where(image, at % side, side + text)])
        samples = []
        for _ in range(count):
            length = int(torch.randint(side * side + 1, self.tokens + 1, (1,), generator=g))
            x = torch.randn(self.tokens, self.d, generator=g)
            samples.append({"x": x.to(self.dtype).to(self.device), "positions": positions.to(self.device),
                            "length": torch.tensor(length, dtype=torch.int32, device=self.device)})
        return samples

    def run_model(self, model: torch.nn.Module, batch: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
        return model(batch["x"], batch["positions"], batch["length"])

    def extract_robot_output(self, output: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
        return output
