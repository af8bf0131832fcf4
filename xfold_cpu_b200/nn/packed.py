"""A pre-norm self-attention layer for packed sequences, to train and to step token by token.

It has no counterpart in the reference.  LayerNorm, the projections, rotary positions and masked
attention all run on the library's kernels, in training (with gradients, on rows that
hold several documents one after another) as in serving (one token at a time over a cache).
"""

from __future__ import annotations

import torch
from torch import nn

from .. import native, training


class PackedAttention(nn.Module):
    """x + output(attention(rotary(q, k), v)) of a LayerNorm'd token track x [B, N, C], bfloat16.

    num_head query heads of head_dim share num_kv_head key / value heads; the first `rotated`
    dims of a head carry rotary positions (stretched by `stretch` for contexts longer than
    the weights were trained at); scores are capped at `softcap` (0: not); with `distance`
    each head's scores also fall with distance, by 2^(-8 (h + 1) / num_head) a token."""

    def __init__(self, c: int, num_head: int, num_kv_head: int | None = None,
                 head_dim: int | None = None, rotated: int | None = None, softcap: float = 0.0,
                 distance: bool = False, stretch: float = 1.0, eps: float = 1e-5):
        super().__init__()
        self.num_head = num_head
        self.num_kv_head = num_head if num_kv_head is None else num_kv_head
        self.head_dim = c // num_head if head_dim is None else head_dim
        self.softcap, self.eps = softcap, eps
        h, g, d = self.num_head, self.num_kv_head, self.head_dim
        if h % g or c % 8 or ((h + 2 * g) * d) % 8 or (h * d) % 8:
            raise ValueError("heads must divide and widths be multiples of 8")
        self.norm_weight = nn.Parameter(torch.ones(c))
        self.norm_bias = nn.Parameter(torch.zeros(c))
        self.qkv = nn.Parameter(torch.randn((h + 2 * g) * d, c) * c ** -0.5)
        self.output = nn.Parameter(torch.randn(c, h * d) * (h * d) ** -0.5)
        self.register_buffer("frequencies", native.rotary_frequencies(
            d if rotated is None else rotated, stretch=stretch), persistent=False)
        slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)],
                              dtype=torch.float32) if distance else None
        self.register_buffer("slopes", slopes, persistent=False)

    def _apply(self, fn, recurse: bool = True):
        """Moves and casts the layer, but keeps frequencies and slopes in float32: an angle is
        position * frequency, and 8 bits of a frequency are a turn off after some thousand tokens."""
        kept = {name: t for name, t in self._buffers.items() if t is not None}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def _heads(self, x: torch.Tensor, positions, offset: int):
        """q [B, H, N, D], k and v [B, G, N, D] as views of one projection, q and k rotated."""
        b, n, _ = x.shape
        h, g, d = self.num_head, self.num_kv_head, self.head_dim
        y = training.layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        qkv = training.linear(y, self.qkv).view(b, n, h + 2 * g, d).transpose(1, 2)
        q, k, v = qkv.split((h, g, g), 1)
        q, k = training.rotary(q, k, self.frequencies, positions=positions, offset=offset)
        return q, k, v

    def _close(self, x: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        b, n, _ = x.shape
        return x + training.linear(out.transpose(1, 2).reshape(b, n, -1), self.output)

    def forward(self, x: torch.Tensor, documents: torch.Tensor | None = None,
                positions: torch.Tensor | None = None,
                prefix: torch.Tensor | None = None) -> torch.Tensor:
        """x [B, N, C] bfloat16; documents int [B, N] (negative: padding), positions int [B, N]
        within them (None: 0, 1, ...), prefix int [B] tokens that see each other both ways."""
        q, k, v = self._heads(x, positions, 0)
        out = training.masked_attention(q, k, v, softcap=self.softcap, slopes=self.slopes,
                                        causal=True, prefix=prefix, documents=documents)
        return self._close(x, out)

    def cache(self, batch: int, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Key and value cache [B, G, length, D] for `step`."""
        shape = (batch, self.num_kv_head, length, self.head_dim)
        return tuple(torch.empty(shape, dtype=torch.bfloat16, device=self.qkv.device)
                     for _ in range(2))

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: tuple[torch.Tensor, torch.Tensor],
             filled: int) -> torch.Tensor:
        """New tokens x [B, n, C] at positions filled, filled + 1, ...: writes their keys and
        values into the cache and attends over what it holds up to them."""
        n = x.shape[1]
        if filled < 0 or x.shape[0] != cache[0].shape[0]:
            raise ValueError("filled counts the cache's tokens, and the cache has a row for each of x")
        if filled + n > cache[0].shape[2]:
            raise ValueError("the cache is full")
        q, k, v = self._heads(x, None, filled)
        cache[0][:, :, filled:filled + n] = k
        cache[1][:, :, filled:filled + n] = v
        out = training.masked_attention(q, cache[0][:, :, :filled + n], cache[1][:, :, :filled + n],
                                        softcap=self.softcap, slopes=self.slopes, causal=True)
        return self._close(x, out)
