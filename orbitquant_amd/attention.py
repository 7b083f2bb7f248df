"""`OrbitCachedAttention`: the self-attention of a decoder layer on quantized linears and the 4-bit key/value cache.

One forward is what a serving step does between the layer's norm and its residual: the q, k and v projections of the new tokens
(`OrbitLinearGroup`: one quantization of the input), norms and rotary positions on the way into the cache (`kv_append`; or a callable of the model's and `kv_write`),
`kv_attend` over what the requests have cached, and the output projection.  Slots and lengths come from one `kv_assign`, positions and masks of
drafted tokens from one `kv_tree`, which all layers of a model share.  (No counterpart in the reference, whose models are diffusion transformers without a cache.)
"""

from __future__ import annotations

from typing import Callable

import torch
from torch import nn

from .kv_cache import KVAssignment, KVTree, OrbitKVCache, kv_append, kv_attend, kv_write
from .layers import OrbitLinear, OrbitLinearGroup
from .qk_rotary import QKNormRotary


class OrbitCachedAttention(nn.Module):
    """`forward(x, assignment, block_table)`: x [tokens, hidden], the new tokens of all requests one behind the other, as `assignment`
    (of `kv_assign`, for this cache's page size) has them; -> [tokens, hidden].

    q, k, v, out: OrbitLinear modules; k and v have the cache's heads, q a multiple of them.  `cache`: the layer's own.  `rotary`: a `QKNormRotary`,
    which `kv_append` applies in one launch with the write; or `rotary(q, k, positions)` -> (q, k), applied to [tokens, heads, D] with the positions
    int32 [tokens], -1 for tokens of no request.  `window`: of the keys that a token sees, the last ones only."""

    def __init__(self, q: OrbitLinear, k: OrbitLinear, v: OrbitLinear, out: OrbitLinear, cache: OrbitKVCache, *,
                 rotary: QKNormRotary | Callable | None = None, window: int | None = None) -> None:
        super().__init__()
        dim, kv_width = cache.head_dim, cache.heads * cache.head_dim
        if k.out_features != kv_width or v.out_features != kv_width:
            raise ValueError(f"k and v must have the cache's {cache.heads} heads of {dim}, got {k.out_features} and {v.out_features} outputs")
        if q.out_features == 0 or q.out_features % kv_width:
            raise ValueError(f"q must have a multiple of the cache's {cache.heads} heads of {dim}, got {q.out_features} outputs")
        if out.in_features != q.out_features:
            raise ValueError(f"out takes {out.in_features} values, q gives {q.out_features}")
        self.q, self.k, self.v, self.out = q, k, v, out
        self.cache = cache
        self.rotary = rotary
        self.window = window

    def forward(self, x: torch.Tensor, assignment: KVAssignment, block_table: torch.Tensor, *, tree: KVTree | None = None, one_each: bool = False,
                max_new: int | None = None, max_length: int | None = None) -> torch.Tensor:
        """`one_each`: every request has exactly one new token, row r of x is request r's (a decoding step, which then need not look
        for a request's rows).  Otherwise rows belong to the requests that `assignment.starts` gives them to, and those of no request attend to nothing.
        `tree`: the new tokens are drafted ones, whose positions and masks it has.
        `max_new` and `max_length` as for `kv_attend`: hints."""
        tokens, dim = x.shape[0], self.cache.head_dim
        if one_each and tokens != assignment.lengths.numel():
            raise ValueError(f"one_each: {tokens} rows for {assignment.lengths.numel()} requests")
        q, k, v = OrbitLinearGroup(self.q, self.k, self.v)(x)
        q, k, v = (t.view(tokens, t.shape[1] // dim, dim) for t in (q, k, v))
        positions, masks = (assignment.positions, None) if tree is None else tree
        if isinstance(self.rotary, QKNormRotary):
            q = kv_append(q, k, v, assignment.slots, self.cache, self.rotary, positions)
        else:
            if self.rotary is not None:
                q, k = self.rotary(q, k, positions)
            kv_write(k, v, assignment.slots, self.cache)
        attended = kv_attend(q, self.cache, block_table, assignment.lengths, starts=None if one_each else assignment.starts, masks=masks, max_new=max_new,
                             max_length=max_length, window=self.window)
        return self.out(attended.flatten(1))
