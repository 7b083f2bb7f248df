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
    int32 [tokens], -1 for tokens of no request.  `window`: of the keys that a token sees, the last ones only.

    A `QKNormRotary`'s weights are the module's parameters `q_norm_weight` and `k_norm_weight`, saved, loaded, moved and converted with its linears; its tables move with
    it, are not saved and stay fp32.  (A state without the weights, as it was saved before they were part of one, leaves them as they are.)  The cache stays where it is."""

    _version = 2   # of the state: 1 has no norms' weights

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
        self._hold(rotary)
        self.window = window

    def _hold(self, rotary) -> None:
        self._rotary = None
        for name in ("_rotary_cos", "_rotary_sin"):
            self.register_buffer(name, None, persistent=False)
        for name in ("q_norm_weight", "k_norm_weight"):
            self.register_parameter(name, None)
        self.rotary = rotary

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        if "_rotary" not in self.__dict__:  # a module pickled whole when its rotary was an attribute like any other
            self._hold(self.__dict__.pop("rotary", None) or self._modules.get("rotary"))

    @property
    def rotary(self) -> QKNormRotary | Callable | None:
        module = self._modules.get("rotary")    # (a callable that is a module is one of this module's)
        if module is not None:
            return module
        if not isinstance(self._rotary, QKNormRotary):
            return self._rotary
        return QKNormRotary(self._rotary_cos, self._rotary_sin, self.q_norm_weight, self.k_norm_weight, self._rotary.eps, self._rotary.interleaved)

    @rotary.setter
    def rotary(self, rotary: QKNormRotary | Callable | None) -> None:
        plan = rotary if isinstance(rotary, QKNormRotary) else QKNormRotary()
        self._rotary = QKNormRotary(eps=plan.eps, interleaved=plan.interleaved) if rotary is plan else rotary
        self._rotary_cos, self._rotary_sin = (None if t is None else t.detach() for t in (plan.cos, plan.sin))
        for name, weight in (("q_norm_weight", plan.q_weight), ("k_norm_weight", plan.k_weight)):
            setattr(self, name, weight if weight is None or isinstance(weight, nn.Parameter) else nn.Parameter(weight.detach(), requires_grad=False))

    def _apply(self, fn, recurse: bool = True):
        tables = self._rotary_cos, self._rotary_sin
        super()._apply(fn, recurse)
        # Nothing saves or rebuilds the tables: what they hold goes along whatever becomes of the weights (another type, memory that is not filled).
        self._rotary_cos, self._rotary_sin = (moved if t is None or t.is_meta or moved.is_meta else t.to(moved.device)
                                              for t, moved in zip(tables, (self._rotary_cos, self._rotary_sin)))
        return self

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        if (local_metadata.get("version") or 1) < 2:
            for name in ("q_norm_weight", "k_norm_weight"):
                if getattr(self, name) is not None and prefix + name not in state_dict:
                    state_dict[prefix + name] = getattr(self, name).detach()
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)

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
        rotary = self.rotary
        if isinstance(rotary, QKNormRotary):
            q = kv_append(q, k, v, assignment.slots, self.cache, rotary, positions)
        else:
            if rotary is not None:
                q, k = rotary(q, k, positions)
            kv_write(k, v, assignment.slots, self.cache)
        attended = kv_attend(q, self.cache, block_table, assignment.lengths, starts=None if one_each else assignment.starts, masks=masks, max_new=max_new,
                             max_length=max_length, window=self.window)
        return self.out(attended.flatten(1))
