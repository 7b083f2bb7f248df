"""The key/value cache of a serving program in four bits, and its operators.

`OrbitKVCache` holds the tensors; `kv_assign` gives new tokens their pages and slots, `kv_write` puts keys and values there (`kv_append`: with the
norms and rotary positions of queries and keys in the same launch), `kv_attend` is the attention of queries over the cache, `kv_read` gives back what the
cache holds.  New tokens may be trees of drafted ones: `kv_tree` gives their positions and masks, `kv_keep` makes the accepted path of each the request's last tokens.  All of them run on the
current stream without synchronizing, so a decoding step (assign, write, attend) can be captured into a HIP graph.  The
functions are also reached as `ops.kv_*`.  (The reference has no cache: its models are diffusion transformers.)

A vector is held in the rotated space of `get_rpbh_rotation(head_dim).signs` and the Walsh-Hadamard transform, as one bf16 scale and
E2M1 codes (include/orbitquant_hip.h states the arithmetic): head_dim / 2 + 2 bytes for a key or a value, 3.76 times less than bf16.
Queries are rotated by the attention itself, and its outputs back: what goes in and comes out is in the model's own basis.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.compiler import is_compiling

from . import _lib
from .ops import _DTYPES, _dt, _OnDevice, _operand, _ptr, _require_gpu, _stream, _workspace
from .qk_rotary import _HOW, QKNormRotary, _plan, _vectors
from .rotations import get_rpbh_rotation


KEEP_ALL = -2   # of `kv_keep`'s lists, as the first entry (OQ_KV_KEEP_ALL)


class OrbitKVCache(NamedTuple):
    """The tensors of a cache, contiguous, on one GPU:

    k_codes uint8 [pages, heads, page, D/2], k_scales bfloat16 [pages, heads, page], v_codes uint8 [pages, heads, D/2, page],
    v_scales bfloat16 [pages, heads, page], signs int8 [D].  D is 64, 128 or 256, a page a power of two from 16 to 1024 tokens.
    """

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    signs: torch.Tensor

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, *, page_size: int = 64, seed: int = 0, device="cuda") -> "OrbitKVCache":
        """A cache of `pages` pages without tokens (its memory is not cleared: what no token was written to is not read as one)."""
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if pages < 1 or heads < 1:
            raise ValueError("pages and heads must be positive")
        signs = get_rpbh_rotation(head_dim, seed).signs.to(device=device, dtype=torch.int8)
        codes = lambda *shape: torch.empty(pages, heads, *shape, dtype=torch.uint8, device=device)  # noqa: E731
        scales = lambda: torch.empty(pages, heads, page_size, dtype=torch.bfloat16, device=device)  # noqa: E731
        return cls(codes(page_size, head_dim // 2), scales(), codes(head_dim // 2, page_size), scales(), signs)

    @property
    def pages(self) -> int:
        return self.k_codes.shape[0]

    @property
    def heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]


class KVAssignment(NamedTuple):
    """What `kv_assign` gives: slots int64 and positions int32 of the new tokens, starts int32 [requests + 1], the lengths
    after the step, int32 [requests], and the number of pages taken from the free list, int32 [1]."""

    slots: torch.Tensor
    positions: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor
    taken: torch.Tensor


class KVTree(NamedTuple):
    """What `kv_tree` gives: positions int32 [tokens] of drafted tokens, and masks int64 [tokens, words]: bit j % 64 of word j / 64 stands for
    the request's new token j."""

    positions: torch.Tensor
    masks: torch.Tensor


class KVKept(NamedTuple):
    """What `kv_keep` gives: the lengths without the forgotten tokens, int32 [requests], and the number of pages that are still taken from the
    free list, int32 [1] (None where no list was given)."""

    lengths: torch.Tensor
    taken: torch.Tensor | None


# For torch.compile the functions below are opaque ops with fake implementations; eager calls do not go through them.
_LIB = torch.library.Library("orbitquant_amd", "FRAGMENT")
_CACHE = "Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor signs"
_LIB.define("kv_assign(Tensor lengths, Tensor new_lengths, Tensor(a!) block_table, Tensor free_pages, Tensor taken, SymInt page_size, SymInt tokens) "
            "-> (Tensor, Tensor)")
_LIB.define("kv_write(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, Tensor signs) -> ()")
_LIB.define(f"kv_read(Tensor slots, {_CACHE}, ScalarType dtype) -> (Tensor, Tensor)")
_LIB.define(f"kv_attend(Tensor q, {_CACHE}, Tensor block_table, Tensor lengths, Tensor? starts, SymInt max_new, SymInt max_length, bool causal, "
            "SymInt window, float scale, bool with_lse) -> (Tensor, Tensor)")
_LIB.define("kv_append(Tensor q, Tensor k, Tensor v, Tensor slots, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, Tensor signs, "
            f"{_HOW}, Tensor? positions) -> Tensor")
_LIB.define("kv_tree(Tensor parents, Tensor starts, Tensor lengths, SymInt words) -> (Tensor, Tensor)")
_LIB.define(f"kv_attend_tree(Tensor q, {_CACHE}, Tensor block_table, Tensor lengths, Tensor? starts, Tensor masks, SymInt max_new, SymInt max_length, "
            "SymInt window, float scale, bool with_lse) -> (Tensor, Tensor)")
_LIB.define("kv_keep(Tensor kept, Tensor lengths, Tensor starts, Tensor slots, Tensor(a!)[] k_codes, Tensor(b!)[] k_scales, Tensor(c!)[] v_codes, Tensor(d!)[] v_scales, "
            "Tensor[] signs, Tensor? block_table, Tensor(e!)? free_pages, Tensor? taken) -> (Tensor, Tensor)")


def _assign_op(lengths, new_lengths, block_table, free_pages, taken, page_size, tokens):
    """-> slots, and the four int32 results one behind the other (`_assigned` parts them: an op's outputs may not share memory)."""
    _require_gpu(lengths, "lengths")
    requests = lengths.numel()
    lengths = _operand(lengths, "lengths", lengths, dtype=torch.int32)
    new_lengths = _operand(new_lengths, "new_lengths", lengths, dtype=torch.int32, numel=requests)
    free_pages = _operand(free_pages, "free_pages", lengths, dtype=torch.int32)
    taken = _operand(taken, "taken", lengths, dtype=torch.int32, numel=1)
    table = _table(block_table, lengths, requests)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    slots, small = _assign_fake(lengths, None, None, None, None, None, tokens)
    _, positions, starts, after, taken_after = _assigned(slots, small, tokens, requests)
    with _OnDevice(lengths):
        rc = _lib.load().oq_kv_assign(
            lengths.data_ptr(), new_lengths.data_ptr(), requests, table.data_ptr(), table.stride(0), table.shape[1], free_pages.data_ptr(),
            free_pages.numel(), taken.data_ptr(), int(page_size), tokens, slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
            after.data_ptr(), taken_after.data_ptr(), _stream(lengths))
    _lib.check(rc, "oq_kv_assign")
    return slots, small


def _assign_fake(lengths, new_lengths, block_table, free_pages, taken, page_size, tokens):
    return (torch.empty(tokens, dtype=torch.int64, device=lengths.device),
            torch.empty(tokens + 2 * lengths.numel() + 2, dtype=torch.int32, device=lengths.device))


def _assigned(slots, small, tokens, requests) -> KVAssignment:
    return KVAssignment(slots, *small.split((tokens, requests + 1, requests, 1)))


def _write_op(k, v, slots, *cache):
    kv_write(k, v, slots, OrbitKVCache(*cache))


def _read_op(slots, k_codes, k_scales, v_codes, v_scales, signs, dtype):
    return kv_read(slots, OrbitKVCache(k_codes, k_scales, v_codes, v_scales, signs), dtype)


def _read_fake(slots, k_codes, k_scales, v_codes, v_scales, signs, dtype):
    shape = (slots.numel(), k_codes.shape[1], signs.shape[0])
    return slots.new_empty(shape, dtype=dtype), slots.new_empty(shape, dtype=dtype)


def _attend_op(q, k_codes, k_scales, v_codes, v_scales, signs, block_table, lengths, starts, max_new, max_length, causal, window, scale, with_lse):
    got = kv_attend(q, OrbitKVCache(k_codes, k_scales, v_codes, v_scales, signs), block_table, lengths, starts=starts, max_new=max_new,
                    max_length=max_length, causal=causal, window=window or None, scale=scale, return_lse=with_lse)
    return got if with_lse else (got, q.new_empty((0, q.shape[1]), dtype=torch.float32))


def _attend_fake(q, k_codes, k_scales, v_codes, v_scales, signs, block_table, lengths, starts, max_new, max_length, causal, window, scale, with_lse):
    return q.new_empty(q.shape), q.new_empty((q.shape[0] if with_lse else 0, q.shape[1]), dtype=torch.float32)


def _append_op(q, k, v, slots, k_codes, k_scales, v_codes, v_scales, signs, cos, sin, q_weight, k_weight, eps, interleaved, positions):
    return kv_append(q, k, v, slots, OrbitKVCache(k_codes, k_scales, v_codes, v_scales, signs), QKNormRotary(cos, sin, q_weight, k_weight, eps, interleaved), positions)


def _tree_op(parents, starts, lengths, words):
    return tuple(_tree(parents, starts, lengths, words))   # (an op's outputs may not share memory)


def _tree_fake(parents, starts, lengths, words):
    return parents.new_empty(parents.shape), parents.new_empty((parents.shape[0], words), dtype=torch.int64)


def _attend_tree_op(q, k_codes, k_scales, v_codes, v_scales, signs, block_table, lengths, starts, masks, max_new, max_length, window, scale, with_lse):
    got = kv_attend(q, OrbitKVCache(k_codes, k_scales, v_codes, v_scales, signs), block_table, lengths, starts=starts, masks=masks, max_new=max_new,
                    max_length=max_length, window=window or None, scale=scale, return_lse=with_lse)
    return got if with_lse else (got, q.new_empty((0, q.shape[1]), dtype=torch.float32))


def _attend_tree_fake(q, k_codes, k_scales, v_codes, v_scales, signs, block_table, lengths, starts, masks, max_new, max_length, window, scale, with_lse):
    return q.new_empty(q.shape), q.new_empty((q.shape[0] if with_lse else 0, q.shape[1]), dtype=torch.float32)


def _keep_op(kept, lengths, starts, slots, k_codes, k_scales, v_codes, v_scales, signs, block_table, free_pages, taken):
    caches = [OrbitKVCache(*c) for c in zip(k_codes, k_scales, v_codes, v_scales, signs, strict=True)]
    after, taken_after = kv_keep(kept, lengths, starts, slots, caches, block_table=block_table, free_pages=free_pages, taken=taken)
    return after, after.new_empty(0) if taken_after is None else taken_after


def _keep_fake(kept, lengths, starts, slots, k_codes, k_scales, v_codes, v_scales, signs, block_table, free_pages, taken):
    return lengths.new_empty(lengths.shape), lengths.new_empty(0 if taken is None else 1)


for _name, _op, _fake in (("kv_assign", _assign_op, _assign_fake), ("kv_write", _write_op, lambda *args: None), ("kv_read", _read_op, _read_fake),
                          ("kv_attend", _attend_op, _attend_fake), ("kv_append", _append_op, lambda q, *args: q.new_empty(q.shape)),
                          ("kv_tree", _tree_op, _tree_fake), ("kv_attend_tree", _attend_tree_op, _attend_tree_fake), ("kv_keep", _keep_op, _keep_fake)):
    _LIB.impl(_name, _op, "CUDA")
    torch.library.register_fake(f"orbitquant_amd::{_name}", _fake, lib=_LIB)


_host = None   # what `_module` has found, to be looked at without a call


def _module():
    """The compiled module (csrc/torch_ops.cpp), which has the usual calls of these functions without Python in between (a cached
    token's slot 13.5 -> 5.4 us, one token decoded 19.5 -> 12.2); None where it is not built.  What it does not take, errors among it, it
    leaves to the Python below."""
    global _host
    _host = _lib.torch_ops()
    if _host is None:
        _lib.warn_without_torch_ops()
    return _host


def _cache_struct(cache, like: torch.Tensor) -> _lib.KvCacheStruct:
    """The cache as the library takes it.  Its tensors are written to, so none is ever copied: what is not contiguous is refused."""
    k_codes, k_scales, v_codes, v_scales, signs = cache
    if k_codes.ndim != 4:
        raise ValueError("k_codes must be [pages, heads, page, D/2]")
    pages, heads, page, half = k_codes.shape
    shapes = ((k_codes, "k_codes", torch.uint8, (pages, heads, page, half)), (k_scales, "k_scales", torch.bfloat16, (pages, heads, page)),
              (v_codes, "v_codes", torch.uint8, (pages, heads, half, page)), (v_scales, "v_scales", torch.bfloat16, (pages, heads, page)),
              (signs, "signs", torch.int8, (2 * half,)))
    for t, name, dtype, shape in shapes:
        if t.device != like.device:
            raise ValueError(f"{name} is on {t.device}, the call's other tensors on {like.device}")
        if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be {dtype} {list(shape)} and contiguous, got {t.dtype} {list(t.shape)}")
    return _lib.KvCacheStruct(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), signs.data_ptr(), pages, heads,
                              page, 2 * half)


def _rows(t: torch.Tensor, name: str, heads: int | None, dim: int) -> torch.Tensor:
    """[tokens, heads, D] with a contiguous last dimension: other strides go to the kernel as they are."""
    if t.ndim != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {dim}], got {list(t.shape)}")
    return t if t.stride(2) == 1 else t.contiguous()


def _table(table: torch.Tensor, like: torch.Tensor, requests: int) -> torch.Tensor:
    if table.device != like.device or table.dtype != torch.int32 or table.ndim != 2 or table.shape[0] != requests:
        raise ValueError(f"block_table must be int32 [{requests}, width] on {like.device}, got {table.dtype} {list(table.shape)} on {table.device}")
    if table.shape[1] > 1 and table.stride(1) != 1 or requests > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("block_table's rows must be contiguous")
    return table


def kv_assign(lengths: torch.Tensor, new_lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor, *,
              page_size: int, tokens: int) -> KVAssignment:
    """Pages and slots for the new tokens of a batch of requests (`oq_kv_assign`), in one launch.

    Request r holds lengths[r] tokens in the first pages of its row of `block_table` and gets new_lengths[r] more.  The pages that
    this needs are taken from the front of `free_pages`, behind the `taken` that are already given out, in request order, and are
    written into the table; a token for which there is no page any more gets the slot -1, which `kv_write` skips and
    `kv_attend` does not see.  `tokens`: the number of new tokens, as the caller's arrays have them; what `new_lengths` leaves of
    it gets slot and position -1.  lengths, new_lengths int32 [requests], block_table int32 [requests, width] (changed in
    place), free_pages int32 [any], taken int32 [1]."""
    if is_compiling():
        return _assigned(*torch.ops.orbitquant_amd.kv_assign(lengths, new_lengths, block_table, free_pages, taken, page_size, tokens), tokens,
                         lengths.numel())
    module = _host or _module()
    if module is not None:
        got = module.kv_assign(lengths, new_lengths, block_table, free_pages, taken, int(page_size), int(tokens))
        if got is not None:
            return KVAssignment._make(got)
    return _assigned(*_assign_op(lengths, new_lengths, block_table, free_pages, taken, page_size, tokens), int(tokens), lengths.numel())


def kv_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: OrbitKVCache) -> None:
    """Keys and values [tokens, heads, D] into the cache at `slots` int64 [tokens] (`oq_kv_write`).  Slots that are negative or
    beyond the last page are skipped; no slot may occur twice.  k and v: one floating type, any strides whose last is 1 (parts of
    a fused projection's output need no copy)."""
    if is_compiling():
        torch.ops.orbitquant_amd.kv_write(k, v, slots, *cache)
        return
    module = _host or _module()
    if module is not None and module.kv_write(k, v, slots, cache):
        return
    _require_gpu(k, "k")
    struct = _cache_struct(cache, k)
    heads, dim = struct.kv_heads, struct.head_dim
    k, v = _rows(k, "k", heads, dim), _rows(v, "v", heads, dim)
    if v.device != k.device or v.dtype != k.dtype or v.shape[0] != k.shape[0]:
        raise ValueError(f"k and v must agree: {k.dtype} {list(k.shape)} on {k.device}, {v.dtype} {list(v.shape)} on {v.device}")
    slots = _operand(slots, "slots", k, dtype=torch.int64, numel=k.shape[0])
    with _OnDevice(k):
        rc = _lib.load().oq_kv_write(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _dt(k), slots.data_ptr(),
                                     k.shape[0], ctypes.byref(struct), _stream(k))
    _lib.check(rc, "oq_kv_write")


def kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: OrbitKVCache, how: QKNormRotary,
              positions: torch.Tensor | None = None) -> torch.Tensor:
    """`qk_norm_rotary` and `kv_write` in one launch (`oq_kv_append`): -> the queries, normed and turned, a new tensor.

    The keys' codes are those of the fp32 result: between the rotation and the cache nothing is rounded.  q [tokens, heads, D], k and v
    [tokens, cache heads, D] of one floating type, any strides whose last is 1; slots int64 [tokens] as for `kv_write`; `how` and
    `positions` as for `qk_norm_rotary`."""
    if is_compiling():
        return torch.ops.orbitquant_amd.kv_append(q, k, v, slots, *cache, *how, positions)
    module = _host or _module()
    if module is not None:
        got = module.kv_append(q, k, v, slots, cache, *how, positions)
        if got is not None:
            return got
    _require_gpu(q, "q")
    struct = _cache_struct(cache, q)
    heads, dim = struct.kv_heads, struct.head_dim
    if q.ndim != 3:
        raise ValueError(f"q must be [tokens, heads, {dim}], got {list(q.shape)}")
    q, k, v = _vectors(q, "q", q, None, dim), _vectors(k, "k", q, heads, dim), _vectors(v, "v", q, heads, dim)
    slots = _operand(slots, "slots", q, dtype=torch.int64, numel=q.shape[0])
    plan, _keep = _plan(how, q, positions)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    with _OnDevice(q):
        rc = _lib.load().oq_kv_append(q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                                      v.stride(1), _dt(q), slots.data_ptr(), q.shape[0], ctypes.byref(plan), ctypes.byref(struct), out.data_ptr(), _stream(q))
    _lib.check(rc, "oq_kv_append")
    return out


def kv_read(slots: torch.Tensor, cache: OrbitKVCache, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds at `slots` int64 [tokens], as keys and values [tokens, heads, D] of `dtype` (`oq_kv_read`); zeros for
    slots that are negative or beyond the last page."""
    if is_compiling():
        return torch.ops.orbitquant_amd.kv_read(slots, *cache, dtype)
    module = _host or _module()
    if module is not None:
        got = module.kv_read(slots, cache, dtype)
        if got is not None:
            return got
    _require_gpu(slots, "slots")
    struct = _cache_struct(cache, slots)
    slots = _operand(slots, "slots", slots, dtype=torch.int64)
    if dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {dtype}")
    tokens = slots.numel()
    k, v = (torch.empty(tokens, struct.kv_heads, struct.head_dim, dtype=dtype, device=slots.device) for _ in range(2))
    with _OnDevice(slots):
        rc = _lib.load().oq_kv_read(slots.data_ptr(), tokens, ctypes.byref(struct), k.data_ptr(), v.data_ptr(), _DTYPES[dtype], _stream(slots))
    _lib.check(rc, "oq_kv_read")
    return k, v


def kv_attend(q: torch.Tensor, cache: OrbitKVCache, block_table: torch.Tensor, lengths: torch.Tensor, *, starts: torch.Tensor | None = None,
              masks: torch.Tensor | None = None, max_new: int | None = None, max_length: int | None = None, causal: bool = True,
              window: int | None = None, scale: float | None = None, return_lse: bool = False):
    """Attention of queries over the cache (`oq_kv_attend`): -> out, of q's shape and type, or (out, lse float32 [tokens, heads]).

    q            [tokens, heads, D]; heads a multiple of the cache's, whose head h // (heads / cache heads) they read
    lengths      int32 [requests]: the cached tokens of each request, its new ones among them (`kv_assign(...).lengths`)
    block_table  int32 [requests, width]
    starts       int32 [requests + 1]: where a request's queries begin in q (`kv_assign(...).starts`); None for one query a request
    masks        int64 [tokens, 1 to 4] (`kv_tree(...).masks`, or any): of its request's new tokens a query sees those whose bit is set, and all
                 tokens before them; a request with more new tokens than the masks have bits is causal.  None: each is causal
    causal       the queries are the last tokens of their request, and see those up to their own; False: all of the request's
    window       of these, only the last `window`
    scale        of the scores; None: 1 / sqrt(D)
    max_new, max_length: the largest number of a request's queries, and the largest of the lengths, as far as the caller knows:
                 they choose launch shapes, and a wrong one costs time only

    A query that sees no token, and a token behind the last request's, gets zeros (lse -inf).  Accumulation, scores and softmax
    are fp32; queries and weights enter the matrix units as fp16 (as two fp16 parts of float32 queries)."""
    if window is not None and (window < 1 or not causal):
        raise ValueError("a window is at least 1 and needs causal attention")
    if masks is not None and not causal:
        raise ValueError("masks need causal attention")
    window = 0 if window is None else int(window)
    max_length = -1 if max_length is None else int(max_length)
    max_new = -1 if max_new is None else int(max_new)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if is_compiling():
        if masks is not None:
            out, lse = torch.ops.orbitquant_amd.kv_attend_tree(q, *cache, block_table, lengths, starts, masks, max_new, max_length, window, scale, return_lse)
        else:
            out, lse = torch.ops.orbitquant_amd.kv_attend(q, *cache, block_table, lengths, starts, max_new, max_length, causal, window, scale, return_lse)
        return (out, lse) if return_lse else out
    module = _host or _module()
    if module is not None:
        got = module.kv_attend(q, cache, block_table, lengths, starts, max_new, max_length, bool(causal), window, scale, bool(return_lse), masks)
        if got is not None:
            return got
    _require_gpu(q, "q")
    struct = _cache_struct(cache, q)
    q = _rows(q, "q", None, struct.head_dim)
    tokens, heads, dim = q.shape
    if heads == 0 or heads % struct.kv_heads:
        raise ValueError(f"q has {heads} heads, the cache {struct.kv_heads}: not a multiple")
    requests = lengths.numel()
    lengths = _operand(lengths, "lengths", q, dtype=torch.int32)
    starts = _operand(starts, "starts", q, dtype=torch.int32, numel=requests + 1)
    if starts is None and requests != tokens:
        raise ValueError(f"{tokens} queries for {requests} requests: starts is needed")
    table = _table(block_table, q, requests)
    if masks is not None:
        if masks.ndim != 2 or masks.shape[0] != tokens or not 1 <= masks.shape[1] <= 4:
            raise ValueError(f"masks must be [{tokens}, 1 to 4 words], got {list(masks.shape)}")
        masks = _operand(masks, "masks", q, dtype=torch.int64)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(tokens, heads, dtype=torch.float32, device=q.device) if return_lse else None
    lib = _lib.load()
    shape = (tokens, heads, struct.kv_heads, dim, struct.page_size, table.shape[1], requests, starts is not None)
    if masks is None:
        needed = lib.oq_kv_attend_workspace_bytes(*shape, window, max_length, max_new)
    else:
        needed = lib.oq_kv_attend_tree_workspace_bytes(_dt(q), *shape, masks.shape[1], window, max_length, max_new)
    workspace, nbytes, _keep = _workspace(needed, q, lambda: (0,))
    which, seen = (lib.oq_kv_attend, (bool(causal),)) if masks is None else (lib.oq_kv_attend_tree, (masks.data_ptr(), masks.shape[1]))
    with _OnDevice(q):
        rc = which(q.data_ptr(), _dt(q), tokens, heads, q.stride(0), q.stride(1), ctypes.byref(struct), table.data_ptr(),
                   table.stride(0), table.shape[1], lengths.data_ptr(), _ptr(starts), requests, *seen, window, scale, max_length, max_new, out.data_ptr(), _ptr(lse),
                   workspace, nbytes, _stream(q))
    _lib.check(rc, "oq_kv_attend")
    return out if lse is None else (out, lse)


def kv_tree(parents: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, *, max_new: int = 64) -> KVTree:
    """Positions and masks of drafted tokens (`oq_kv_tree`), once a step for all layers.

    parents  int32 [tokens]: of each token the index, among its request's new ones, of the one it hangs on, which stands before it; -1 for one that
             hangs on what the request has cached
    starts, lengths   int32 [requests + 1] and [requests], as `kv_assign` gives them for these tokens
    max_new  the largest number of new tokens of a request that is a tree, at most 256: it decides on the masks' words.  A request with more than
             these have bits is a prompt, whose tokens follow each other whatever its parents say: a tree of 70 nodes needs max_new=70, and is a chain without it

    A token's position is its depth behind the cached ones: what `kv_append` wants for it, where `kv_assign`'s are its place's.  Tokens of no request have
    position -1 and empty masks."""
    words = -(-int(max_new) // 64)
    if not 1 <= words <= 4:
        raise ValueError(f"max_new must be from 1 to 256, got {max_new}")
    if is_compiling():
        return KVTree(*torch.ops.orbitquant_amd.kv_tree(parents, starts, lengths, words))
    module = _host or _module()
    if module is not None:
        got = module.kv_tree(parents, starts, lengths, words)
        if got is not None:
            return KVTree._make(got)
    return _tree(parents, starts, lengths, words)


def _tree(parents, starts, lengths, words) -> KVTree:
    _require_gpu(parents, "parents")
    if parents.ndim != 1:
        raise ValueError(f"parents must be [tokens], got {list(parents.shape)}")
    tokens, requests = parents.numel(), lengths.numel()
    parents = _operand(parents, "parents", parents, dtype=torch.int32)
    lengths = _operand(lengths, "lengths", parents, dtype=torch.int32)
    starts = _operand(starts, "starts", parents, dtype=torch.int32, numel=requests + 1)
    positions = torch.empty(tokens, dtype=torch.int32, device=parents.device)
    masks = torch.empty(tokens, words, dtype=torch.int64, device=parents.device)
    with _OnDevice(parents):
        rc = _lib.load().oq_kv_tree(parents.data_ptr(), starts.data_ptr(), lengths.data_ptr(), requests, tokens, words, positions.data_ptr(), masks.data_ptr(),
                                    _stream(parents))
    _lib.check(rc, "oq_kv_tree")
    return KVTree(positions, masks)


def kv_keep(kept: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, slots: torch.Tensor, caches, *, block_table: torch.Tensor | None = None,
            free_pages: torch.Tensor | None = None, taken: torch.Tensor | None = None) -> KVKept:
    """After a step of drafted tokens: of each request's new tokens the `kept` ones stay, as if they had been its only ones (`oq_kv_keep`).

    kept     int32 [requests, most], most at most 256: which of the request's new tokens, in rising order, -1 behind the last.  A list ends at the first
             entry that does not rise, is none of the request's new tokens, has no slot or would go where there is none.  The i-th one's entries move to where its i-th new token's are
             A list that begins with `KEEP_ALL` keeps all of the request's new tokens, however many: a prompt beside trees
    lengths, starts, slots   as `kv_assign` gave them for the step
    caches   the OrbitKVCaches of all layers, of one shape, changed in place (one launch for every 64 of them); one that layers share, once; caches that
             share memory otherwise are refused
    block_table, free_pages, taken   as they are after that `kv_assign` (`taken`: its result), all or none of them.  Pages behind the kept tokens go back
             onto the list, in place, in front of those that it gives out next.  The table's columns behind the kept pages stand for nothing from then on.
             Pages that `kv_assign` drew for columns that the table does not have go back too, if the call is for all of its requests; only of a step in which the list ran out
             and no column got a page is it not known which these were (a table with room for every new token never has any)"""
    if (block_table is None) != (free_pages is None) or (free_pages is None) != (taken is None):
        raise ValueError("block_table, free_pages and taken go together")
    caches = list(caches)
    if not caches:
        raise ValueError("kv_keep needs the caches of at least one layer")
    if is_compiling():
        after, taken_after = torch.ops.orbitquant_amd.kv_keep(kept, lengths, starts, slots, *(list(t) for t in zip(*caches)), block_table, free_pages, taken)
        return KVKept(after, None if taken is None else taken_after)
    module = _host or _module()
    if module is not None:
        got = module.kv_keep(kept, lengths, starts, slots, caches, block_table, free_pages, taken)
        if got is not None:
            return KVKept._make(got)
    _require_gpu(lengths, "lengths")
    structs = (_lib.KvCacheStruct * len(caches))(*(_cache_struct(c, lengths) for c in caches))
    requests = lengths.numel()
    if kept.ndim != 2 or kept.shape[0] != requests:
        raise ValueError(f"kept must be [{requests}, most], got {list(kept.shape)}")
    lengths = _operand(lengths, "lengths", lengths, dtype=torch.int32)
    kept = _operand(kept, "kept", lengths, dtype=torch.int32)
    starts = _operand(starts, "starts", lengths, dtype=torch.int32, numel=requests + 1)
    slots = _operand(slots, "slots", lengths, dtype=torch.int64)
    after = torch.empty(requests, dtype=torch.int32, device=lengths.device)
    taken_after, pages = None, (None, 0, 0, None, 0, None)
    if taken is not None:
        table = _table(block_table, lengths, requests)
        taken = _operand(taken, "taken", lengths, dtype=torch.int32, numel=1)
        if free_pages.device != lengths.device or free_pages.dtype != torch.int32 or free_pages.ndim != 1 or not free_pages.is_contiguous():
            raise ValueError(f"free_pages must be int32 [any], contiguous, on {lengths.device}, got {free_pages.dtype} {list(free_pages.shape)} on {free_pages.device}")
        taken_after = torch.empty(1, dtype=torch.int32, device=lengths.device)
        pages = (table.data_ptr(), table.stride(0), table.shape[1], free_pages.data_ptr(), free_pages.numel(), taken.data_ptr())
    with _OnDevice(lengths):
        rc = _lib.load().oq_kv_keep(kept.data_ptr(), kept.shape[1], lengths.data_ptr(), starts.data_ptr(), slots.data_ptr(), requests, slots.numel(), structs, len(caches),
                                    *pages, after.data_ptr(), _ptr(taken_after), _stream(lengths))
    _lib.check(rc, "oq_kv_keep")
    return KVKept(after, taken_after)
