"""The key/value cache of a serving program in four bits, and its operators.

`OrbitKVCache` holds the tensors; `kv_assign` gives new tokens their pages and slots, `kv_write` puts keys and values there,
`kv_attend` is the attention of queries over the cache, `kv_read` gives back what the cache holds.  All of them run on the
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
from .rotations import get_rpbh_rotation


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


# For torch.compile the functions below are opaque ops with fake implementations; eager calls do not go through them.
_LIB = torch.library.Library("orbitquant_amd", "FRAGMENT")
_CACHE = "Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor signs"
_LIB.define("kv_assign(Tensor lengths, Tensor new_lengths, Tensor(a!) block_table, Tensor free_pages, Tensor taken, SymInt page_size, SymInt tokens) "
            "-> (Tensor, Tensor)")
_LIB.define("kv_write(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, Tensor signs) -> ()")
_LIB.define(f"kv_read(Tensor slots, {_CACHE}, ScalarType dtype) -> (Tensor, Tensor)")
_LIB.define(f"kv_attend(Tensor q, {_CACHE}, Tensor block_table, Tensor lengths, Tensor? starts, SymInt max_new, SymInt max_length, bool causal, "
            "SymInt window, float scale, bool with_lse) -> (Tensor, Tensor)")


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


for _name, _op, _fake in (("kv_assign", _assign_op, _assign_fake), ("kv_write", _write_op, lambda *args: None), ("kv_read", _read_op, _read_fake),
                          ("kv_attend", _attend_op, _attend_fake)):
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
              max_new: int | None = None, max_length: int | None = None, causal: bool = True, window: int | None = None,
              scale: float | None = None, return_lse: bool = False):
    """Attention of queries over the cache (`oq_kv_attend`): -> out, of q's shape and type, or (out, lse float32 [tokens, heads]).

    q            [tokens, heads, D]; heads a multiple of the cache's, whose head h // (heads / cache heads) they read
    lengths      int32 [requests]: the cached tokens of each request, its new ones among them (`kv_assign(...).lengths`)
    block_table  int32 [requests, width]
    starts       int32 [requests + 1]: where a request's queries begin in q (`kv_assign(...).starts`); None for one query a request
    causal       the queries are the last tokens of their request, and see those up to their own; False: all of the request's
    window       of these, only the last `window`
    scale        of the scores; None: 1 / sqrt(D)
    max_new, max_length: the largest number of a request's queries, and the largest of the lengths, as far as the caller knows:
                 they choose launch shapes, and a wrong one costs time only

    A query that sees no token, and a token behind the last request's, gets zeros (lse -inf).  Accumulation, scores and softmax
    are fp32; queries and weights enter the matrix units as fp16 (as two fp16 parts of float32 queries)."""
    if window is not None and (window < 1 or not causal):
        raise ValueError("a window is at least 1 and needs causal attention")
    window = 0 if window is None else int(window)
    max_length = -1 if max_length is None else int(max_length)
    max_new = -1 if max_new is None else int(max_new)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if is_compiling():
        out, lse = torch.ops.orbitquant_amd.kv_attend(q, *cache, block_table, lengths, starts, max_new, max_length, causal, window, scale, return_lse)
        return (out, lse) if return_lse else out
    module = _host or _module()
    if module is not None:
        got = module.kv_attend(q, cache, block_table, lengths, starts, max_new, max_length, bool(causal), window, scale, bool(return_lse))
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
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(tokens, heads, dtype=torch.float32, device=q.device) if return_lse else None
    lib = _lib.load()
    needed = lib.oq_kv_attend_workspace_bytes(tokens, heads, struct.kv_heads, dim, struct.page_size, table.shape[1], requests, starts is not None,
                                              window, max_length, max_new)
    workspace, nbytes, _keep = _workspace(needed, q, lambda: (0,))
    with _OnDevice(q):
        rc = lib.oq_kv_attend(q.data_ptr(), _dt(q), tokens, heads, q.stride(0), q.stride(1), ctypes.byref(struct), table.data_ptr(),
                              table.stride(0), table.shape[1], lengths.data_ptr(), _ptr(starts), requests, bool(causal), window, scale, max_length, max_new, out.data_ptr(), _ptr(lse),
                              workspace, nbytes, _stream(q))
    _lib.check(rc, "oq_kv_attend")
    return out if lse is None else (out, lse)
