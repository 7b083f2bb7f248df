"""Sizes whose launches the runtime cannot make (2^32 threads and more) are refused as such, before anything is launched; no GPU is needed."""

import ctypes

import pytest

from orbitquant_amd import _lib
from test_kv_cache_refusals import NOWHERE, _attend, _cache_struct

UNSUPPORTED = 2


@pytest.mark.parametrize("dim,heads,write_threads", [(64, 1, 128), (64, 7, 128), (128, 1, 256), (128, 8, 256), (256, 3, 256), (256, 65535, 256)])
def test_writes_and_reads(dim, heads, write_threads):
    """A workgroup has one head of sixteen tokens."""
    lib, cache = _lib.load(), ctypes.byref(_cache_struct(head_dim=dim, kv_heads=heads))
    most = lambda threads: ((1 << 32) - 1) // (threads * heads) * 16   # tokens  # noqa: E731
    for tokens in (most(write_threads) + 1, 2 * most(write_threads), 1 << 40):
        assert lib.oq_kv_write(NOWHERE, dim, dim, NOWHERE, dim, dim, 2, NOWHERE, tokens, cache, None) == UNSUPPORTED
        assert b"kv_write" in lib.oq_last_error() and str(tokens).encode() in lib.oq_last_error()
    for tokens in (most(256) + 1, 1 << 40):
        assert lib.oq_kv_read(NOWHERE, tokens, cache, NOWHERE, NOWHERE, 2, None) == UNSUPPORTED
        assert b"kv_read" in lib.oq_last_error()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens(dim):
    lib, cache = _lib.load(), ctypes.byref(_cache_struct(head_dim=dim))
    requests = 1 << 23                                              # two key heads, 256 threads for each request and head
    size = lambda requests: lib.oq_kv_attend_workspace_bytes(requests, 4, 2, dim, 64, 100, requests, 0, 0, -1, -1)  # noqa: E731
    assert _attend(lib, cache=cache, tokens=requests, requests=requests, stride=100, width=100) == UNSUPPORTED and b"kv_attend" in lib.oq_last_error()
    assert size(requests) == 0 and size(requests - 2000) > 0        # (a workspace is asked for where requests are cut: of what is refused, none)


@pytest.mark.parametrize("dim,threads", [(64, 256), (128, 256), (256, 512)])
def test_prompts(dim, threads):
    """One request of many tokens, 128 rows a workgroup; 65535 heads that share nothing."""
    lib, cache = _lib.load(), ctypes.byref(_cache_struct(head_dim=dim, kv_heads=65535))
    tiles = (1 << 32) // threads // 65535 + 1
    tokens = tiles * 128
    if tokens * 65535 <= 0x7fffffff:
        assert _attend(lib, cache=cache, tokens=tokens, heads=65535, starts=NOWHERE, requests=1, width=1, stride=1) == UNSUPPORTED
    assert _attend(lib, cache=cache, tokens=0x7fffffff // 65535, heads=65535, starts=NOWHERE, requests=100, width=1, stride=1) == UNSUPPORTED
