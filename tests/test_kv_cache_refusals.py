"""What the key/value cache's entry points refuse; no GPU is needed to be refused."""

import ctypes

import pytest
import torch

from orbitquant_amd import OrbitKVCache, _lib, kv_assign, kv_attend, kv_read, kv_write

NOWHERE = 0x1000   # an address that no refused call looks at


def _cache_struct(**kw):
    values = {"k_codes": NOWHERE, "k_scales": NOWHERE, "v_codes": NOWHERE, "v_scales": NOWHERE, "signs": NOWHERE, "pages": 4, "kv_heads": 2,
              "page_size": 64, "head_dim": 128}
    return _lib.KvCacheStruct(**{**values, **kw})


BAD_CACHES = [({"head_dim": 96}, 2), ({"head_dim": 0}, 2), ({"page_size": 48}, 2), ({"page_size": 8}, 2), ({"page_size": 2048}, 2), ({"page_size": 0}, 2),
              ({"pages": 0}, 1), ({"pages": 1 << 31}, 1), ({"kv_heads": 0}, 1), ({"kv_heads": 65536}, 1), ({"k_codes": None}, 1), ({"v_scales": None}, 1),
              ({"signs": None}, 1), ({"k_codes": NOWHERE + 8}, 1), ({"v_codes": NOWHERE + 4}, 1), ({"signs": NOWHERE + 1}, 1)]


@pytest.mark.parametrize("bad,status", BAD_CACHES)
def test_bad_caches(bad, status):
    lib = _lib.load()
    cache = ctypes.byref(_cache_struct(**bad))
    assert lib.oq_kv_write(NOWHERE, 256, 128, NOWHERE, 256, 128, 2, NOWHERE, 1, cache, None) == status
    assert lib.oq_kv_read(NOWHERE, 1, cache, NOWHERE, NOWHERE, 2, None) == status
    assert _attend(lib, cache=cache) == status
    assert b"kv_attend" in lib.oq_last_error()


def _attend(lib, **kw):
    a = {"q": NOWHERE, "dtype": 2, "tokens": 2, "heads": 4, "ts": 512, "hs": 128, "cache": ctypes.byref(_cache_struct()), "table": NOWHERE, "stride": 8,
         "width": 8, "lengths": NOWHERE, "starts": None, "requests": 2, "causal": 1, "window": 0, "out": NOWHERE, "ws": None} | kw
    return lib.oq_kv_attend(a["q"], a["dtype"], a["tokens"], a["heads"], a["ts"], a["hs"], a["cache"], a["table"], a["stride"], a["width"], a["lengths"],
                            a["starts"], a["requests"], a["causal"], a["window"], 1.0, -1, -1, a["out"], None, a["ws"], 0, None)


@pytest.mark.parametrize("bad,status", [
    ({"dtype": 3}, 1), ({"tokens": -1}, 1), ({"heads": 3}, 1), ({"heads": 0}, 1), ({"requests": 3}, 1), ({"requests": -1}, 1), ({"window": -1}, 1),
    ({"window": 5, "causal": 0}, 1), ({"stride": 7}, 1), ({"width": -1}, 1), ({"q": None}, 1), ({"out": None}, 1), ({"lengths": None}, 1),
    ({"table": None}, 1), ({"out": NOWHERE + 8}, 1), ({"ws": NOWHERE + 8}, 1), ({"tokens": 1 << 30, "requests": 1 << 30}, 2),
    ({"width": 1 << 25, "stride": 1 << 25}, 2), ({"heads": 65536}, 2)])
def test_bad_attention(bad, status):
    assert _attend(_lib.load(), **bad) == status


@pytest.mark.parametrize("bad,status", [({"page": 24}, 2), ({"requests": 8193}, 2), ({"requests": -1}, 1), ({"tokens": -1}, 1), ({"stride": 3}, 1),
                                        ({"free": -1}, 1), ({"lengths": None}, 1), ({"table": None}, 1), ({"taken": None}, 1), ({"slots": None}, 1)])
def test_bad_assignments(bad, status):
    a = {"lengths": NOWHERE, "requests": 2, "table": NOWHERE, "stride": 4, "width": 4, "free": 3, "taken": NOWHERE, "page": 16, "tokens": 2,
         "slots": NOWHERE} | bad
    assert _lib.load().oq_kv_assign(a["lengths"], NOWHERE, a["requests"], a["table"], a["stride"], a["width"], NOWHERE, a["free"], a["taken"], a["page"],
                                    a["tokens"], a["slots"], NOWHERE, NOWHERE, NOWHERE, NOWHERE, None) == status


def test_bad_writes_and_reads():
    lib, cache = _lib.load(), ctypes.byref(_cache_struct())
    write = lambda k=NOWHERE, dtype=2, slots=NOWHERE, tokens=1: lib.oq_kv_write(k, 256, 128, NOWHERE, 256, 128, dtype, slots, tokens, cache, None)  # noqa: E731
    assert write(k=None) == write(dtype=7) == write(slots=None) == write(tokens=-1) == 1 and write(tokens=1 << 41) == 2 and write(tokens=0) == 0
    read = lambda slots=NOWHERE, tokens=1, k=NOWHERE, dtype=2: lib.oq_kv_read(slots, tokens, cache, k, NOWHERE, dtype, None)  # noqa: E731
    assert read(slots=None) == read(k=None) == read(k=NOWHERE + 2) == read(dtype=-1) == read(tokens=-1) == 1 and read(tokens=0) == 0
    assert lib.oq_kv_write(NOWHERE, 256, 128, NOWHERE, 256, 128, 2, NOWHERE, 1, None, None) == 1


def test_workspace_sizes():
    """None where there is nothing to cut, and nothing for what the call refuses."""
    size = _lib.load().oq_kv_attend_workspace_bytes
    assert size(1, 32, 8, 128, 64, 2048, 1, 0, 0, -1, -1) > 0
    assert size(1, 32, 8, 128, 64, 2048, 1, 0, 0, 100, -1) == 0          # two steps of keys
    assert size(8192, 32, 8, 128, 64, 128, 1, 1, 0, -1, 8192) == 0       # rows enough
    assert size(0, 32, 8, 128, 64, 2048, 0, 0, 0, -1, -1) == 0
    assert size(1, 32, 7, 128, 64, 2048, 1, 0, 0, -1, -1) == size(1, 32, 8, 100, 64, 2048, 1, 0, 0, -1, -1) == size(1, 32, 8, 128, 60, 2048, 1, 0, 0, -1, -1) == 0


def test_tensors_on_the_host_are_refused():
    cache = OrbitKVCache.empty(2, 2, 64, page_size=16, device="cpu")
    assert (cache.pages, cache.heads, cache.page_size, cache.head_dim) == (2, 2, 16, 64)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    slots, i32 = torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: kv_write(x, x, slots, cache), lambda: kv_read(slots, cache), lambda: kv_attend(x, cache, i32.view(1, 1), i32),
                 lambda: kv_assign(i32, i32, i32.view(1, 1), i32, i32, page_size=16, tokens=1)):
        with pytest.raises(RuntimeError, match="must live on an AMD GPU"):
            call()


@pytest.mark.parametrize("kw", [{"head_dim": 72}, {"page_size": 20}, {"page_size": 8}, {"pages": 0}, {"heads": 0}])
def test_caches_that_cannot_be_made(kw):
    with pytest.raises(ValueError):
        OrbitKVCache.empty(**{"pages": 2, "heads": 2, "head_dim": 64, "device": "cpu", **kw})


@pytest.mark.gpu
def test_operands_that_do_not_fit():
    cache = OrbitKVCache.empty(4, 2, 64, page_size=16)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    i32 = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    other = OrbitKVCache(cache.k_codes.transpose(0, 1), *cache[1:])
    for bad in (lambda: kv_write(x[:, :1], x[:, :1], slots, cache), lambda: kv_write(x, x[:2], slots, cache), lambda: kv_write(x, x.float(), slots, cache),
                lambda: kv_write(x, x, slots.int(), cache), lambda: kv_write(x, x, slots[:2], cache), lambda: kv_write(x, x, slots.cpu(), cache),
                lambda: kv_write(x, x, slots, other), lambda: kv_write(x.double(), x.double(), slots, cache),
                lambda: kv_write(x, x, slots, OrbitKVCache(cache[0], cache[1].float(), *cache[2:])), lambda: kv_read(slots.int(), cache),
                lambda: kv_read(slots, cache, torch.float64), lambda: kv_attend(x[:, :, :32], cache, table, i32),
                lambda: kv_attend(torch.zeros(3, 3, 64, device="cuda"), cache, table, i32), lambda: kv_attend(x, cache, table.long(), i32),
                lambda: kv_attend(x, cache, table[:2], i32), lambda: kv_attend(x, cache, table.t(), i32), lambda: kv_attend(x, cache, table, i32.long()),
                lambda: kv_attend(x, cache, table[:2], i32[:2]), lambda: kv_attend(x, cache, table, i32, starts=i32), lambda: kv_attend(x, cache, table, i32, window=0),
                lambda: kv_attend(x, cache, table, i32, window=3, causal=False), lambda: kv_assign(i32, i32[:2], table, i32, i32[:1], page_size=16, tokens=3),
                lambda: kv_assign(i32, i32, table[:, ::2], i32, i32[:1], page_size=16, tokens=3), lambda: kv_assign(i32, i32, table, i32, i32, page_size=16, tokens=3),
                lambda: kv_assign(i32, i32, table, i32.cpu(), i32[:1], page_size=16, tokens=3), lambda: kv_assign(i32, i32, table, i32, i32[:1], page_size=16, tokens=-1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.OrbitQuantHipError, match="page_size"):
        kv_assign(i32, i32, table, i32, i32[:1], page_size=17, tokens=3)
