"""What norms and rotary positions, the append, and the operators of drafted trees refuse; no GPU is needed to be refused."""

import ctypes

import pytest
import torch

from orbitquant_amd import OrbitKVCache, QKNormRotary, _lib, kv_append, kv_attend, kv_keep, kv_tree, qk_norm_rotary
from test_kv_cache_refusals import BAD_CACHES, NOWHERE, _cache_struct

INVALID, UNSUPPORTED = 1, 2


def _plan(**kw):
    values = {"cos": NOWHERE, "sin": NOWHERE, "rows": 100, "rotary_dim": 64, "positions": NOWHERE, "q_weight": NOWHERE, "k_weight": NOWHERE, "weight_dtype": 2, "norm": 1,
              "eps": 1e-6, "interleaved": 0}
    return _lib.QkPlanStruct(**{**values, **kw})


def _rotary(plan=None, **kw):
    a = {"q": NOWHERE, "heads": 4, "k": NOWHERE, "kv_heads": 2, "dtype": 2, "tokens": 3, "dim": 128, "q_out": NOWHERE, "k_out": NOWHERE} | kw
    return _lib.load().oq_qk_norm_rotary(a["q"], 512, 128, a["heads"], a["k"], 256, 128, a["kv_heads"], a["dtype"], a["tokens"], a["dim"],
                                         None if plan == "none" else ctypes.byref(plan or _plan()), a["q_out"], a["k_out"], None)


def _append(plan=None, cache=None, **kw):
    a = {"q": NOWHERE, "heads": 4, "k": NOWHERE, "v": NOWHERE, "dtype": 2, "slots": NOWHERE, "tokens": 3, "q_out": NOWHERE} | kw
    return _lib.load().oq_kv_append(a["q"], 512, 128, a["heads"], a["k"], 256, 128, a["v"], 256, 128, a["dtype"], a["slots"], a["tokens"],
                                    None if plan == "none" else ctypes.byref(plan or _plan()), ctypes.byref(cache or _cache_struct()), a["q_out"], None)


@pytest.mark.parametrize("bad,status", [({"cos": None}, 1), ({"sin": None}, 1), ({"rotary_dim": 0}, 1), ({"rotary_dim": 7}, 1), ({"rotary_dim": 130}, 1), ({"rotary_dim": -2}, 1),
                                        ({"rows": -1}, 1), ({"rows": 1 << 31}, 2), ({"cos": NOWHERE + 2}, 1), ({"norm": 0}, 1), ({"weight_dtype": 3}, 1), ({"eps": -1e-6}, 1),
                                        ({"eps": float("nan")}, 1), ({"eps": float("inf")}, 1)])
def test_bad_plans(bad, status):
    assert _rotary(_plan(**bad)) == status and b"qk_norm_rotary" in _lib.load().oq_last_error()
    assert _append(_plan(**bad)) == status and b"kv_append" in _lib.load().oq_last_error()


@pytest.mark.parametrize("bad,status", [({"plan": "none"}, 1), ({"dtype": 3}, 1), ({"tokens": -1}, 1), ({"heads": 0}, 1), ({"kv_heads": 0}, 1), ({"heads": 65536}, 1), ({"dim": 0}, 1),
                                        ({"dim": 63}, 1), ({"dim": 514}, 2), ({"q": None}, 1), ({"k": None}, 1), ({"q_out": None}, 1), ({"k_out": None}, 1), ({"q_out": NOWHERE + 8}, 1),
                                        ({"k_out": NOWHERE + 2}, 1), ({"tokens": 1 << 30}, 2), ({"tokens": 1 << 20, "heads": 1024}, 2), ({"tokens": 1 << 20, "kv_heads": 1024}, 2)])
def test_bad_norms_and_rotations(bad, status):
    assert _rotary(**bad) == status


@pytest.mark.parametrize("bad,status", BAD_CACHES)
def test_bad_caches(bad, status):
    lib, cache = _lib.load(), _cache_struct(**bad)
    assert _append(cache=cache) == status
    assert _keep(cache) == status
    assert _keep(_cache_struct(), cache) != 0
    assert _attend_tree(cache=ctypes.byref(cache)) == status
    assert lib.oq_last_error()


@pytest.mark.parametrize("bad,status", [({"plan": "none"}, 1), ({"dtype": 5}, 1), ({"tokens": -1}, 1), ({"heads": 0}, 1), ({"q": None}, 1), ({"k": None}, 1), ({"v": None}, 1),
                                        ({"slots": None}, 1), ({"q_out": None}, 1), ({"q_out": NOWHERE + 4}, 1), ({"tokens": 1 << 40}, 2), ({"tokens": 1 << 28}, 2)])
def test_bad_appends(bad, status):
    assert _append(**bad) == status


def test_nothing_to_do():
    """No tokens: nothing is looked at, and nothing is launched."""
    assert _rotary(tokens=0, q=None, k=None) == 0 and _append(tokens=0, q=None, k=None, v=None, slots=None) == 0
    assert _tree(tokens=0, parents=None) == 0 and _keep(_cache_struct(), requests=0, **NO_PAGES) == 0 and _attend_tree(tokens=0, requests=0, q=None) == 0


def _tree(**kw):
    a = {"parents": NOWHERE, "starts": NOWHERE, "lengths": NOWHERE, "requests": 2, "tokens": 5, "words": 1, "positions": NOWHERE, "masks": NOWHERE} | kw
    return _lib.load().oq_kv_tree(a["parents"], a["starts"], a["lengths"], a["requests"], a["tokens"], a["words"], a["positions"], a["masks"], None)


@pytest.mark.parametrize("bad,status", [({"requests": -1}, 1), ({"tokens": -1}, 1), ({"words": 0}, 1), ({"words": 5}, 2), ({"tokens": 1 << 30}, 2), ({"requests": 1 << 24}, 2),
                                        ({"parents": None}, 1), ({"starts": None}, 1), ({"lengths": None}, 1), ({"positions": None}, 1), ({"masks": None}, 1), ({"masks": NOWHERE + 4}, 1)])
def test_bad_trees(bad, status):
    assert _tree(**bad) == status


def _attend_tree(**kw):
    a = {"q": NOWHERE, "tokens": 2, "heads": 4, "cache": ctypes.byref(_cache_struct()), "requests": 2, "masks": NOWHERE, "words": 1, "starts": None, "window": 0} | kw
    return _lib.load().oq_kv_attend_tree(a["q"], 2, a["tokens"], a["heads"], 512, 128, a["cache"], NOWHERE, 8, 8, NOWHERE, a["starts"], a["requests"], a["masks"], a["words"],
                                         a["window"], 1.0, -1, -1, NOWHERE, None, None, 0, None)


@pytest.mark.parametrize("bad,status", [({"words": 0}, 1), ({"words": 5}, 2), ({"masks": None}, 1), ({"masks": NOWHERE + 4}, 1), ({"heads": 3}, 1), ({"requests": 3}, 1), ({"q": None}, 1),
                                        ({"window": -1}, 1), ({"tokens": 1 << 30, "requests": 1 << 30}, 2)])
def test_bad_attention(bad, status):
    assert _attend_tree(**bad) == status


def _keep(*caches, **kw):
    a = {"kept": NOWHERE, "most": 3, "lengths": NOWHERE, "starts": NOWHERE, "slots": NOWHERE, "requests": 2, "tokens": 5, "count": len(caches), "table": NOWHERE, "stride": 4, "width": 4,
         "free": NOWHERE, "free_count": 9, "taken": NOWHERE, "after": NOWHERE, "taken_after": NOWHERE} | kw
    structs = (_lib.KvCacheStruct * max(1, len(caches)))(*caches)
    return _lib.load().oq_kv_keep(a["kept"], a["most"], a["lengths"], a["starts"], a["slots"], a["requests"], a["tokens"], structs if caches else None, a["count"], a["table"],
                                  a["stride"], a["width"], a["free"], a["free_count"], a["taken"], a["after"], a["taken_after"], None)


NO_PAGES = {"table": None, "free": None, "free_count": 0, "taken": None, "taken_after": None}


@pytest.mark.parametrize("bad,status", [({"most": -1}, 1), ({"most": 257}, 2), ({"requests": -1}, 1), ({"requests": 8193}, 2), ({"tokens": -1}, 1), ({"tokens": 1 << 30}, 2), ({"count": 0}, 1),
                                        ({"stride": 3}, 1), ({"width": -1}, 1), ({"free_count": -1}, 1), ({"kept": None}, 1), ({"lengths": None}, 1), ({"starts": None}, 1), ({"slots": None}, 1),
                                        ({"after": None}, 1), ({"taken": None}, 1), ({"taken_after": None}, 1), ({"free": None}, 1), ({"table": None}, 1)])
def test_bad_paths(bad, status):
    assert _keep(_cache_struct(), **bad) == status


@pytest.mark.parametrize("other", [{"pages": 5}, {"kv_heads": 3}, {"page_size": 32}, {"head_dim": 64}])
def test_caches_of_different_shapes(other):
    assert _keep(_cache_struct(), _cache_struct(**other)) == INVALID


@pytest.mark.parametrize("first,again", [(0, 1), (0, 3), (1, 2), (2, 3)])
def test_a_cache_twice(first, again):
    """Two wavefronts would move the same entries, one of them what the other has moved already."""
    layers = [_cache_struct(k_codes=NOWHERE + 4096 * i) for i in range(4)]
    layers[again] = layers[first]
    assert _keep(*layers) == INVALID and b"cache %d is cache %d again" % (again, first) in _lib.load().oq_last_error()


def test_python_refuses_the_host():
    """Tensors on the host, and what is wrong whatever they are on."""
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    cache = OrbitKVCache.empty(2, 2, 64, page_size=16, device="cpu")
    slots = torch.arange(3)
    i32 = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: qk_norm_rotary(q, k, QKNormRotary()), lambda: kv_append(q, k, k, slots, cache, QKNormRotary()), lambda: kv_tree(i32, i32[:2], i32[:1]),
                 lambda: kv_keep(i32[:2, None], i32[:2], i32, slots, [cache])):
        with pytest.raises(RuntimeError, match="AMD GPU"):
            call()
    for max_new in (0, 257, -1):
        with pytest.raises(ValueError, match="max_new"):
            kv_tree(i32, i32[:2], i32[:1], max_new=max_new)
    with pytest.raises(ValueError, match="at least one layer"):
        kv_keep(i32[:2, None], i32[:2], i32, slots, [])
    with pytest.raises(ValueError, match="go together"):
        kv_keep(i32[:2, None], i32[:2], i32, slots, [cache], taken=i32[:1])
    with pytest.raises(ValueError, match="masks need causal"):
        kv_attend(q, cache, i32[:, None], i32, masks=torch.zeros(3, 1, dtype=torch.int64), causal=False)
