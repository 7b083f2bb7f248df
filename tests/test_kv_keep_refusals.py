"""Caches that share memory are refused by `oq_kv_keep`; no GPU is needed to be refused.  (Two wavefronts of a launch would move the same entries, one of them what the
other has moved already.)"""

import itertools

import pytest

from orbitquant_amd import _lib
from test_kv_cache_refusals import _cache_struct
from test_kv_tree_refusals import INVALID, _keep

PARTS = ("k_codes", "k_scales", "v_codes", "v_scales")
APART = 1 << 20     # between parts that do not touch


def _layers(count):
    """Of the shapes of `_cache_struct`: 4 pages of 2 heads of 64 tokens of 128: 32 KiB of codes, 1 KiB of scales."""
    return [{part: APART * (1 + 4 * i + j) for j, part in enumerate(PARTS)} for i in range(count)]


def _refused(layers):
    assert _keep(*(_cache_struct(**layer) for layer in layers)) == INVALID
    return _lib.load().oq_last_error()


@pytest.mark.parametrize("part", PARTS)
@pytest.mark.parametrize("first,again", [(0, 1), (0, 3), (1, 2), (2, 3)])
def test_a_part_twice(part, first, again):
    layers = _layers(4)
    layers[again][part] = layers[first][part]
    assert b"cache" in _refused(layers)


@pytest.mark.parametrize("one,other", itertools.product(PARTS, PARTS))
def test_parts_that_overlap(one, other):
    """Of whatever kind they are, by their last and first sixteen bytes."""
    size = {"k_codes": 4 * 2 * 64 * 64, "v_codes": 4 * 2 * 64 * 64, "k_scales": 4 * 2 * 64 * 2, "v_scales": 4 * 2 * 64 * 2}
    layers = _layers(3)
    layers[2][other] = layers[0][one] + size[one] - 16
    _refused(layers)
    layers = _layers(3)
    layers[0][other] = layers[2][one] - size[other] + 16
    _refused(layers)


@pytest.mark.parametrize("one,other", itertools.combinations(PARTS, 2))
def test_parts_of_one_cache(one, other):
    layers = _layers(1)
    layers[0][one] = layers[0][other]
    _refused(layers)


def test_many_caches():
    """More than one launch takes; the two stand in different ones."""
    layers = _layers(130)
    layers[129]["v_scales"] = layers[3]["v_scales"]
    assert b"129" in _refused(layers)
