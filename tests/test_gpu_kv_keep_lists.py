"""`kv_keep`: lists that name what has no place to go, and caches whose parts touch."""

import numpy as np
import pytest
import torch

import kv_oracle
from test_gpu_kv_cache import _cache, _i32

pytestmark = pytest.mark.gpu


def _random(cache):
    for t in cache[:4]:
        t.view(torch.uint8).random_(0, 255)
    return cache


def _check_moves(caches, was, moves, page):
    for c, old in zip(caches, was):
        for x, y in zip(kv_oracle.cache_codes(c), old):
            want = y.copy()
            for source, to in moves:
                want[to // page, :, to % page] = y[source // page, :, source % page]
            np.testing.assert_array_equal(x.view(np.int32) if x.dtype == np.float32 else x, want.view(np.int32) if want.dtype == np.float32 else want)


@pytest.mark.parametrize("slots,kept,count,moves", [
    ([-1, 5, 6], [1, 2], 0, []),                                        # the first has nowhere to go
    ([-1, 5, 6], [0, 1], 0, []),
    ([3, -1, 5, 6], [0, 2, 3], 1, []),                                  # the second
    ([3, 4, -1, 6, 7], [1, 3, 4], 2, [(4, 3), (6, 4)]),
    ([3, 4, 10 ** 9, 6, 7], [1, 3, 4], 2, [(4, 3), (6, 4)]),            # (a slot that the cache does not have)
    ([3, 4, 5, 6, 7], [1, 3, 4], 3, [(4, 3), (6, 4), (7, 5)]),
    ([3, 4, 5, 6, -1], [1, 3, 4], 2, [(4, 3), (6, 4)]),
])
def test_an_entry_without_a_place_to_go_ends_the_list(slots, kept, count, moves):
    """The length stands for entries that are there: a token that cannot move is not kept."""
    from orbitquant_amd import kv_keep

    caches = [_random(_cache(2, 3, 64, 16)) for _ in range(2)]
    was = [kv_oracle.cache_codes(c) for c in caches]
    n = len(slots)
    got = kv_keep(_i32([kept, kept]), _i32([6 + n, 9]), _i32([0, n, n]), torch.tensor(slots, device="cuda"), caches)
    assert got.lengths.tolist() == [6 + count, 9]
    _check_moves(caches, was, moves, 16)


def test_a_long_list_that_ends_behind_its_first_batch():
    """Places without a page behind the 64th entry of a list, and pages behind them back on the list."""
    from orbitquant_amd import kv_keep

    rng = np.random.RandomState(1)
    for hole in (63, 64, 65, 90):
        cache = _random(_cache(16, 1, 64, 16))
        was = [kv_oracle.cache_codes(cache)]
        slots = rng.permutation(256)[:200]
        slots[hole] = -1
        kept = sorted(rng.permutation(np.delete(np.arange(200), [hole]))[:100].tolist())
        table = _i32([list(range(16))])
        free = _i32(list(range(16, 40)))
        got = kv_keep(_i32([kept]), _i32([230]), _i32([0, 200]), torch.from_numpy(slots).cuda(), [cache], block_table=table, free_pages=free, taken=_i32([20]))
        assert got.lengths.tolist() == [30 + hole] and got.taken.tolist() == [20 - (-(-230 // 16) - -(-(30 + hole) // 16))]
        _check_moves([cache], was, [(int(slots[k]), int(slots[i])) for i, k in enumerate(kept[:hole])], 16)


def test_caches_side_by_side():
    """Layers that are parts of one tensor touch, and do not overlap."""
    from orbitquant_amd import OrbitKVCache, kv_keep

    whole = _random(_cache(12, 2, 64, 16))
    layers = [OrbitKVCache(*(t[4 * i:4 * i + 4] for t in whole[:4]), whole.signs) for i in range(3)]
    was = [kv_oracle.cache_codes(c) for c in layers]
    got = kv_keep(_i32([[0, 2]]), _i32([9]), _i32([0, 3]), torch.tensor([20, 21, 40], device="cuda"), layers)
    assert got.lengths.tolist() == [8]
    _check_moves(layers, was, [(40, 21)], 16)


def test_caches_that_share_a_part_are_refused():
    from orbitquant_amd import kv_keep

    one, other = _cache(4, 2, 64, 16), _cache(4, 2, 64, 16)
    slots = torch.tensor([20, 21, 40], device="cuda")
    for at in range(4):
        shared = other._replace(**{one._fields[at]: one[at]})
        for caches in ([one, shared], [_cache(4, 2, 64, 16), one, _cache(4, 2, 64, 16), shared]):
            with pytest.raises(ValueError, match="cache"):
                kv_keep(_i32([[0, 2]]), _i32([9]), _i32([0, 3]), slots, caches)
