"""Steps that hold drafted trees and prompts: the trees' accepted paths stay, and of the prompts everything."""

import numpy as np
import pytest
import torch

import kv_oracle
from test_gpu_kv_cache import _cache, _i32, _queries
from test_gpu_kv_tree import _parents
from test_gpu_qk_rotary import _how

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.mark.parametrize("words", [1, 4])
def test_trees_beside_prompts(words):
    """Prompts of 300 and 70 tokens (one longer than any list, one shorter) before, between and behind trees: each request goes on as it would alone, and no page is
    lost."""
    from orbitquant_amd import KEEP_ALL, kv_append, kv_assign, kv_attend, kv_keep, kv_tree

    rng = np.random.RandomState(words)
    before, new = [5, 40, 0, 17, 33], [300, 9, 70, 13, 290]
    whole = [True, False, True, False, True]
    pages, width = 80, 24
    table = torch.full((5, width), -1, dtype=torch.int32, device="cuda")
    free = _i32(rng.permutation(pages).tolist())
    cache = _cache(pages, 2, 64, PAGE, fill=0xFF)
    how = _how(rng, 64, 64, False, "weights")
    got = kv_assign(_i32([0] * 5), _i32(before), table, free, _i32([0]), page_size=PAGE, tokens=sum(before))
    q, k, v = (_queries(rng, sum(before), h, 64, torch.bfloat16) for h in (4, 2, 2))
    kv_append(q, k, v, got.slots, cache, how, got.positions)
    step = kv_assign(got.lengths, _i32(new), table, free, got.taken, page_size=PAGE, tokens=sum(new))
    tree = kv_tree(_i32(_parents(rng, new, "chain")), step.starts, step.lengths, max_new=64 * words)
    q, k, v = (_queries(rng, sum(new), h, 64, torch.bfloat16) for h in (4, 2, 2))
    q = kv_append(q, k, v, step.slots, cache, how, tree.positions)
    kv_attend(q, cache, table, step.lengths, starts=step.starts, masks=tree.masks)
    was = kv_oracle.cache_codes(cache)
    rows = [[KEEP_ALL, -1, -1], [0, 3, 8], [KEEP_ALL, 0, 1], [0, -1, -1], [KEEP_ALL, -1, -1]]
    kept = kv_keep(_i32(rows), step.lengths, step.starts, step.slots, [cache], block_table=table, free_pages=free, taken=step.taken)
    want = [b + n if all_ else b + sum(x >= 0 for x in row) for b, n, all_, row in zip(before, new, whole, rows)]
    assert kept.lengths.tolist() == want
    held = [p for row, n in zip(table.tolist(), want) for p in row[:-(-n // PAGE)]]
    assert sorted(held + free[int(kept.taken):].tolist()) == list(range(pages))
    slots, first = step.slots.tolist(), step.starts.tolist()[1]
    moves = {slots[first + 1]: slots[first + 3], slots[first + 2]: slots[first + 8]}
    for x, y in zip(kv_oracle.cache_codes(cache), was):
        y = y.copy()
        fresh = {to: y[source // PAGE, :, source % PAGE].copy() for to, source in moves.items()}
        for to, z in fresh.items():
            y[to // PAGE, :, to % PAGE] = z
        np.testing.assert_array_equal(x.view(np.int32) if x.dtype == np.float32 else x, y.view(np.int32) if y.dtype == np.float32 else y)


def test_all_of_a_request_that_has_no_page():
    """A request that stays as the step left it keeps its length whatever its slots are, and of its pages none comes back."""
    from orbitquant_amd import KEEP_ALL, kv_assign, kv_keep

    cache = _cache(6, 1, 64, PAGE)
    was = cache.k_codes.clone()
    for before, new, width, pages in (([0, 3], [90, 40], 8, 6), ([60, 10], [30, 9], 4, 12), ([-5, 0], [3, 0], 2, 4)):
        table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
        free = _i32(list(range(pages)))
        got = kv_assign(_i32(before), _i32(new), table, free, _i32([0]), page_size=PAGE, tokens=sum(new))
        for rows in ([[KEEP_ALL]] * 2, torch.full((2, 70), KEEP_ALL).tolist()):
            kept = kv_keep(_i32(rows), got.lengths, got.starts, got.slots, [cache], block_table=table, free_pages=free, taken=got.taken)
            assert torch.equal(kept.lengths, got.lengths) and torch.equal(kept.taken, got.taken) and free.tolist() == list(range(pages))
    assert torch.equal(cache.k_codes, was)


def test_behind_other_entries_the_mark_ends_the_list():
    from orbitquant_amd import KEEP_ALL, kv_keep

    cache = _cache(2, 1, 64, PAGE)
    slots = torch.arange(5, device="cuda")
    got = kv_keep(_i32([[0, KEEP_ALL, 2], [-3, KEEP_ALL, -1]]), _i32([7, 9]), _i32([0, 3, 5]), slots, [cache])
    assert got.lengths.tolist() == [5, 7]
