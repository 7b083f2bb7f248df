"""Trees of drafted tokens over the 4-bit cache against their definitions: positions and masks, the attention under masks, the accepted path, and
a run of all of them as a program that drafts uses them."""

import numpy as np
import pytest
import torch

import kv_oracle
import tree_oracle as oracle
from test_gpu_kv_cache import DTYPES, _cache, _filled, _i32, _queries

pytestmark = pytest.mark.gpu


def _starts(new):
    return np.concatenate(([0], np.cumsum(new))).astype(int).tolist()


def _masks(rows):
    return torch.tensor(oracle.signed(rows), dtype=torch.int64, device="cuda")


# ---------------------------------------------------------------- positions and masks

def _parents(rng, counts, kind):
    parents = []
    for n in counts:
        if kind == "chain":
            parents += list(range(-1, n - 1))
        elif kind == "roots":
            parents += [-1] * n
        elif kind == "random":
            parents += [int(rng.randint(-1, i)) if i else -1 for i in range(n)]
        else:   # anything: behind the token, itself, far away
            parents += rng.choice([-1, -100, 0, 1, 2, 5, 63, 64, 255, 256, 10 ** 6, 2 ** 31 - 1, -2 ** 31], n).tolist()
    return parents


@pytest.mark.parametrize("kind", ["chain", "roots", "random", "anything"])
@pytest.mark.parametrize("max_new", [1, 64, 65, 192, 256])
def test_tree(kind, max_new):
    from orbitquant_amd import kv_tree

    rng = np.random.RandomState(max_new)
    counts = [1, 0, 2, 63, 64, 65, 7, 128, 191, 0, 256, 300, 1]
    starts = _starts(counts)
    tokens = starts[-1] + 5                     # five tokens of no request
    lengths = [n + int(rng.randint(0, 50)) for n in counts]
    lengths[3] = 10                             # fewer tokens than new ones
    lengths[6] = -4
    parents = _parents(rng, counts, kind) + [0] * 5
    words = -(-max_new // 64)
    want, masks = oracle.tree(parents, starts, lengths, words, tokens)
    got = kv_tree(_i32(parents), _i32(starts), _i32(lengths), max_new=max_new)
    assert got.positions.tolist() == want and got.masks.tolist() == oracle.signed(masks)


def test_tree_edges():
    from orbitquant_amd import kv_tree

    none = torch.empty(0, dtype=torch.int32, device="cuda")
    got = kv_tree(none, _i32([0]), none)
    assert got.positions.shape == (0,) and got.masks.shape == (0, 1)
    got = kv_tree(_i32([3, 3]), _i32([0]), none)
    assert got.positions.tolist() == [-1, -1] and got.masks.tolist() == [[0], [0]]
    # starts that do not fit are cut to the tokens that there are
    got = kv_tree(_i32([-1, 0, 1]), _i32([-5, 2, 99]), _i32([10, 10]), max_new=64)
    assert got.positions.tolist() == [8, 9, 9] and got.masks.tolist() == [[1], [3], [1]]


@pytest.mark.parametrize("requests", [257, 5000])
def test_tree_many_requests(requests):
    from orbitquant_amd import kv_tree

    rng = np.random.RandomState(requests)
    counts = rng.randint(0, 20, requests).tolist()
    starts, lengths = _starts(counts), [n + int(rng.randint(0, 9)) for n in counts]
    parents = _parents(rng, counts, "random")
    want, masks = oracle.tree(parents, starts, lengths, 1, starts[-1])
    got = kv_tree(_i32(parents), _i32(starts), _i32(lengths))
    assert got.positions.tolist() == want and got.masks.tolist() == masks


# ---------------------------------------------------------------- attention

def _check(got, q, cache, table, lengths, starts, masks, window=None, scale=None):
    out, lse = got
    want, want_lse, bound = oracle.attend(q, cache, table, lengths, starts, masks, window, scale)
    far, far_lse = kv_oracle.allowed(bound, want, q.dtype)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    broken, empty = np.isnan(want).any(-1), np.isneginf(want_lse)
    np.testing.assert_array_equal(np.isnan(out).any(-1), broken)
    assert (out[empty] == 0).all() and np.isneginf(lse[empty]).all()
    fine = ~broken & ~empty
    off = np.linalg.norm(out - want, axis=-1)[fine]
    assert (off <= far[fine]).all(), (off / far[fine]).max()
    off = np.abs(lse[fine] - want_lse[fine])
    assert (off <= far_lse[fine]).all(), (off / far_lse[fine]).max()


def _random_masks(rng, counts, words, tokens):
    """Of every kind: paths, single bits, none, all, bits of tokens that the request does not have."""
    rows = oracle.tree(_parents(rng, counts, "random"), _starts(counts), [10 ** 6] * len(counts), words, tokens)[1]
    for i in range(tokens):
        pick = rng.randint(8)
        if pick == 0:
            rows[i] = [0] * words
        elif pick == 1:
            rows[i] = [2 ** 64 - 1] * words
        elif pick == 2:
            rows[i] = [int(rng.randint(0, 2 ** 62)) for _ in range(words)]
    return rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 4, 16), (128, 1, 6, 64), (128, 2, 1, 32), (256, 1, 2, 64), (128, 1, 17, 1024)])
@pytest.mark.parametrize("window", [None, 1, 5, 50])
def test_attend_masks(dim, heads, group, page, window, dtype):
    """Trees behind cached tokens and on their own, of one token and of a hundred and more, a request without new ones, rows that see nothing, tokens of
    no request; few rows and many in one call."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(dim + group)
    new, before = [60, 1, 13, 0, 5, 9, 64, 70], [130, 40, 0, 33, 64, 59, 3, 200]
    lengths = [a + b for a, b in zip(new, before)]
    cache, table = _filled(rng, lengths, heads, dim, page)
    starts = _starts(new)
    tokens = starts[-1] + 3
    q = _queries(rng, tokens, heads * group, dim, dtype)
    for words in (1, 2):                    # with one word the last request is a prompt
        masks = _random_masks(rng, new, words, tokens)
        for max_new in (None, 70, 1):
            got = kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), masks=_masks(masks), window=window, max_new=max_new, return_lse=True)
            _check(got, q, cache, table, lengths, starts, masks, window)


@pytest.mark.parametrize("dim,page,dtype", [(64, 16, torch.float16), (128, 64, torch.bfloat16), (256, 128, torch.float32)])
@pytest.mark.parametrize("window", [None, 3, 700])
def test_attend_masks_long(dim, page, dtype, window):
    """Contexts that are cut into parts: trees of few rows and of many, alone and in a batch, the widest of 250 tokens, at every place in a step of keys."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(dim)
    for new, before in (([5], [2000]), ([250], [1100]), ([3, 100, 1, 7], [1500, 2200, 1029, 8]), ([2] * 9, [1024 + 7 * i for i in range(9)])):
        lengths, starts = [a + b for a, b in zip(new, before)], _starts(new)
        cache, table = _filled(rng, lengths, 2, dim, page)
        q = _queries(rng, starts[-1], 4, dim, dtype)
        masks = _random_masks(rng, new, 4, starts[-1])
        got = kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), masks=_masks(masks), window=window, max_new=max(new), max_length=max(lengths),
                        return_lse=True)
        _check(got, q, cache, table, lengths, starts, masks, window)
        # and without the hints, cut otherwise
        got = kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), masks=_masks(masks), window=window, return_lse=True)
        _check(got, q, cache, table, lengths, starts, masks, window)


@pytest.mark.parametrize("dim,page,dtype", [(64, 64, torch.bfloat16), (128, 16, torch.float16), (256, 64, torch.float32)])
def test_hints_and_windows_of_any_size(dim, page, dtype):
    """Wrong hints cost time only, windows may be longer than anything, and a call gives the same bits every time."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(14)
    new, before = [40, 2, 90], [1300, 0, 2]
    lengths, starts = [a + b for a, b in zip(new, before)], _starts(new)
    cache, table = _filled(rng, lengths, 2, dim, page)
    q = _queries(rng, starts[-1], 6, dim, dtype)
    masks = _random_masks(rng, new, 2, starts[-1])
    call = lambda **kw: kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), masks=_masks(masks), return_lse=True, **kw)  # noqa: E731
    for hints in ({"max_length": 1}, {"max_length": 10 ** 6, "max_new": 10 ** 6}, {"max_length": 0, "max_new": 0}, {"max_new": 3, "max_length": 1300}):
        _check(call(**hints), q, cache, table, lengths, starts, masks)
    for window in (1341, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
        _check(call(window=window), q, cache, table, lengths, starts, masks, window)
    first = call(max_new=90)
    for _ in range(5):
        for a, b in zip(first, call(max_new=90)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("before", [[1500, 900], [5500, 900]])     # whole by themselves; cut where there is a workspace
def test_attend_masks_without_workspace(before, dtype):
    """The library's call without a workspace leaves requests whole; with less than it asks for, too."""
    import ctypes

    from orbitquant_amd import _lib, kv_cache

    rng = np.random.RandomState(15)
    new = [30, 70]
    lengths, starts = [a + b for a, b in zip(new, before)], _starts(new)
    cache, table = _filled(rng, lengths, 2, 64, 64)
    q = _queries(rng, 100, 4, 64, dtype)
    masks = _random_masks(rng, new, 2, 100)
    held = [_i32(lengths), _i32(starts), _masks(masks), torch.empty(1024, dtype=torch.uint8, device="cuda")]
    lib, struct = _lib.load(), kv_cache._cache_struct(cache, q)
    shape = (100, 4, 2, 64, 64, table.shape[1], 2, 1)
    needed = lib.oq_kv_attend_tree_workspace_bytes(kv_cache._dt(q), *shape, 2, 0, -1, 70)
    assert needed == 0 if before[0] == 1500 else needed > 1024
    for workspace, size in ((None, 0), (held[3].data_ptr(), 1024)):
        out, lse = torch.empty_like(q), torch.empty(100, 4, device="cuda")
        rc = lib.oq_kv_attend_tree(q.data_ptr(), kv_cache._dt(q), 100, 4, q.stride(0), q.stride(1), ctypes.byref(struct), table.data_ptr(), table.stride(0), table.shape[1],
                                   held[0].data_ptr(), held[1].data_ptr(), 2, held[2].data_ptr(), 2, 0, 0.125, -1, 70, out.data_ptr(), lse.data_ptr(), workspace, size,
                                   kv_cache._stream(q))
        assert rc == 0
        _check((out, lse), q, cache, table, lengths, starts, masks, scale=0.125)


def test_a_chain_is_causal_attention():
    """Masks of chains see what no masks see.  (Not bit for bit: the two may be launched otherwise, and then add up in another order.  So both are held
    to the bound of the same definition.)"""
    from orbitquant_amd import kv_attend, kv_tree

    rng = np.random.RandomState(8)
    new, before = [1, 30, 64, 7, 200], [900, 70, 0, 1500, 100]
    lengths, starts = [a + b for a, b in zip(new, before)], _starts(new)
    cache, table = _filled(rng, lengths, 2, 128, 64)
    q = _queries(rng, starts[-1], 8, 128, torch.bfloat16)
    tree = kv_tree(_i32(_parents(rng, new, "chain")), _i32(starts), _i32(lengths), max_new=200)
    positions = np.concatenate([np.arange(b, b + n) for b, n in zip(before, new)])
    assert tree.positions.tolist() == positions.tolist()
    masks = oracle.tree(_parents(rng, new, "chain"), starts, lengths, 4, starts[-1])[1]
    for got in (kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), masks=tree.masks, return_lse=True),
                kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), return_lse=True)):
        _check(got, q, cache, table, lengths, starts, masks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_query_a_request(dtype):
    """Without starts a mask has one bit that counts."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(9)
    lengths = [1, 5, 64, 65, 1, 0, 700]
    cache, table = _filled(rng, lengths, 2, 64, 16)
    q = _queries(rng, 7, 6, 64, dtype)
    masks = [[1], [0], [1], [2 ** 64 - 2], [0], [1], [2 ** 63 + 1]]
    for window in (None, 1, 20):
        got = kv_attend(q, cache, table, _i32(lengths), masks=_masks(masks), window=window, return_lse=True)
        _check(got, q, cache, table, lengths, list(range(8)), masks, window)


def test_missing_pages_and_narrow_tables():
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(10)
    new, lengths = [20, 9], [100, 70]
    cache, table = _filled(rng, lengths, 2, 64, 16)
    table[0, 5] = -1                            # places 80 to 95: the request's first new ones
    table[1, 1] = 10 ** 6
    starts = _starts(new)
    q = _queries(rng, 29, 4, 64, torch.float32)
    masks = _random_masks(rng, new, 1, 29)
    for t in (table, table[:, :4].contiguous()):
        got = kv_attend(q, cache, t, _i32(lengths), starts=_i32(starts), masks=_masks(masks), return_lse=True)
        _check(got, q, cache, t, lengths, starts, masks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 8])
def test_nan_where_it_is_not_seen(dtype, group):
    """A drafted token with a broken key and value changes only the rows whose masks have it (few rows, and many)."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(11)
    new, lengths = [20], [150]
    cache, table = _filled(rng, lengths, 1, 64, 16)
    at = int(table[0, 135 // 16]), 135 % 16     # new token 5
    for which in (1, 3):
        cache[which][at[0], :, at[1]] = float("nan")
    q = _queries(rng, 20, group, 64, dtype)
    masks = [[int(rng.randint(0, 2 ** 20)) | 1 << i] for i in range(20)]
    got = kv_attend(q, cache, table, _i32(lengths), starts=_i32([0, 20]), masks=_masks(masks))
    for i in range(20):
        assert torch.isnan(got[i]).all() == bool(masks[i][0] >> 5 & 1) and torch.isnan(got[i]).any() == torch.isnan(got[i]).all()


def test_attend_refuses():
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(12)
    cache, table = _filled(rng, [20], 2, 64, 16)
    q = _queries(rng, 3, 4, 64, torch.bfloat16)
    call = lambda masks, **kw: kv_attend(q, cache, table, _i32([20]), starts=_i32([0, 3]), masks=masks, **kw)  # noqa: E731
    ones = torch.ones(3, 1, dtype=torch.int64, device="cuda")
    for bad in (ones[:2], ones[:, 0], ones.expand(3, 5), ones[:, :0], ones.int(), ones.cpu()):
        with pytest.raises(ValueError, match="masks"):
            call(bad)
    with pytest.raises(ValueError, match="masks need causal"):
        call(ones, causal=False)
    assert torch.equal(call(ones.expand(3, 4)), call(ones.expand(3, 4).contiguous()))     # (strided masks are copied)


# ---------------------------------------------------------------- the accepted path

def _kept_rows(rng, new, most):
    """Random rising lists, whole ones, empty ones, and ones that end at a wrong entry."""
    rows = []
    for n in new:
        count = min(n, int(rng.randint(0, most + 1)))
        row = sorted(rng.permutation(n)[:count].tolist())
        kind = rng.randint(6)
        if kind == 0:
            row = list(range(min(n, most)))
        row += [-1] * (most - len(row))
        if kind == 1 and most > 2:
            row[2] = row[0]                     # does not rise
        if kind == 2:
            row[-1] = n                         # none of the request's
        if kind == 3 and most > 1:
            row[1] = -5
        rows.append(row[:most])
    return rows


@pytest.mark.parametrize("dim,heads,page", [(64, 1, 16), (128, 3, 64), (256, 2, 32)])
@pytest.mark.parametrize("layers,most", [(1, 1), (3, 9), (2, 70)])
def test_keep(dim, heads, page, layers, most):
    from orbitquant_amd import kv_assign, kv_keep

    rng = np.random.RandomState(dim + most)
    new = [1, 40, 0, 64, 130, 7, 20, 33]
    before = [30, 0, 16, 5, 100, 15, 63, 64]
    width = 16
    table = torch.full((len(new), width), -1, dtype=torch.int32, device="cuda")
    pages = 8 * width + 4
    free = _i32(rng.permutation(pages).tolist())
    first = kv_assign(_i32([0] * 8), _i32(before), table, free, _i32([0]), page_size=page, tokens=sum(before))
    got = kv_assign(first.lengths, _i32(new), table, free, first.taken, page_size=page, tokens=sum(new))
    caches = [_cache(pages, heads, dim, page) for _ in range(layers)]
    for c in caches:
        for t in c[:4]:
            t.view(torch.uint8).random_(0, 255)
    was = [kv_oracle.cache_codes(c) for c in caches]
    kept = _kept_rows(rng, new, most)
    slots, starts, lengths = got.slots.tolist(), got.starts.tolist(), got.lengths.tolist()
    moves, after, want_free, want_taken = oracle.keep(kept, lengths, starts, slots, table.tolist(), free.tolist(), int(got.taken), page)
    old_table = table.clone()
    kept_lengths, taken = kv_keep(_i32(kept), got.lengths, got.starts, got.slots, caches, block_table=table, free_pages=free, taken=got.taken)
    assert kept_lengths.tolist() == after and free.tolist() == want_free and taken.tolist() == [want_taken] and torch.equal(table, old_table)
    for c, old in zip(caches, was):
        for x, y in zip(kv_oracle.cache_codes(c), old):
            y = y.copy()
            fresh = [y[s // page, :, s % page].copy() for s, _ in moves]
            for (_, to), z in zip(moves, fresh):
                y[to // page, :, to % page] = z
            np.testing.assert_array_equal(x.view(np.int32) if x.dtype == np.float32 else x, y.view(np.int32) if y.dtype == np.float32 else y)


def test_keep_without_pages_and_slots():
    """No free list; tokens that got no page end a list."""
    from orbitquant_amd import kv_keep

    cache = _cache(4, 2, 64, 16)
    cache[0].random_(0, 255)
    was = cache[0].clone()
    slots = torch.tensor([0, 1, 2, -1, -1, 17, 18], device="cuda")
    got = kv_keep(_i32([[0, 2, 3], [0, 1, -1]]), _i32([25, 10]), _i32([0, 5, 7]), slots, [cache])
    assert got.lengths.tolist() == [22, 10] and got.taken is None
    assert torch.equal(cache[0][0, :, 1], was[0, :, 2]) and torch.equal(cache[0][1:], was[1:]) and torch.equal(cache[0][0, :, 2:], was[0, :, 2:])
    assert kv_keep(torch.empty(2, 0, dtype=torch.int32, device="cuda"), _i32([25, 10]), _i32([0, 5, 7]), slots, [cache]).lengths.tolist() == [20, 8]


def test_keep_many_requests_and_caches():
    """More requests than a workgroup has threads, and more layers than one launch takes."""
    from orbitquant_amd import kv_assign, kv_keep

    rng = np.random.RandomState(13)
    requests, page = 700, 16
    before, new = rng.randint(0, 40, requests).tolist(), rng.randint(0, 50, requests).tolist()
    table = torch.full((requests, 6), -1, dtype=torch.int32, device="cuda")
    free = _i32(rng.permutation(requests * 6).tolist())
    first = kv_assign(_i32([0] * requests), _i32(before), table, free, _i32([0]), page_size=page, tokens=sum(before))
    got = kv_assign(first.lengths, _i32(new), table, free, first.taken, page_size=page, tokens=sum(new))
    caches = [_cache(requests * 6, 1, 64, page, fill=i + 1) for i in range(66)]
    caches[65][0].random_(0, 255)
    was = caches[65][0].cpu().numpy()
    kept = _kept_rows(rng, new, 6)
    moves, after, want_free, want_taken = oracle.keep(kept, got.lengths.tolist(), got.starts.tolist(), got.slots.tolist(), table.tolist(), free.tolist(), int(got.taken), page)
    lengths, taken = kv_keep(_i32(kept), got.lengths, got.starts, got.slots, caches, block_table=table, free_pages=free, taken=got.taken)
    assert lengths.tolist() == after and free.tolist() == want_free and taken.tolist() == [want_taken]
    want = was.copy()
    for source, to in moves:
        want[to // page, :, to % page] = was[source // page, :, source % page]
    np.testing.assert_array_equal(caches[65][0].cpu().numpy(), want)
    assert all((c[0] == i + 1).all() for i, c in enumerate(caches[:65]))
    # the pages that came back are given out again, each once
    again = kv_assign(lengths, _i32(new), table, free, taken, page_size=page, tokens=sum(new))
    held = [int(table[r, c]) for r, n in enumerate(again.lengths.tolist()) for c in range(min(6, -(-n // page)))]
    assert min(held) >= 0 and len(set(held)) == len(held)


def test_keep_beyond_32_bits():
    """Entries whose codes lie behind 4 GiB."""
    from orbitquant_amd import OrbitKVCache, kv_keep

    cache = OrbitKVCache.empty(5 * 2 ** 13, 16, 128, page_size=128)      # 2^13 pages of 16 heads: 1 GiB of keys
    slots = torch.tensor([5, 2 ** 20 + 70, 5 * 2 ** 20 - 1, 2 ** 22 + 3], device="cuda")
    at, place = slots // 128, slots % 128
    for t in cache[:4]:
        where = (at, slice(None), place) if t.ndim == 3 or t is cache[0] else (at, slice(None), slice(None), place)
        t[where] = torch.randint(1, 100, t[where].shape, device="cuda").to(t.dtype)
    was = _entries(cache, at, place)
    got = kv_keep(_i32([[0, 2, 3]]), _i32([4]), _i32([0, 4]), slots, [cache])
    assert got.lengths.tolist() == [3]
    for x, y in zip(_entries(cache, at, place), was):
        assert torch.equal(x[[0, 1, 2, 3]], y[[0, 2, 3, 3]])


def _entries(cache, at, place):
    """The entries' codes and scales."""
    return [cache[0][at, :, place], cache[1][at, :, place], cache[2][at, :, :, place], cache[3][at, :, place]]


def test_keep_no_requests():
    """Nothing moves, the count stays; also with more caches than one launch takes."""
    from orbitquant_amd import kv_keep

    cache = _cache(2, 1, 64, 16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    for caches in ([cache], [cache] * 65):
        got = kv_keep(none.view(0, 3), none, _i32([0]), torch.empty(0, dtype=torch.int64, device="cuda"), caches, block_table=none.view(0, 4), free_pages=_i32([4, 5, 6]),
                      taken=_i32([2]))
        assert got.lengths.shape == (0,) and got.taken.tolist() == [2]
    assert (cache[0] == 0xA5).all()


def test_keep_refuses():
    from orbitquant_amd import kv_keep

    cache, slots = _cache(4, 2, 64, 16), torch.arange(5, device="cuda")
    call = lambda kept=_i32([[0], [1]]), caches=(cache,), **kw: kv_keep(kept, _i32([5, 6]), _i32([0, 2, 5]), slots, caches, **kw)  # noqa: E731
    table, free, taken = _i32([[0], [1]]), _i32([2, 3]), _i32([1])
    for bad in ({"kept": _i32([[0]])}, {"kept": _i32([0, 1])}, {"kept": _i32([[0], [1]]).long()}, {"kept": _i32([[0], [1]]).cpu()}, {"caches": ()},
                {"caches": (cache, _cache(4, 1, 64, 16))}, {"caches": (cache, _cache(4, 2, 64, 32))}, {"caches": (cache, _cache(5, 2, 64, 16))},
                {"caches": (cache, _cache(4, 2, 128, 16))}, {"block_table": table}, {"block_table": table, "free_pages": free}, {"free_pages": free, "taken": taken},
                {"block_table": table[:1], "free_pages": free, "taken": taken}, {"block_table": table, "free_pages": free.long(), "taken": taken},
                {"block_table": table, "free_pages": _i32([1, 2, 3, 4])[::2], "taken": taken}, {"block_table": table, "free_pages": free, "taken": _i32([1, 2])}):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(RuntimeError):
        call(kept=torch.zeros(2, 257, dtype=torch.int32, device="cuda"))
