"""The attention's bits do not depend on what stands in places that hold no token: behind a request's last one, in pages that are nobody's or missing."""

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import _cache, _i32, _queries, _vectors
from test_gpu_kv_tree import _masks, _parents, _starts

import tree_oracle

pytestmark = pytest.mark.gpu

FILLS = (0x00, 0x3f, 0x7f, 0xff, 0xa5, 0x01, None)      # as scales: 0, 0.75, 3.4e38, NaN, a small negative one, a tiny one; anything


def _fill(cache, fill, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in cache[:4]:
        if fill is None:
            t.view(torch.uint8).random_(0, 256, generator=g)
        else:
            t.view(torch.uint8).fill_(fill)


def _calls(dim, page, dtype, masked, missing):
    """The same tokens in caches that were filled with different things before: -> the results of a call on each."""
    from orbitquant_amd import kv_attend, kv_write

    rng = np.random.RandomState(dim + page)
    new = [23, 46, 70, 1, 5, 130]
    before = [0, 0, 70, 90, 200, 65]
    lengths, starts = [a + b for a, b in zip(new, before)], _starts(new)
    width = max(-(-n // page) for n in lengths) + 1
    table, at = torch.full((len(new), width), -1, dtype=torch.int32), 3
    for r, n in enumerate(lengths):
        count = -(-n // page)
        table[r, :count] = torch.arange(at, at + count)
        at += count
    slots = torch.cat([table[r, torch.arange(n) // page].long() * page + torch.arange(n) % page for r, n in enumerate(lengths)]).cuda()
    if missing:
        table[2, 0] = table[5, 1 if page < 128 else 0] = -1
    table = table.cuda()
    k, v = (_vectors(rng, len(slots), 2, dim, torch.float32).cuda() for _ in range(2))
    v *= torch.from_numpy(2.0 ** rng.randint(-2, 4, (len(slots), 1, 1))).float().cuda()      # (of different sizes, within 2^8)
    q = _queries(rng, starts[-1] + 2, 8, dim, dtype)
    masks = _masks(tree_oracle.tree(_parents(rng, new, "random"), starts, lengths, 3, starts[-1] + 2)[1]) if masked else None
    for i, fill in enumerate(FILLS):
        cache = _cache(at + 2, 2, dim, page)
        _fill(cache, fill, i)
        kv_write(k, v, slots, cache)
        yield fill, [kv_attend(q, cache, table, _i32(lengths), starts=_i32(starts), masks=masks, return_lse=True, **hints)
                     for hints in ({}, {"max_new": 130, "max_length": 265}, {"window": 30}, {"max_new": 1})]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 64), (128, 64), (128, 1024), (256, 32), (256, 128)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("missing", [False, True])
def test_places_without_a_token_change_nothing(dim, page, dtype, masked, missing):
    want = None
    for fill, results in _calls(dim, page, dtype, masked, missing):
        want = want or results
        for a, b in zip(want, results):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), fill


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens(dim):
    from orbitquant_amd import kv_attend, kv_write

    rng = np.random.RandomState(dim)
    lengths = [1, 23, 64, 65, 700, 0]
    table = torch.arange(6 * 12, dtype=torch.int32).view(6, 12)
    slots = torch.cat([table[r, torch.arange(n) // 64].long() * 64 + torch.arange(n) % 64 for r, n in enumerate(lengths)]).cuda()
    k, v = (_vectors(rng, len(slots), 2, dim, torch.float32).cuda() for _ in range(2))
    v *= torch.from_numpy(2.0 ** rng.randint(-2, 4, (len(slots), 1, 1))).float().cuda()
    q, want = _queries(rng, 6, 8, dim, torch.bfloat16), None
    for i, fill in enumerate(FILLS):
        cache = _cache(72, 2, dim, 64)
        _fill(cache, fill, i)
        kv_write(k, v, slots, cache)
        got = [kv_attend(q, cache, table.cuda(), _i32(lengths), return_lse=True, max_length=longest) for longest in (None, 700, 64)]
        want = want or got
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), fill
