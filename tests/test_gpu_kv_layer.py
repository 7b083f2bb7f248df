"""`OrbitCachedAttention` where requests do not have one new token each, and the decoding example's caches, tables and pages."""

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import _cache, _check, _i32
from test_gpu_kv_serving import _layer

pytestmark = pytest.mark.gpu


def _prompted(window=None):
    """A layer whose cache holds prompts of three requests."""
    from orbitquant_amd import kv_assign

    rng = np.random.RandomState(30)
    cache = _cache(20, 2, 64, 16, fill=0xFF)
    layer = _layer(cache, 4, 256, window=window)
    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    free = _i32(rng.permutation(20).tolist())
    got = kv_assign(_i32([0, 0, 0]), _i32([30, 17, 60]), table, free, _i32([0]), page_size=16, tokens=107)
    layer(_inputs(rng, 107), got, table, max_new=60)
    return rng, layer, table, free, got


def _inputs(rng, tokens):
    return torch.from_numpy(rng.standard_normal((tokens, 256)).astype(np.float32)).to("cuda", torch.bfloat16)


@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("new,tokens", [([1, 0, 1], 3), ([0, 0, 1], 3), ([2, 0, 1], 3), ([2, 1, 0], 3), ([0, 0, 0], 3), ([1, 1, 1], 3), ([1, 1, 0], 2), ([0, 3, 1], 5)])
@pytest.mark.parametrize("hints", [{}, {"max_new": 1}, {"max_new": 3, "max_length": 90}, {"max_length": 10}])
def test_rows_belong_to_the_requests_that_starts_names(new, tokens, window, hints):
    """As many rows as requests does not mean a row each: requests without new tokens in a batch of a fixed size, and several tokens of one."""
    from orbitquant_amd import kv_assign, kv_attend

    rng, layer, table, free, before = _prompted(window)
    got = kv_assign(before.lengths, _i32(new), table, free, before.taken, page_size=16, tokens=tokens)
    x = _inputs(rng, tokens)
    y = layer(x, got, table, **hints)
    q = layer.q(x).view(tokens, 4, 64)
    attended = kv_attend(q, layer.cache, table, got.lengths, starts=got.starts, window=window, return_lse=True)
    _check(attended, q, layer.cache, table, got.lengths, starts=got.starts, window=window)
    assert (attended[0][sum(new):] == 0).all()
    assert torch.equal(y, layer.out(attended[0].reshape(tokens, -1)))


def test_one_row_each_where_the_caller_says_so():
    from orbitquant_amd import kv_assign, kv_attend

    rng, layer, table, free, before = _prompted()
    got = kv_assign(before.lengths, _i32([1, 1, 1]), table, free, before.taken, page_size=16, tokens=3)
    x = _inputs(rng, 3)
    y = layer(x, got, table, one_each=True)
    q = layer.q(x).view(3, 4, 64)
    attended = kv_attend(q, layer.cache, table, got.lengths, return_lse=True)
    _check(attended, q, layer.cache, table, got.lengths)
    assert torch.equal(y, layer.out(attended[0].reshape(3, -1)))
    with pytest.raises(ValueError, match="one_each"):
        layer(_inputs(rng, 2), got, table, one_each=True)


def test_decode_example_caches():
    """After replayed steps every layer's cache holds what the same steps leave there when they are run eagerly, at the same pages."""
    from orbitquant_amd import kv_read
    from orbitquant_amd.examples import decode

    prompts = [20, 70, 61]
    eager, replayed = (decode.Decoder(2, 3, 80) for _ in range(2))
    ids = torch.randint(0, decode.VOCABULARY, (sum(prompts),), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    for m in (eager, replayed):
        m.step(ids, _i32(prompts), max_new=max(prompts))
    graph = replayed.captured_step()
    for steps in range(1, 6):
        eager.step(eager.last.clone(), _i32([1, 1, 1]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.last, replayed.last) and torch.equal(eager.taken, replayed.taken) and torch.equal(eager.block_table, replayed.block_table)
        assert replayed.lengths.tolist() == [n + steps for n in prompts]
        held = [int(eager.block_table[r, t // decode.PAGE]) * decode.PAGE + t % decode.PAGE for r, n in enumerate(prompts) for t in range(n + steps)]
        assert min(held) >= 0 and len(set(held)) == len(held)
        slots = torch.tensor(held, device="cuda")
        for a, b in zip(eager.layers, replayed.layers):
            for x, y in zip(kv_read(slots, a.attention.cache, torch.float32), kv_read(slots, b.attention.cache, torch.float32)):
                assert torch.equal(x, y) and torch.isfinite(x).all() and x.abs().sum() > 0


@pytest.mark.parametrize("one_each", [False, True])
def test_no_rows(one_each):
    """A step without tokens: of requests that have none, or of no requests."""
    from orbitquant_amd import kv_assign

    rng, layer, table, free, before = _prompted()
    if one_each:
        none = torch.empty(0, dtype=torch.int32, device="cuda")
        table, got = table[:0], kv_assign(none, none, table[:0], free, before.taken, page_size=16, tokens=0)
    else:
        got = kv_assign(before.lengths, _i32([0, 0, 0]), table, free, before.taken, page_size=16, tokens=0)
    held = [t.clone() for t in layer.cache]
    y = layer(_inputs(rng, 0), got, table, one_each=one_each)
    assert y.shape == (0, 256) and y.dtype == torch.bfloat16
    for was, now in zip(held, layer.cache):
        assert torch.equal(was.view(torch.uint8), now.view(torch.uint8))
