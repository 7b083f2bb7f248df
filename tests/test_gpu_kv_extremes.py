"""The cache's attention where numbers of very different sizes meet: queries of one tile, values of one step, what a mask hides, and broken
vectors; and positions at the end of what a table can hold."""

import math

import numpy as np
import pytest
import torch

import kv_oracle as oracle
from test_gpu_kv_cache import DTYPES, _cache, _check, _filled, _i32, _queries

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- queries of one tile

FACTORS = {torch.bfloat16: (2.0 ** 20, 2.0 ** 33, 1e10, 1e30), torch.float16: (2.0 ** 14,), torch.float32: (2.0 ** 12, 2.0 ** 20, 2.0 ** 36, 1e20, 1e30)}
OF_TYPE = [(dtype, factor) for dtype in DTYPES for factor in FACTORS[dtype]]


@pytest.mark.parametrize("dtype,factor", OF_TYPE)
@pytest.mark.parametrize("dim,page", [(64, 64), (128, 16), (256, 64)])
def test_a_row_is_its_own(dim, page, dtype, factor):
    """A prompt with queries far larger and far smaller than the others, zeros, an infinity and a NaN: every other row as without them."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(dim)
    lengths, new = [180], [100]
    cache, table = _filled(rng, lengths, 1, dim, page)
    q = _queries(rng, 100, 2, dim, torch.float32)
    q[7, 1] *= factor
    q[70, 0] *= -factor
    q[33, 0] *= 1e-4
    q[34, 1] = 0
    q[50, 0, 5] = float("inf")
    q[51, 1, 6] = float("nan")
    q = q.to(dtype)
    starts = _i32([0, 100])
    for window in (None, 60):
        _check(kv_attend(q, cache, table, _i32(lengths), starts=starts, window=window, return_lse=True), q, cache, table, _i32(lengths), starts=starts,
               window=window)


@pytest.mark.parametrize("dtype,factor", [(torch.bfloat16, 1e10), (torch.float16, 2.0 ** 14), (torch.float32, 1e20)])
def test_a_row_is_its_own_in_parts(dtype, factor):
    """The same where tiles are cut, and where a tile has several requests' neighbours beside it."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(31)
    lengths, new = [1500, 1290, 130], [80, 90, 1]
    cache, table = _filled(rng, lengths, 1, 64, 32)
    starts = _i32(np.concatenate(([0], np.cumsum(new))).tolist())
    q = _queries(rng, sum(new), 1, 64, torch.float32)
    q[3] *= factor
    q[100] *= factor
    q[101] /= factor if dtype != torch.float16 else 64
    q = q.to(dtype)
    _check(kv_attend(q, cache, table, _i32(lengths), starts=starts, return_lse=True), q, cache, table, _i32(lengths), starts=starts)


# ---------------------------------------------------------------- values of one step

def _check_with_overflow(got, q, cache, table, lengths, **kw):
    """`_check`, where outputs may pass the largest number of their type: an entry is right to be infinite where what its row may be off (the bound
    is the row's, whose other entries may be far larger) reaches beyond that number."""
    want, _, bound = oracle.attend(q, cache, table, lengths, **kw)
    far = oracle.allowed(bound, want, q.dtype)[0][..., None]
    out = got[0].double().cpu().numpy()
    fine = np.isinf(out) & (np.sign(out) * want + far > torch.finfo(q.dtype).max)
    _check((torch.where(torch.from_numpy(fine), torch.from_numpy(want).to(q.dtype), got[0].cpu()), got[1]), q, cache, table, lengths, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,new,at", [(64, 90, 50), (128, 90, 50), (256, 90, 50), (128, 12, 84), (256, 12, 84), (64, 2, 89)])
@pytest.mark.parametrize("window", [None, 3, 20])
def test_a_large_value_changes_only_the_rows_that_see_it(window, dim, new, at, dtype):
    """By both kernels; with a window the rows behind it see past it again."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(new)
    cache, table = _filled(rng, [90], 1, dim, 32)
    cache.v_scales[int(table[0, at // 32]), 0, at % 32] *= 2.0 ** 40
    starts = _i32([0, new])
    q = _queries(rng, new, 4, dim, dtype)
    got = kv_attend(q, cache, table, _i32([90]), starts=starts, window=window, return_lse=True)
    _check_with_overflow(got, q, cache, table, _i32([90]), starts=starts, window=window)


def _by_weights(q, cache, table, length):
    """One request's last token: out, and the mean of |v| over the weights; a relative error of e in every weight moves out by at most 2 e of that."""
    kc, ks, vc, vs = oracle.cache_codes(cache)
    dim = kc.shape[-1]
    turn = oracle.sylvester(dim) / dim * cache[4].cpu().numpy().astype(np.float64)
    rows = tuple(np.array(x) for x in zip(*[(int(table[0, t // cache.page_size]), 0, t % cache.page_size) for t in range(length)]))
    k, v = ((oracle.decode(c[rows]) * s[rows][:, None]) @ turn for c, s in ((kc, ks), (vc, vs)))
    s = q[0].double().cpu().numpy() @ k.T / math.sqrt(dim)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    return w @ v, w @ np.linalg.norm(v, axis=-1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** 15, 2.0 ** 30, 2.0 ** 60])
def test_a_large_value_without_weight_changes_nothing(size, dtype):
    from orbitquant_amd import OrbitKVCache, kv_attend, kv_write

    rng = np.random.RandomState(32)
    cache = OrbitKVCache.empty(3, 1, 64, page_size=32)
    q = _queries(rng, 1, 1, 64, dtype)
    k, v = (_queries(rng, 90, 1, 64, torch.float32) for _ in range(2))
    k[60] = -20 * q[0].float()          # a score 20 |q|^2 / 8, some 160, below the others
    v[60] *= size
    kv_write(k, v, torch.arange(90, device="cuda"), cache)
    table = _i32([[0, 1, 2]])
    out = kv_attend(q, cache, table, _i32([90]))
    want, mean = _by_weights(q, cache, table, 90)
    (size_of, _, count, dim), = (oracle.attend(q, cache, table, _i32([90]))[2],)
    far, _ = oracle.allowed((size_of, mean[None], count, dim), want[None], dtype)
    off = np.linalg.norm(out.double().cpu().numpy() - want, axis=-1)
    assert (off <= far).all(), (off, far)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("sizes", [(1e22, 1e22), (1e25, 1e25), (1e30, 1e30), (1e33, 1e33), (1.0, 1e30), (1e30, 1.0), (1e-30, 1e25), (1e25, 1e-30), (1e-25, 1e25), (1e-30, 1.0)])
def test_values_of_any_size(sizes, new, dtype):
    """Numbers of the types that a value's scale holds, large and small ones side by side: in one step, in different steps, by different wavefronts
    and in different parts."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(33)
    for length, first in ((60, 25), (400, 64), (400, 350), (1800, 900)):
        cache, table = _filled(rng, [length], 1, 64, 64)
        v = torch.where(torch.arange(cache.page_size * table.shape[1], device="cuda") < first, sizes[0], sizes[1])
        for column in range(-(-length // 64)):
            cache.v_scales[int(table[0, column]), 0] *= v[64 * column:64 * column + 64]
        q = _queries(rng, new, 4, 64, dtype)
        starts = _i32([0, new])
        for window in (None, 30):
            _check(kv_attend(q, cache, table, _i32([length]), starts=starts, window=window, return_lse=True), q, cache, table, _i32([length]), starts=starts,
                   window=window)


# ---------------------------------------------------------------- broken values

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,length,new,at", [(64, 90, 90, 50), (128, 200, 100, 130), (256, 90, 90, 10), (128, 300, 1, 20), (64, 300, 1, 299), (256, 300, 12, 290), (64, 1800, 30, 700), (64, 1500, 90, 700)])
@pytest.mark.parametrize("window", [None, 40])
def test_a_broken_value_leaves_the_scores_alone(window, dim, length, new, at, dtype):
    """A NaN among the values makes the outputs NaN that see it; the sum of the weights, which lse is, has no value in it.  In steps that a mask goes through and in
    others, by both kernels and in parts."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(34)
    cache, table = _filled(rng, [length], 1, dim, 64)
    cache.v_scales[int(table[0, at // 64]), 0, at % 64] = float("nan")
    q = _queries(rng, new, 4, dim, dtype)
    starts, lengths = _i32([0, new]), _i32([length])
    out, lse = kv_attend(q, cache, table, lengths, starts=starts, window=window, return_lse=True)
    want, want_lse, bound = oracle.attend(q, cache, table, lengths, starts=starts, window=window)
    _check((out, torch.where(torch.from_numpy(np.isnan(want).any(-1)).cuda(), torch.from_numpy(want_lse).float().cuda(), lse)), q, cache, table, lengths, starts=starts,
           window=window)
    far = oracle.allowed(bound, want, dtype)[1]
    assert (np.abs(lse.double().cpu().numpy() - want_lse) <= far).all()


# ---------------------------------------------------------------- positions at the end of what a table holds

@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("window,sees", [((1 << 30) - 1, 1023), (1 << 30, 1024), ((1 << 30) + 1, 1024), (1 << 31, 1024), (1 << 40, 1024)])
def test_windows_as_long_as_a_table(window, sees, new):
    """A request of 2^30 tokens, as many as a table may have, whose pages are missing but for the first: its last token sees that page's, but for
    the one in front of a window of 2^30 - 1."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(35)
    cache, _ = _filled(rng, [1024], 1, 64, 1024)
    first = next(p for p in range(cache.pages) if not torch.isnan(cache.v_scales[p]).any())
    cache.k_scales[first] = 0                   # all scores are equal: lse is the logarithm of the number of keys
    table = torch.full((1, 1 << 20), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = first
    q = _queries(rng, new, 2, 64, torch.bfloat16)
    out, lse = kv_attend(q, cache, table, _i32([1 << 30]), starts=_i32([0, new]), window=window, return_lse=True)
    _check((out[-1:], lse[-1:]), q[-1:], cache, _i32([[first]]), _i32([1024]), window=sees)


# ---------------------------------------------------------------- scores of any size

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,new", [(64, 1), (64, 100), (128, 1), (256, 20), (128, 100)])
@pytest.mark.parametrize("length", [1, 100, 1500, 9000])
@pytest.mark.parametrize("one_key", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
def test_outputs_are_means_however_large_the_scores_are(sign, one_key, length, dim, new, dtype):
    """All values are one value, which is then every row's output, whatever its weights: for scores from 1 to what fp32 holds, above and below zero, of
    keys that are one key or differ.  A weight is rounded once, and the sum of the weights is not."""
    from orbitquant_amd import OrbitKVCache, kv_attend, kv_write

    rng = np.random.RandomState(36)
    pages = -(-length // 64) + 1
    cache = OrbitKVCache.empty(pages, 1, dim, page_size=64, seed=3)
    k = torch.from_numpy(rng.standard_normal((1 if one_key else 64 * pages, 1, dim)).astype(np.float32)).cuda()
    v = torch.from_numpy(rng.standard_normal((1, 1, dim)).astype(np.float32)).cuda()
    kv_write(k.expand(64 * pages, 1, dim), v.expand(64 * pages, 1, dim), torch.arange(64 * pages, device="cuda"), cache)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1)
    heads = 16
    q = k[:1].expand(new, heads, dim) * sign * 2.0 ** (torch.arange(new * heads, device="cuda").view(new, heads, 1) * (117 / (new * heads)))
    q = (q * (1 + torch.rand(q.shape[:2], device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))[..., None])).to(dtype)
    out, lse = kv_attend(q, cache, table, _i32([length]), starts=_i32([0, new]), causal=False, return_lse=True)
    want, _, (_, largest, _, _) = oracle.attend(q[:1] * 0, cache, table, _i32([1]), starts=_i32([0, 1]), causal=False)
    zeros = np.zeros((new, heads))
    far, _ = oracle.allowed((zeros, zeros + largest[0, 0], zeros + length, dim), np.broadcast_to(want[:1], (new, heads, dim)), dtype)
    off = np.linalg.norm(out.double().cpu().numpy() - want[0, 0], axis=-1)
    assert (off <= far).all(), (off / far).max()
    assert torch.isfinite(lse).all()
