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
