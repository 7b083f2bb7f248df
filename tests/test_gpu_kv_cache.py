"""The 4-bit key/value cache on the GPU against its definition: pages and slots, what is written, what is read back, and the
attention over it, at the sizes, strides and masks where these can go wrong."""

import numpy as np
import pytest
import torch

import kv_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- pages and slots

ASSIGN = {
    "one token into a new page": ([0], [1], 16, 4, 1, 0),
    "one token into the last place": ([15], [1], 16, 4, 1, 0),
    "one token behind a full page": ([16], [1], 16, 4, 1, 0),
    "ragged": ([5, 0, 64, 63, 100, 0, 17], [1, 130, 1, 2, 0, 0, 64], 64, 9, 0, 2),
    "nothing new": ([3, 9], [0, 0], 16, 3, 0, 0),
    "negative counts": ([-4, 20], [5, -7], 16, 5, 0, 0),
    "the free list runs out": ([0, 10, 30], [40, 40, 40], 16, 8, 3, 1),
    "no free page at all": ([0, 15], [4, 3], 16, 2, 0, 0),
    "the table is too narrow": ([30, 0], [20, 70], 16, 2, 20, 0),
    "more tokens asked for than come": ([2, 2], [3, 4], 32, 2, 2, -9),
}


@pytest.mark.parametrize("name", ASSIGN)
@pytest.mark.parametrize("extra", [0, 5, -3])
def test_assign(name, extra):
    from orbitquant_amd import kv_assign

    lengths, new, page, width, short, taken = ASSIGN[name]
    total = sum(max(n, 0) for n in new)
    tokens = max(0, total + extra)
    rng = np.random.RandomState(len(name))
    need = sum(-(-max(n, 0) // page) + 1 for n in new) + 3
    pool = rng.permutation(1000)
    free = pool[:need + max(taken, 0)].tolist() if name not in ("the free list runs out", "no free page at all") else pool[:short].tolist()
    table = np.full((len(lengths), width), -7)
    for r, was in enumerate(lengths):
        have = min(width, -(-max(was, 0) // page))
        table[r, :have] = pool[500 + 20 * r: 500 + 20 * r + have]
    want = oracle.assign(lengths, new, table, free, taken, page, tokens)
    big = torch.full((len(lengths), width + 3), -5, dtype=torch.int32, device="cuda")     # rows are further apart than they are long
    big[:, :width] = torch.from_numpy(table).cuda()
    got = kv_assign(_i32(lengths), _i32(new), big[:, :width], _i32(free), _i32([taken]), page_size=page, tokens=tokens)
    assert got.slots.tolist() == want[0] and got.positions.tolist() == want[1] and got.starts.tolist() == want[2]
    assert got.lengths.tolist() == want[3] and got.taken.tolist() == [want[4]]
    assert big[:, :width].tolist() == want[5] and (big[:, width:] == -5).all()


@pytest.mark.parametrize("requests", [1, 63, 64, 65, 255, 257, 1000, 8192])
def test_assign_many(requests):
    from orbitquant_amd import kv_assign

    rng = np.random.RandomState(requests)
    page, width = 32, 12
    lengths = rng.randint(0, 300, requests).tolist()
    new = np.where(rng.rand(requests) < 0.5, 1, rng.randint(0, 60, requests)).tolist()
    table = np.full((requests, width), -1)
    for r, was in enumerate(lengths):
        table[r, :-(-was // page)] = rng.randint(0, 100000, -(-was // page))
    free = rng.permutation(4 * requests + 50).tolist()
    want = oracle.assign(lengths, new, table, free, 7, page, sum(new))
    device_table = _i32(table.tolist())
    got = kv_assign(_i32(lengths), _i32(new), device_table, _i32(free), _i32([7]), page_size=page, tokens=sum(new))
    assert got.slots.tolist() == want[0] and got.positions.tolist() == want[1] and got.starts.tolist() == want[2]
    assert got.lengths.tolist() == want[3] and got.taken.tolist() == [want[4]] and device_table.tolist() == want[5]


def test_assign_without_requests():
    from orbitquant_amd import kv_assign

    got = kv_assign(_i32([]), _i32([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), _i32([1, 2]), _i32([1]), page_size=16, tokens=3)
    assert got.slots.tolist() == [-1] * 3 and got.starts.tolist() == [0] and got.taken.tolist() == [1] and got.lengths.numel() == 0


# ---------------------------------------------------------------- into the cache and back

def _vectors(rng, tokens, heads, dim, dtype):
    x = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    x[:, :, 1] *= 8
    return torch.from_numpy(x).to(dtype)


def _cache(pages, heads, dim, page, fill=0xA5):
    from orbitquant_amd import OrbitKVCache

    cache = OrbitKVCache.empty(pages, heads, dim, page_size=page, seed=3)
    for t in cache[:4]:
        t.view(torch.uint8).fill_(fill)      # what no token was written to is anything: as scales, a large negative number
    return cache


def _check_written(cache, k, v, slots):
    page = cache.page_size
    signs = cache.signs.cpu().numpy()
    kc, ks, vc, vs = oracle.cache_codes(cache)
    for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
        want_codes, want_scales = oracle.encode(x.float().cpu().numpy(), signs)
        for t, slot in enumerate(slots):
            if slot >= 0:
                at = (slot // page, slice(None), slot % page)
                np.testing.assert_array_equal(scales[at], want_scales[t])
                np.testing.assert_array_equal(codes[at], want_codes[t])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,page", [(64, 1, 16), (64, 5, 64), (128, 3, 32), (128, 8, 1024), (256, 2, 16), (256, 3, 128)])
@pytest.mark.parametrize("tokens", [1, 37])
def test_write_and_read(tokens, dim, heads, page, dtype):
    from orbitquant_amd import kv_read, kv_write

    rng = np.random.RandomState(tokens + dim)
    pages = -(-tokens // page) + 2
    cache = _cache(pages, heads, dim, page)
    before = [t.clone() for t in cache]
    slots = rng.permutation(pages * page)[:tokens].tolist()
    if tokens > 1:
        slots[3], slots[-1] = -1, pages * page       # skipped
    k, v = _vectors(rng, tokens, heads, dim, dtype), _vectors(rng, tokens, heads, dim, dtype)
    device_slots = torch.tensor(slots, dtype=torch.int64, device="cuda")
    kv_write(k.cuda(), v.cuda(), device_slots, cache)
    live = [s if 0 <= s < pages * page else -1 for s in slots]
    _check_written(cache, k, v, live)
    # nothing else was touched
    touched = torch.zeros(pages * page, dtype=torch.bool)
    touched[[s for s in live if s >= 0]] = True
    touched = touched.view(pages, 1, page).cuda()
    for t, was, mask in ((cache.k_codes, before[0], touched[..., None]), (cache.k_scales, before[1], touched),
                         (cache.v_codes, before[2], touched[:, :, None]), (cache.v_scales, before[3], touched)):
        assert torch.equal(torch.where(mask, 0, t.view(torch.uint8) if t.dtype == torch.uint8 else t.view(torch.int16)),
                           torch.where(mask, 0, was.view(torch.uint8) if was.dtype == torch.uint8 else was.view(torch.int16)))
    for out_dtype in DTYPES:
        got = kv_read(device_slots, cache, out_dtype)
        for x, y in zip((k, v), got):
            codes, scales = oracle.encode(x.float().numpy(), cache.signs.cpu().numpy())
            want = torch.from_numpy(oracle.held32(codes, scales, cache.signs.cpu().numpy())).to(out_dtype)
            want[[i for i, s in enumerate(live) if s < 0]] = 0
            assert y.dtype == out_dtype and torch.equal(y.cpu(), want)


@pytest.mark.parametrize("page", [16, 64])
def test_write_a_run_of_tokens(page):
    """A prompt's tokens lie side by side in their pages, and begin and end inside one."""
    from orbitquant_amd import kv_write

    rng = np.random.RandomState(0)
    cache = _cache(9, 3, 128, page)
    order = rng.permutation(9)
    slots = [int(order[t // page]) * page + t % page for t in range(5, 5 + 7 * 16 + 11) if t // page < 9]
    k, v = _vectors(rng, len(slots), 3, 128, torch.bfloat16), _vectors(rng, len(slots), 3, 128, torch.bfloat16)
    kv_write(k.cuda(), v.cuda(), torch.tensor(slots, device="cuda"), cache)
    _check_written(cache, k, v, slots)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_strides(dtype):
    """Parts of a fused projection, heads in another order than tokens, and vectors that begin anywhere."""
    from orbitquant_amd import kv_write

    rng = np.random.RandomState(1)
    tokens, heads, dim = 19, 2, 64
    slots = list(range(tokens))
    device_slots = torch.tensor(slots, device="cuda")
    fused = _vectors(rng, tokens, 3 * heads, dim, dtype).cuda()
    shifted = torch.empty(tokens * heads * dim + 3, dtype=dtype, device="cuda")[3:].view(tokens, heads, dim).copy_(fused[:, :heads])
    heads_first = fused[:, heads:2 * heads].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    spread = torch.stack((fused[:, :heads], fused[:, :heads]), -1)[..., 0]       # the last dimension is not contiguous
    for k, v in ((fused[:, heads:2 * heads], fused[:, 2 * heads:]), (shifted, heads_first), (spread, shifted), (fused[:1, :heads].expand(tokens, heads, dim), shifted)):
        cache = _cache(3, heads, dim, 16)
        kv_write(k, v, device_slots, cache)
        _check_written(cache, k, v, slots)


def test_write_extremes():
    """Zeros, single spikes, ties, the largest and smallest numbers, infinities and NaN."""
    from orbitquant_amd import kv_read, kv_write

    dim = 64
    rows = [np.zeros(dim), np.full(dim, -0.0), np.eye(dim)[7], np.ones(dim), np.full(dim, 1e-42), np.full(dim, 3e-39), np.full(dim, 1e-37),
            np.full(dim, 1e36), np.arange(dim) - 31.5, np.eye(dim)[3] * np.inf, np.eye(dim)[3] * np.nan, np.full(dim, np.inf),
            np.where(np.arange(dim) == 5, 2e38, 1e38), np.tile([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dim // 8)]
    ties = oracle.hadamard32(np.tile([6.0, -0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0], dim // 8)[None])[0] / dim
    x = np.nan_to_num(np.stack(rows + [ties]).astype(np.float32), nan=np.nan, posinf=np.inf, neginf=-np.inf)
    x[9][np.arange(dim) != 3] = 1.0
    x[10][np.arange(dim) != 3] = 1.0
    x = torch.from_numpy(x).view(len(x), 1, dim)
    cache = _cache(2, 1, dim, 16)
    cache.signs.fill_(1)                          # so that the row of ties is one
    slots = list(range(len(x)))
    kv_write(x.cuda(), x.flip(0).contiguous().cuda(), torch.tensor(slots, device="cuda"), cache)
    _check_written(cache, x, x.flip(0), slots)
    kc, ks, _, _ = oracle.cache_codes(cache)
    assert ks.reshape(-1)[len(x) - 1] == 1.0 and kc.reshape(-1, dim)[len(x) - 1][:8].tolist() == [7, 8, 2, 10, 4, 4, 14, 6]
    k, _ = kv_read(torch.tensor(slots, device="cuda"), cache, torch.float32)
    k = k.view(len(x), dim).cpu()
    assert (k[0] == 0).all() and torch.isnan(k[9:13]).all() and torch.isfinite(k[:9]).all() and torch.isfinite(k[13:]).all()


def test_no_tokens():
    from orbitquant_amd import kv_attend, kv_read, kv_write

    cache = _cache(2, 2, 64, 16)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    x = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    kv_write(x, x, none, cache)
    k, v = kv_read(none, cache)
    assert k.shape == v.shape == (0, 2, 64)
    out, lse = kv_attend(x, cache, torch.empty(0, 3, dtype=torch.int32, device="cuda"), _i32([]), return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


# ---------------------------------------------------------------- attention

def _filled(rng, lengths, heads, dim, page, dtype=torch.bfloat16, extra_columns=1, scale_v=1.0):
    """A cache with `lengths` tokens a request, their pages anywhere; what no token was written to is NaN."""
    from orbitquant_amd import kv_write

    have = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(have) + 2
    cache = _cache(pages, heads, dim, page, fill=0xFF)
    order = rng.permutation(pages)
    table = np.full((len(lengths), max(have, default=0) + extra_columns), -1)
    slots, at = [], 0
    for r, n in enumerate(lengths):
        table[r, :have[r]] = order[at:at + have[r]]
        at += have[r]
        slots += [int(table[r, t // page]) * page + t % page for t in range(n)]
    if slots:
        k, v = _vectors(rng, len(slots), heads, dim, dtype), _vectors(rng, len(slots), heads, dim, dtype) * scale_v
        kv_write(k.cuda(), v.cuda(), torch.tensor(slots, device="cuda"), cache)
    return cache, _i32(table.tolist()).view(len(lengths), -1)


def _check(got, q, cache, table, lengths, **kw):
    out, lse = got
    want, want_lse, bound = oracle.attend(q, cache, table, lengths, **kw)
    far, far_lse = oracle.allowed(bound, want, q.dtype)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    # what the type cannot hold is infinite in it
    out = np.where(np.isinf(out) & (np.abs(want) > 0.99 * torch.finfo(q.dtype).max) & (np.sign(out) == np.sign(want)), want, out)
    broken = np.isnan(want).any(-1)
    np.testing.assert_array_equal(np.isnan(out).all(-1), broken)
    assert not np.isnan(out[~broken]).any()
    empty = np.isneginf(want_lse)
    assert (out[empty] == 0).all() and np.isneginf(lse[empty]).all()
    off = np.linalg.norm(out - want, axis=-1)[~broken & ~empty]
    assert (off <= far[~broken & ~empty]).all(), (off / far[~broken & ~empty]).max()
    off = np.abs(lse - want_lse)[~broken & ~empty]
    assert (off <= far_lse[~broken & ~empty]).all(), (off / far_lse[~broken & ~empty]).max()


def _queries(rng, tokens, heads, dim, dtype):
    return torch.from_numpy(rng.standard_normal((tokens, heads, dim)).astype(np.float32)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,page", [(2, 1, 16), (1, 3, 64), (3, 4, 32), (2, 16, 128), (1, 17, 64), (1, 40, 16)])
def test_attend_single_tokens(dim, heads, group, page, dtype):
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(dim + group)
    lengths = [1, 0, 16, 17, 64, 65, 127, 300, 1030]
    cache, table = _filled(rng, lengths, heads, dim, page)
    q = _queries(rng, len(lengths), heads * group, dim, dtype)
    _check(kv_attend(q, cache, table, _i32(lengths), return_lse=True), q, cache, table, _i32(lengths))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 4, 16), (128, 1, 6, 64), (128, 2, 1, 32), (256, 1, 2, 64)])
@pytest.mark.parametrize("window", [None, 1, 50])
def test_attend_prompts(dim, heads, group, page, window, dtype):
    """Chunks behind cached tokens, whole prompts, single tokens among them, a request without queries and one whose
    lengths leave its first queries nothing to see."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(dim + group)
    lengths, new = [130, 70, 1, 200, 33, 5, 90], [60, 70, 1, 1, 0, 9, 17]
    cache, table = _filled(rng, lengths, heads, dim, page)
    starts = _i32(np.concatenate(([0], np.cumsum(new))).tolist())
    q = _queries(rng, sum(new) + 3, heads * group, dim, dtype)     # three tokens belong to no request
    for max_new in (None, 70, 1):
        _check(kv_attend(q, cache, table, _i32(lengths), starts=starts, window=window, max_new=max_new, return_lse=True), q, cache, table,
               _i32(lengths), starts=starts, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_all_tokens(dtype):
    """Not causal: every query sees all of its request, new or not."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(5)
    lengths, new = [77, 0, 300], [77, 40, 5]
    cache, table = _filled(rng, lengths, 2, 128, 64)
    starts = _i32(np.concatenate(([0], np.cumsum(new))).tolist())
    q = _queries(rng, sum(new), 6, 128, dtype)
    _check(kv_attend(q, cache, table, _i32(lengths), starts=starts, causal=False, return_lse=True), q, cache, table, _i32(lengths), starts=starts,
           causal=False)


def test_attend_lengths_from_one_on():
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(6)
    lengths = list(range(1, 200))
    cache, table = _filled(rng, lengths, 1, 64, 16)
    q = _queries(rng, len(lengths), 2, 64, torch.float32)
    for window in (None, 37):
        _check(kv_attend(q, cache, table, _i32(lengths), window=window, return_lse=True), q, cache, table, _i32(lengths), window=window)


def test_attend_missing_pages():
    """Entries of the table that are -1, not the cache's, or beyond its width: their tokens are not there."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(7)
    lengths = [300, 300, 300, 40]
    cache, table = _filled(rng, lengths, 2, 128, 16)
    table[0, 3] = -1
    table[1, 5:9] = cache.pages
    table[2, :] = -1
    table[3, 0] = -2147483648
    for width, starts in ((table.shape[1], None), (11, None), (table.shape[1], _i32([0, 1, 2, 3, 4]))):
        t = table[:, :width]
        q = _queries(rng, 4, 4, 128, torch.bfloat16)
        _check(kv_attend(q, cache, t, _i32(lengths), starts=starts, max_new=64, return_lse=True), q, cache, t, _i32(lengths), starts=starts)


@pytest.mark.parametrize("what", ["k", "v"])
def test_attend_nan_where_it_is_not_seen(what):
    """A broken token makes the queries NaN that see it, and no other."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(8)
    lengths = [90]
    cache, table = _filled(rng, lengths, 1, 128, 32)
    page = int(table[0, 50 // 32])
    (cache.k_scales if what == "k" else cache.v_scales)[page, 0, 50 % 32] = float("nan")
    starts = _i32([0, 90])
    q = _queries(rng, 90, 4, 128, torch.bfloat16)
    for window in (None, 20):
        got = kv_attend(q, cache, table, _i32(lengths), starts=starts, window=window, return_lse=True)
        want = oracle.attend(q, cache, table, _i32(lengths), starts=starts, window=window)[0]
        seen = np.array([p >= 50 and (window is None or p < 50 + window) for p in range(90)])
        assert np.isnan(want[seen]).all() and not np.isnan(want[~seen]).any()
        out = got[0].float().cpu().numpy()
        assert np.isnan(out[seen]).all() and not np.isnan(out[~seen]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_size,v_size", [(1e-6, 1.0), (30.0, 1.0), (1.0, 1e-5), (1.0, 3e4), (0.0, 1.0), (1.0, 1e-30), (1.0, 1e20)])
def test_attend_sizes_of_numbers(q_size, v_size, dtype):
    """Scores near zero and far apart, values beyond fp16's range on both sides."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(9)
    lengths = [150, 3]
    cache, table = _filled(rng, lengths, 2, 64, 16, dtype=torch.bfloat16, scale_v=v_size)
    q = (_queries(rng, 2, 4, 64, torch.float32) * q_size).to(dtype)
    if dtype == torch.float16 and v_size > 1e10 or dtype == torch.float16 and v_size < 1e-4:
        pytest.skip("not numbers of this type")
    _check(kv_attend(q, cache, table, _i32(lengths), return_lse=True), q, cache, table, _i32(lengths))


def test_attend_values_of_mixed_scales():
    """A first token with most of the weight and a value of almost nothing."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(10)
    lengths = [500]
    cache, table = _filled(rng, lengths, 1, 128, 64)
    cache.v_scales[int(table[0, 0]), 0, 0] *= 2.0 ** -12
    cache.k_scales[int(table[0, 0]), 0, 0] *= 12
    q = _queries(rng, 1, 8, 128, torch.float32)
    _check(kv_attend(q, cache, table, _i32(lengths), return_lse=True), q, cache, table, _i32(lengths))


def test_attend_broken_queries():
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(11)
    lengths = [40, 40, 40]
    cache, table = _filled(rng, lengths, 1, 64, 16)
    q = _queries(rng, 3, 2, 64, torch.float32)
    q[0, 0, 3] = float("nan")
    q[1, 1, 5] = float("inf")
    out = kv_attend(q, cache, table, _i32(lengths))
    broken = torch.isnan(out).all(-1).cpu()
    assert broken.tolist() == [[True, False], [False, True], [False, False]] and torch.isfinite(out[~broken.cuda()]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_strides(dtype):
    """Queries as part of a fused projection, with any beginning, and a table that is part of a wider one."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(12)
    lengths = [70, 200, 5]
    cache, table = _filled(rng, lengths, 2, 64, 16)
    wide = torch.full((3, table.shape[1] + 9), 99999, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    table = wide[:, :table.shape[1]]
    fused = _queries(rng, 3, 10, 64, dtype)
    shifted = torch.empty(3 * 4 * 64 + 5, dtype=dtype, device="cuda")[5:].view(3, 4, 64).copy_(fused[:, :4])
    heads_first = fused[:, 2:6].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    spread = torch.stack((fused[:, :4], fused[:, :4]), -1)[..., 0]
    for q in (fused[:, 4:8], shifted, heads_first, spread, fused[:1, :4].expand(3, 4, 64)):
        _check(kv_attend(q, cache, table, _i32(lengths), return_lse=True), q, cache, table, _i32(lengths))


@pytest.mark.parametrize("scale", [0.05, -0.1, 0.0, 1.0])
def test_attend_scale(scale):
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(13)
    cache, table = _filled(rng, [333], 1, 128, 64)
    q = _queries(rng, 1, 4, 128, torch.bfloat16)
    _check(kv_attend(q, cache, table, _i32([333]), scale=scale, return_lse=True), q, cache, table, _i32([333]), scale=scale)


@pytest.mark.parametrize("max_length", [None, 1, 700, 5000])
def test_attend_hints_cost_time_only(max_length):
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(14)
    lengths = [2500, 640]
    cache, table = _filled(rng, lengths, 1, 64, 64)
    q = _queries(rng, 2, 4, 64, torch.float32)
    _check(kv_attend(q, cache, table, _i32(lengths), max_length=max_length, return_lse=True), q, cache, table, _i32(lengths))


def test_attend_is_the_same_every_time():
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(15)
    lengths, new = [3000, 900, 64], [1, 30, 64]
    cache, table = _filled(rng, lengths, 2, 128, 64)
    starts = _i32(np.concatenate(([0], np.cumsum(new))).tolist())
    q = _queries(rng, sum(new), 8, 128, torch.bfloat16)
    first = kv_attend(q, cache, table, _i32(lengths), starts=starts, return_lse=True)
    for _ in range(5):
        again = kv_attend(q, cache, table, _i32(lengths), starts=starts, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_beyond_32_bits():
    """A cache whose codes pass 2^32 bytes, read and written at its end."""
    from orbitquant_amd import OrbitKVCache, kv_attend, kv_read, kv_write

    rng = np.random.RandomState(16)
    page, heads, dim = 64, 8, 128
    pages = (1 << 32) // (heads * page * dim // 2) + 5
    cache = OrbitKVCache.empty(pages, heads, dim, page_size=page, seed=3)
    table = _i32([[pages - 1, 0, pages - 3]])
    slots = torch.tensor([int(table[0, t // page]) * page + t % page for t in range(150)], device="cuda")
    k, v = (_vectors(rng, 150, heads, dim, torch.bfloat16).cuda() for _ in range(2))
    kv_write(k, v, slots, cache)
    for x, y in zip((k, v), kv_read(slots, cache, torch.float32)):
        codes, scales = oracle.encode(x.float().cpu().numpy(), cache.signs.cpu().numpy())
        np.testing.assert_array_equal(y.cpu().numpy(), oracle.held32(codes, scales, cache.signs.cpu().numpy()))
    q = _queries(rng, 1, 8, dim, torch.bfloat16)
    got = kv_attend(q, cache, table, _i32([150]), return_lse=True)
    small = OrbitKVCache(*(t[[pages - 1, 0, pages - 3]].contiguous() for t in cache[:4]), cache.signs)
    _check(got, q, small, _i32([[0, 1, 2]]), _i32([150]))


# ---------------------------------------------------------------- together, on streams and in graphs

def _step(state):
    from orbitquant_amd import kv_assign, kv_attend, kv_write

    got = kv_assign(state["lengths"], state["new"], state["table"], state["free"], state["taken"], page_size=64, tokens=len(state["k"]))
    kv_write(state["k"], state["v"], got.slots, state["cache"])
    return got, kv_attend(state["q"], state["cache"], state["table"], got.lengths, return_lse=True)


def _step_state(rng, lengths):
    heads, dim = 2, 128
    cache, table = _filled(rng, lengths, heads, dim, 64, extra_columns=2)
    # pages of new tokens: behind the ones in use
    grown = [torch.cat((t, t[:len(lengths)]), 0).contiguous() for t in cache[:4]]
    free = list(range(cache.pages, cache.pages + len(lengths)))
    n = len(lengths)
    return {"lengths": _i32(lengths), "new": _i32([1] * n), "table": table, "free": _i32(free), "taken": _i32([0]), "cache": type(cache)(*grown, cache.signs),
            "q": _queries(rng, n, 8, dim, torch.bfloat16), "k": _queries(rng, n, heads, dim, torch.bfloat16), "v": _queries(rng, n, heads, dim, torch.bfloat16)}


def test_step_on_a_stream_and_in_a_graph():
    """A decoding step captured once and replayed, its lengths and pages moving on between the replays, against the same steps run eagerly on
    another stream."""
    rng = np.random.RandomState(17)
    lengths = [63, 64, 700, 0, 128]
    eager, captured = (_step_state(np.random.RandomState(17), lengths) for _ in range(2))
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _step(captured)
    torch.cuda.current_stream().wait_stream(warm)
    captured = _step_state(np.random.RandomState(17), lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, out = _step(captured)
    side = torch.cuda.Stream()
    for i in range(4):
        fresh = [_queries(rng, 5, s, 128, torch.bfloat16) for s in (8, 2, 2)]
        for state in (eager, captured):
            for name, x in zip("qkv", fresh):
                state[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want_got, want = _step(eager)
        torch.cuda.synchronize()
        for x, y in zip((*got, *out), (*want_got, *want)):
            assert torch.equal(x, y)
        _check(out, captured["q"], captured["cache"], captured["table"], got.lengths)
        for state, g in ((eager, want_got), (captured, got)):
            state["lengths"].copy_(g.lengths)
            state["taken"].copy_(g.taken)
        torch.cuda.synchronize()
    assert captured["taken"].item() >= 3 and captured["lengths"].tolist() == [n + 4 for n in lengths]
