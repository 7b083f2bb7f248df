"""Norms and rotary positions on the GPU against their definition, outside of a cache and on the way into one: bit for bit, since every product and
sum of the definition is one IEEE operation in fp32."""

import numpy as np
import pytest
import torch

import kv_oracle
import tree_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _numpy(t):
    return None if t is None else t.float().cpu().numpy()


def _inputs(rng, tokens, heads, dim, dtype):
    x = rng.standard_normal((tokens, heads, dim))
    x[:, :, 1 % dim] *= 8
    return torch.from_numpy(x.astype(np.float32)).to("cuda", dtype)


def _how(rng, dim, rotary, interleaved, norm, dtype=torch.bfloat16, rows=500):
    from orbitquant_amd import QKNormRotary

    cos = sin = q_weight = k_weight = None
    if rotary:
        angle = np.arange(rows)[:, None] * 100.0 ** (-np.arange(rotary // 2) / (rotary // 2))
        cos, sin = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    if norm == "weights":
        q_weight, k_weight = (torch.from_numpy((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32)).to("cuda", dtype) for _ in range(2))
    return QKNormRotary(cos, sin, q_weight, k_weight, None if norm == "none" else 1e-5, interleaved)


def _want(x, how, which, positions):
    """fp32, before the rounding to the output's type."""
    weight = how.q_weight if which == "q" else how.k_weight
    return oracle.norm_rotary32(_numpy(x), _numpy(how.cos), _numpy(how.sin), _numpy(weight), how.eps, how.interleaved,
                                np.arange(len(x)) if positions is None else positions.cpu().numpy())


def _same(got, want):
    want = torch.from_numpy(want).to(got.dtype)
    got = got.cpu()
    both = torch.isnan(got) & torch.isnan(want)
    assert torch.equal(torch.where(both, 0, got), torch.where(both, 0, want))


FORMS = [(128, 128, False, "weights"), (128, 128, True, "weights"), (64, 32, False, "none"), (64, 32, True, "plain"), (256, 0, False, "weights"), (256, 64, False, "weights"),
         (128, 0, False, "none"), (128, 0, True, "plain")]
ODD = [(2, 2, False, "plain"), (2, 2, True, "weights"), (6, 4, False, "weights"), (10, 2, True, "none"), (16, 16, False, "weights"), (18, 18, True, "weights"), (32, 16, False, "weights"),
       (40, 20, False, "weights"), (72, 72, False, "weights"), (72, 36, True, "weights"), (80, 80, True, "weights"), (96, 48, False, "none"), (112, 112, False, "plain"),
       (320, 64, False, "weights"), (510, 250, False, "weights"), (512, 512, True, "weights"), (512, 512, False, "weights")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary,interleaved,norm", FORMS + ODD)
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 5, 2), (37, 9, 4)])
def test_qk_norm_rotary(tokens, heads, kv_heads, dim, rotary, interleaved, norm, dtype):
    from orbitquant_amd import qk_norm_rotary

    rng = np.random.RandomState(dim + rotary + tokens)
    q, k = _inputs(rng, tokens, heads, dim, dtype), _inputs(rng, tokens, kv_heads, dim, dtype)
    how = _how(rng, dim, rotary, interleaved, norm, dtype)
    positions = torch.from_numpy(rng.randint(0, 500, tokens)).to("cuda", torch.int32)
    got = qk_norm_rotary(q, k, how, positions)
    for x, out, which in zip((q, k), got, "qk"):
        assert out.dtype == dtype and out.shape == x.shape and out.is_contiguous()
        want = _want(x, how, which, positions)
        _same(out, want)
        # and the fp32 steps against 64 bits: some ten roundings, each of half a step, on values that are as large as their pair
        weight = how.q_weight if which == "q" else how.k_weight
        real = oracle.norm_rotary64(_numpy(x), _numpy(how.cos), _numpy(how.sin), _numpy(weight), how.eps, how.interleaved, positions.cpu().numpy())
        size = np.abs(real).max(-1, keepdims=True)
        assert (np.abs(want - real) <= 2.0 ** -24 * (12 + np.log2(dim)) * 2 * size).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 72])
def test_positions(dtype, dim):
    """Negative ones turn nothing (a row of infinities stays one), those behind the tables are NaN, and without any a token has its own row."""
    from orbitquant_amd import qk_norm_rotary

    rng = np.random.RandomState(1)
    q, k = _inputs(rng, 6, 3, dim, dtype), _inputs(rng, 6, 1, dim, dtype)
    q[1, 0, 3] = float("inf")
    how = _how(rng, dim, dim // 2, False, "none", dtype, rows=50)
    positions = torch.tensor([-1, -7, 0, 49, 50, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got = qk_norm_rotary(q, k, how, positions)
    for x, out, which in zip((q, k), got, "qk"):
        _same(out, _want(x, how, which, positions))
        assert torch.equal(out[:2], x[:2]) and torch.isnan(out[4:, :, :dim // 2]).all() and torch.equal(out[4:, :, dim // 2:], x[4:, :, dim // 2:])
    for x, out, which in zip((q, k), qk_norm_rotary(q, k, how), "qk"):
        _same(out, _want(x, how, which, None))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_alignment(dtype, interleaved):
    """Parts of a fused projection's output, transposed heads, vectors that begin anywhere, broadcast ones, and a last dimension that is not contiguous."""
    from orbitquant_amd import qk_norm_rotary

    rng = np.random.RandomState(2)
    dim, tokens = 64, 13
    how = _how(rng, dim, dim, interleaved, "weights", torch.float32)
    base = _inputs(rng, tokens, 12, dim + 5, dtype)
    flat = torch.randn(tokens * 9 * dim + 3, device="cuda").to(dtype)
    views = [(base[:, :7, 3:dim + 3], base[:, 8:10, 1:dim + 1]), (_inputs(rng, 7, tokens, dim, dtype).transpose(0, 1), _inputs(rng, 2, tokens, dim, dtype).transpose(0, 1)),
             (flat[3:].view(tokens, 9, dim)[:, 2:], flat[1:-2].view(tokens, 9, dim)[:, ::4]), (_inputs(rng, 1, 5, dim, dtype).expand(tokens, -1, -1), base[:, :1, :dim]),
             (base[..., :2 * (dim // 2)], _inputs(rng, tokens, dim, 3, dtype).transpose(1, 2)), (base[:, :3, 2:dim + 2].flip(0), base[:, 3:4, :dim])]
    shifted = torch.randn(2 * 500 * dim, device="cuda")[1:1 + 500 * dim // 2].view(500, dim // 2)     # tables that begin anywhere
    weight = torch.randn(dim + 1, device="cuda")[1:]
    for q, k in views:
        for plan in (how, how._replace(cos=shifted, sin=shifted), how._replace(q_weight=weight, k_weight=None)):
            positions = torch.from_numpy(rng.randint(0, 500, tokens)).to("cuda", torch.int32)
            for x, out, which in zip((q, k), qk_norm_rotary(q, k, plan, positions), "qk"):
                _same(out, _want(x.contiguous(), plan, which, positions))


def test_sizes_of_numbers():
    """Zeros (of a norm without eps they are NaN, as 0 / 0 is), tiny, huge, infinite and broken values: each row its own affair."""
    from orbitquant_amd import QKNormRotary, qk_norm_rotary

    x = torch.randn(8, 2, 64, device="cuda")
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 2.0 ** 58
    x[3, 0, 5] = float("inf")
    x[4, 1, 6] = float("nan")
    x[5] *= 1e-42
    for eps in (1e-6, 0.0):
        how = QKNormRotary(eps=eps)
        got = qk_norm_rotary(x, x, how)
        for out, which in zip(got, "qk"):
            _same(out, _want(x, how, which, None))
        assert torch.isfinite(got[0][6:]).all() and torch.isfinite(got[0][2]).all()


@pytest.mark.parametrize("heads", [1, 2, 3, 4, 5, 31, 33, 130])
def test_heads(heads):
    from orbitquant_amd import qk_norm_rotary

    rng = np.random.RandomState(heads)
    q, k = _inputs(rng, 70, heads, 32, torch.bfloat16), _inputs(rng, 70, 131 - heads, 32, torch.bfloat16)
    how = _how(rng, 32, 16, False, "weights")
    positions = torch.arange(70, dtype=torch.int32, device="cuda")
    for x, out, which in zip((q, k), qk_norm_rotary(q, k, how, positions), "qk"):
        _same(out, _want(x, how, which, positions))


def test_no_tokens():
    from orbitquant_amd import OrbitKVCache, QKNormRotary, kv_append, qk_norm_rotary

    q, k = (torch.empty(0, h, 64, device="cuda") for h in (4, 2))
    got = qk_norm_rotary(q, k, QKNormRotary(eps=1e-6))
    assert got[0].shape == q.shape and got[1].shape == k.shape
    cache = OrbitKVCache.empty(2, 2, 64)
    assert kv_append(q, k, k, torch.empty(0, dtype=torch.int64, device="cuda"), cache, QKNormRotary()).shape == q.shape


def test_refuses():
    from orbitquant_amd import QKNormRotary, kv_append, qk_norm_rotary

    cache, slots = _cache(2, 2, 64, 16), torch.arange(5, device="cuda")
    q, k = torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 2, 64, device="cuda")
    table, weight, positions = torch.zeros(9, 32, device="cuda"), torch.ones(64, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    fine = QKNormRotary(table, table, weight, weight, 1e-6)

    def both(how, positions, q=q, k=k):
        return (lambda: qk_norm_rotary(q, k, how, positions)), (lambda: kv_append(q, k, k, slots, cache, how, positions))

    for how, at in ((fine._replace(sin=None), positions), (fine._replace(cos=table[:8]), positions), (fine._replace(cos=table[0], sin=table[0]), positions),
                    (fine._replace(cos=table.repeat(1, 2), sin=table.repeat(1, 2)), positions), (fine._replace(cos=table[:, :0], sin=table[:, :0]), positions),
                    (fine._replace(cos=table.half()), positions), (fine._replace(cos=table.cpu()), positions), (fine._replace(q_weight=weight[:63]), positions),
                    (fine._replace(k_weight=weight.half()), positions), (fine._replace(k_weight=weight.int(), q_weight=None), positions), (fine._replace(q_weight=weight.cpu()), positions),
                    (fine._replace(eps=None), positions), (fine._replace(eps=-1.0), positions), (fine._replace(eps=float("nan")), positions),
                    (fine._replace(eps=float("inf")), positions), (fine, positions[:4]), (fine, positions.long()), (fine, positions.cpu()),
                    (fine._replace(cos=table[:4], sin=table[:4]), None)):
        for call in both(how, at):
            with pytest.raises(ValueError):
                call()
    for bad_q, bad_k in ((q[0], k), (q, k[0]), (q, k[:4]), (q, k.half()), (q, k.cpu()), (q, k[..., :32]), (q[:, :0], k), (q, k[:, :0]), (q.double(), k.double()), (q.int(), k.int())):
        for call in both(fine, positions, bad_q, bad_k):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        qk_norm_rotary(q[..., :63], k[..., :63], QKNormRotary())
    with pytest.raises(RuntimeError):
        qk_norm_rotary(torch.zeros(1, 1, 514, device="cuda"), torch.zeros(1, 1, 514, device="cuda"), QKNormRotary())
    for v, where in ((k[:4], slots), (k.half(), slots), (torch.zeros(5, 3, 64, device="cuda"), slots), (k, slots[:4]), (k, slots.int()), (k, slots.cpu())):
        with pytest.raises(ValueError):
            kv_append(q, k, v, where, cache, fine, positions)
    with pytest.raises(ValueError):
        kv_append(q, torch.zeros(5, 3, 64, device="cuda"), torch.zeros(5, 3, 64, device="cuda"), slots, cache, fine, positions)


# ---------------------------------------------------------------- into the cache

def _cache(pages, heads, dim, page, fill=0xA5):
    from orbitquant_amd import OrbitKVCache

    cache = OrbitKVCache.empty(pages, heads, dim, page_size=page)
    for t in cache[:4]:
        t.view(torch.uint8).fill_(fill)
    return cache


def _check_appended(cache, before, k32, v, slots):
    """The tokens' codes and scales are those of the fp32 keys and of the values, and nothing else has changed."""
    signs = cache.signs.cpu().numpy()
    now, was = kv_oracle.cache_codes(cache), kv_oracle.cache_codes(before)
    page = cache.page_size
    touched = np.zeros(was[1].shape, bool)
    for x, codes, scales, old_codes, old_scales in ((k32, now[0], now[1], was[0], was[1]), (v, now[2], now[3], was[2], was[3])):
        want_codes, want_scales = kv_oracle.encode(x, signs)
        for t, slot in enumerate(slots):
            if not 0 <= slot < cache.pages * page:
                continue
            touched[slot // page, :, slot % page] = True
            np.testing.assert_array_equal(codes[slot // page, :, slot % page], want_codes[t])
            np.testing.assert_array_equal(scales[slot // page, :, slot % page], want_scales[t])
        np.testing.assert_array_equal(codes[~touched], old_codes[~touched])
        np.testing.assert_array_equal(scales[~touched], old_scales[~touched])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary,interleaved,norm", FORMS + [(64, 64, False, "plain"), (64, 20, False, "weights"), (128, 64, False, "weights"), (256, 256, False, "weights"),
                                                                 (256, 256, True, "none"), (256, 100, True, "weights"), (128, 96, False, "plain"), (64, 64, True, "weights")])
@pytest.mark.parametrize("tokens,heads,kv_heads,page", [(1, 6, 3, 16), (37, 8, 2, 64)])
def test_kv_append(tokens, heads, kv_heads, page, dim, rotary, interleaved, norm, dtype):
    from orbitquant_amd import kv_append

    rng = np.random.RandomState(dim + rotary + tokens + page)
    both = _inputs(rng, tokens, heads + 2 * kv_heads, dim, dtype)
    q, k, v = both.split((heads, kv_heads, kv_heads), 1)
    how = _how(rng, dim, rotary, interleaved, norm, dtype)
    positions = torch.from_numpy(rng.randint(0, 500, tokens)).to("cuda", torch.int32)
    cache = _cache(6, kv_heads, dim, page)
    before = type(cache)(*(t.clone() for t in cache))
    slots = rng.permutation(6 * page)[:tokens]
    if tokens > 20:
        slots[:20] = np.arange(7, 27)       # a run over a page's end
        slots[20:] = rng.permutation(np.arange(28, 6 * page))[:tokens - 20]
        slots[25], slots[30] = -1, 6 * page
    got = kv_append(q, k, v, torch.from_numpy(slots).cuda(), cache, how, positions)
    _same(got, _want(q, how, "q", positions))
    _check_appended(cache, before, _want(k, how, "k", positions), _numpy(v), slots.tolist())


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_is_the_steps_one_by_one(dtype):
    """`qk_norm_rotary` of the values in fp32, then `kv_write`: the same bits, whatever the strides."""
    from orbitquant_amd import kv_append, kv_write, qk_norm_rotary

    rng = np.random.RandomState(3)
    for dim, rotary, interleaved in ((64, 64, False), (128, 128, True), (128, 32, False), (256, 256, False)):
        how = _how(rng, dim, rotary, interleaved, "weights", dtype)
        base = _inputs(rng, 50, 9, dim + 3, dtype)
        q, k, v = base[:, :4, 1:dim + 1], base[:, 4:6, 2:dim + 2], base[:, 6:8, :dim]
        slots = torch.randperm(4 * 32, device="cuda")[:50]
        positions = torch.randint(0, 500, (50,), dtype=torch.int32, device="cuda")
        one, two = _cache(4, 2, dim, 32), _cache(4, 2, dim, 32)
        got = kv_append(q, k, v, slots, one, how, positions)
        q32, k32 = qk_norm_rotary(q.float(), k.float(), how, positions)
        kv_write(k32, v.float(), slots, two)
        assert torch.equal(got, q32.to(dtype))
        for a, b in zip(one, two):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_broken_keys():
    """A key with an infinity or a position behind the tables is held as NaN, its neighbours as they are."""
    from orbitquant_amd import kv_append, kv_read

    rng = np.random.RandomState(4)
    how = _how(rng, 64, 64, False, "weights", torch.float32, rows=20)
    q, k, v = (_inputs(rng, 5, h, 64, torch.float32) for h in (2, 1, 1))
    k[1, 0, 3] = float("inf")
    positions = torch.tensor([3, 4, 20, -1, 19], dtype=torch.int32, device="cuda")
    cache = _cache(1, 1, 64, 16)
    slots = torch.arange(5, device="cuda")
    kv_append(q, k, v, slots, cache, how, positions)
    held_k, held_v = kv_read(slots, cache, torch.float32)
    assert torch.isnan(held_k[[1, 2]]).all() and torch.isfinite(held_k[[0, 3, 4]]).all() and torch.isfinite(held_v).all()


def test_offsets_beyond_32_bits():
    """Slots whose codes lie behind 4 GiB, in a cache of 5 GiB of keys and as many of values."""
    from orbitquant_amd import OrbitKVCache, kv_append, kv_read

    rng = np.random.RandomState(5)
    cache = OrbitKVCache.empty(5 * 2 ** 13, 16, 128, page_size=128)       # 2^13 pages of 16 heads: 1 GiB of keys
    how = _how(rng, 128, 128, False, "weights")
    q, k, v = (_inputs(rng, 3, h, 128, torch.bfloat16) for h in (16, 16, 16))
    positions = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    slots = torch.tensor([5 * 2 ** 20 - 1, 2 ** 20 + 5, 2 ** 22 + 77], device="cuda")
    kv_append(q, k, v, slots, cache, how, positions)
    signs = cache.signs.cpu().numpy()
    for held, x in zip(kv_read(slots, cache, torch.float32), (_want(k, how, "k", positions), _numpy(v))):
        codes, scales = kv_oracle.encode(x, signs)
        np.testing.assert_array_equal(held.cpu().numpy(), kv_oracle.held32(codes, scales, signs))
