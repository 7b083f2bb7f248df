"""The cache's attention where a launch cuts many tiles into parts, the ways into the operators (Python, compiled host code,
`torch.compile`) against each other, and the attention layer and the decoding example that run them together."""

import numpy as np
import pytest
import torch

import kv_oracle as oracle
from test_gpu_kv_cache import _cache, _check, _filled, _i32, _queries, _step, _step_state, _vectors

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- many tiles in parts

@pytest.mark.parametrize("requests,longest,heads,window", [(65, 3000, 1, None), (70, 2500, 3, 1200), (257, 1500, 1, None), (530, 1300, 1, None)])
def test_attend_many_requests_in_parts(requests, longest, heads, window):
    """More tiles than a wavefront has lanes, and more than a workgroup has threads: single tokens of lengths from nothing to long."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(requests)
    lengths = rng.randint(0, longest, requests)
    lengths[rng.rand(requests) < 0.3] //= 50
    lengths[[0, requests // 2, -1]] = longest, 0, longest
    lengths = lengths.tolist()
    cache, table = _filled(rng, lengths, heads, 64, 32)
    q = _queries(rng, requests, 2 * heads, 64, torch.bfloat16)
    for max_length in (None, longest):
        _check(kv_attend(q, cache, table, _i32(lengths), window=window, max_length=max_length, return_lse=True), q, cache, table, _i32(lengths),
               window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("requests,longest,window", [(3, 60, None), (140, 120, 50), (530, 480, None)])
def test_attend_short_and_many(requests, longest, window, dim, page, dtype):
    """A few steps of very many requests, groups of other sizes than the tile's, none and one token among the lengths."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(requests + dim)
    lengths = rng.randint(0, longest + 1, requests)
    lengths[:3] = longest, 0, 1
    lengths = lengths.tolist()
    cache, table = _filled(rng, lengths, 2, dim, page, extra_columns=0)
    q = _queries(rng, requests, 2 * 5, dim, dtype)
    _check(kv_attend(q, cache, table, _i32(lengths), window=window, max_length=longest, return_lse=True), q, cache, table, _i32(lengths), window=window)


@pytest.mark.parametrize("requests,heads", [(40, 16), (65, 8), (300, 2), (400, 1)])
def test_attend_long_requests_in_parts(requests, heads):
    """The same where requests are so long that they are always cut: the tiles of a wavefront, of a few a lane, of the
    whole workgroup, with more parts than the chip holds and with fewer."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(heads)
    lengths = rng.randint(0, 4300, requests)
    lengths[rng.rand(requests) < 0.5] //= 40
    lengths[[0, -1]] = 4300, 4299
    lengths = lengths.tolist()
    cache, table = _filled(rng, lengths, heads, 64, 64)
    q = _queries(rng, requests, heads, 64, torch.float16)
    _check(kv_attend(q, cache, table, _i32(lengths), return_lse=True), q, cache, table, _i32(lengths))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 128)])
@pytest.mark.parametrize("requests", [3, 70])
def test_attend_prompts_and_tokens_in_parts(requests, dim, page, dtype):
    """Chunks of prompts behind long contexts, chunks of a few rows and single tokens in one call, both kernels' tiles in parts."""
    from orbitquant_amd import kv_attend

    rng = np.random.RandomState(requests + dim)
    new = [(1, 150, 5, 0, 40)[i % 5] if requests > 3 else (1, 300, 20)[i] for i in range(requests)]
    lengths = [n + (1100, 1400, 0, 50, 3)[i % 5] for i, n in enumerate(new)]
    cache, table = _filled(rng, lengths, 1, dim, page)
    starts = _i32(np.concatenate(([0], np.cumsum(new))).tolist())
    q = _queries(rng, sum(new), 2, dim, dtype)
    for window in (None, 1250):
        _check(kv_attend(q, cache, table, _i32(lengths), starts=starts, window=window, return_lse=True), q, cache, table, _i32(lengths), starts=starts,
               window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_without_workspace(dtype):
    """The C entry without memory for parts: every tile whole."""
    import ctypes

    from orbitquant_amd import _lib, kv_cache

    rng = np.random.RandomState(20)
    lengths, new = [1500, 1300, 40], [1, 200, 40]
    cache, table = _filled(rng, lengths, 2, 128, 64)
    device_lengths, starts = _i32(lengths), _i32([0, 1, 201, 241])
    q = _queries(rng, 241, 4, 128, dtype)
    out, lse = torch.empty_like(q), torch.empty(241, 4, device="cuda")
    struct = kv_cache._cache_struct(cache, q)
    rc = _lib.load().oq_kv_attend(
        q.data_ptr(), kv_cache._dt(q), 241, 4, q.stride(0), q.stride(1), ctypes.byref(struct), table.data_ptr(), table.stride(0), table.shape[1],
        device_lengths.data_ptr(), starts.data_ptr(), 3, True, 0, 128 ** -0.5, -1, -1, out.data_ptr(), lse.data_ptr(), None, 0,
        kv_cache._stream(q))
    assert rc == 0
    _check((out, lse), q, cache, table, device_lengths, starts=starts)


# ---------------------------------------------------------------- the ways in

def _all_results(state):
    from orbitquant_amd import kv_read

    got, (out, lse) = _step(state)
    keys, values = kv_read(got.slots, state["cache"], torch.float16)
    return [*got, out, lse, keys, values, state["table"]]


def test_python_and_compiled_host_code_agree(monkeypatch):
    from orbitquant_amd import kv_cache

    lengths = [63, 64, 2000, 0, 128]
    compiled = _all_results(_step_state(np.random.RandomState(21), lengths))
    monkeypatch.setattr(kv_cache, "_host", None)
    monkeypatch.setattr(kv_cache, "_module", lambda: None)
    for a, b in zip(compiled, _all_results(_step_state(np.random.RandomState(21), lengths))):
        assert torch.equal(a, b)


def test_under_torch_compile():
    """One graph without breaks, the cache and the table written in place, the same bits."""
    lengths = [63, 64, 700, 0, 128]
    eager, traced = (_step_state(np.random.RandomState(22), lengths) for _ in range(2))
    call = torch.compile(_all_results, fullgraph=True)
    for _ in range(2):
        want, got = _all_results(eager), call(traced)
        for a, b in zip(want, got):
            assert a.dtype == b.dtype and torch.equal(a, b)
        for a, b in zip(eager["cache"], traced["cache"]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for state, result in ((eager, want), (traced, got)):
            state["lengths"].copy_(result[3])
            state["taken"].copy_(result[4])


def test_ops_pass_opcheck():
    rng = np.random.RandomState(23)
    cache, table = _filled(rng, [70, 20], 2, 64, 16)
    q = _queries(rng, 2, 4, 64, torch.bfloat16)
    k = _queries(rng, 2, 2, 64, torch.bfloat16)
    ops = torch.ops.orbitquant_amd
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.kv_assign, (_i32([70, 20]), _i32([1, 1]), table, _i32([3]), _i32([0]), 16, 2), test_utils=tests)
    torch.library.opcheck(ops.kv_write, (k, k, torch.tensor([3, 40], device="cuda"), *cache), test_utils=tests)
    torch.library.opcheck(ops.kv_read, (torch.tensor([3, -1], device="cuda"), *cache, torch.float16), test_utils=tests)
    for with_lse in (False, True):
        torch.library.opcheck(ops.kv_attend, (q, *cache, table, _i32([70, 20]), None, -1, -1, True, 0, 0.125, with_lse), test_utils=tests)


# ---------------------------------------------------------------- the layer and the example

def _layer(cache, heads, hidden, dtype=torch.bfloat16, **kw):
    from orbitquant_amd import OrbitCachedAttention, OrbitLinear, recipe

    generator = torch.Generator(device="cuda").manual_seed(5)

    def linear(inputs, outputs):
        weight = torch.randn(outputs, inputs, generator=generator, device="cuda") / inputs ** 0.5
        return OrbitLinear.from_weight(weight.to(dtype), bias=None, config=recipe("w4a4"))

    width, kv = heads * cache.head_dim, cache.heads * cache.head_dim
    return OrbitCachedAttention(linear(hidden, width), linear(hidden, kv), linear(hidden, kv), linear(width, hidden), cache, **kw)


@pytest.mark.parametrize("window", [None, 40])
def test_layer(window):
    """Prompts, then single tokens: what the cache holds is what the projections gave, and the output is that of the attention
    over it by its definition, through the last projection."""
    from orbitquant_amd import kv_assign, kv_read

    rng = np.random.RandomState(24)
    hidden, heads, page = 256, 4, 16
    cache = _cache(20, 2, 64, page, fill=0xFF)
    calls = []

    def rotary(q, k, positions):
        calls.append(positions.tolist())
        return q * 0.5, k + positions[:, None, None].clamp(max=3).to(k.dtype)

    layer = _layer(cache, heads, hidden, rotary=rotary, window=window)
    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    lengths, taken, free = _i32([0, 0, 0]), _i32([0]), _i32(rng.permutation(20).tolist())
    for new in ([30, 1, 70], [1, 1, 1], [3, 0, 2]):
        x = torch.from_numpy(rng.standard_normal((sum(new), hidden)).astype(np.float32)).to("cuda", torch.bfloat16)
        got = kv_assign(lengths, _i32(new), table, free, taken, page_size=page, tokens=sum(new))
        y = layer(x, got, table, max_new=max(new))
        assert calls[-1] == got.positions.tolist()
        keys = layer.k(x).view(-1, 2, 64) + got.positions[:, None, None].clamp(max=3).to(x.dtype)
        held = kv_read(got.slots, cache, torch.float32)
        for t, plain in zip(held, (keys, layer.v(x).view(-1, 2, 64))):
            codes, scales = oracle.encode(plain.float().cpu().numpy(), cache.signs.cpu().numpy())
            np.testing.assert_array_equal(t.cpu().numpy(), oracle.held32(codes, scales, cache.signs.cpu().numpy()))
        from orbitquant_amd import kv_attend

        q = layer.q(x).view(-1, heads, 64) * 0.5
        attended = kv_attend(q, cache, table, got.lengths, starts=got.starts, window=window, return_lse=True)
        _check(attended, q, cache, table, got.lengths, starts=got.starts, window=window)
        assert y.shape == x.shape
        if max(new) > 1:
            assert torch.equal(y, layer.out(attended[0].reshape(len(x), -1)))
        else:           # single tokens: their queries are counted another way, and parts may be cut elsewhere
            one_each = kv_attend(q, cache, table, got.lengths, max_new=1, window=window)
            assert torch.equal(y, layer.out(one_each.reshape(len(x), -1)))
        lengths, taken = got.lengths, got.taken


def test_layer_refuses():
    from orbitquant_amd import OrbitCachedAttention

    cache = _cache(2, 2, 64, 16)
    fine = _layer(cache, 4, 256)
    with pytest.raises(ValueError, match="cache's 2 heads"):
        OrbitCachedAttention(fine.q, fine.q, fine.v, fine.out, cache)
    with pytest.raises(ValueError, match="multiple of the cache's"):
        OrbitCachedAttention(_layer(_cache(2, 1, 64, 16), 3, 256).q, fine.k, fine.v, fine.out, cache)
    with pytest.raises(ValueError, match="out takes"):
        OrbitCachedAttention(fine.q, fine.k, fine.v, _layer(cache, 2, 256).out, cache)


def test_decode_example(capsys):
    """Replayed steps choose the tokens that the same steps choose when they are run eagerly."""
    from orbitquant_amd.examples import decode

    got = decode.main(["--layers", "2", "--requests", "3", "--tokens", "5", "--prompt", "70"])
    assert "tokens/s" in capsys.readouterr().out and got["bytes_per_token_and_layer"] == 264
    prompts = got["prompts"]
    assert got["pages_taken"] == sum(-(-(n + 5) // decode.PAGE) for n in prompts)
    model, again = (decode.Decoder(2, 3, 70 + 5 + 2) for _ in range(2))
    ids = torch.randint(0, decode.VOCABULARY, (sum(prompts),), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for m in (model, again):
        m.step(ids, _i32(prompts), max_new=max(prompts))
    graph = again.captured_step()
    for _ in range(4):
        want = model.step(model.last.clone(), _i32([1, 1, 1])).clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, again.last) and torch.equal(model.lengths, again.lengths)
        for a, b in zip(model.layers, again.layers):
            used = model.block_table[model.block_table >= 0].long()
            assert used.numel() == int(model.taken)
