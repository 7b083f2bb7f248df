"""`OrbitCachedAttention` with norms and tables of its own on the GPU: moved away and back, converted, loaded, compiled."""

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import _cache, _i32
from test_gpu_kv_serving import _layer
from test_gpu_qk_rotary import _how

pytestmark = pytest.mark.gpu


def _step(layer, x):
    from orbitquant_amd import kv_assign

    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    got = kv_assign(_i32([0, 0, 0]), _i32([3, 1, 9]), table, _i32(list(range(20))), _i32([0]), page_size=16, tokens=13)
    with torch.no_grad():
        return layer(x, got, table)


def _new(seed):
    rng = np.random.RandomState(seed)
    torch.manual_seed(seed)
    return _layer(_cache(20, 2, 64, 16, fill=0xFF), 4, 256, rotary=_how(rng, 64, 32, False, "weights"))


def test_moved_converted_and_loaded():
    layer, x = _new(1), torch.randn(13, 256, device="cuda", dtype=torch.bfloat16)
    want = _step(layer, x)
    layer.to("cpu")
    assert all(t.device.type == "cpu" for t in layer.rotary[:4])
    layer.to("cuda")
    assert all(t.device.type == "cuda" for t in layer.rotary[:4]) and torch.equal(_step(layer, x), want)
    other = _new(2)
    assert not torch.equal(_step(other, x), want)
    other.load_state_dict(layer.state_dict())
    other.rotary = other.rotary._replace(cos=layer.rotary.cos, sin=layer.rotary.sin)
    assert torch.equal(_step(other, x), want)
    layer.half()
    assert layer.rotary.q_weight.dtype == torch.float16 and layer.rotary.cos.dtype == torch.float32


def test_compiled():
    layer, x = _new(3), torch.randn(13, 256, device="cuda", dtype=torch.bfloat16)
    want = _step(layer, x)
    from orbitquant_amd import kv_assign

    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    got = kv_assign(_i32([0, 0, 0]), _i32([3, 1, 9]), table, _i32(list(range(20))), _i32([0]), page_size=16, tokens=13)
    with torch.no_grad():
        assert torch.equal(torch.compile(layer, fullgraph=True)(x, got, table), want)
