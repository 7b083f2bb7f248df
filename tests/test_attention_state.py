"""`OrbitCachedAttention`'s norms and tables belong to the module: they are saved, loaded, moved and copied with its linears."""

import copy
import io

import pytest
import torch
from torch import nn

from orbitquant_amd import OrbitCachedAttention, OrbitKVCache, OrbitLinear, QKNormRotary, recipe


def _how(weights=True, tables=True, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    angle = torch.arange(50.0)[:, None] * 10.0 ** -torch.arange(16.0)
    cos, sin = (angle.cos(), angle.sin()) if tables else (None, None)
    q, k = ((1 + torch.randn(64, generator=g) / 8).to(dtype) for _ in range(2)) if weights else (None, None)
    return QKNormRotary(cos, sin, q, k, 1e-6 if weights else None, True)


def _layer(rotary, seed=0):
    g = torch.Generator().manual_seed(seed)
    linear = lambda i, o: OrbitLinear.from_weight(torch.randn(o, i, generator=g).to(torch.bfloat16), bias=None, config=recipe("w4a4"))  # noqa: E731
    cache = OrbitKVCache.empty(2, 2, 64, page_size=16, device="cpu")
    return OrbitCachedAttention(linear(128, 256), linear(128, 128), linear(128, 128), linear(256, 128), cache, rotary=rotary)


def _equal(a, b):
    for x, y in zip(a, b, strict=True):
        assert torch.equal(x, y) and x.dtype == y.dtype if isinstance(x, torch.Tensor) else x == y


def test_the_plan_is_what_was_given():
    for how in (_how(), _how(weights=False), _how(tables=False), QKNormRotary(), QKNormRotary(eps=0.5)):
        layer = _layer(how)
        assert isinstance(layer.rotary, QKNormRotary)
        _equal(layer.rotary, how)


def test_weights_are_saved_and_loaded():
    how, other = _how(), _how(seed=1)
    saved, fresh = _layer(how), _layer(other)
    assert not torch.equal(how.q_weight, other.q_weight)
    buffer = io.BytesIO()
    torch.save(saved.state_dict(), buffer)
    buffer.seek(0)
    fresh.load_state_dict(torch.load(buffer, weights_only=True))
    _equal(fresh.rotary, how)
    # one of them alone
    fresh = _layer(other._replace(k_weight=None))
    fresh.load_state_dict(_layer(how._replace(k_weight=None)).state_dict())
    _equal(fresh.rotary, how._replace(k_weight=None))


def test_a_state_without_them_leaves_them_as_they_are():
    """States saved before they were part of one; as strict as ever about the linears."""
    how = _how()
    state = {name: t for name, t in _layer(_how(weights=False)).state_dict().items()}
    layer = _layer(how, seed=1)
    layer.load_state_dict(state)
    _equal(layer.rotary, how)
    del state["q.row_norms"]
    with pytest.raises(RuntimeError, match="q.row_norms"):
        _layer(how).load_state_dict(state)


def test_they_move_with_the_module():
    layer = _layer(_how()).to("meta")
    assert all(t.device.type == "meta" for t in layer.rotary[:4])


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.to(torch.float32), lambda m: m.double().to(torch.bfloat16), lambda m: m.to("cpu", torch.float16)])
def test_tables_stay_fp32(convert):
    """A conversion takes the norms' weights along; tables are fp32 whatever the model is, and lose nothing on the way."""
    how = _how()
    layer = convert(_layer(how))
    assert layer.rotary.q_weight.dtype == layer.rotary.k_weight.dtype != torch.float64
    _equal(layer.rotary[:2], how[:2])
    torch.testing.assert_close(layer.rotary.q_weight.float(), how.q_weight.float(), rtol=0, atol=0)


def test_memory_that_is_not_filled():
    """A skeleton that a state is loaded into: the tables, which no state has, are what they were."""
    how = _how()
    layer, saved = _layer(how), _layer(how).state_dict()
    layer.to_empty(device="cpu")
    layer.load_state_dict(saved)
    _equal(layer.rotary, how)


def test_copies_are_their_own():
    layer = _layer(_how())
    other = copy.deepcopy(layer)
    _equal(other.rotary, layer.rotary)
    with torch.no_grad():
        other.rotary.q_weight.zero_()
    assert layer.rotary.q_weight.abs().sum() > 0 and other.rotary.q_weight.abs().sum() == 0


def test_a_models_own_parameters_stay_those():
    """Weights that are parameters elsewhere in the model are the same ones, updated there and seen here."""
    norm = nn.Parameter(torch.ones(64))
    layer = _layer(QKNormRotary(q_weight=norm, k_weight=norm, eps=1e-6))
    assert layer.rotary.q_weight is norm and layer.rotary.k_weight is norm
    with torch.no_grad():
        norm.mul_(3)
    assert (layer.rotary.k_weight == 3).all()


def test_tables_are_shared_between_layers():
    how = _how()
    layers = nn.ModuleList(_layer(how) for _ in range(3))
    assert len({layer.rotary.cos.data_ptr() for layer in layers}) == 1
    layers.to(torch.bfloat16)
    assert len({layer.rotary.cos.data_ptr() for layer in layers}) == 1
    assert not any("cos" in name or "sin" in name for name in layers.state_dict())


def test_another_one_later():
    layer = _layer(_how())
    how = _how(seed=3)
    layer.rotary = how
    _equal(layer.rotary, how)
    assert torch.equal(layer.state_dict()["q_norm_weight"], how.q_weight)
    layer.rotary = None
    assert layer.rotary is None and "q_norm_weight" not in layer.state_dict()
    call = lambda q, k, positions: (q, k)  # noqa: E731
    layer.rotary = call
    assert layer.rotary is call
    layer.rotary = how
    _equal(layer.rotary, how)


def test_callables_are_as_before():
    call = lambda q, k, positions: (q, k)  # noqa: E731
    assert _layer(call).rotary is call and _layer(None).rotary is None

    class Turn(nn.Module):
        def __init__(self):
            super().__init__()
            self.scale = nn.Parameter(torch.ones(3))

        def forward(self, q, k, positions):
            return q, k

    turn = Turn()
    layer = _layer(turn)
    assert layer.rotary is turn and "rotary.scale" in layer.state_dict() and turn in list(layer.modules())


def test_modules_pickled_before():
    """Whole, when the plan was an attribute like any other."""
    class Turn(nn.Module):
        def forward(self, q, k, positions):
            return q, k

    how, turn = _how(), Turn()
    for rotary in (how, None, turn):
        layer = _layer(rotary)
        state = {name: dict(value) if name in ("_parameters", "_buffers", "_modules") else value for name, value in layer.__dict__.items()}
        for name in ("q_norm_weight", "k_norm_weight"):
            del state["_parameters"][name]
        for name in ("_rotary_cos", "_rotary_sin"):
            del state["_buffers"][name]
        del state["_rotary"]
        if rotary is not turn:
            state["rotary"] = rotary
        old = OrbitCachedAttention.__new__(OrbitCachedAttention)
        old.__setstate__(state)
        if rotary is how:
            _equal(old.rotary, how)
            assert torch.equal(old.state_dict()["k_norm_weight"], how.k_weight)
        else:
            assert old.rotary is rotary
        old.to(torch.float16)
