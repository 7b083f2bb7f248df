"""Norms of queries and keys for each head and their rotary positions, in one launch.

`QKNormRotary` holds what a model's attention has of them (tables of cosines and sines, the norms' weights); `qk_norm_rotary` applies it to
queries and keys, as they come from the projections, for an attention of the model's own; `kv_append` (`kv_cache.py`) does the same on the
way into the 4-bit cache.  For inference: results carry no gradient.  (The reference leaves both to its models' torch code.)
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch.compiler import is_compiling

from . import _lib
from .ops import _DTYPES, _FLOATS, _dt, _OnDevice, _operand, _ptr, _require_gpu, _stream


class QKNormRotary(NamedTuple):
    """How a layer's queries and keys are normed and turned.

    cos, sin     float32 [rows, R/2], R even and at most D: a row for each position; None: nothing is turned
    q_weight, k_weight   [D] of one floating type, or None: the norm has no weight
    eps          of the norms x / sqrt(mean(x^2) + eps) of each head; None: there is no norm
    interleaved  pairs are dimensions 2p and 2p + 1; otherwise p and p + R/2 of the first R

    The norm is each head's own (a model that norms all heads of a projection together needs its own).  Squares are fp32: it is right for values below 2^59
    where mean square + eps is at least 2^-126, which any usual eps sees to.

    Dimensions behind the first R are not turned.  The arithmetic is fp32, rounded once in the end, and stated in include/orbitquant_hip.h."""

    cos: torch.Tensor | None = None
    sin: torch.Tensor | None = None
    q_weight: torch.Tensor | None = None
    k_weight: torch.Tensor | None = None
    eps: float | None = None
    interleaved: bool = False


_LIB = torch.library.Library("orbitquant_amd", "FRAGMENT")
_HOW = "Tensor? cos, Tensor? sin, Tensor? q_weight, Tensor? k_weight, float? eps, bool interleaved"
_LIB.define(f"qk_norm_rotary(Tensor q, Tensor k, {_HOW}, Tensor? positions) -> (Tensor, Tensor)")


def _op(q, k, cos, sin, q_weight, k_weight, eps, interleaved, positions):
    return _general(q, k, QKNormRotary(cos, sin, q_weight, k_weight, eps, interleaved), positions)   # (an op's outputs may not share memory)


_LIB.impl("qk_norm_rotary", _op, "CUDA")
torch.library.register_fake("orbitquant_amd::qk_norm_rotary", lambda q, k, *how: (q.new_empty(q.shape), k.new_empty(k.shape)), lib=_LIB)


_host = None   # what `_module` has found, to be looked at without a call


def _module():
    """The compiled module (csrc/torch_ops.cpp), which has the usual calls without Python in between; None where it is not built."""
    global _host
    _host = _lib.torch_ops()
    if _host is None:
        _lib.warn_without_torch_ops()
    return _host


def _vectors(t: torch.Tensor, name: str, like: torch.Tensor, heads: int | None, dim: int) -> torch.Tensor:
    """[tokens, heads, D] like `like`, with a contiguous last dimension: other strides go to the kernel as they are."""
    if t.ndim != 3 or t.shape[0] != like.shape[0] or t.shape[2] != dim or t.shape[1] == 0 or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [{like.shape[0]}, {'heads' if heads is None else heads}, {dim}], got {list(t.shape)}")
    if t.device != like.device or t.dtype != like.dtype:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, q {like.dtype} on {like.device}")
    return t if t.stride(2) == 1 else t.contiguous()


def _plan(how: QKNormRotary, q: torch.Tensor, positions: torch.Tensor | None) -> tuple[_lib.QkPlanStruct, list]:
    """The plan as the library takes it, and what has to live until the call is made."""
    tokens, _, dim = q.shape
    cos, sin, q_weight, k_weight, eps, interleaved = how
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    rows = rotary = 0
    if cos is None:
        positions = None
    else:
        if cos.ndim != 2 or cos.shape != sin.shape or not 0 < 2 * cos.shape[1] <= dim:
            raise ValueError(f"cos and sin must be [rows, at most {dim // 2}], got {list(cos.shape)} and {list(sin.shape)}")
        rows, rotary = cos.shape[0], 2 * cos.shape[1]
        cos, sin = (_operand(t, name, q, dtype=torch.float32) for t, name in ((cos, "cos"), (sin, "sin")))
        positions = _operand(positions, "positions", q, dtype=torch.int32, numel=tokens)
        if positions is None and rows < tokens:
            raise ValueError(f"{tokens} tokens without positions, and tables of {rows} rows")
    weights = [t for t in (q_weight, k_weight) if t is not None]
    if eps is None and weights:
        raise ValueError("weights of a norm need its eps")
    if eps is not None and not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be a number from 0 on, got {eps}")
    if len({t.dtype for t in weights}) > 1:
        raise ValueError(f"q_weight and k_weight must be of one type, got {weights[0].dtype} and {weights[1].dtype}")
    q_weight, k_weight = (_operand(t, name, q, dtype=_FLOATS, numel=dim) for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")))
    plan = _lib.QkPlanStruct(_ptr(cos), _ptr(sin), rows, rotary, _ptr(positions), _ptr(q_weight), _ptr(k_weight), _DTYPES[weights[0].dtype] if weights else 0,
                             eps is not None, eps or 0.0, bool(interleaved))
    return plan, [cos, sin, positions, q_weight, k_weight]


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, how: QKNormRotary, positions: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries [tokens, heads, D] and keys [tokens, kv_heads, D] normed and turned to their positions (`oq_qk_norm_rotary`): two new tensors.

    q and k: one floating type, any strides whose last is 1 (parts of a fused projection's output need no copy).  D even, at most 512.
    positions: int32 [tokens], rows of the tables; a token at a negative one (of no request) is normed and not turned, one behind
    the tables becomes NaN.  None: token t has row t, as an image's patches have theirs."""
    if is_compiling():
        return torch.ops.orbitquant_amd.qk_norm_rotary(q, k, *how, positions)
    module = _host or _module()
    if module is not None:
        got = module.qk_norm_rotary(q, k, *how, positions)
        if got is not None:
            return got
    return _general(q, k, how, positions)


def _general(q, k, how, positions):
    _require_gpu(q, "q")
    if q.ndim != 3:
        raise ValueError(f"q must be [tokens, heads, D], got {list(q.shape)}")
    tokens, heads, dim = q.shape
    q, k = _vectors(q, "q", q, None, dim), _vectors(k, "k", q, None, dim)
    plan, _keep = _plan(how, q, positions)
    outs = tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    with _OnDevice(q):
        rc = _lib.load().oq_qk_norm_rotary(q.data_ptr(), q.stride(0), q.stride(1), heads, k.data_ptr(), k.stride(0), k.stride(1), k.shape[1], _dt(q), tokens, dim,
                                           ctypes.byref(plan), outs[0].data_ptr(), outs[1].data_ptr(), _stream(q))
    _lib.check(rc, "oq_qk_norm_rotary")
    return outs
