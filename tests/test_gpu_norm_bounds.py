"""Norms of small and large heads against 64 bits: right wherever mean square plus eps is a normal fp32 number and squares are finite."""

import numpy as np
import pytest
import torch

import tree_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 512])
@pytest.mark.parametrize("square,eps", [(2.0 ** -126, 0.0), (2.0 ** -125, 0.0), (2.0 ** -110, 0.0), (2.0 ** -60, 0.0), (2.0 ** -149, 2.0 ** -126), (2.0 ** -200, 2.0 ** -126),
                                        (2.0 ** -126, 2.0 ** -126), (2.0 ** -140, 1e-6), (1.0, 0.0), (2.0 ** 106, 0.0), (2.0 ** 106, 1e-6)])
def test_norms_over_the_range_that_is_stated(dim, square, eps):
    """Each square is off by 2^-24 of itself or, where it is no normal number, by 2^-150 (half the smallest step); sums of such are exact.  Over the head's mean that is 2^-150 beside
    at least 2^-126: one rounding more than the twelve and log2(D) of a head whose squares are all normal."""
    from orbitquant_amd import QKNormRotary, qk_norm_rotary

    rng = np.random.RandomState(dim)
    x = rng.standard_normal((40, 3, dim))
    x[:, :, 1] *= 8
    x *= np.sqrt(square * 1.001 / (x * x).mean(-1, keepdims=True))
    x = torch.from_numpy(x.astype(np.float32)).cuda()
    if eps == 0.0:
        assert ((x.double() ** 2).mean(-1) >= 2.0 ** -126).all()
    assert (x.abs() < 2.0 ** 59).all()
    got = qk_norm_rotary(x, x, QKNormRotary(eps=eps))
    want = oracle.norm_rotary64(x.cpu().numpy(), None, None, None, eps, False, None)
    size = np.abs(want).max(-1, keepdims=True)
    for out in got:
        # (an output may be no normal number itself, where eps is the larger part: half of the smallest step)
        assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -24 * (13 + np.log2(dim)) * 2 * size + 2.0 ** -150).all()
