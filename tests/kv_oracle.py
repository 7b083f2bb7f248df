"""The 4-bit key/value cache and its attention by their definitions: plain loops and 64-bit arithmetic on the host, apart
from the steps that the definition itself states in fp32 (the rotation and the scale of a vector)."""

import math

import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EVEN_FIRST = [0, 2, 4, 6, 1, 3, 5, 7]   # codes in the order in which a tie prefers them


def hadamard32(x: np.ndarray) -> np.ndarray:
    """The unnormalised transform over the last axis, every butterfly one fp32 add or subtract."""
    y = x.astype(np.float32).copy()
    d = 1
    while d < y.shape[-1]:
        p = y.reshape(*y.shape[:-1], -1, 2, d)
        with np.errstate(all="ignore"):
            a, b = p[..., 0, :] + p[..., 1, :], p[..., 0, :] - p[..., 1, :]
        y = np.stack((a, b), -2).reshape(y.shape)
        d *= 2
    return y


def sylvester(dim: int) -> np.ndarray:
    h = np.ones((1, 1))
    while len(h) < dim:
        h = np.block([[h, h], [h, -h]])
    return h


def bf16(x: np.ndarray) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).float().numpy()


def encode(x: np.ndarray, signs: np.ndarray):
    """x fp32 [..., D] -> (codes uint8 [..., D], scales fp32 of bf16 values [...])."""
    y = hadamard32(x.astype(np.float32) * signs.astype(np.float32))
    finite = np.isfinite(y).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(y), y, 0)).max(-1), 0).astype(np.float32)
    scale = bf16(top * np.float32(1.0 / 6.0))
    scale = np.where(scale < 2.0 ** -126, np.float32(0), scale)
    with np.errstate(all="ignore"):
        inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
        z = np.where(finite[..., None], (y * inv[..., None]).astype(np.float32), np.float32(0))
    away = np.abs(np.abs(z)[..., None].astype(np.float64) - GRID[EVEN_FIRST])
    code = np.array(EVEN_FIRST, dtype=np.uint8)[away.argmin(-1)]     # the first of equals: the even one
    code |= (np.signbit(z) & finite[..., None]).astype(np.uint8) << 3
    return code, np.where(finite, scale, np.float32(np.nan))


def decode(codes: np.ndarray) -> np.ndarray:
    return np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]


def held32(codes: np.ndarray, scales: np.ndarray, signs: np.ndarray) -> np.ndarray:
    """What a vector stands for, in the fp32 steps of its definition."""
    y = hadamard32((decode(codes).astype(np.float32) * scales[..., None].astype(np.float32)).astype(np.float32))
    return (y * np.float32(1.0 / codes.shape[-1]) * signs.astype(np.float32)).astype(np.float32)


def cache_codes(cache):
    """(k codes, k scales, v codes, v scales) of an OrbitKVCache as [pages, heads, page, D] and [pages, heads, page]."""
    k, ks, v, vs = (t.cpu() for t in cache[:4])
    v = v.transpose(2, 3)
    nibbles = lambda t: torch.stack((t & 15, t >> 4), -1).flatten(-2).numpy()  # noqa: E731
    return nibbles(k), ks.float().numpy(), nibbles(v), vs.float().numpy()


def assign(lengths, new, table, free, taken, page, tokens):
    """By counting."""
    table = [list(map(int, row)) for row in table]
    width = len(table[0]) if table else 0
    slots, positions, starts, after = [], [], [0], []
    given = max(taken, 0)
    for r, (was, more) in enumerate(zip(lengths, new)):
        was, more = max(was, 0), max(more, 0)
        first_fresh = -(-was // page)
        for column in range(first_fresh, -(-(was + more) // page)):
            if column < width:
                table[r][column] = free[given] if given < len(free) else -1
            given += 1
        for position in range(was, was + more):
            column = position // page
            at = table[r][column] if column < width else -1
            slots.append(at * page + position % page if at >= 0 else -1)
            positions.append(position)
        starts.append(starts[-1] + more)
        after.append(was + more)
    pad = max(0, tokens - len(slots))
    return (slots + [-1] * pad)[:tokens], (positions + [-1] * pad)[:tokens], starts, after, min(given, len(free)), table


def attend(q, cache, table, lengths, starts=None, causal=True, window=None, scale=None):
    """-> (out float64 [tokens, heads, D], lse, bound): `bound` [tokens, heads] has the factors of the error bound, see `allowed`."""
    kc, ks, vc, vs = cache_codes(cache)
    signs = cache[4].cpu().numpy().astype(np.float64)
    pages, kv_heads, page, dim = kc.shape
    turn = sylvester(dim) / dim * signs
    q = q.double().cpu().numpy()
    tokens, heads, _ = q.shape
    group = heads // kv_heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    table, lengths = table.cpu().numpy(), lengths.cpu().tolist()
    starts = list(range(len(lengths) + 1)) if starts is None else starts.cpu().tolist()
    out, lse = np.zeros((tokens, heads, dim)), np.full((tokens, heads), -np.inf)
    size, largest, count = (np.zeros((tokens, heads)) for _ in range(3))
    for r, length in enumerate(lengths):
        length = max(length, 0)
        there = [t for t in range(min(length, table.shape[1] * page)) if 0 <= table[r, t // page] < pages]
        for h in range(kv_heads):
            at = [(table[r, t // page], h, t % page) for t in there]
            if not at:
                continue
            rows = tuple(np.array(x) for x in zip(*at))
            k = (decode(kc[rows]) * ks[rows][:, None]) @ turn
            v = (decode(vc[rows]) * vs[rows][:, None]) @ turn
            place = np.array(there)
            for i in range(starts[r], starts[r + 1]):
                position = length - (starts[r + 1] - starts[r]) + i - starts[r]
                seen = place <= position if causal else np.ones(len(place), bool)
                if window is not None:
                    seen &= place > position - window
                if not seen.any():
                    continue
                for j in range(h * group, (h + 1) * group):
                    with np.errstate(all="ignore"):
                        s = scale * (k[seen] @ q[i, j])
                        m = s.max()
                        w = np.exp(s - m)
                        out[i, j] = (w / w.sum()) @ v[seen]
                        lse[i, j] = m + np.log(w.sum())
                    size[i, j] = abs(scale) * np.linalg.norm(q[i, j]) * np.linalg.norm(k[seen], axis=1).max()
                    largest[i, j] = np.linalg.norm(v[seen], axis=1).max()
                    count[i, j] = seen.sum()
    return out, lse, (size, largest, count, dim)


def allowed(bound, want, dtype):
    """How far a row of the output may be off in the 2-norm, and its lse.

    A query enters the product with a relative error e_q an entry (2^-12 as one fp16, 2^-22 as two parts), which moves a score by
    at most e_q * scale |q| |k|; a weight has e_w; fp32 has its own error in the product over D entries and in sums over the keys.  Weights off by a
    relative e move the normalised sum by at most 2 e max|v|; the output is rounded once."""
    size, largest, count, dim = bound
    e_q = {torch.bfloat16: 2.0 ** -12}.get(dtype, 2.0 ** -21)
    e_w = {torch.float32: 2.0 ** -21}.get(dtype, 2.0 ** -12)
    own = 2.0 ** -23 * (2 * dim + 8) * (size + 1)
    scores = e_q * size + own
    weights = scores + e_w + 2.0 ** -23 * (count / 16 + 64)
    rounding = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12, torch.float32: 2.0 ** -24}[dtype]
    return 2 * weights * largest + 2 * rounding * np.linalg.norm(want, axis=-1) + 1e-7 * (dtype == torch.float16), scores + 2.0 ** -21 * (size + 16)
