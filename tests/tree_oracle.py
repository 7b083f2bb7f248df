"""Norms and rotary positions, trees of drafted tokens and the accepted path by their definitions, on the host: the fp32 steps that the
definitions state in numpy's fp32, everything else in 64 bits or by counting."""

import math

import numpy as np

from kv_oracle import cache_codes, decode, sylvester

F = np.float32


def pairs(dim, rotary, interleaved):
    """[2, dim / 2]: the dimensions of every pair."""
    p = np.arange(dim // 2)
    if interleaved:
        return np.stack((2 * p, 2 * p + 1))
    if rotary == 0:
        return np.stack((p, p + dim // 2))
    half = rotary // 2
    return np.where(p < half, np.stack((p, p + half)), np.stack((p + half, p + dim // 2)))


def square_sum(a, b):
    """fp32: the squares of a pair, pairs 4, 2, 1 apart of each eight, then eights 1, 2, 4, ... apart."""
    s = a * a + b * b
    width = 8
    while width < s.shape[-1]:
        width *= 2
    s = np.concatenate((s, np.zeros((*s.shape[:-1], width - s.shape[-1]), F)), -1).reshape(*s.shape[:-1], -1, 8)
    for d in (4, 2, 1):
        s = s[..., :d] + s[..., d:2 * d]
    s = s[..., 0]
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    return s


def norm_rotary32(x, cos, sin, weight, eps, interleaved, positions):
    """x [tokens, heads, D], cos and sin [rows, R / 2] or None, weight [D] or None, eps or None, positions [tokens]: all fp32 -> fp32."""
    x = x.astype(F)
    dim = x.shape[-1]
    rotary = 0 if cos is None else 2 * cos.shape[1]
    first, second = pairs(dim, rotary, interleaved)
    a, b = x[..., first], x[..., second]
    with np.errstate(all="ignore"):
        if eps is not None:
            r = F(1) / np.sqrt(square_sum(a, b) * F(1.0 / dim) + F(eps))
            w = np.ones(dim, F) if weight is None else weight.astype(F)
            a, b = (a * r) * w[first], (b * r) * w[second]
        if rotary:
            half = rotary // 2
            at = np.clip(positions, 0, max(0, len(cos) - 1))
            c, s = (np.where((positions >= len(cos))[:, None], F(np.nan), t[at])[:, None].astype(F) for t in (cos, sin))
            u, v = a[..., :half], b[..., :half]
            still = (positions < 0)[:, None, None]
            a = np.concatenate((np.where(still, u, u * c - v * s), a[..., half:]), -1)
            b = np.concatenate((np.where(still, v, v * c + u * s), b[..., half:]), -1)
    out = np.empty_like(x)
    out[..., first], out[..., second] = a, b
    return out


def norm_rotary64(x, cos, sin, weight, eps, interleaved, positions):
    """The same in 64 bits, a pair as a complex number; positions within the tables."""
    x = x.astype(np.float64)
    if eps is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 if weight is None else weight.astype(np.float64))
    if cos is None:
        return x
    turn = (cos.astype(np.float64) + 1j * sin.astype(np.float64))[positions][:, None]
    rotary = 2 * cos.shape[1]
    out = x.copy()
    if interleaved:
        z = (x[..., 0:rotary:2] + 1j * x[..., 1:rotary:2]) * turn
        out[..., 0:rotary:2], out[..., 1:rotary:2] = z.real, z.imag
    else:
        z = (x[..., :rotary // 2] + 1j * x[..., rotary // 2:rotary]) * turn
        out[..., :rotary // 2], out[..., rotary // 2:rotary] = z.real, z.imag
    return out


def tree(parents, starts, lengths, words, tokens):
    """-> (positions, masks as rows of unsigned words)."""
    positions, masks = [-1] * tokens, [[0] * words for _ in range(tokens)]
    for r, length in enumerate(lengths):
        first, count = starts[r], starts[r + 1] - starts[r]
        before = max(length, 0) - count
        paths = []
        for i in range(count):
            if count > 64 * words:
                positions[first + i] = before + i
                continue
            parent = parents[first + i]
            paths.append((paths[parent] if 0 <= parent < i else []) + [i])
            positions[first + i] = before + len(paths[i]) - 1
            for j in paths[i]:
                masks[first + i][j // 64] |= 1 << (j % 64)
    return positions, masks


def signed(masks):
    return [[w - (1 << 64) if w >> 63 else w for w in row] for row in masks]


def seen_by(mask_row, before, new, length, window):
    """The places that a query sees of a request's `length`, `new` of them drafted, by its mask."""
    places = list(range(before)) + [before + j for j in range(new) if mask_row[j // 64] >> (j % 64) & 1]
    return places if window is None else places[-window:]


def attend(q, cache, table, lengths, starts, masks, window=None, scale=None):
    """-> (out float64, lse, bound) as `kv_oracle.attend`; masks: rows of unsigned words."""
    kc, ks, vc, vs = cache_codes(cache)
    signs = cache[4].cpu().numpy().astype(np.float64)
    pages, kv_heads, page, dim = kc.shape
    turn = sylvester(dim) / dim * signs
    q = q.double().cpu().numpy()
    tokens, heads, _ = q.shape
    group = heads // kv_heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    table = table.cpu().numpy()
    words = len(masks[0]) if masks else 1
    out, lse = np.zeros((tokens, heads, dim)), np.full((tokens, heads), -np.inf)
    size, largest, count = (np.zeros((tokens, heads)) for _ in range(3))
    for r, length in enumerate(lengths):
        new = starts[r + 1] - starts[r]
        before = length - new
        there = np.array([t < table.shape[1] * page and 0 <= table[r, t // page] < pages for t in range(length)], bool)
        where = [(table[r, t // page], t % page) if there[t] else (0, 0) for t in range(length)]
        blocks, places = np.array([w[0] for w in where], int), np.array([w[1] for w in where], int)
        for h in range(kv_heads):
            k = (decode(kc[blocks, h, places]) * ks[blocks, h, places][:, None]) @ turn if length else None
            v = (decode(vc[blocks, h, places]) * vs[blocks, h, places][:, None]) @ turn if length else None
            for i in range(starts[r], starts[r + 1]):
                if new > 64 * words:
                    last = before + i - starts[r]
                    own = [t for t in range(max(0, last + 1)) if window is None or t > last - window]
                else:
                    own = seen_by(masks[i], before, new, length, window)
                own = [t for t in own if 0 <= t < length and there[t]]
                if not own:
                    continue
                for j in range(h * group, (h + 1) * group):
                    with np.errstate(all="ignore"):
                        s = scale * (k[own] @ q[i, j])
                        m = s.max()
                        w = np.exp(s - m)
                        out[i, j] = (w / w.sum()) @ v[own]
                        lse[i, j] = m + np.log(w.sum())
                    size[i, j] = abs(scale) * np.linalg.norm(q[i, j]) * np.linalg.norm(k[own], axis=1).max()
                    largest[i, j] = np.linalg.norm(v[own], axis=1).max()
                    count[i, j] = len(own)
    return out, lse, (size, largest, count, dim)


def keep(kept, lengths, starts, slots, table, free, taken, page):
    """-> (moves (from, to) in order, lengths, free list, taken)."""
    free = list(free)
    moves, after, back = [], [], []
    for r, length in enumerate(lengths):
        new = starts[r + 1] - starts[r]
        last, count = -1, 0
        for k in kept[r]:
            if k <= last or k >= new or slots[starts[r] + k] < 0:
                break
            moves.append((slots[starts[r] + k], slots[starts[r] + count]))
            last, count = k, count + 1
        after.append(max(length - new, 0) + count)
        width = len(table[r])
        back += [p for p in table[r][min(width, -(-after[-1] // page)): min(width, -(-length // page))] if p >= 0]
    begin = taken - len(back)
    for i, p in enumerate(back):
        if begin + i >= 0:
            free[begin + i] = p
    return moves, after, free, max(begin, 0)
