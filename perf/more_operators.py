"""Norms and rotary positions on their way into the 4-bit key/value cache, and trees of drafted tokens over it, as measurable cases.

A case is a dict of plain values.  `listed()` gives the named ones, `draw(rng)` one more of the same ranges,
`prepare(case, seed)` what a program holds before the call, `run(state)` one pass (the package's calls where `own` is true,
elementary torch operations in 32 bits where it is not), `exact(case, seed)` the definition in 64 bits, and `work(case)` the
bytes and operations that one pass cannot do without.

Kinds of work:
  rotary   queries and keys [tokens, heads, D]: each head's root-mean-square norm with a weight, then the rotary positions.  The D
           values of a head are D/2 pairs: 2p and 2p+1 (interleaved), or p and p + R/2 of the first R and likewise of the rest.
             y = x * (1 / sqrt(sum(x^2) / D + eps)) * w;  a pair (y0, y1), of the first R/2, becomes (y0 c - y1 s, y1 c + y0 s)
           in fp32, every product and sum rounded by itself; a head's squares are added pair by pair, then pairs 4, 2, 1, 8, 16, ... apart.
  append   the same, and the key goes into the cache as it is, without a rounding in between; with it the value, unrotated
  tree     positions and masks of drafted tokens from their parents: token i of a request's new ones sees those on its path
  attend   attention of drafted tokens over the cache: what was there before, and of the new tokens those of the query's mask
  keep     the accepted path of every tree: its entries move together in the caches of all layers, the other pages are given back

The cache.  A token's key (or value) of one head, x[D], is held as y = H(signs * x) with H the unnormalised Walsh-Hadamard
transform (butterflies of distance 1, 2, 4, ...): one scale a = bf16(max|y| / 6) and D codes in four bits, the nearest E2M1
value (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign, ties to the even code) of y / a.  It stands for signs * H(a * code) / D.
Pages of `page` tokens; a slot is page index * page + place in the page:
  k_codes [pages, heads, page, D/2] uint8    byte j of a token: dimensions 2j (low four bits) and 2j+1
  v_codes [pages, heads, D/2, page] uint8    the same bytes, a page's tokens side by side
  k_scales, v_scales [pages, heads, page] bfloat16
"""

from __future__ import annotations

import math
from functools import reduce

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
MOST = 64        # drafted tokens of a word of a mask


def _case(kind, name=None, **kw):
    case = {"kind": kind, **kw}
    return case if name is None else {"name": name, **case}


def listed() -> list[dict]:
    return [
        # the next token of one conversation through a 4096-wide layer with eight shared heads, outside of a cache: latency
        _case("rotary", "rotary one", tokens=1, queries=32, heads=8, dim=128, rotary=128, interleaved=False, norm=True, dtype="bf16"),
        # the largest by bytes: a video DiT's queries and keys, 21 latent frames of 30 x 52 patches, 40 heads of their own
        _case("rotary", "rotary video", tokens=32760, queries=40, heads=40, dim=128, rotary=128, interleaved=True, norm=True, dtype="bf16"),
        # the same token into the cache
        _case("append", "append one", tokens=1, queries=32, heads=8, dim=128, rotary=128, interleaved=False, norm=True, page=64, dtype="bf16"),
        # a prompt of odd length in half precision: short heads, half of their dimensions turned, no norms, small pages
        _case("append", "append odd fp16", tokens=333, queries=15, heads=5, dim=64, rotary=32, interleaved=False, norm=False, page=16, dtype="fp16"),
        # a long prompt's queries, keys and values
        _case("append", "append prompt", tokens=8192, queries=32, heads=8, dim=128, rotary=128, interleaved=False, norm=True, page=64, dtype="bf16"),
        # a small tree of one conversation
        _case("tree", "tree one", requests=1, longest=2000, nodes=26),
        # trees of a full serving batch, ragged, the widest of 250 nodes
        _case("tree", "tree many", requests=64, longest=16384, nodes=250),
        # one conversation, a context of a thousand tokens, a small tree: latency
        _case("attend", "drafts one", requests=1, longest=1003, nodes=26, queries=32, heads=8, dim=128, page=64, dtype="bf16", window=0),
        # wide heads in single precision over a sliding window, a group of three, a few drafts each, ragged
        _case("attend", "drafts window fp32", requests=7, longest=5000, nodes=13, queries=12, heads=4, dim=256, page=32, dtype="fp32", window=1500),
        # the largest by operations: a serving batch, long ragged contexts, full trees
        _case("attend", "drafts batch", requests=16, longest=16384, nodes=60, queries=32, heads=8, dim=128, page=64, dtype="bf16", window=0),
        # one conversation of a small model of two layers
        _case("keep", "keep one", requests=1, longest=1003, nodes=26, depth=5, layers=2, heads=8, dim=128, page=16, dtype="bf16"),
        # a serving batch, eight layers' caches
        _case("keep", "keep batch", requests=64, longest=4096, nodes=60, depth=8, layers=8, heads=8, dim=128, page=64, dtype="bf16"),
    ]


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "rotary", "append", "append", "tree", "attend", "attend", "attend", "keep"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    wide = 2 if dtype == "fp32" else 1
    if kind == "tree":
        return _case(kind, requests=_log_int(rng, 1, 64), longest=_log_int(rng, 256, 16384), nodes=_log_int(rng, 1, 250))
    heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16, 32])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 6, 7, 8])
    page = rng.choice([16, 32, 64, 64, 128])
    if kind in ("rotary", "append"):
        dim = rng.choice([64, 128, 128, 256]) if kind == "append" else rng.choice([40, 64, 72, 80, 96, 128, 128, 256])
        rotary = rng.choice([dim, dim, dim, dim // 2, 0])
        rotary -= rotary % 2
        interleaved = rng.random() < 0.4
        queries = heads * group
        most = 32760 * 80 * 128 if kind == "rotary" else 8192 * 48 * 128
        tokens = _log_int(rng, 1, max(1, most // ((queries + heads * (1 if kind == "rotary" else 2)) * dim * wide)))
        case = _case(kind, tokens=min(tokens, 40000), queries=queries, heads=heads, dim=dim, rotary=rotary, interleaved=interleaved,
                     norm=rotary == 0 or rng.random() < 0.7, dtype=dtype)
        return case if kind == "rotary" else case | {"page": page}
    dim = rng.choice([64, 128, 128, 256])
    nodes = _log_int(rng, 1, 250)
    same = {"nodes": nodes, "heads": heads, "dim": dim, "page": page, "dtype": dtype}
    if kind == "keep":
        layers = _log_int(rng, 1, 8)
        requests = _log_int(rng, 1, 64)
        longest = max(nodes, _log_int(rng, 64, max(64, min(16384, 64 * 4096 * 8 * 8 * 128 // (requests * heads * dim * layers)))))
        return _case(kind, requests=requests, longest=longest, depth=rng.randint(1, min(12, nodes)), layers=layers, **same)
    requests = _log_int(rng, 1, 64)
    pairs = 16 * 60 * 16384 * 32 * 128 // (2 * heads * group * dim * wide * wide)     # half of the largest listed case's operations
    longest = max(nodes, _log_int(rng, nodes, max(nodes, min(131101, pairs // (requests * nodes)))))
    return _case(kind, requests=requests, longest=longest, queries=heads * group, window=_log_int(rng, 16, 4096) if rng.random() < 0.25 else 0, **same)


# ---------------------------------------------------------------- sizes that follow from a case

def _ragged(case: dict) -> tuple[list[int], list[int]]:
    """(tokens cached before the pass, drafted tokens) of each request: by the case alone, so that `work` knows them.  One
    request has the longest context and the widest tree; the others spread below it.  `longest` counts the drafted tokens."""
    n, longest, nodes = case["requests"], case["longest"], case["nodes"]
    before, new = [], []
    for r in range(n):
        share = 1.0 if r == n // 2 else 0.2 + 0.8 * ((r * 0.6180339887) % 1.0)
        count = nodes if r == n // 2 else max(1, round(nodes * (0.3 + 0.7 * ((r * 0.7548776662) % 1.0))))
        before.append(max(0, round(longest * share) - count))
        new.append(count)
    return before, new


def _words(case: dict) -> int:
    return -(-case["nodes"] // MOST)


def _pages(case: dict) -> list[int]:
    return [-(-(b + n) // case["page"]) for b, n in zip(*_ragged(case))]


def work(case: dict) -> dict:
    kind = case["kind"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if kind in ("rotary", "append"):
        t, dim, heads, queries = case["tokens"], case["dim"], case["heads"], case["queries"]
        table = t * (4 * case["rotary"] + 4)
        a_value = 6 * case["norm"] + 3 * case["rotary"] / dim
        if kind == "rotary":
            values = t * (queries + heads) * dim
            return {"bytes": 2 * values * size + table, "flops": a_value * values}
        held = heads * (dim + 4)                            # bytes of a token: two times D/2 codes and two scales
        return {"bytes": t * ((2 * queries + 2 * heads) * dim * size + held + 8) + table,
                "flops": t * (a_value * (queries + heads) * dim + heads * dim * 2.0 * (math.log2(dim) + 6))}
    before, new = _ragged(case)
    if kind == "tree":
        return {"bytes": sum(new) * (8 + 8 * _words(case)) + 8 * len(new) + 4, "flops": 4.0 * sum(new)}
    heads, dim = case["heads"], case["dim"]
    held = heads * (dim + 4)
    if kind == "keep":
        kept = sum(_kept_counts(case))
        return {"bytes": case["layers"] * kept * 2 * held + 8 * kept + 16 * len(new), "flops": float(kept)}
    window = case["window"] or case["longest"]
    tokens = sum(min(b, window) + n for b, n in zip(before, new))
    pairs = sum(n * min(b + 1, window) for b, n in zip(before, new))
    return {"bytes": tokens * held + sum(new) * (2 * case["queries"] * dim * size + 8 * _words(case)) + 4 * tokens // case["page"],
            "flops": 4.0 * pairs * case["queries"] * dim}


def _kept_counts(case: dict) -> list[int]:
    """Accepted tokens of each request, the last certain one among them."""
    return [min(n, 1 + (r * 5 + 3) % case["depth"]) if case["requests"] > 1 else min(n, case["depth"]) for r, n in enumerate(_ragged(case)[1])]


# ---------------------------------------------------------------- inputs

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _vectors(g, tokens: int, heads: int, dim: int, keys: bool, dtype=torch.float32) -> torch.Tensor:
    """Keys: N(0, 1) with two channels of a head eight times as large, as rotary models show; values: N(0, 1)."""
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda")
    if keys:
        x[:, :, 1] *= 8
        x[:, :, dim // 2 + 1] *= 8
    return x.to(dtype)


def _empty_cache(pages: int, heads: int, dim: int, page: int, signs) -> tuple:
    codes = torch.zeros(2, pages, heads, page * dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, pages, heads, page, dtype=torch.bfloat16, device="cuda")
    return (codes[0].view(pages, heads, page, dim // 2), scales[0], codes[1].view(pages, heads, dim // 2, page), scales[1], signs)


def _filled_cache(g, pages: int, heads: int, dim: int, page: int) -> tuple:
    cache = _empty_cache(pages, heads, dim, page, (torch.randint(0, 2, (dim,), generator=g, device="cuda") * 2 - 1).to(torch.int8))
    chunk = max(1, (1 << 27) // (heads * page * dim))
    for at in range(0, pages, chunk):
        slots = torch.arange(at * page, min(at + chunk, pages) * page, device="cuda")
        v = _vectors(g, len(slots), heads, dim, False)
        _plain_write(_vectors(g, len(slots), heads, dim, True), v, slots, cache)
    return cache


def _put(values, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(values, dtype=dtype, device="cuda")


def _norm_rotary(g, case: dict) -> dict:
    """q, k (and v), parts of one projection's output; the tables of the positions that the model has, norms' weights."""
    t, dim, queries, heads, dtype = case["tokens"], case["dim"], case["queries"], case["heads"], DTYPES[case["dtype"]]
    parts = [_vectors(g, t, queries, dim, True, dtype), _vectors(g, t, heads, dim, True, dtype)]
    if case["kind"] == "append":
        parts.append(_vectors(g, t, heads, dim, False, dtype))
    both = torch.cat(parts, 1)
    state = dict(zip(("q", "k", "v"), both.split([p.shape[1] for p in parts], 1)))
    state |= {"cos": None, "sin": None, "positions": None, "q_weight": None, "k_weight": None, "eps": None, "interleaved": case["interleaved"]}
    if case["rotary"]:
        rows, half = t + 1000, case["rotary"] // 2
        speed = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * speed
        first = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        state |= {"cos": angle.cos().float(), "sin": angle.sin().float(), "positions": torch.arange(first, first + t, dtype=torch.int32, device="cuda")}
    if case["norm"]:
        weight = lambda: (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype)  # noqa: E731
        state |= {"q_weight": weight(), "k_weight": weight(), "eps": EPS}
    return state


def _parents(g, counts: list[int]) -> list[int]:
    """Drafted tokens in the order of their depth: each hangs on one of the few in front of it."""
    parents = []
    for n in counts:
        back = torch.randint(1, 9, (n,), generator=g, device="cuda").tolist()
        parents += [max(0, i - b) if i else -1 for i, b in enumerate(back)]
    return parents


def _batch(g, case: dict) -> dict:
    """Lengths, starts and trees of a batch; its pages anywhere in the pool."""
    before, new = _ragged(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    parents = _parents(g, new)
    state = {"parents": _put(parents), "starts": _put(starts), "lengths": _put([b + n for b, n in zip(before, new)]), "tokens": starts[-1],
             "nodes": case["nodes"], "longest": case["longest"], "counts": (before, new)}
    if "page" in case:
        need = _pages(case)
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32).cpu()
        table = torch.full((len(before), max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        # the free list as it stands after the step that drafted: first what it has given out
        state |= {"pages": pages, "page": case["page"], "table": table.cuda(), "free": order.cuda(), "taken": _put([at])}
    return state


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    kind = case["kind"]
    state = {"kind": kind}
    if kind in ("rotary", "append"):
        state |= _norm_rotary(g, case)
        if kind == "append":
            t, page, heads, dim = case["tokens"], case["page"], case["heads"], case["dim"]
            pages = -(-t // page) + 3
            state["cache"] = _empty_cache(pages, heads, dim, page, (torch.randint(0, 2, (dim,), generator=g, device="cuda") * 2 - 1).to(torch.int8))
            # the tokens' slots: runs of a page in a row, the pages anywhere
            order = torch.randperm(pages, generator=g, device="cuda")[: -(-t // page)]
            state["slots"] = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:t].contiguous()
            state["dtype"] = DTYPES[case["dtype"]]
        return state
    state |= _batch(g, case)
    if kind == "tree":
        return state
    heads, dim, page, dtype = case["heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    if kind == "attend":
        state["cache"] = _filled_cache(g, state["pages"], heads, dim, page)
        firsts = state["table"][:, 0].clamp(min=0).long()
        state["cache"][3][firsts, :, 0] *= 0.0625           # a first token's value is small
        state["q"] = torch.randn(state["tokens"], case["queries"], dim, generator=g, device="cuda").to(dtype)
        state["masks"] = _plain_tree(state)[1]
        return state | {"window": case["window"] or None, "scale": 1.0 / math.sqrt(dim)}
    state["caches"] = [_filled_cache(g, state["pages"], heads, dim, page) for _ in range(case["layers"])]
    # slots as the step's assignment gave them, and a path down each tree: past its first token somewhere behind the places that it moves to
    before, new = state["counts"]
    position = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)])
    request = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    state["slots"] = (state["table"].cpu()[request, position // page].long() * page + position % page).cuda()
    kept = torch.full((len(new), case["depth"]), -1, dtype=torch.int32)
    for r, (n, count) in enumerate(zip(new, _kept_counts(case))):
        path = torch.arange(count)
        if n >= 2 * count:
            path[1:] = torch.randperm(n - count, generator=g, device="cuda").cpu()[:count - 1].sort().values + count
        kept[r, :count] = path
    return state | {"kept": kept.cuda(), "dtype": dtype}


# ---------------------------------------------------------------- one pass

def run(s: dict):
    return (_run_own if own else _run_plain)(s)


def _run_own(s: dict):
    from orbitquant_amd import OrbitKVCache, QKNormRotary, ops

    kind = s["kind"]
    if kind in ("rotary", "append"):
        how = QKNormRotary(s["cos"], s["sin"], s["q_weight"], s["k_weight"], s["eps"], s["interleaved"])
        if kind == "rotary":
            return ops.qk_norm_rotary(s["q"], s["k"], how, s["positions"])
        cache = OrbitKVCache(*s["cache"])
        q = ops.kv_append(s["q"], s["k"], s["v"], s["slots"], cache, how, s["positions"])
        return (q, *ops.kv_read(s["slots"], cache, s["dtype"]))
    if kind == "tree":
        return tuple(ops.kv_tree(s["parents"], s["starts"], s["lengths"], max_new=s["nodes"]))
    if kind == "attend":
        return ops.kv_attend(s["q"], OrbitKVCache(*s["cache"]), s["table"], s["lengths"], starts=s["starts"], masks=s["masks"], max_new=s["nodes"],
                             max_length=s["longest"], window=s["window"], scale=s["scale"])
    caches = [OrbitKVCache(*c) for c in s["caches"]]
    lengths, taken = ops.kv_keep(s["kept"], s["lengths"], s["starts"], s["slots"], caches, block_table=s["table"], free_pages=s["free"], taken=s["taken"])
    where = _targets(s)
    return lengths, taken, s["free"], *(x for c in caches for x in ops.kv_read(where, c, s["dtype"]))


def _run_plain(s: dict):
    kind = s["kind"]
    if kind == "rotary":
        return tuple(_plain_norm_rotary(s[x], s, s[x + "_weight"]).to(s[x].dtype) for x in ("q", "k"))
    if kind == "append":
        q = _plain_norm_rotary(s["q"], s, s["q_weight"]).to(s["q"].dtype)
        _plain_write(_plain_norm_rotary(s["k"], s, s["k_weight"]), s["v"], s["slots"], s["cache"])
        return (q, *_plain_read(s["slots"], s["cache"], s["dtype"]))
    if kind == "tree":
        return _plain_tree(s)
    if kind == "attend":
        return _plain_attend(s)
    lengths, taken = _plain_keep(s)
    where = _targets(s)
    return lengths, taken, s["free"], *(x for c in s["caches"] for x in _plain_read(where, c, s["dtype"]))


def _targets(s: dict) -> torch.Tensor:
    """The slots that a request's first new tokens have, as many as may be kept; -1 behind them."""
    at = s["starts"][:-1, None] + torch.arange(s["kept"].shape[1], dtype=torch.int32, device="cuda")
    return torch.where(at < s["starts"][1:, None], s["slots"][at.clamp(max=len(s["slots"]) - 1).long()], -1).reshape(-1)


# ---------------------------------------------------------------- the plain forms

def _pairs(dim: int, rotary: int, interleaved: bool) -> torch.Tensor:
    """[2, D/2]: the first and second dimension of every pair."""
    p = torch.arange(dim // 2, device="cuda")
    if interleaved:
        return torch.stack((2 * p, 2 * p + 1))
    half, rest = rotary // 2, (dim - rotary) // 2
    if half == 0:
        return torch.stack((p, p + dim // 2))
    first = torch.where(p < half, p, p + half)
    return torch.stack((first, first + torch.where(p < half, half, rest)))


def _tree_sum(x: torch.Tensor) -> torch.Tensor:
    """Sums over the last axis: entries 4, 2, 1 apart of each eight, then neighbours of what is left."""
    width = 8
    while width < x.shape[-1]:
        width *= 2
    x = torch.nn.functional.pad(x, (0, width - x.shape[-1])).unflatten(-1, (-1, 8))
    x = x[..., :4] + x[..., 4:]
    x = x[..., :2] + x[..., 2:]
    x = x[..., 0] + x[..., 1]
    while x.shape[-1] > 1:
        x = x[..., 0::2] + x[..., 1::2]
    return x


def _plain_norm_rotary(x: torch.Tensor, s: dict, weight) -> torch.Tensor:
    dim = x.shape[-1]
    rotary = 0 if s["cos"] is None else 2 * s["cos"].shape[1]
    first, second = _pairs(dim, rotary, s["interleaved"])
    x = x.float()
    a, b = x[..., first], x[..., second]
    if s["eps"] is not None:
        share = torch.reciprocal(torch.sqrt(_tree_sum(a * a + b * b) * (1.0 / dim) + s["eps"]))
        a, b = a * share * weight.float()[first], b * share * weight.float()[second]
    if rotary:
        rows = s["positions"].long()
        cos, sin = s["cos"][rows][:, None], s["sin"][rows][:, None]
        half = rotary // 2
        u, v = a[..., :half], b[..., :half]
        a, b = torch.cat((u * cos - v * sin, a[..., half:]), -1), torch.cat((v * cos + u * sin, b[..., half:]), -1)
    out = torch.empty_like(x)
    out[..., first], out[..., second] = a, b
    return out


def _plain_tree(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """By the path's steps: every token looks at its parent's parent until nobody has one."""
    starts, parents = s["starts"].long(), s["parents"].long()
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(starts[1:], token, right=True)
    index = token - starts[request]
    words = -(-s["nodes"] // MOST)
    word = torch.arange(words, device="cuda")
    bit = lambda i: torch.where(i[:, None] // MOST == word, torch.ones_like(i)[:, None] << (i % MOST)[:, None], 0)  # noqa: E731
    masks, depth, at = bit(index), torch.zeros_like(index), parents.clone()
    for _ in range(s["nodes"]):
        there = at >= 0
        masks = masks | torch.where(there[:, None], bit(at.clamp(min=0)), 0)
        depth += there
        at = torch.where(there, parents[(starts[request] + at).clamp(min=0)], -1)
    new = starts[1:] - starts[:-1]
    return ((s["lengths"].long() - new)[request] + depth).int(), masks


def _butterfly(x: torch.Tensor, distance: int) -> torch.Tensor:
    pairs = x.view(*x.shape[:-1], -1, 2, distance)
    a, b = pairs[..., 0, :], pairs[..., 1, :]
    return torch.stack((a + b, a - b), -2).view(x.shape)


def _hadamard(x: torch.Tensor) -> torch.Tensor:
    return reduce(_butterfly, [1 << i for i in range(x.shape[-1].bit_length() - 1)], x.contiguous())


def _plain_quantize(x: torch.Tensor, signs: torch.Tensor):
    """(bytes [..., D/2], scales [...]) of vectors."""
    y = _hadamard(x.float() * signs)
    top = y.abs().amax(-1)
    scale = (top * (1.0 / 6.0)).to(torch.bfloat16)
    scale = torch.where(scale.float() < 2.0 ** -126, 0.0, scale)
    scale = torch.where(torch.isfinite(top), scale, math.nan).to(torch.bfloat16)
    a = scale.float()
    z = (y * torch.where(a > 0, torch.reciprocal(a), 0.0)[..., None])
    m = z.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)) | ((z < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _values_table(device) -> torch.Tensor:
    """[256, 2]: what the two codes of a byte stand for."""
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    v = torch.cat((v, -v))
    return torch.stack((v.repeat(16), v.repeat_interleave(16)), 1)


def _plain_write(k, v, slots, cache) -> None:
    k_codes, k_scales, v_codes, v_scales, signs = cache
    page = k_codes.shape[2]
    at, place = slots // page, slots % page
    codes, scales = _plain_quantize(k, signs)
    k_codes[at, :, place], k_scales[at, :, place] = codes, scales
    codes, scales = _plain_quantize(v, signs)
    v_codes[at, :, :, place], v_scales[at, :, place] = codes, scales


def _plain_read(slots, cache, dtype):
    """Zeros where a slot is negative."""
    k_codes, k_scales, v_codes, v_scales, signs = cache
    page, dim = k_codes.shape[2], len(signs)
    there = (slots >= 0)[:, None, None]
    at, place = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    table = _values_table(signs.device)
    out = ((k_codes[at, :, place], k_scales[at, :, place]), (v_codes[at, :, :, place], v_scales[at, :, place]))
    back = lambda c, a: torch.where(there, _hadamard(table[c.int()].flatten(-2) * a.float()[..., None]) * (1.0 / dim) * signs, 0.0).to(dtype)  # noqa: E731
    return back(*out[0]), back(*out[1])


def _plain_attend(s: dict) -> torch.Tensor:
    """Request by request, its pages gathered."""
    k_codes, k_scales, v_codes, v_scales, signs = s["cache"]
    dim, heads, page = len(signs), k_codes.shape[1], s["page"]
    group = s["q"].shape[1] // heads
    table = _values_table(signs.device)
    queries = _hadamard(s["q"].float() * signs) * (s["scale"] / dim)
    out = torch.empty_like(queries)
    start = 0
    for r, (before, new) in enumerate(zip(*s["counts"])):
        length = before + new
        # pages that lie wholly before every query's window are not looked at
        skip = max(0, before - s["window"]) // page * page if s["window"] else 0
        pages = s["table"][r, skip // page: -(-length // page)].long()
        keys = table[k_codes[pages].transpose(0, 1).flatten(1, 2).int()].flatten(-2) * k_scales[pages].transpose(0, 1).flatten(1, 2).float()[..., None]
        masks = s["masks"][start: start + new]
        place = torch.arange(skip, skip + keys.shape[1], device="cuda")
        drafted = (place - before).clamp(min=0, max=new - 1)
        bits = (masks[:, drafted // MOST] >> (drafted % MOST)) & 1
        seen = (place < before) | ((place < length) & (bits == 1))
        if s["window"]:
            seen &= seen.flip(-1).cumsum(-1).flip(-1) <= s["window"]
        q = queries[start: start + new].view(new, heads, group, dim).permute(1, 0, 2, 3).reshape(heads, new * group, dim)
        score = torch.matmul(q, keys.transpose(1, 2).contiguous()).view(heads, new, group, -1)
        del keys
        score.masked_fill_(~seen[:, None], -math.inf)
        score -= score.amax(-1, keepdim=True).clamp(min=-3e38)
        score.exp_()
        total = score.sum(-1, keepdim=True)
        values = (table[v_codes[pages].permute(1, 0, 3, 2).flatten(1, 2).int()].flatten(-2)) * v_scales[pages].transpose(0, 1).flatten(1, 2).float()[..., None]
        o = torch.matmul(score.flatten(1, 2), values).view(heads, new, group, dim) / total.clamp(min=1e-30)
        out[start: start + new] = o.permute(1, 0, 2, 3).reshape(new, heads * group, dim)
        start += new
    return (_hadamard(out) * (1.0 / dim) * signs).to(s["q"].dtype)


def _plain_keep(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    kept, starts, page, table, free = s["kept"].long(), s["starts"].long(), s["page"], s["table"], s["free"]
    new = starts[1:] - starts[:-1]
    before = s["lengths"].long() - new
    # a list goes on as long as it goes up, within the request, to tokens that have a place
    ahead = torch.nn.functional.pad(kept, (1, 0), value=-1)[:, :-1]
    source = s["slots"][(starts[:-1, None] + kept).clamp(min=0, max=len(s["slots"]) - 1)]
    good = (kept > ahead) & (kept < new[:, None]) & (source >= 0)
    good = torch.cumprod(good.long(), 1).bool()
    count = good.sum(1)
    target = s["slots"][(starts[:-1, None] + torch.arange(kept.shape[1], device="cuda")).clamp(max=len(s["slots"]) - 1)]
    # what does not move is written to where it is
    rest = torch.where(good, source, source[:, :1].clamp(min=0))
    to = torch.where(good, target, source[:, :1].clamp(min=0))
    rest_at, rest_in, to_at, to_in = rest // page, rest % page, to // page, to % page
    for k_codes, k_scales, v_codes, v_scales, _ in s["caches"]:
        moved = k_codes[rest_at, :, rest_in], k_scales[rest_at, :, rest_in], v_codes[rest_at, :, :, rest_in], v_scales[rest_at, :, rest_in]
        k_codes[to_at, :, to_in], k_scales[to_at, :, to_in], v_codes[to_at, :, :, to_in], v_scales[to_at, :, to_in] = moved
    lengths = before + count
    column = torch.arange(table.shape[1], device="cuda")
    given = (column >= ((lengths + page - 1) // page)[:, None]) & (column < ((before + new + page - 1) // page)[:, None]) & (table >= 0)
    order = torch.cumsum(given.flatten().long(), 0)
    taken = (s["taken"].long() - order[-1]).clamp(min=0)
    at = torch.where(given.flatten(), s["taken"].long() - order[-1] + order - 1, len(free))
    free.copy_(torch.cat((free, free[:1])).index_put((at,), table.flatten())[: len(free)])
    return lengths.int(), taken.int()


# ---------------------------------------------------------------- the definition in 64 bits

def _sylvester(dim: int) -> torch.Tensor:
    h = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    while len(h) < dim:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h


def _exact_held(x: torch.Tensor, signs: torch.Tensor) -> torch.Tensor:
    """What the cache holds for vectors, in the rotated space: [..., D], before the division by D."""
    y = torch.matmul(x.double() * signs.double(), _sylvester(x.shape[-1]))
    a = (y.abs().amax(-1, keepdim=True) / 6).float().to(torch.bfloat16).double()
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    z = y / torch.where(a > 0, a, 1.0)
    nearest = torch.bucketize(z.abs(), (grid[1:] + grid[:-1]) / 2)
    return a * torch.copysign(grid[nearest], z)


def _exact_codes(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Codes [..., D/2] and scales [...] as what they stand for in the rotated space."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return torch.where(both >= 8, -1.0, 1.0) * grid[(both & 7).long()] * scales.double()[..., None]


def _exact_norm_rotary(x: torch.Tensor, s: dict, weight) -> torch.Tensor:
    """By complex numbers: a pair is one, and turns by one."""
    x = x.double()
    dim = x.shape[-1]
    if s["eps"] is not None:
        x = x / (x.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * weight.double()
    if s["cos"] is None:
        return x
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
    rotary = 2 * turn.shape[-1]
    head, rest = x[..., :rotary], x[..., rotary:]
    if s["interleaved"]:
        head = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(head[..., : rotary // 2].contiguous(), head[..., rotary // 2:].contiguous()) * turn
        head = torch.cat((z.real, z.imag), -1)
    return torch.cat((head, rest), -1) if rotary < dim else head


def _exact_paths(case: dict, s: dict) -> list[list[list[int]]]:
    """Request by request, token by token: the tokens on its path, itself the last one."""
    parents, at, paths = s["parents"].tolist(), 0, []
    for n in _ragged(case)[1]:
        own_paths = []
        for i in range(n):
            parent = parents[at + i]
            own_paths.append((own_paths[parent] if parent >= 0 else []) + [i])
        paths.append(own_paths)
        at += n
    return paths


def _exact_tree(case: dict, s: dict):
    positions, masks = [], []
    for before, paths in zip(_ragged(case)[0], _exact_paths(case, s)):
        for path in paths:
            positions.append(before + len(path) - 1)
            whole = sum(1 << i for i in path)
            words = [whole >> (MOST * w) & ((1 << MOST) - 1) for w in range(_words(case))]
            masks.append([w - (1 << MOST) if w >> (MOST - 1) else w for w in words])
    return torch.tensor(positions, dtype=torch.int32), torch.tensor(masks, dtype=torch.int64)


def _exact_keep(case: dict, s: dict):
    page, slots, table, free, taken = case["page"], s["slots"].tolist(), s["table"].tolist(), s["free"].tolist(), int(s["taken"])
    lengths, moves, back, start = [], [], [], 0
    before, new = _ragged(case)
    where = []
    for r, (b, n) in enumerate(zip(before, new)):
        count = 0
        for i, token in enumerate(s["kept"][r].tolist()):
            if token < 0:
                break
            moves.append((slots[start + token], slots[start + i]))
            count += 1
        lengths.append(b + count)
        back += table[r][-(-(b + count) // page): -(-(b + n) // page)]
        where += [slots[start + i] if i < n else -1 for i in range(case["depth"])]
        start += n
    free[taken - len(back): taken] = back
    came_from = dict((to, source) for source, to in moves)
    out = []
    for k_codes, k_scales, v_codes, v_scales, signs in s["caches"]:
        turn = _sylvester(len(signs)) / len(signs) * signs.double()
        at = torch.tensor([came_from.get(w, w) for w in where], device="cuda")
        there = (at >= 0)[:, None, None]
        block, place = at.clamp(min=0) // page, at.clamp(min=0) % page
        out.append(torch.where(there, torch.matmul(_exact_codes(k_codes[block, :, place], k_scales[block, :, place]), turn), 0.0))
        out.append(torch.where(there, torch.matmul(_exact_codes(v_codes[block, :, :, place], v_scales[block, :, place]), turn), 0.0))
    small = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return small(lengths), small([taken - len(back)]), small(free), *out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return tuple(_exact_norm_rotary(s[x], s, s[x + "_weight"]) for x in ("q", "k"))
    if kind == "append":
        signs = s["cache"][4].double()
        turn = _sylvester(len(signs)) / len(signs) * signs
        k = _exact_norm_rotary(s["k"], s, s["k_weight"])
        return _exact_norm_rotary(s["q"], s, s["q_weight"]), *(torch.matmul(_exact_held(x, signs), turn) for x in (k, s["v"]))
    if kind == "tree":
        return _exact_tree(case, s)
    if kind == "keep":
        return _exact_keep(case, s)
    k_codes, k_scales, v_codes, v_scales, signs = s["cache"]
    dim, page, heads = case["dim"], case["page"], case["heads"]
    group, turn = case["queries"] // heads, _sylvester(dim) / dim * signs.double()
    out = torch.empty(s["tokens"], case["queries"], dim, dtype=torch.float64, device="cuda")
    start = 0
    for r, (before, new, paths) in enumerate(zip(*_ragged(case), _exact_paths(case, s))):
        length = before + new
        first = max(0, before - case["window"]) // page if case["window"] else 0
        pages = s["table"][r, first: -(-length // page)].long()
        k = _exact_codes(k_codes[pages], k_scales[pages]).transpose(0, 1).reshape(heads, -1, dim)
        v = _exact_codes(v_codes[pages].transpose(2, 3), v_scales[pages]).transpose(0, 1).reshape(heads, -1, dim)
        seen = torch.zeros(new, k.shape[1], dtype=torch.bool)
        for i, path in enumerate(paths):
            window = case["window"] or length
            path = path[-window:]
            seen[i, torch.tensor(path) + before - first * page] = True
            low = max(0, before - (window - len(path)))
            seen[i, low - first * page: before - first * page] = True
        seen = seen.cuda()
        q = s["q"][start: start + new].double()
        for h in range(heads):
            score = torch.matmul(q[:, h * group:(h + 1) * group].reshape(-1, dim), torch.matmul(k[h], turn).t().contiguous()).view(new, group, -1) / math.sqrt(dim)
            weight = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1)
            out[start: start + new, h * group:(h + 1) * group] = torch.matmul(weight, torch.matmul(v[h], turn))
        start += new
    return out
