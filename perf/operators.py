"""The 4-bit key/value cache of a serving program and the attention that reads it, as measurable cases.

A case is a dict of plain values.  `listed()` gives the named ones, `draw(rng)` one more of the same ranges,
`prepare(case, seed)` what a program holds before the call, `run(state)` one pass (the package's calls where `own` is true,
elementary torch operations in 32 bits where it is not), `exact(case, seed)` the definition in 64 bits, and `work(case)` the
bytes and operations that one pass cannot do without.

The cache.  A token's key (or value) of one head, x[D], is held as y = H(signs * x) with H the unnormalised Walsh-Hadamard
transform (butterflies of distance 1, 2, 4, ...): one scale a = bf16(max|y| / 6) and D codes in four bits, the nearest E2M1
value (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign, ties to the even code) of y / a.  It stands for signs * H(a * code) / D.
Pages of `page` tokens; a slot is page index * page + place in the page:
  k_codes [pages, heads, page, D/2] uint8    byte j of a token: dimensions 2j (low four bits) and 2j+1
  v_codes [pages, heads, D/2, page] uint8    the same bytes, a page's tokens side by side
  k_scales, v_scales [pages, heads, page] bfloat16

Kinds of work:
  assign   pages and slots for the new tokens of a batch of requests, from their lengths
  write    new keys and values into the cache, and read back as the values they are held as
  attend   queries over the cache: one token a request, or `new` tokens of a prompt (ragged), causal, perhaps with a window
  step     a serving step: assign, write, attend
"""

from __future__ import annotations

import math
from functools import reduce

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(kind, name=None, **kw):
    case = {"kind": kind, **kw}
    return case if name is None else {"name": name, **case}


def listed() -> list[dict]:
    return [
        # the smallest call: the next token of a single conversation gets its slot
        _case("assign", "assign one", requests=1, longest=2000, new=1, page=16, width=256),
        # a busy scheduler: hundreds of requests, some in their prompt and most decoding, a ragged batch
        _case("assign", "assign many", requests=509, longest=16384, new=1024, page=64, width=300),
        # one decoded token of a 4096-wide layer with 32 heads of its own
        _case("write", "write one", tokens=1, heads=32, dim=128, page=64, dtype="bf16"),
        # a prompt of odd length in single precision, short heads, small pages
        _case("write", "write odd fp32", tokens=333, heads=5, dim=64, page=16, dtype="fp32"),
        # a long prompt's keys and values, eight shared heads
        _case("write", "write prompt", tokens=8192, heads=8, dim=128, page=64, dtype="bf16"),
        # one conversation, a 4096-wide layer with 32 heads, a context of a thousand tokens: latency
        _case("attend", "decode one", requests=1, longest=1003, new=1, queries=32, heads=32, dim=128, page=16, dtype="bf16", window=0),
        # one conversation over a long document, heads shared by four
        _case("attend", "decode long", requests=1, longest=131101, new=1, queries=32, heads=8, dim=128, page=64, dtype="bf16", window=0),
        # wide heads in single precision over a sliding window, a group of three, ragged lengths
        _case("attend", "decode window fp32", requests=7, longest=5000, new=1, queries=12, heads=4, dim=256, page=32, dtype="fp32", window=1500),
        # the largest by bytes: a full serving batch with long ragged contexts
        _case("attend", "decode batch", requests=64, longest=16384, new=1, queries=32, heads=8, dim=128, page=64, dtype="bf16", window=0),
        # chunks of several prompts behind cached prefixes, half precision, short heads, ragged
        _case("attend", "prompt chunks fp16", requests=6, longest=6000, new=700, queries=16, heads=4, dim=64, page=64, dtype="fp16", window=0),
        # the largest by operations: a whole prompt of eight thousand tokens
        _case("attend", "prompt", requests=1, longest=8192, new=8192, queries=32, heads=8, dim=128, page=64, dtype="bf16", window=0),
        # sixteen sequences decoded together, as the decode stack is: slots, write and attention
        _case("step", "step", requests=16, longest=4096, new=1, queries=32, heads=8, dim=128, page=64, dtype="bf16", window=0),
    ]


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["assign", "write", "attend", "attend", "attend", "step"])
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "assign":
        longest = _log_int(rng, 1, 16384)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 1024)
        return _case(kind, requests=_log_int(rng, 1, 509), longest=longest, new=new, page=page, width=-(-(longest + new) // page) + rng.randrange(9))
    dim, dtype = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16, 32])
    if kind == "write":
        return _case(kind, tokens=_log_int(rng, 1, max(1, min(8192, 8192 * 8 * 128 // (heads * dim * (2 if dtype == "fp32" else 1))))),
                     heads=heads, dim=dim, page=page, dtype=dtype)
    group = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 16])
    window = _log_int(rng, 16, 4096) if rng.random() < 0.25 else 0
    same = {"queries": heads * group, "heads": heads, "dim": dim, "page": page, "dtype": dtype, "window": window}
    budget = 64 * 16384 * 8 * 128 // (heads * dim)     # cached tokens of the largest listed case, at this width
    if kind == "step" or rng.random() < 0.6:
        requests = _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, max(1, min(131101, budget // requests)))
        return _case(kind, requests=requests, longest=longest, new=1, **same)
    pairs = 32 * 8192 * 8192 // (4 * heads * group) * 128 // dim * (1 if dtype == "bf16" else 2) // 2   # a fraction of the largest prompt's
    requests = _log_int(rng, 1, 8)
    new = _log_int(rng, 2, max(2, min(4096, math.isqrt(pairs // requests))))
    longest = max(new, min(_log_int(rng, new, 16384), pairs // (requests * new), budget // requests))
    return _case(kind, requests=requests, longest=longest, new=new, **same)


# ---------------------------------------------------------------- sizes that follow from a case

def _ragged(case: dict) -> tuple[list[int], list[int]]:
    """(tokens cached before the pass, new tokens) of each request: by the case alone, so that `work` knows them.  One
    request has the longest context; the others spread below it.  `longest` counts the new tokens for "attend"."""
    n, longest, new = case["requests"], case["longest"], case["new"]
    before, fresh = [], []
    for r in range(n):
        share = 1.0 if r == n // 2 else 0.2 + 0.8 * ((r * 0.6180339887) % 1.0)
        count = new if new == 1 or r == n // 2 else max(1, round(new * (0.1 + 0.9 * ((r * 0.7548776662) % 1.0))))
        if case["kind"] == "assign":
            count = 1 if new > 1 and r % 4 else count       # most requests decode, one in four is in its prompt
            before.append(round(longest * share) if r % 16 != 3 else 0)     # and some have just come in
        elif case["kind"] == "step":
            before.append(max(0, round(longest * share) - 1))
        else:
            before.append(max(0, round(longest * share) - count))
        fresh.append(count)
    return before, fresh


def _visible(case: dict) -> tuple[int, int]:
    """(cached tokens that a pass reads, query-key pairs) over all requests."""
    tokens = pairs = 0
    for before, new in zip(*_ragged(case)):
        window = case["window"] or before + new
        first = max(0, before + 1 - window)
        tokens += before + new - first
        full = max(0, min(new, window - before))            # queries whose window is not full yet
        pairs += full * before + full * (full + 1) // 2 + (new - full) * window
    return tokens, pairs


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "assign":
        return _assign_work(case)
    size = 4 if case["dtype"] == "fp32" else 2
    held = case["heads"] * (case["dim"] + 4)                # bytes of a token: two times D/2 codes and two scales
    row = case["heads"] * case["dim"] * 2 * size            # bytes of a token's key and value
    if kind == "write":
        t, stages = case["tokens"], int(math.log2(case["dim"]))
        return {"bytes": t * (2 * row + 2 * held + 16), "flops": 2.0 * t * case["heads"] * case["dim"] * (2 * stages + 6)}
    tokens, pairs = _visible(case)
    new = sum(_ragged(case)[1])
    w = {"bytes": tokens * held + 2 * new * case["queries"] * case["dim"] * size + 4 * tokens // case["page"] + 4 * case["requests"],
         "flops": 4.0 * pairs * case["queries"] * case["dim"]}
    if kind == "step":
        w["bytes"] += new * (row + held) + _assign_work(case)["bytes"]
    return w


def _assign_work(case: dict) -> dict:
    before, new = _ragged(case)
    page = case["page"]
    fresh = sum(-(-(b + n) // page) - -(-b // page) for b, n in zip(before, new))
    # lengths in and out, new counts, starts; a fresh page's index in and out; a token's slot and position
    return {"bytes": 16 * len(before) + 16 + 8 * fresh + 12 * sum(new), "flops": 8.0 * (sum(new) + len(before))}


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


def _empty_cache(pages: int, heads: int, dim: int, page: int, g) -> tuple:
    codes = torch.zeros(2, pages, heads, page * dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, pages, heads, page, dtype=torch.bfloat16, device="cuda")
    signs = (torch.randint(0, 2, (dim,), generator=g, device="cuda") * 2 - 1).to(torch.int8)
    return (codes[0].view(pages, heads, page, dim // 2), scales[0], codes[1].view(pages, heads, dim // 2, page), scales[1], signs)


def _requests(g, case: dict) -> dict:
    """Lengths, pages and the block table of a batch, its pages anywhere in the pool, some of them free."""
    before, new = _ragged(case)
    page = case["page"]
    serving = case["kind"] != "attend"                      # the pages of new tokens are not assigned yet
    have = [-(-(b if serving else b + n) // page) for b, n in zip(before, new)]
    need = [-(-(b + n) // page) for b, n in zip(before, new)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32).cpu()
    width = case.get("width", max(need) + 1)
    table = torch.full((len(before), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(have):
        table[r, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    put = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"pages": pages, "before": put(before), "new": put(new), "after": put([b + n for b, n in zip(before, new)]), "starts": put(starts),
            "table": table.cuda(), "free": order[at:].cuda(), "taken": put([0]), "tokens": starts[-1], "most": max(new),
            "longest": max(b + n for b, n in zip(before, new))}


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    state = {"kind": case["kind"], "page": case["page"]}
    if case["kind"] == "assign":
        return state | _requests(g, case)
    heads, dim, page, dtype = case["heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    state["dtype"] = dtype
    if case["kind"] == "write":
        t = case["tokens"]
        pages = -(-t // page) + 3
        state["cache"] = _empty_cache(pages, heads, dim, page, g)
        # the tokens' slots: runs of a page in a row, the pages anywhere; keys and values are parts of one projection's output
        order = torch.randperm(pages, generator=g, device="cuda")[: -(-t // page)]
        state["slots"] = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:t].contiguous()
        both = torch.cat((_vectors(g, t, heads, dim, True, dtype), _vectors(g, t, heads, dim, False, dtype)), 1)
        return state | {"k": both[:, :heads], "v": both[:, heads:]}
    state |= _requests(g, case)
    state["cache"] = cache = _empty_cache(state["pages"], heads, dim, page, g)
    chunk = max(1, (1 << 27) // (heads * page * dim))
    for at in range(0, state["pages"], chunk):
        slots = torch.arange(at * page, min(at + chunk, state["pages"]) * page, device="cuda")
        v = _vectors(g, len(slots), heads, dim, False)
        _plain_write(_vectors(g, len(slots), heads, dim, True), v, slots, cache)
    firsts = state["table"][:, 0].clamp(min=0).long()
    cache[3][firsts, :, 0] *= 0.0625                        # a first token's value is small
    state["q"] = torch.randn(state["tokens"], case["queries"], dim, generator=g, device="cuda").to(dtype)
    state["window"] = case["window"] or None
    state["scale"] = 1.0 / math.sqrt(dim)
    if case["kind"] == "step":
        both = torch.cat((_vectors(g, state["tokens"], heads, dim, True, dtype), _vectors(g, state["tokens"], heads, dim, False, dtype)), 1)
        state |= {"k": both[:, :heads], "v": both[:, heads:]}
    return state


# ---------------------------------------------------------------- one pass

def run(s: dict):
    return (_run_own if own else _run_plain)(s)


def _run_own(s: dict):
    from orbitquant_amd import OrbitKVCache, ops

    kind = s["kind"]
    if kind == "assign":
        return (*ops.kv_assign(s["before"], s["new"], s["table"], s["free"], s["taken"], page_size=s["page"], tokens=s["tokens"]), s["table"])
    cache = OrbitKVCache(*s["cache"])
    if kind == "write":
        ops.kv_write(s["k"], s["v"], s["slots"], cache)
        return ops.kv_read(s["slots"], cache, s["dtype"])
    if kind == "attend":
        starts = s["starts"] if s["most"] > 1 else None
        return ops.kv_attend(s["q"], cache, s["table"], s["after"], starts=starts, max_new=s["most"], max_length=s["longest"],
                             window=s["window"], scale=s["scale"])
    slots, positions, _, after, taken = ops.kv_assign(s["before"], s["new"], s["table"], s["free"], s["taken"], page_size=s["page"],
                                                      tokens=s["tokens"])
    ops.kv_write(s["k"], s["v"], slots, cache)
    out = ops.kv_attend(s["q"], cache, s["table"], after, max_length=s["longest"], window=s["window"], scale=s["scale"])
    return out, slots, positions, after, taken


def _run_plain(s: dict):
    kind = s["kind"]
    if kind == "assign":
        return (*_plain_assign(s), s["table"])
    if kind == "write":
        _plain_write(s["k"], s["v"], s["slots"], s["cache"])
        return _plain_read(s["slots"], s["cache"], s["dtype"])
    if kind == "attend":
        return _plain_attend(s, s["after"])
    slots, positions, _, after, taken = _plain_assign(s)
    _plain_write(s["k"], s["v"], slots, s["cache"])
    return _plain_attend(s, after), slots, positions, after, taken


# ---------------------------------------------------------------- the plain forms

def _plain_assign(s: dict):
    before, new, table, free, page = s["before"].clamp(min=0), s["new"].clamp(min=0), s["table"], s["free"], s["page"]
    starts = torch.nn.functional.pad(torch.cumsum(new, 0, dtype=torch.int32), (1, 0))
    after = before + new
    have, need = (before + (page - 1)) // page, (after + (page - 1)) // page
    fresh = need - have
    upto = torch.cumsum(fresh, 0, dtype=torch.int32)
    column = torch.arange(table.shape[1], dtype=torch.int32, device=table.device)
    at = (s["taken"] + upto - fresh - have)[:, None] + column
    page_of = torch.where(at < len(free), free[at.clamp(0, max(0, len(free) - 1)).long()], -1) if len(free) else torch.full_like(table, -1)
    table.copy_(torch.where((column >= have[:, None]) & (column < need[:, None]), page_of, table))
    token = torch.arange(s["tokens"], dtype=torch.int32, device=table.device)
    request = torch.searchsorted(starts[1:], token, right=True).clamp(max=len(before) - 1)
    there = token < starts[-1]
    position = torch.where(there, before[request] + token - starts[request], -1)
    place = (position // page).clamp(min=0).long()
    mapped = torch.where(there & (place < table.shape[1]), table[request, place.clamp(max=table.shape[1] - 1)], -1).long()
    slots = torch.where(mapped >= 0, mapped * page + position % page, -1)
    return slots, position, starts, after, torch.minimum(s["taken"] + upto[-1:], torch.full_like(s["taken"], len(free)))


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
    k_codes, k_scales, v_codes, v_scales, signs = cache
    page, dim = k_codes.shape[2], len(signs)
    at, place = slots // page, slots % page
    table = _values_table(signs.device)
    out = ((k_codes[at, :, place], k_scales[at, :, place]), (v_codes[at, :, :, place], v_scales[at, :, place]))
    back = lambda c, a: (_hadamard(table[c.int()].flatten(-2) * a.float()[..., None]) * (1.0 / dim) * signs).to(dtype)  # noqa: E731
    return back(*out[0]), back(*out[1])


def _plain_attend(s: dict, lengths) -> torch.Tensor:
    """Every request padded to the widest: its pages gathered, its queries in rows of `most`."""
    k_codes, k_scales, v_codes, v_scales, signs = s["cache"]
    q, most, dim, heads = s["q"], s["most"], len(signs), k_codes.shape[1]
    requests = len(lengths)
    group = q.shape[1] // heads
    table = _values_table(q.device)
    pages = s["table"][:, : -(-s["longest"] // s["page"])].clamp(min=0).long()
    keys = (table[k_codes[pages].transpose(1, 2).flatten(2, 3).int()].flatten(-2)) * k_scales[pages].transpose(1, 2).flatten(2, 3).float()[..., None]
    starts = s["starts"][:-1].long()
    count = s["starts"][1:].long() - starts
    row = torch.arange(most, device=q.device)
    rows = (starts[:, None] + row).clamp(max=len(q) - 1)
    qr = _hadamard(q.float() * signs) * (s["scale"] / dim)
    qr = qr[rows].view(requests, most, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, heads, most * group, dim)
    position = (lengths.long() - count)[:, None] + row
    place = torch.arange(keys.shape[2], device=q.device)
    seen = place <= position[..., None]
    if s["window"] is not None:
        seen &= place > position[..., None] - s["window"]
    score = torch.matmul(qr, keys.transpose(2, 3)).view(requests, heads, most, group, -1)
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-3e38)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    del keys
    values = (table[v_codes[pages].permute(0, 2, 1, 4, 3).flatten(2, 3).int()].flatten(-2)) * v_scales[pages].transpose(1, 2).flatten(2, 3).float()[..., None]
    out = torch.matmul(score.flatten(2, 3), values).view(requests, heads, most, group, dim) / total.clamp(min=1e-30)
    out = (_hadamard(out) * (1.0 / dim) * signs).permute(0, 2, 1, 3, 4).reshape(requests, most, heads * group, dim)
    token = torch.arange(len(q), device=q.device)
    request = torch.searchsorted(s["starts"][1:].long(), token, right=True)
    return out[request, token - starts[request]].to(q.dtype)


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


def _exact_assign(case: dict, s: dict):
    """By counting, on the host."""
    page, free, table = case["page"], s["free"].tolist(), s["table"].cpu().clone()
    slots, positions, starts, after, taken = [], [], [0], [], 0
    for r, (before, new) in enumerate(zip(*_ragged(case))):
        for pos in range(before, before + new):
            if pos % page == 0:
                if pos // page < table.shape[1]:
                    table[r, pos // page] = free[taken] if taken < len(free) else -1
                taken += 1
            at = int(table[r, pos // page]) if pos // page < table.shape[1] else -1
            slots.append(at * page + pos % page if at >= 0 else -1)
            positions.append(pos)
        starts.append(starts[-1] + new)
        after.append(before + new)
    small = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return torch.tensor(slots, dtype=torch.int64), small(positions), small(starts), small(after), small([min(taken, len(free))]), table


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "assign":
        return _exact_assign(case, s)
    signs = s["cache"][4].double()
    dim, page, heads = len(signs), case["page"], case["heads"]
    turn = _sylvester(dim) / dim * signs                    # rotated space -> the original one
    if case["kind"] == "write":
        return tuple(torch.matmul(_exact_held(s[x], signs), turn) for x in ("k", "v"))
    k_codes, k_scales, v_codes, v_scales, _ = s["cache"]
    group = case["queries"] // heads
    out = torch.empty(s["tokens"], case["queries"], dim, dtype=torch.float64, device="cuda")
    if case["kind"] == "step":
        slots, positions, _, after, taken, table = _exact_assign(case, s)
        new_k, new_v = _exact_held(s["k"], signs), _exact_held(s["v"], signs)
    else:
        table = s["table"].cpu()
    starts = s["starts"].tolist()
    for r, (before, new) in enumerate(zip(*_ragged(case))):
        n = before + new
        first = max(0, before + 1 - case["window"]) if case["window"] else 0
        pages = table[r, first // page: -(-n // page)].long().cuda()
        skip = first // page * page
        k = _exact_codes(k_codes[pages], k_scales[pages])                                       # [pages, heads, page, D]
        v = _exact_codes(v_codes[pages].transpose(2, 3), v_scales[pages])
        k, v = (x.transpose(0, 1).reshape(heads, -1, dim)[:, : n - skip].clone() for x in (k, v))
        if case["kind"] == "step":
            k[:, before - skip:], v[:, before - skip:] = (x[starts[r]:starts[r + 1]].transpose(0, 1) for x in (new_k, new_v))
        q = s["q"][starts[r]:starts[r + 1]].double()
        place = torch.arange(skip, n, device="cuda")
        for at in range(0, new, 1024):
            rows = q[at:at + 1024]
            position = before + at + torch.arange(len(rows), device="cuda")
            seen = place <= position[:, None]
            if case["window"]:
                seen &= place > position[:, None] - case["window"]
            for h in range(heads):
                kh, vh = torch.matmul(k[h], turn), torch.matmul(v[h], turn)
                score = torch.matmul(rows[:, h * group:(h + 1) * group].reshape(-1, dim), kh.t().contiguous()).view(len(rows), group, -1) / math.sqrt(dim)
                score = score.masked_fill(~seen[:, None], -math.inf)
                weight = torch.softmax(score, -1)
                out[starts[r] + at: starts[r] + at + len(rows), h * group:(h + 1) * group] = torch.matmul(weight, vh)
    if case["kind"] == "step":
        return out, slots, positions, after, taken
    return out
