"""Drafted tokens from end to end: the operators together as a program runs them, on streams, in graphs, from compiled and Python host code and under
torch.compile; the layer; the example."""

import numpy as np
import pytest
import torch

import kv_oracle
import tree_oracle as oracle
from test_gpu_kv_cache import _cache, _i32, _queries
from test_gpu_kv_serving import _layer
from test_gpu_kv_tree import _check, _masks, _parents, _starts
from test_gpu_qk_rotary import _how

pytestmark = pytest.mark.gpu

PAGE, HEADS, GROUP, DIM, LAYERS = 16, 2, 3, 64, 2


def _state(seed, before=(20, 0, 47, 3), new=(9, 1, 17, 5)):
    """Requests whose prompts are cached, and the drafted tokens of a step: two layers' queries, keys and values."""
    from orbitquant_amd import kv_append, kv_assign

    rng = np.random.RandomState(seed)
    requests, width = len(before), 8
    how = _how(rng, DIM, DIM, False, "weights")
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    free = _i32(rng.permutation(requests * width).tolist())
    caches = [_cache(requests * width, HEADS, DIM, PAGE, fill=0xFF) for _ in range(LAYERS)]
    got = kv_assign(_i32([0] * requests), _i32(list(before)), table, free, _i32([0]), page_size=PAGE, tokens=sum(before))
    for c in caches:
        q, k, v = (_queries(rng, sum(before), h, DIM, torch.bfloat16) for h in (HEADS * GROUP, HEADS, HEADS))
        kv_append(q, k, v, got.slots, c, how, got.positions)
    tokens = sum(new)
    state = {"lengths": got.lengths.clone(), "new": _i32(list(new)), "table": table, "free": free, "taken": got.taken.clone(), "caches": caches, "how": how,
             "parents": _i32(_parents(rng, new, "random")), "kept": _i32(_paths(rng, new, 4))}
    _fresh(state, rng, tokens)
    return state


def _paths(rng, new, most):
    rows = []
    for n in new:
        count = int(rng.randint(1, min(n, most) + 1))
        row = [0] + sorted((1 + rng.permutation(n - 1)[:count - 1]).tolist())
        rows.append(row + [-1] * (most - count))
    return rows


def _fresh(state, rng, tokens):
    state["rows"] = [[_queries(rng, tokens, h, DIM, torch.bfloat16) for h in (HEADS * GROUP, HEADS, HEADS)] for _ in range(LAYERS)]


def _step(s):
    from orbitquant_amd import kv_append, kv_assign, kv_attend, kv_keep, kv_tree

    got = kv_assign(s["lengths"], s["new"], s["table"], s["free"], s["taken"], page_size=PAGE, tokens=len(s["parents"]))
    tree = kv_tree(s["parents"], got.starts, got.lengths)
    results = [*got, *tree]
    for c, (q, k, v) in zip(s["caches"], s["rows"]):
        q = kv_append(q, k, v, got.slots, c, s["how"], tree.positions)
        results += [q, *kv_attend(q, c, s["table"], got.lengths, starts=got.starts, masks=tree.masks, return_lse=True)]
    kept = kv_keep(s["kept"], got.lengths, got.starts, got.slots, s["caches"], block_table=s["table"], free_pages=s["free"], taken=got.taken)
    return results + list(kept)


def test_a_step_leaves_what_its_path_alone_would_have_left():
    """After a step and `kv_keep` the caches hold, bit for bit, what appending the path's tokens one behind the other leaves there; their rows of the attention are
    those of the path; and a second step goes on from there."""
    from orbitquant_amd import kv_append, kv_assign, kv_attend

    s, plain = _state(1), _state(1)
    rng = np.random.RandomState(2)
    for _ in range(3):
        new = s["new"].tolist()
        before = s["lengths"].tolist()
        results = _step(s)
        starts, kept = _starts(new), s["kept"].tolist()
        positions, masks = oracle.tree(s["parents"].tolist(), starts, results[3].tolist(), 1, sum(new))
        assert results[5].tolist() == positions and results[6].tolist() == masks
        counts = [sum(k >= 0 for k in row) for row in kept]
        # the same tokens one behind the other, at the positions that their nodes have (a list of nodes that is no path has gaps in these)
        rows = torch.tensor([starts[r] + k for r, row in enumerate(kept) for k in row if k >= 0], device="cuda")
        got = kv_assign(plain["lengths"], _i32(counts), plain["table"], plain["free"], plain["taken"], page_size=PAGE, tokens=sum(counts))
        assert results[-2].tolist() == got.lengths.tolist() == [b + c for b, c in zip(before, counts)] and results[-1].tolist() == got.taken.tolist()
        for layer, c in enumerate(plain["caches"]):
            q, k, v = (x[rows] for x in plain["rows"][layer])
            kv_append(q, k, v, got.slots, c, plain["how"], results[5][rows])
        for a, b in zip(s["caches"], plain["caches"]):
            where_a, where_b = (_held(st["table"], got.lengths.tolist()) for st in (s, plain))
            for x, y in zip(kv_oracle.cache_codes(a), kv_oracle.cache_codes(b)):
                np.testing.assert_array_equal(x[where_a[0], :, where_a[1]], y[where_b[0], :, where_b[1]])
        for st, r in ((s, results[-2:]), (plain, (got.lengths, got.taken))):
            st["lengths"].copy_(r[0])
            st["taken"].copy_(r[1])
            assert len(set(_pages(st))) == len(_pages(st))
        parents, paths = _i32(_parents(rng, new, "random")), _i32(_paths(rng, new, 4))
        for st in (s, plain):
            st["parents"], st["kept"] = parents, paths
        _fresh(s, rng, sum(new))
        plain["rows"] = s["rows"]


def _held(table, lengths):
    at = [(int(table[r, t // PAGE]), t % PAGE) for r, n in enumerate(lengths) for t in range(n)]
    return np.array([a[0] for a in at]), np.array([a[1] for a in at])


def _pages(s):
    """All pages that are in use or will be given out."""
    held = [int(s["table"][r, c]) for r, n in enumerate(s["lengths"].tolist()) for c in range(-(-n // PAGE))]
    return held + s["free"][int(s["taken"]):].tolist()


def test_rows_of_a_step():
    """The attention of every drafted token, by its definition."""
    s = _state(3)
    results = _step(s)
    before_keep = _state(3)
    from orbitquant_amd import kv_append, kv_assign, kv_tree

    got = kv_assign(before_keep["lengths"], before_keep["new"], before_keep["table"], before_keep["free"], before_keep["taken"], page_size=PAGE, tokens=32)
    tree = kv_tree(before_keep["parents"], got.starts, got.lengths)
    masks = [[w[0]] for w in tree.masks.tolist()]
    for layer, (c, (q, k, v)) in enumerate(zip(before_keep["caches"], before_keep["rows"])):
        q = kv_append(q, k, v, got.slots, c, before_keep["how"], tree.positions)
        assert torch.equal(q, results[7 + 3 * layer])
        _check((results[8 + 3 * layer], results[9 + 3 * layer]), q, c, before_keep["table"], got.lengths.tolist(), got.starts.tolist(), masks)


def _same(a, b):
    for x, y in zip(a, b, strict=True):
        assert x.dtype == y.dtype and torch.equal(x, y)


def _same_caches(a, b):
    for c, d in zip(a["caches"], b["caches"]):
        for x, y in zip(c, d):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_on_a_stream_and_in_a_graph():
    """A step captured once and replayed, its state moving on between the replays, with eager work of the program's in between, against the same steps run eagerly
    on another stream."""
    eager, captured = _state(4), _state(4)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _step(captured)
    torch.cuda.current_stream().wait_stream(warm)
    captured = _state(4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(captured)
    rng, side = np.random.RandomState(5), torch.cuda.Stream()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = _step(eager)
        torch.cuda.synchronize()
        _same(out, want)
        _same_caches(eager, captured)
        assert torch.equal(eager["free"], captured["free"]) and torch.equal(eager["table"], captured["table"])
        new = eager["new"].tolist()
        parents, kept = _i32(_parents(rng, new, "random")), _i32(_paths(rng, new, 4))
        rows = [[torch.randn_like(x) for x in r] for r in eager["rows"]]
        for st, result in ((eager, want), (captured, out)):
            st["lengths"].copy_(result[-2])
            st["taken"].copy_(result[-1])
            st["parents"].copy_(parents)
            st["kept"].copy_(kept)
            for r, fresh in zip(st["rows"], rows):
                for x, y in zip(r, fresh):
                    x.copy_(y)
        torch.cuda.synchronize()


def test_two_graphs_of_one_state_do_not_share_what_they_write():
    """Long contexts, whose parts need workspaces: two captured calls, replayed on two streams at once, each give their own result."""
    from orbitquant_amd import kv_attend
    from test_gpu_kv_cache import _filled

    rng = np.random.RandomState(6)
    cache, table = _filled(rng, [2500], 2, 64, 64)
    masks = _masks([[1 << i | 1] for i in range(20)])
    queries = [_queries(rng, 20, 4, 64, torch.bfloat16) for _ in range(2)]
    call = lambda q: kv_attend(q, cache, table, _i32([2500]), starts=_i32([0, 20]), masks=masks, max_new=20, return_lse=True)  # noqa: E731
    want = [call(q) for q in queries]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    lengths, starts = _i32([2500]), _i32([0, 20])
    call = lambda q: kv_attend(q, cache, table, lengths, starts=starts, masks=masks, max_new=20, return_lse=True)  # noqa: E731
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(q))
        graphs.append(graph)
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            _same(got, w)


def test_python_and_compiled_host_code_agree(monkeypatch):
    from orbitquant_amd import kv_cache, qk_rotary

    def everything(s):
        return _step(s) + list(qk_rotary.qk_norm_rotary(*s["rows"][0][:2], s["how"], s["lengths"].repeat(8))) + [s["free"], s["table"]]

    a, b = _state(7), _state(7)
    compiled = everything(a)
    for module in (kv_cache, qk_rotary):
        monkeypatch.setattr(module, "_host", None)
        monkeypatch.setattr(module, "_module", lambda: None)
    _same(compiled, everything(b))
    _same_caches(a, b)


def test_under_torch_compile():
    """One graph without breaks, the caches and the free list written in place, the same bits."""
    from orbitquant_amd import qk_norm_rotary

    def everything(s):
        results = _step(s)
        return results + list(qk_norm_rotary(s["rows"][0][0], s["rows"][0][1], s["how"], results[5]))

    eager, traced = _state(8), _state(8)
    call = torch.compile(everything, fullgraph=True)
    for _ in range(2):
        want, got = everything(eager), call(traced)
        _same(want, got)
        _same_caches(eager, traced)
        assert torch.equal(eager["free"], traced["free"])
        for st, result in ((eager, want), (traced, got)):
            st["lengths"].copy_(result[-4])
            st["taken"].copy_(result[-3])


def test_ops_pass_opcheck():
    s = _state(9)
    q, k, v = s["rows"][0]
    how = tuple(s["how"])
    ops = torch.ops.orbitquant_amd
    tests = ("test_schema", "test_faketensor")
    starts = _i32(_starts([9, 1, 17, 5]))
    after, positions, slots = s["lengths"] + s["new"], torch.arange(32, dtype=torch.int32, device="cuda"), torch.arange(100, 132, device="cuda")
    torch.library.opcheck(ops.qk_norm_rotary, (q, k, *how, positions), test_utils=tests)
    torch.library.opcheck(ops.qk_norm_rotary, (q, k, None, None, None, None, None, True, None), test_utils=tests)
    torch.library.opcheck(ops.kv_append, (q, k, v, slots, *s["caches"][0], *how, positions), test_utils=tests)
    torch.library.opcheck(ops.kv_tree, (s["parents"], starts, after, 2), test_utils=tests)
    masks = torch.ones(32, 1, dtype=torch.int64, device="cuda")
    for with_lse in (False, True):
        torch.library.opcheck(ops.kv_attend_tree, (q, *s["caches"][0], s["table"], after, starts, masks, -1, -1, 0, 0.125, with_lse), test_utils=tests)
    lists = [list(t) for t in zip(*s["caches"])]
    torch.library.opcheck(ops.kv_keep, (s["kept"], after, starts, slots, *lists, s["table"], s["free"], s["taken"]), test_utils=tests)
    torch.library.opcheck(ops.kv_keep, (s["kept"], after, starts, slots, *lists, None, None, None), test_utils=tests)


# ---------------------------------------------------------------- the layer and the example

@pytest.mark.parametrize("window", [None, 12])
def test_layer(window):
    """`QKNormRotary` in a layer: prompts, single tokens and trees go through `kv_append`, and the attention has the masks."""
    from orbitquant_amd import kv_append, kv_assign, kv_attend, kv_tree

    rng = np.random.RandomState(10)
    how = _how(rng, 64, 32, False, "weights")
    layer = _layer(_cache(20, 2, 64, 16, fill=0xFF), 4, 256, rotary=how, window=window)
    other = _cache(20, 2, 64, 16, fill=0xFF)
    table = torch.full((3, 6), -1, dtype=torch.int32, device="cuda")
    lengths, taken, free = _i32([0, 0, 0]), _i32([0]), _i32(rng.permutation(20).tolist())
    for new, drafted in (([30, 1, 20], False), ([1, 1, 1], False), ([7, 1, 13], True)):
        x = torch.from_numpy(rng.standard_normal((sum(new), 256)).astype(np.float32)).to("cuda", torch.bfloat16)
        got = kv_assign(lengths, _i32(new), table, free, taken, page_size=16, tokens=sum(new))
        tree = kv_tree(_i32(_parents(rng, new, "random")), got.starts, got.lengths) if drafted else None
        y = layer(x, got, table, tree=tree, max_new=max(new))
        q, k, v = (p(x).view(len(x), -1, 64) for p in (layer.q, layer.k, layer.v))
        q = kv_append(q, k, v, got.slots, other, how, tree.positions if drafted else got.positions)
        attended = kv_attend(q, other, table, got.lengths, starts=got.starts, masks=tree.masks if drafted else None, max_new=max(new), window=window)
        assert torch.equal(y, layer.out(attended.reshape(len(x), -1)))
        lengths, taken = got.lengths, got.taken


def test_accepted():
    from orbitquant_amd.examples.draft import accepted

    parents = _i32([-1, 0, 0, 1, 2, 3, 4])
    ids = torch.tensor([[5, 1, 2, 3, 4, 8, 9], [5, 1, 1, 3, 4, 8, 9], [5, 7, 2, 3, 4, 8, 9], [5, 1, 2, 3, 4, 8, 9]], device="cuda")
    chosen = torch.tensor([[2, 0, 4, 0, 9, 0, 0], [1, 3, 0, 8, 0, 0, 0], [0, 0, 0, 0, 0, 0, 0], [1, 4, 3, 0, 0, 0, 0]], device="cuda")
    assert accepted(ids, chosen, parents, 3).tolist() == [[0, 2, 4, 6], [0, 1, 3, 5], [0, -1, -1, -1], [0, 1, -1, -1]]


def test_draft_example(capsys):
    """Steps say at least a token each, lengths and pages follow, and replays are the eager steps."""
    from orbitquant_amd.examples import draft

    got = draft.main(["--layers", "2", "--requests", "3", "--steps", "6", "--prompt", "70", "--depth", "3"])
    assert "tokens a step" in capsys.readouterr().out
    said = np.array(got["said"])
    counts = (said >= 0).sum(-1)
    assert (counts >= 1).all() and (said[..., 0] >= 0).all() and got["tokens"] == counts.sum()
    assert got["lengths"] == [n + int(c) for n, c in zip(got["prompts"], counts.sum(-1))]
    assert got["pages_taken"] == sum(-(-n // draft.PAGE) for n in got["lengths"])
    prompts = got["prompts"]
    eager, again = (draft.Drafter(2, 3, 200, 3) for _ in range(2))
    ids = torch.randint(0, draft.VOCABULARY, (sum(prompts),), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for m in (eager, again):
        m.step(ids, _i32(prompts), max_new=max(prompts))
    graph = again.captured_draft_step()
    for _ in range(4):
        want = eager.draft_step().clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, again.said) and torch.equal(eager.lengths, again.lengths) and torch.equal(eager.taken, again.taken)


def test_draft_example_follows_the_model():
    """Where the guesses are what the model says next, all of them are kept: told its own continuation, it says the same."""
    from orbitquant_amd.examples import draft

    plain, drafter = (draft.Drafter(1, 1, 120, 3) for _ in range(2))
    ids = torch.randint(0, draft.VOCABULARY, (40,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    for m in (plain, drafter):
        m.step(ids, _i32([40]), max_new=40)
    first = int(plain.last)
    said = [int(plain.draft_step()[0, 0])]          # nothing is known yet: a wrong guess, one token
    assert plain.lengths.tolist()[0] >= 41
    # the tree's second level is what followed: the certain token's row of the attention does not see the guesses
    drafter.followed[0, first, 0] = said[0]
    told = drafter.draft_step()[0].tolist()
    assert told[0] == said[0] and told[1] >= 0 and int(drafter.lengths) >= 42
