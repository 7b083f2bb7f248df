"""Where the pages of drafted steps go: after every step the pages that requests hold and those that the list still gives out are the whole pool, each
once; also where a request is at its table's end, where the list has run out, and both."""

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import _cache, _i32

pytestmark = pytest.mark.gpu

PAGE = 16


class Pool:
    """Requests over one list of pages, and what is known of them on the host."""

    def __init__(self, rng, before, width, pages):
        from orbitquant_amd import kv_assign

        self.rng, self.width, self.pages = rng, width, pages
        self.table = torch.full((len(before), width), -1, dtype=torch.int32, device="cuda")
        self.free, self.taken = _i32(rng.permutation(pages).tolist()), _i32([0])
        self.caches = [_cache(pages, 1, 64, PAGE)]
        got = kv_assign(_i32([0] * len(before)), _i32([min(n, width * PAGE) for n in before]), self.table, self.free, self.taken, page_size=PAGE, tokens=0)
        # (what lies behind the table was never given a page here)
        self.lengths, self.taken = _i32(before), got.taken.clone()

    def held(self):
        rows = self.table.tolist()
        return [p for row, n in zip(rows, self.lengths.tolist()) for p in row[:min(self.width, -(-n // PAGE))] if p >= 0]

    def listed(self):
        return self.free[int(self.taken):].tolist()

    def step(self, new, most=4, kept=None):
        """Drafted tokens for every request, of which the first that have a slot stay (or the `kept` ones); -> the tokens that stayed."""
        from orbitquant_amd import kv_assign, kv_keep

        got = kv_assign(self.lengths, _i32(new), self.table, self.free, self.taken, page_size=PAGE, tokens=sum(new))
        if kept is None:
            kept = [list(range(int(self.rng.randint(0, most + 1)))) for _ in new]
        rows = [row + [-1] * (most - len(row)) for row in kept]
        after = kv_keep(_i32(rows), got.lengths, got.starts, got.slots, self.caches, block_table=self.table, free_pages=self.free, taken=got.taken)
        slots, starts = got.slots.tolist(), got.starts.tolist()
        stay = []
        for r, row in enumerate(kept):
            count = 0
            while count < len(row) and row[count] < new[r] and slots[starts[r] + row[count]] >= 0:
                count += 1
            stay.append(count)
        assert after.lengths.tolist() == [n + c for n, c in zip(self.lengths.tolist(), stay)]
        self.lengths, self.taken = after.lengths, after.taken
        return stay

    def whole(self):
        pages = self.held() + self.listed()
        return sorted(pages) == list(range(self.pages))


TABLES = {
    "one request at its table's end": ([60], [26], 4),
    "one that is there already": ([64], [40], 4),
    "one that is behind it": ([75], [20], 4),
    "among others": ([60, 3, 64, 70, 30, 0, 33], [26, 26, 40, 20, 5, 0, 17], 4),
    "the first and the last": ([63, 0, 5, 40, 62], [30, 9, 33, 1, 50], 4),
    "a table of one page": ([15, 2, 16], [33, 40, 1], 1),
    "a table without columns": ([0, 5], [20, 3], 0),
    "more pages behind it than threads": ([16], [256 * 20 + 7], 1),
}


@pytest.mark.parametrize("name", TABLES)
@pytest.mark.parametrize("spare", [600, 3])
def test_no_page_is_lost_at_the_tables_end(name, spare):
    """The list has more than is asked for; or hardly so much, and nothing stays."""
    before, new, width = TABLES[name]
    need = sum(-(-(b + n) // PAGE) - -(-b // PAGE) for b, n in zip(before, new)) + sum(min(width, -(-b // PAGE)) for b in before)
    pool = Pool(np.random.RandomState(len(name)), before, width, need + spare)
    assert pool.whole()
    for _ in range(8):
        pool.step(new, kept=None if spare > 3 else [[]] * len(new))
        assert pool.whole()


def test_the_count_of_taken_pages_stays():
    """Nothing is kept, step after step: the count is what it was."""
    pool = Pool(np.random.RandomState(1), [1020, 40], 64, 100)
    taken, free = int(pool.taken), set(pool.listed())
    for _ in range(12):
        pool.step([26, 26], kept=[[], []])
        assert int(pool.taken) == taken and set(pool.listed()) == free and pool.whole()


@pytest.mark.parametrize("seed", range(4))
def test_many_requests_some_at_their_tables_end(seed):
    """More requests than a workgroup has threads."""
    rng = np.random.RandomState(seed)
    requests, width = 700, 3
    before, new = rng.randint(0, 55, requests).tolist(), rng.randint(0, 30, requests).tolist()
    pool = Pool(rng, before, width, requests * 5 + 50)
    assert pool.whole()
    for _ in range(3):
        pool.step(new)
        assert pool.whole()


@pytest.mark.parametrize("pages", [9, 10, 11, 13, 16])
def test_the_list_runs_out(pages):
    """A table wide enough, a list that is not: tokens without a page end a path, and nothing is lost or given twice."""
    pool = Pool(np.random.RandomState(2), [30, 3, 64, 20], 8, pages)
    assert pool.whole()
    for _ in range(10):
        pool.step([26, 40, 20, 9])
        assert pool.whole()


@pytest.mark.parametrize("order", [[60, 3, 64, 20], [3, 60, 20, 64], [20, 3, 64, 60]])
@pytest.mark.parametrize("short", range(1, 9))
def test_the_list_runs_out_at_the_tables_end(order, short):
    """Both at once.  Only where all that the list still had went to columns that there are not is it not known what that was."""
    new = [40, 26, 26, 30]
    fresh = [c < 4 for b, n in zip(order, new) for c in range(-(-b // PAGE), -(-(b + n) // PAGE))]      # of a step's pages: whether there is a column
    given = len(fresh) - short
    pool = Pool(np.random.RandomState(short), order, 4, sum(-(-b // PAGE) for b in order) + given)
    assert pool.whole()
    listed = pool.listed()
    pool.step(new, kept=[[0]] * 4)
    if given == 0 or any(fresh[:given]):
        assert pool.whole()
    else:
        pages = pool.held() + pool.listed()
        assert len(set(pages)) == len(pages) and set(range(pool.pages)) - set(pages) <= set(listed)


PARTS = {"one by one": [(0, 1), (1, 2), (2, 3), (3, 4), (4, 5)], "from the last": [(4, 5), (3, 4), (2, 3), (1, 2), (0, 1)], "the middle first": [(1, 4), (4, 5), (0, 1)],
         "two halves": [(0, 2), (2, 5)], "the second half first": [(2, 5), (0, 2)]}


@pytest.mark.parametrize("order", PARTS)
@pytest.mark.parametrize("before", [[60, 3, 64, 40, 62], [64, 64, 20, 64, 3], [64, 60, 64, 3, 64]])
def test_a_part_of_the_requests(before, order):
    """A step that is ended by several calls: no page is listed that a request holds, and none twice."""
    from orbitquant_amd import kv_assign, kv_keep

    pool = Pool(np.random.RandomState(3), before, 4, 60)
    new = [26, 40, 20, 30, 9]
    got = kv_assign(pool.lengths, _i32(new), pool.table, pool.free, pool.taken, page_size=PAGE, tokens=sum(new))
    rows, taken = pool.table.tolist(), got.taken
    others = {p for row, n in zip(rows, pool.lengths.tolist()) for p in row[:min(4, -(-(n + 1) // PAGE))] if p >= 0}
    for first, last in PARTS[order]:
        after = kv_keep(_i32([[0]] * (last - first)), got.lengths[first:last], got.starts[first:last + 1], got.slots, pool.caches, block_table=pool.table[first:last],
                        free_pages=pool.free, taken=taken)
        taken = after.taken
        listed = pool.free[int(taken):].tolist()
        assert len(set(listed)) == len(listed) and not others & set(listed)


@pytest.mark.parametrize("before", [[60, 3, 64, 40, 62], [20, 60, 3, 64], [3, 64, 20], [64, 62]])
@pytest.mark.parametrize("kept", [[], [0], [0, 1, 2, 3, 4]])
def test_a_call_repeated(before, kept):
    """With the count that it was first given, over the list that it has changed: no page is listed that a request holds, and none twice."""
    from orbitquant_amd import kv_assign, kv_keep

    pool = Pool(np.random.RandomState(4), before, 4, 60)
    new = [26, 40, 20, 30, 9][:len(before)]
    got = kv_assign(pool.lengths, _i32(new), pool.table, pool.free, pool.taken, page_size=PAGE, tokens=sum(new))
    rows = _i32([kept + [-1] * (5 - len(kept))] * len(before))
    for again in range(3):
        after = kv_keep(rows, got.lengths, got.starts, got.slots, pool.caches, block_table=pool.table, free_pages=pool.free, taken=got.taken)
        pool.lengths, pool.taken = after.lengths, after.taken
        pages = pool.held() + pool.listed()
        assert len(set(pages)) == len(pages) and (again > 0 or pool.whole())


def test_captured_at_the_tables_end():
    """A step at a row's end captured once and replayed, the state moving on, against the eager steps."""
    from orbitquant_amd import kv_assign, kv_keep

    eager, graphed = (Pool(np.random.RandomState(5), [60, 3, 64, 20], 4, 40) for _ in range(2))
    new, rows = _i32([26, 9, 20, 30]), _i32([[0, -1]] * 4)

    def step(pool):
        got = kv_assign(pool.lengths, new, pool.table, pool.free, pool.taken, page_size=PAGE, tokens=85)
        after = kv_keep(rows, got.lengths, got.starts, got.slots, pool.caches, block_table=pool.table, free_pages=pool.free, taken=got.taken)
        pool.lengths.copy_(after.lengths)
        pool.taken.copy_(after.taken)

    state = (graphed.lengths, graphed.taken, graphed.table, graphed.free)
    was = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    for t, old in zip(state, was):
        t.copy_(old)
    for _ in range(8):
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert eager.whole() and graphed.whole()
        for a, b in zip((eager.lengths, eager.taken, eager.table, eager.free), state):
            assert torch.equal(a, b)


def test_the_example_at_its_tables_end():
    """The drafting example's steps where a request has as many tokens as its row has places."""
    from orbitquant_amd import OrbitKVCache
    from orbitquant_amd.examples import decode, draft

    model = draft.Drafter(1, 2, 200, 3)
    width = model.block_table.shape[1]
    longest, pages = width * draft.PAGE - 1, 2 * width + 20
    model.free_pages = torch.randperm(pages, device="cuda", dtype=torch.int32)
    attention = model.layers[0].attention
    attention.cache = OrbitKVCache.empty(pages, decode.KV_HEADS, draft.HEAD_DIM, page_size=draft.PAGE)
    attention.rotary = draft.rotary_tables(width * draft.PAGE + 8)
    ids = torch.randint(0, draft.VOCABULARY, (longest + 60,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    model.step(ids, _i32([longest, 60]), max_new=longest)
    for _ in range(4):
        was = model.lengths.tolist()
        model.draft_step()
        held = [p for row, n in zip(model.block_table.tolist(), model.lengths.tolist()) for p in row[:min(width, -(-n // draft.PAGE))]]
        assert sorted(held + model.free_pages[int(model.taken):].tolist()) == list(range(pages))
        assert model.lengths.tolist()[0] == width * draft.PAGE and model.lengths.tolist()[1] > was[1]
