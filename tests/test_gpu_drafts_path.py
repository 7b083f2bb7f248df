"""A drafted path against the same tokens said one behind the other: rows of the attention, and what the drafting example says."""

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import _check, _i32, _queries
from test_gpu_kv_drafts import GROUP, HEADS, DIM, LAYERS, PAGE, _state

pytestmark = pytest.mark.gpu


def _path(rng, parents):
    """From a root down to some node, the nodes' indices."""
    node, path = int(rng.randint(len(parents))), []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


def test_rows_of_a_path_are_those_of_its_tokens_alone():
    """Three steps: of each tree a path from its root; the path's tokens appended and attended to as a chain, over a cache of their own, have the rows that the tree gave
    them, within what both may be off."""
    from orbitquant_amd import kv_append, kv_assign, kv_attend, kv_keep, kv_tree
    from test_gpu_kv_tree import _parents

    s, plain = _state(21), _state(21)
    rng = np.random.RandomState(22)
    new = s["new"].tolist()
    for _ in range(3):
        parents = _parents(rng, new, "random")
        step = kv_assign(s["lengths"], s["new"], s["table"], s["free"], s["taken"], page_size=PAGE, tokens=sum(new))
        starts = step.starts.tolist()
        tree = kv_tree(_i32(parents), step.starts, step.lengths)
        paths = [_path(rng, parents[starts[r]:starts[r + 1]]) for r in range(len(new))]
        counts = [len(p) for p in paths]
        rows = torch.tensor([starts[r] + n for r, p in enumerate(paths) for n in p], device="cuda")
        chain = kv_assign(plain["lengths"], _i32(counts), plain["table"], plain["free"], plain["taken"], page_size=PAGE, tokens=sum(counts))
        assert torch.equal(tree.positions[rows], chain.positions)           # a path's nodes stand where its tokens would
        for layer in range(LAYERS):
            q, k, v = (_queries(rng, sum(new), h, DIM, torch.bfloat16) for h in (HEADS * GROUP, HEADS, HEADS))
            turned = kv_append(q, k, v, step.slots, s["caches"][layer], s["how"], tree.positions)
            out, lse = kv_attend(turned, s["caches"][layer], s["table"], step.lengths, starts=step.starts, masks=tree.masks, return_lse=True)
            alone = kv_append(q[rows], k[rows], v[rows], chain.slots, plain["caches"][layer], plain["how"], chain.positions)
            assert torch.equal(turned[rows], alone)
            _check((out[rows], lse[rows]), alone, plain["caches"][layer], plain["table"], chain.lengths, starts=chain.starts)
        most = max(counts)
        kept = kv_keep(_i32([p + [-1] * (most - len(p)) for p in paths]), step.lengths, step.starts, step.slots, s["caches"], block_table=s["table"], free_pages=s["free"],
                       taken=step.taken)
        assert torch.equal(kept.lengths, chain.lengths) and torch.equal(kept.taken, chain.taken)
        for st, got in ((s, kept), (plain, chain)):
            st["lengths"], st["taken"] = got.lengths, got.taken


def _continuation(seed, steps):
    """What the example's model says after a prompt, one token a step: the first token, the tokens after it, and how clear each choice was: the distance of the two
    largest logits over the logits' standard deviation."""
    from orbitquant_amd.examples import draft

    model = draft.Drafter(1, 1, 120, 3)
    clear = []
    model.head.register_forward_hook(lambda module, args, logits: clear.append(float(logits[0].float().topk(2).values.diff().abs() / logits[0].float().std())))
    ids = torch.randint(0, draft.VOCABULARY, (40,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    model.step(ids, _i32([40]), max_new=40)
    first, said = int(model.last), []
    for _ in range(steps):
        model.followed.zero_()                  # (no guess but token 0, nothing is known)
        told = model.draft_step()[0].tolist()
        said.append(told[0])
        if told[1] >= 0:
            return None                         # the model says 0: a guess that was right
    return ids, first, said, min(clear)


def test_the_example_says_all_that_it_was_told():
    """Told its own continuation, the drafter keeps every guess: four tokens in one step, the ones that it says one by one.  Of sixteen prompts those are taken whose tokens are
    followed by one token each (the guesses know no more), and whose choices are no near ties."""
    from orbitquant_amd.examples import draft

    tried = 0
    for seed in range(16):
        found = _continuation(seed, 4)
        if found is None:
            continue
        ids, first, said, clear = found
        follows = dict(zip([first, *said[:-2]], said[:-1]))
        if clear < 0.05 or any(follows[a] != b for a, b in zip([first, *said[:-2]], said[:-1])):
            continue
        tried += 1
        drafter = draft.Drafter(1, 1, 120, 3)
        drafter.step(ids, _i32([40]), max_new=40)
        assert int(drafter.last) == first
        for token, after in follows.items():
            drafter.followed[0, token, 0] = after
        assert drafter.draft_step()[0].tolist() == said and drafter.lengths.tolist() == [44] and int(drafter.last) == said[-1]
        # and a wrong guess in the middle: what stands before it is kept
        drafter = draft.Drafter(1, 1, 120, 3)
        drafter.step(ids, _i32([40]), max_new=40)
        for token, after in follows.items():
            drafter.followed[0, token, 0] = after
        if len({first, *said[:3]}) == 4:
            drafter.followed[0, said[0], 0] = (said[1] + 1) % draft.VOCABULARY
            assert drafter.draft_step()[0].tolist() == [*said[:2], -1, -1] and drafter.lengths.tolist() == [42]
    assert tried >= 3
