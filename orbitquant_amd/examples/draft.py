"""Serving with drafted tokens: every step checks a small tree of guesses per request at once and keeps the path that the model agrees with.

    python -m orbitquant_amd.examples.draft [--layers 4] [--requests 8] [--steps 64] [--depth 4]

The decoder of `decode.py`, its rotary positions applied by `kv_append`.  Guesses are the two tokens that have last followed a token in what the model
itself has said, and after each of them a chain of what last followed: a tree of 1 + 2 * depth tokens, the first of which is the certain one.  A step
is `kv_assign` and `kv_tree`, the layers over all nodes, the walk down the tree as far as the model's own choice is among the children, and `kv_keep`: the path's
entries become the request's last tokens in all layers' caches, and pages that only held wrong guesses go back.  Nothing comes to the host, so a
step is a graph.
"""

from __future__ import annotations

import argparse
import time

import torch
from torch import nn

from orbitquant_amd import QKNormRotary, kv_assign, kv_keep, kv_tree
from orbitquant_amd.examples.decode import HEAD_DIM, HIDDEN, PAGE, VOCABULARY, Decoder


def rotary_tables(positions: int, device="cuda") -> QKNormRotary:
    half = HEAD_DIM // 2
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    return QKNormRotary(angle.cos().float(), angle.sin().float())


def accepted(ids: torch.Tensor, chosen: torch.Tensor, parents: torch.Tensor, depth: int) -> torch.Tensor:
    """The path down each tree [requests, nodes] on which every token is what the model chose after the one before: int32 [requests, depth + 1] nodes, -1
    behind its end.  Where two children of a node are the same token, the first is taken."""
    at = torch.zeros(len(ids), dtype=torch.int64, device=ids.device)
    path = [at]
    node = torch.arange(ids.shape[1], device=ids.device)
    for _ in range(depth):
        fits = (parents == at[:, None]) & (ids == chosen.gather(1, at.clamp(min=0)[:, None])) & (at >= 0)[:, None]
        at = torch.where(fits, node, ids.shape[1]).amin(1)
        at = torch.where(at < ids.shape[1], at, -1)
        path.append(at)
    return torch.stack(path, 1).int()


class Drafter(Decoder):
    def __init__(self, layers: int, requests: int, longest: int, depth: int, device="cuda", seed: int = 0) -> None:
        # (wrong guesses need room behind the last kept token until their step is over)
        super().__init__(layers, requests, longest + 2 * depth + 1, device, seed, rotary=rotary_tables(longest + depth + 1, device))
        self.depth, self.nodes = depth, 1 + 2 * depth
        parents = torch.tensor([-1, 0, 0] + list(range(1, self.nodes - 2)), dtype=torch.int32, device=device)[: self.nodes]
        self.parents, self.parents_of_all = parents, parents.repeat(requests)
        self.each_new = torch.full((requests,), self.nodes, dtype=torch.int32, device=device)
        self.rows = torch.arange(requests, device=device)
        self.followed = torch.zeros(requests, VOCABULARY, 2, dtype=torch.int64, device=device)      # what has last followed each token, and before that
        self.said = torch.zeros(requests, depth + 1, dtype=torch.int64, device=device)              # of the last step, -1 behind the end

    def guesses(self) -> torch.Tensor:
        """[requests, nodes]: the certain token, and level by level the two chains."""
        level = self.followed[self.rows, self.last]
        ids = [self.last[:, None]]
        for _ in range(self.depth):
            ids.append(level)
            level = self.followed[self.rows[:, None], level, 0]
        return torch.cat(ids, 1)

    def note(self, before: torch.Tensor, after: torch.Tensor) -> None:
        """That `after` has followed `before` [requests], where it is not negative."""
        was = self.followed[self.rows, before]
        new = (after >= 0) & (after != was[:, 0])
        self.followed[self.rows, before] = torch.where(new[:, None], torch.stack((after, was[:, 0]), 1), was)

    @torch.no_grad()
    def draft_step(self, **hints) -> torch.Tensor:
        """-> `said`: what each request has said in this step, one token and as many as were guessed."""
        ids = self.guesses()
        requests = len(ids)
        assignment = kv_assign(self.lengths, self.each_new, self.block_table, self.free_pages, self.taken, page_size=PAGE, tokens=ids.numel())
        tree = kv_tree(self.parents_of_all, assignment.starts, assignment.lengths, max_new=self.nodes)
        x = self.embedding[ids.flatten()]
        for layer in self.layers:
            x = layer(x, assignment, self.block_table, tree=tree, max_new=self.nodes, **hints)
        chosen = self.head(nn.functional.rms_norm(x, (HIDDEN,))).argmax(-1).view(requests, -1)
        path = accepted(ids, chosen, self.parents, self.depth)
        kept = kv_keep(path, assignment.lengths, assignment.starts, assignment.slots, [layer.attention.cache for layer in self.layers],
                       block_table=self.block_table, free_pages=self.free_pages, taken=assignment.taken)
        self.said.copy_(torch.where(path >= 0, chosen.gather(1, path.clamp(min=0).long()), -1))
        before = ids.gather(1, path.clamp(min=0).long())
        for i in range(self.depth + 1):
            self.note(before[:, i], self.said[:, i])
        self.last.copy_(self.said.gather(1, (path >= 0).sum(1, keepdim=True) - 1)[:, 0])
        self.lengths.copy_(kept.lengths)
        self.taken.copy_(kept.taken)
        return self.said

    def captured_draft_step(self, **hints) -> torch.cuda.CUDAGraph:
        """The step as a graph.  The state is left as it was (but for cache entries behind the requests' tokens)."""
        state = (self.lengths, self.taken, self.last, self.block_table, self.free_pages, self.followed, self.said)
        was = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.draft_step(**hints)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.draft_step(**hints)
        for t, old in zip(state, was):
            t.copy_(old)
        return graph


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--depth", type=int, default=4, help="of the trees: tokens that are guessed one behind the other")
    ap.add_argument("--prompt", type=int, default=500, help="the longest prompt; the others are shorter")
    opts = ap.parse_args(argv)
    prompts = [max(1, opts.prompt * (i + 1) // opts.requests) for i in range(opts.requests)]
    longest = opts.prompt + (opts.steps + 1) * (opts.depth + 1)
    model = Drafter(opts.layers, opts.requests, longest, opts.depth)
    ids = torch.randint(0, VOCABULARY, (sum(prompts),), device="cuda")
    first = model.step(ids, torch.tensor(prompts, dtype=torch.int32, device="cuda"), max_new=max(prompts)).tolist()
    graph = model.captured_draft_step(max_length=longest)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    said = []
    for _ in range(opts.steps):
        graph.replay()
        said.append(model.said.clone())
    torch.cuda.synchronize()
    each = (time.perf_counter() - begin) / opts.steps
    said = torch.stack(said, 1)
    tokens = int((said >= 0).sum())
    result = {"prompts": prompts, "first": first, "said": said.tolist(), "tokens": tokens, "ms_per_step": each * 1e3, "lengths": model.lengths.tolist(),
              "pages_taken": int(model.taken)}
    print(f"{opts.requests} requests, prompts of {prompts[0]} to {prompts[-1]} tokens, {opts.layers} layers, trees of {model.nodes}: {each * 1e3:.3f} ms a step, "
          f"{tokens / opts.steps / opts.requests:.2f} tokens a step and request, {tokens / opts.steps / each:.0f} tokens/s")
    return result


if __name__ == "__main__":
    main()
