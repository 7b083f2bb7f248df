"""Serving with the 4-bit key/value cache: ragged prompts in one pass, then tokens one by one as a replayed HIP graph.

    python -m orbitquant_amd.examples.decode [--layers 4] [--requests 8] [--tokens 64]

A decoder of random weights (there is no checkpoint to load here), hidden size 1024, eight heads of 128 over two key heads, every
matrix in four bits.  All layers share one `kv_assign` a step; each has a cache of its own, with the same pages.  Lengths, pages and
the last tokens live on the GPU, so that a step is the same launches every time and needs no host in between.
"""

from __future__ import annotations

import argparse
import time

import torch
from torch import nn

from orbitquant_amd import OrbitCachedAttention, OrbitKVCache, OrbitLinear, kv_assign, recipe

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, VOCABULARY, PAGE = 1024, 8, 2, 128, 4096, 64


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor):
    """Rotary positions: the halves of a head's dimensions turned by the position times a frequency."""
    half = q.shape[-1] // 2
    angle = positions.clamp(min=0)[:, None, None] * 10000.0 ** (-torch.arange(half, device=q.device) / half)
    cos, sin = angle.cos(), angle.sin()

    def turn(x):
        a, b = x[..., :half].float(), x[..., half:].float()
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)

    return turn(q), turn(k)


def linear(inputs: int, outputs: int, generator: torch.Generator, device) -> OrbitLinear:
    weight = torch.randn(outputs, inputs, generator=generator, device=device) / inputs ** 0.5
    return OrbitLinear.from_weight(weight.to(torch.bfloat16), bias=None, config=recipe("w4a4"))


class Layer(nn.Module):
    def __init__(self, pages: int, generator: torch.Generator, device) -> None:
        super().__init__()
        cache = OrbitKVCache.empty(pages, KV_HEADS, HEAD_DIM, page_size=PAGE, device=device)
        wide, kv = HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
        shapes = (HIDDEN, wide), (HIDDEN, kv), (HIDDEN, kv), (wide, HIDDEN), (HIDDEN, 4 * HIDDEN), (4 * HIDDEN, HIDDEN)
        *projections, self.up, self.down = (linear(*shape, generator, device) for shape in shapes)
        self.attention = OrbitCachedAttention(*projections, cache, rotary=rotary)
        self.up.fuse_output_activation(nn.functional.gelu, dtype=torch.bfloat16)

    def forward(self, x, assignment, block_table, **hints):
        x = x + self.attention(nn.functional.rms_norm(x, (HIDDEN,)), assignment, block_table, **hints)
        return x + self.down(self.up(nn.functional.rms_norm(x, (HIDDEN,))))


class Decoder(nn.Module):
    """`requests` rows of a block table over a pool of pages, and the tokens that they hold."""

    def __init__(self, layers: int, requests: int, longest: int, device="cuda", seed: int = 0) -> None:
        super().__init__()
        generator = torch.Generator(device=device).manual_seed(seed)
        width = -(-longest // PAGE)
        self.layers = nn.ModuleList(Layer(requests * width, generator, device) for _ in range(layers))
        self.head = linear(HIDDEN, VOCABULARY, generator, device)
        self.embedding = torch.randn(VOCABULARY, HIDDEN, generator=generator, device=device).to(torch.bfloat16)
        counts = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=device)  # noqa: E731
        self.block_table = counts(requests, width) - 1
        self.free_pages = torch.randperm(requests * width, generator=generator, device=device, dtype=torch.int32)
        self.lengths, self.taken, self.last = counts(requests), counts(1), torch.zeros(requests, dtype=torch.int64, device=device)
        self.one_new = counts(requests) + 1      # (held here: a graph reads it at every replay)

    @torch.no_grad()
    def step(self, ids: torch.Tensor, new_lengths: torch.Tensor, **hints) -> torch.Tensor:
        """The new tokens of all requests, one request behind the other -> the next token of each."""
        assignment = kv_assign(self.lengths, new_lengths, self.block_table, self.free_pages, self.taken, page_size=PAGE, tokens=len(ids))
        x = self.embedding[ids]
        for layer in self.layers:
            x = layer(x, assignment, self.block_table, **hints)
        ends = (assignment.starts[1:] - 1).long()
        self.last.copy_(self.head(nn.functional.rms_norm(x[ends], (HIDDEN,))).argmax(-1))
        self.lengths.copy_(assignment.lengths)
        self.taken.copy_(assignment.taken)
        return self.last

    def captured_step(self) -> torch.cuda.CUDAGraph:
        """A decoding step (one token of every request, the last one chosen) as a graph.  The state is left as it was."""
        state = [t.clone() for t in (self.lengths, self.taken, self.last, self.block_table)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step(self.last, self.one_new, one_each=True)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.step(self.last, self.one_new, one_each=True)
        for t, was in zip((self.lengths, self.taken, self.last, self.block_table), state):
            t.copy_(was)
        return graph


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=64, help="to decode for each request")
    ap.add_argument("--prompt", type=int, default=500, help="the longest prompt; the others are shorter")
    opts = ap.parse_args(argv)
    prompts = [max(1, opts.prompt * (i + 1) // opts.requests) for i in range(opts.requests)]
    model = Decoder(opts.layers, opts.requests, opts.prompt + opts.tokens + 2)
    ids = torch.randint(0, VOCABULARY, (sum(prompts),), device="cuda")
    first = model.step(ids, torch.tensor(prompts, dtype=torch.int32, device="cuda"), max_new=max(prompts)).tolist()
    graph = model.captured_step()
    torch.cuda.synchronize()
    begin = time.perf_counter()
    chosen = []
    for _ in range(opts.tokens):
        graph.replay()
        chosen.append(model.last.clone())
    torch.cuda.synchronize()
    each = (time.perf_counter() - begin) / opts.tokens
    cache = model.layers[0].attention.cache
    held = sum(t.numel() * t.element_size() for t in cache[:4]) / (cache.pages * PAGE)
    result = {"prompts": prompts, "first": first, "tokens": torch.stack(chosen, 1).tolist(), "ms_per_step": each * 1e3,
              "bytes_per_token_and_layer": held, "pages_taken": int(model.taken)}
    print(f"{opts.requests} requests, prompts of {prompts[0]} to {prompts[-1]} tokens, {opts.layers} layers: {each * 1e3:.3f} ms a step, "
          f"{opts.requests / each:.0f} tokens/s; {held:.0f} bytes of cache a token and layer ({4 * KV_HEADS * HEAD_DIM} in bfloat16)")
    return result


if __name__ == "__main__":
    main()
