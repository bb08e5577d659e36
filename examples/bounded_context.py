"""Streaming attention layers over a paged cache that stays within a budget.

    python examples/bounded_context.py --requests 4 --prompt 1500 --new 200 --budget 1024

Each layer's prompt goes through the cache in chunks (``paged_window_attention``:
a sliding window, the first tokens stay visible), its last ``--look`` tokens and
then every new token one at a time.  Each of those attends to what its request
holds (``paged_decode_attention``, which gathers each position's attention
weight), so that a prompt past the budget is cut by what its last tokens looked
at.  Whenever a request holds ``--budget`` plus ``--slack`` positions its cache
is cut back to the budget (``evict_paged_context``).  Keys and values are
written by the serving operators' ``write_context_kv``: a key is normed and
rotated at the position its token has in the text, and keeps that rotation when
its row moves.

The model is a stack of attention layers with random weights: what it computes
is of no use, the calls are a serving loop's.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from flashmap_b200 import cache_ops, serving_ops  # noqa: E402


class PagedLayers:
    """The paged caches of a stack of attention layers with what they hold."""

    def __init__(self, layers, requests, heads, kv_heads, head_dim, capacity, page=16, device="cuda"):
        self.layers, self.requests, self.heads, self.kv_heads, self.head_dim = layers, requests, heads, kv_heads, head_dim
        self.page, self.capacity = page, capacity
        cols = -(-capacity // page)
        order = torch.randperm(requests * cols, device=device).to(torch.int32)
        self.table = order.view(requests, cols)
        # one pool per layer in vLLM's layout: a row holds a token's key, then its value
        self.pools = [torch.zeros(requests * cols, kv_heads, page, 2 * head_dim, dtype=torch.bfloat16, device=device)
                      for _ in range(layers)]
        self.pool_ptrs = torch.tensor([p.data_ptr() for p in self.pools], dtype=torch.int64, device=device)
        self.held = torch.zeros(requests, dtype=torch.int32, device=device)  # positions of each request in the cache
        self.most = 0                                                         # and the most of any, known on the host
        self.sums = [torch.zeros(requests, kv_heads, capacity, device=device) for _ in range(layers)]
        self.norm = torch.ones(layers, head_dim, dtype=torch.bfloat16, device=device)
        self.rope = serving_ops.rope_table(1 << 16, head_dim, 1e6, device)

    def views(self, layer):
        pool = self.pools[layer]
        return pool[..., : self.head_dim], pool[..., self.head_dim:]

    def append(self, kv, positions, rows_each):
        """``kv (requests * rows_each, layers, 2, kv_heads, head_dim)``, each request's next rows, whose tokens stand
        at ``positions`` of the text."""
        at = self.held.long()[:, None] + torch.arange(rows_each, device=kv.device)[None]
        pages = self.table.gather(1, at // self.page)
        slots = (pages.long() * self.page + at % self.page).flatten()
        p = self.pools[0]
        serving_ops.write_context_kv(kv, positions.flatten(), slots, self.norm, self.rope, self.pool_ptrs,
                                     (p.stride(0), p.stride(1), p.stride(2), self.head_dim), self.page, 1e-6,
                                     heads_per_cache=self.kv_heads)
        self.held += rows_each
        self.most += rows_each

    def evict(self, budget, sinks, recent):
        held = self.held
        for layer in range(self.layers):
            k, v = self.views(layer)
            _, self.held, sums = cache_ops.evict_paged_context(k, v, held, self.table, self.sums[layer], budget,
                                                               sinks=sinks, recent=recent)
            self.sums[layer].zero_()
            self.sums[layer][..., :budget] = sums
        self.most = min(self.most, budget)


def run(requests=4, prompt=1500, new=200, budget=1024, slack=64, window=512, sinks=4, chunk=512, look=32, layers=2,
        heads=16, kv_heads=4, head_dim=128, seed=0):
    """Runs the loop; returns the last step's output and the positions held after every step."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = PagedLayers(layers, requests, heads, kv_heads, head_dim, max(prompt, budget + slack) + 1)
    scale = head_dim ** -0.5

    def project(rows):  # queries, and all layers' keys and values, of `rows` new tokens to a request
        q = torch.randn(requests * rows, heads, head_dim, generator=g, device="cuda").to(torch.bfloat16)
        kv = torch.randn(requests * rows, layers, 2, kv_heads, head_dim, generator=g, device="cuda").to(torch.bfloat16)
        return q, kv

    def rotated(q, positions):
        return serving_ops.vllm_rms_norm_rope(q, cache.norm[0], cache.rope, positions.flatten(), 1e-6)

    def token(position):  # one new token of every request, which gathers weights
        q, kv = project(1)
        positions = torch.full((requests, 1), position, device="cuda")
        cache.append(kv, positions, 1)
        x = rotated(q, positions)
        for layer in range(layers):
            x = cache_ops.paged_decode_attention(x, *cache.views(layer), cache.held, cache.table, cache.most, scale,
                                                 weight_sums=cache.sums[layer])
        return x

    # the prompt: chunk by chunk up to its last tokens, whose weights the first eviction goes by
    x = None
    body = prompt - min(max(look, 0), prompt)
    for begin in range(0, body, chunk):
        rows = min(chunk, body - begin)
        q, kv = project(rows)
        positions = (begin + torch.arange(rows, device="cuda")).repeat(requests, 1)
        cache.append(kv, positions, rows)
        cu = torch.arange(requests + 1, dtype=torch.int32, device="cuda") * rows
        x = rotated(q, positions)
        for layer in range(layers):
            x = cache_ops.paged_window_attention(x, *cache.views(layer), cu, cache.held, cache.table, rows, cache.most,
                                                 scale, window=window, sinks=sinks)
    for position in range(body, prompt):
        x = token(position)
    # new tokens, one at a time
    held = []
    for step in range(new):
        if cache.most >= budget + slack:
            cache.evict(budget, sinks, recent=min(window, budget - sinks))
        x = token(prompt + step)
        held.append(cache.most)
    return x, held


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("requests", 4), ("prompt", 1500), ("new", 200), ("budget", 1024), ("slack", 64), ("window", 512),
                        ("sinks", 4), ("chunk", 512), ("look", 32), ("layers", 2)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args(argv)
    x, held = run(**vars(args))
    torch.cuda.synchronize()
    print(f"{args.requests} requests, {args.prompt} + {args.new} tokens: {held[0]} positions held after the first new "
          f"token, {held[-1]} after the last, {max(held)} at most; output norm {float(x.float().norm()):.4g}")


if __name__ == "__main__":
    main()
