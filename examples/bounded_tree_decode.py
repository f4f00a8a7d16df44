"""Tree-drafted decoding over a latent cache that keeps a bound: the operators as a serving loop uses them.

    python examples/bounded_tree_decode.py [--steps 12] [--requests 4] [--budget 512]

Every step of every request: a tree of drafted tokens is rotated and written behind the committed ones
(`rope_kv_cache_update`), all its nodes attend to the cache together (`tree_attention`), a path
of the tree is accepted and its rows take the places of the next committed tokens, the accepted tokens
add their attention weights to the cache's (`accumulate_attention_weights`), and a request that outgrew
its budget is cut back (`evict_cache`).  A request's tokens keep their own rotary positions
wherever their rows end up.  Projections and sampling are stand-ins (random draws): the point is the
cache.
"""
from __future__ import annotations

import argparse
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))

from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights, evict_cache  # noqa: E402
from qwen_mla_vllm_b200.rotary import rope_kv_cache_update, rotary_steps  # noqa: E402
from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks  # noqa: E402

HEADS, RANK, GROUPS, ROT, PAGE = 24, 768, 4, 58, 16  # the plugin's tp1 layer
ROPE = GROUPS * ROT
QK, WIDTH = RANK + ROPE, RANK + ROPE + HEADS
SM_SCALE = 1 / 16
PARENTS = [-1, 0, 0, 1, 1, 2, 3, 5]  # a tree of eight nodes
SINKS, RECENT = 4, 64


class BoundedCache:
    """The paged rows of a batch, with every token's rotary position and accumulated weight."""

    def __init__(self, requests: int, budget: int, headroom: int, device: torch.device):
        self.budget, self.cols = budget, budget + headroom
        pages = -(-self.cols // PAGE)
        self.rows = torch.zeros(requests * pages, PAGE, 1, WIDTH, dtype=torch.bfloat16, device=device)
        self.block_table = torch.randperm(requests * pages, device=device).reshape(requests, pages).to(torch.int32)
        self.weights = torch.zeros(requests, self.cols, device=device)
        self.positions = torch.full((requests, self.cols), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.next_position = torch.zeros(requests, dtype=torch.int32, device=device)

    def slots(self, tokens: torch.Tensor) -> torch.Tensor:
        """Cache slots of tokens [requests, n] (numbers within each request)."""
        page = torch.gather(self.block_table, 1, tokens.long() // PAGE).long()
        return (page * PAGE + tokens.long() % PAGE).reshape(-1)

    def commit(self, path: torch.Tensor) -> None:
        """Accept the drafted nodes path [requests, n] (ascending): their rows become the next tokens."""
        n = path.shape[1]
        order = torch.arange(n, device=path.device)
        src, dst = self.slots(self.lens[:, None] + path), self.slots(self.lens[:, None] + order)
        flat = self.rows.view(-1, WIDTH)
        flat[dst] = flat[src].clone()
        at = (self.lens[:, None] + order).long()
        self.positions.scatter_(1, at, (self.next_position[:, None] + order).to(torch.int32))
        self.weights.scatter_(1, at, 0.0)
        self.lens += n
        self.next_position += n

    def bound(self) -> None:
        """Cut every request back to the budget; its oldest and newest tokens stay."""
        w, p, lens = evict_cache(self.rows, self.weights, self.positions, self.block_table, self.lens, self.budget,
                                 page_size=PAGE, sinks=SINKS, recent_from=(self.next_position - RECENT).to(torch.int32))
        self.weights.zero_()
        self.weights[:, :w.shape[1]] = w
        self.positions.fill_(-1)
        self.positions[:, :p.shape[1]] = p
        self.lens = lens


def step(cache: BoundedCache, steps: torch.Tensor, mask: torch.Tensor, depth: torch.Tensor, paths: list[list[int]],
         g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """One verify step: returns the drafted nodes' attention outputs and their log-sum-exp."""
    dev = cache.rows.device
    R, N = cache.lens.shape[0], mask.shape[-1]
    # stand-ins for the layer's projections of the R * N drafted tokens
    q = torch.randn(R * N, HEADS, QK, generator=g, device=dev).to(torch.bfloat16)
    latent = torch.randn(R * N, RANK, generator=g, device=dev).to(torch.bfloat16)
    rms = torch.rand(R * N, HEADS, generator=g, device=dev) + 0.5
    k_pe = torch.cat([torch.randn(R * N, ROPE, generator=g, device=dev), rms], 1).to(torch.bfloat16)
    # a node's position is its depth past the committed tokens, its row lies in the order of the nodes
    positions = (cache.next_position[:, None] + depth).reshape(-1).to(torch.int32)
    slots = cache.slots(cache.lens[:, None] + torch.arange(N, device=dev))
    rope_kv_cache_update(q[..., RANK:], k_pe, latent, positions, slots, steps, cache.rows, packed_rope=ROPE, local_heads=HEADS)
    o = torch.empty(R * N, HEADS, RANK, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(R * N, HEADS, device=dev)
    tree_attention(q, cache.rows, o, lse, cache.block_table, cache.lens, mask, rank=RANK, sm_scale=SM_SCALE, page_size=PAGE,
                   rms_offset=QK)
    # stand-in for the sampler: every request accepts one path of the tree
    path = torch.tensor(paths[int(torch.randint(len(paths), (1,), generator=g, device=dev))], device=dev).repeat(R, 1)
    n = path.shape[1]
    cache.commit(path)
    rows = (torch.arange(R, device=dev)[:, None] * N + path).reshape(-1)
    lens = (cache.lens[:, None] - n + 1 + torch.arange(n, device=dev)).reshape(-1).to(torch.int32)
    accumulate_attention_weights(q[rows], cache.rows, cache.weights, lse[rows], cache.block_table, lens, sm_scale=SM_SCALE,
                                 page_size=PAGE, rms_offset=QK, qrows=n, decay=0.98)
    cache.bound()
    return o, lse


def main(argv=None) -> BoundedCache:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=12)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--budget", type=int, default=512)
    a = ap.parse_args(argv)
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(0)
    mask = tree_masks(torch.tensor(PARENTS, device=dev))
    depth = torch.tensor([bin(m).count("1") - 1 for m in mask.tolist()], device=dev)
    leaves = [i for i in range(len(PARENTS)) if i not in PARENTS]
    paths = [[j for j in range(len(PARENTS)) if mask[i].item() >> j & 1] for i in leaves]
    steps, _ = rotary_steps(ROT, 1e7, device=dev)
    cache = BoundedCache(a.requests, a.budget, 64, dev)
    for i in range(a.steps):
        o, lse = step(cache, steps, mask, depth, paths, g)
        print(f"step {i}: tokens kept {cache.lens.tolist()}, positions up to {cache.next_position.max().item()}, "
              f"mean lse {lse.mean().item():.3f}")
    return cache


if __name__ == "__main__":
    main()
