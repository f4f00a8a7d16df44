"""Who owns the operators' scratch: a stream, a graph, or the caller."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200 import _lib, ops, tree_attention as ta  # noqa: F401
from qwen_mla_vllm_b200.cache_eviction import (accumulate_attention_weights, accumulate_attention_weights_workspace_bytes,
                                               evict_cache, evict_cache_workspace_bytes)
from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_attention_workspace_bytes, tree_masks
from tree_util import SM, build_case

pytestmark = pytest.mark.gpu


class Calls:
    """One call of each operator on a cache of its own; out() is what it left behind."""

    def __init__(self, dev, reqs, nodes, ctx, seed=0):
        self.c, self.q, self.bt, self.ctx, _ = build_case(dev, reqs, nodes, 12, 384, 116, 16, [ctx + 3 * r for r in range(reqs)], seed=seed)
        self.mask = tree_masks((torch.arange(nodes) - 1).to(dev))
        self.o = torch.empty(reqs * nodes, 12, 384, dtype=torch.bfloat16, device=dev)
        self.lse = torch.full((reqs * nodes, 12), 5.0, device=dev)
        self.lens = (self.ctx[:, None] + torch.arange(1, nodes + 1, dtype=torch.int32, device=dev)).flatten().contiguous()
        cols = ctx + 3 * reqs + nodes
        g = torch.Generator().manual_seed(seed)
        self.w = torch.rand(reqs, cols, generator=g).to(dev)
        self.w1 = self.w.clone()
        self.pos = torch.arange(cols, dtype=torch.int32, device=dev).repeat(reqs, 1)
        self.rows = self.c.clone()
        self.new = (torch.empty(reqs, ctx // 2, device=dev), torch.empty(reqs, ctx // 2, dtype=torch.int32, device=dev),
                    torch.empty(reqs, dtype=torch.int32, device=dev))
        self.kw = dict(sm_scale=SM, page_size=16, rms_offset=500)
        self.nodes = nodes

    def tree(self, **kw):
        tree_attention(self.q, self.c, self.o, self.lse, self.bt, self.ctx, self.mask, rank=384, **self.kw, **kw)

    def weights(self, **kw):
        self.w1.copy_(self.w)
        accumulate_attention_weights(self.q, self.c, self.w1, torch.full_like(self.lse, 5.0), self.bt, self.lens, qrows=self.nodes,
                                     **self.kw, **kw)

    def evict(self, **kw):
        self.rows.copy_(self.c)
        evict_cache(self.rows, self.w, self.pos, self.bt, self.ctx, self.new[0].shape[1], page_size=16, out=self.new, **kw)

    def out(self, name):
        return [t.clone() for t in {"tree": (self.o, self.lse), "weights": (self.w1,), "evict": (self.rows, *self.new)}[name]]

    def wipe(self):
        for t in (self.o, self.lse, self.w1, self.rows, *self.new):
            t.zero_()


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bigger", ["tree", "weights", "evict"])
@pytest.mark.parametrize("name", ["tree", "weights", "evict"])
def test_a_graph_outlives_a_larger_call(cuda_device, name, bigger):
    """Captured, then the stream's scratch grows, then others take the memory that a grown scratch leaves."""
    small, big = Calls(cuda_device, 2, 3, 200), Calls(cuda_device, 48, 8, 6000, seed=1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        getattr(small, name)()
        want = small.out(name)
        kept = dict(ta._ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            getattr(small, name)()
        assert ta._ws.keys() == kept.keys() and all(ta._ws[k] is kept[k] for k in kept)  # a capture leaves them alone
        size = kept[(0, st.cuda_stream)].numel()
        del kept
        getattr(big, bigger)()
        others = [torch.full((size,), 77, dtype=torch.uint8, device=cuda_device) for _ in range(8)]
        small.wipe()
        g.replay()
        st.synchronize()
        assert equal(small.out(name), want)
        assert all((t == 77).all() for t in others)
        if bigger == "tree":  # the largest scratch of the three: it did grow
            assert ta._ws[(0, st.cuda_stream)].numel() > size


def test_a_first_call_inside_a_capture(cuda_device):
    """Nothing was kept for the stream yet; two graphs captured on it may run side by side."""
    a, b = Calls(cuda_device, 3, 4, 500), Calls(cuda_device, 5, 2, 900, seed=2)
    a.tree(), b.tree()
    want = a.out("tree"), b.out("tree")
    a.wipe(), b.wipe()
    st, s1, s2 = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for x in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            x.tree()
    assert (0, st.cuda_stream) not in ta._ws
    for _ in range(20):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert equal(a.out("tree"), want[0]) and equal(b.out("tree"), want[1])


def test_a_workspace_of_the_stated_size(cuda_device):
    c = Calls(cuda_device, 4, 5, 700)
    args = (c.q, c.c, c.o, c.lse, c.bt, c.ctx, c.mask)
    need = {"tree": tree_attention_workspace_bytes(*args, rank=384, page_size=16, rms_offset=500),
            "weights": accumulate_attention_weights_workspace_bytes(c.q, c.c, c.w1, c.lse, c.bt, c.lens, page_size=16, rms_offset=500, qrows=5),
            "evict": evict_cache_workspace_bytes(4, c.w.shape[1], c.new[0].shape[1])}
    for name, n in need.items():
        getattr(c, name)()
        want = c.out(name)
        c.wipe()
        guard = torch.full((n + 1024,), 0xA5, dtype=torch.uint8, device=cuda_device)
        getattr(c, name)(workspace=guard[:n])
        assert equal(c.out(name), want) and (guard[n:] == 0xA5).all()
        with pytest.raises(_lib.QmlaError):
            getattr(c, name)(workspace=guard[:n - 1])
        for bad in (torch.empty(n, dtype=torch.uint8), guard[::2]):
            with pytest.raises(ValueError):
                getattr(c, name)(workspace=bad)
    assert tree_attention_workspace_bytes(c.q[:0], c.c, c.o[:0], c.lse[:0], c.bt, c.ctx[:0], c.mask, rank=384, page_size=16, rms_offset=500) == 0


def test_ops_take_a_workspace(cuda_device):
    c = Calls(cuda_device, 2, 3, 300)
    c.tree(), c.weights(), c.evict()
    want = [c.out(n) for n in ("tree", "weights", "evict")]
    c.wipe()
    c.w1.copy_(c.w), c.rows.copy_(c.c)
    ws = torch.empty(1 << 26, dtype=torch.uint8, device=cuda_device)
    kept = dict(ta._ws)
    t = torch.ops.qmla
    t.tree_attention(c.q, c.c, c.o, c.lse, c.bt, c.ctx, c.mask, 384, SM, 16, 500, False, False, 0.0, None, workspace=ws)
    t.accumulate_attention_weights(c.q, c.c, c.w1, torch.full_like(c.lse, 5.0), c.bt, c.lens, SM, 16, 500, False, False, 0.0, None, 3, 1.0,
                                   workspace=ws)
    t.evict_cache(c.rows, c.w, c.pos, c.bt, c.ctx, *c.new, c.new[0].shape[1], 16, 0, None, workspace=ws)
    assert all(equal(c.out(n), x) for n, x in zip(("tree", "weights", "evict"), want))
    assert ta._ws.keys() == kept.keys() and all(ta._ws[k] is kept[k] for k in kept)
