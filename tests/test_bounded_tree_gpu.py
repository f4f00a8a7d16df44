"""The operators together, as the example's serving loop and as torch.library ops, on the GPU."""
from __future__ import annotations

import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_serving_loop_keeps_its_bound(cuda_device):
    sys.path.insert(0, str(ROOT / "examples"))
    import bounded_tree_decode as ex
    cache = ex.main(["--steps", "60", "--requests", "3", "--budget", "128"])
    assert cache.lens.tolist() == [128] * 3 and int(cache.next_position.max()) > 160
    kept = cache.positions[:, :128]
    for r in range(3):
        p = kept[r].sort().values
        assert torch.equal(p, p.unique())  # no token twice
        last = int(cache.next_position[r])
        assert p[:ex.SINKS].tolist() == list(range(ex.SINKS))
        assert p[-ex.RECENT:].tolist() == list(range(last - ex.RECENT, last))
    assert cache.weights.isfinite().all() and (cache.weights[:, :128] > 0).any()
    # a committed tree's rows carry their own rotation: the cache holds no NaN and no stale zero row
    rows = cache.rows.view(-1, ex.WIDTH)[cache.slots(torch.arange(128, device=cuda_device).repeat(3, 1))]
    assert rows.isfinite().all() and (rows.abs().amax(dim=1) > 0).all()


def test_accumulated_weights_follow_the_tree(cuda_device):
    """A path accepted from a tree, then decoded as a chain over the committed rows, has the same lse."""
    sys.path.insert(0, str(ROOT / "examples"))
    import bounded_tree_decode as ex
    from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights
    from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks
    g = torch.Generator().manual_seed(2)
    cache = ex.BoundedCache(2, 256, 64, cuda_device)
    cache.lens += 100
    cache.rows.copy_(torch.randn(cache.rows.shape, generator=g).to(torch.bfloat16))
    cache.rows[..., ex.QK:] = cache.rows[..., ex.QK:].abs() + 0.5
    mask = tree_masks(torch.tensor(ex.PARENTS, device=cuda_device))
    q = torch.randn(16, ex.HEADS, ex.QK, generator=g).to(torch.bfloat16).to(cuda_device)
    o = torch.empty(16, ex.HEADS, ex.RANK, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.empty(16, ex.HEADS, device=cuda_device)
    tree_attention(q, cache.rows, o, lse, cache.block_table, cache.lens, mask, rank=ex.RANK, sm_scale=ex.SM_SCALE,
                   page_size=ex.PAGE, rms_offset=ex.QK)
    path = torch.tensor([[0, 2, 5, 7]] * 2, device=cuda_device)
    cache.commit(path)
    rows = (torch.arange(2, device=cuda_device)[:, None] * 8 + path).reshape(-1)
    lens = (cache.lens[:, None] - 3 + torch.arange(4, device=cuda_device)).reshape(-1).to(torch.int32)
    cache.weights.zero_()
    accumulate_attention_weights(q[rows], cache.rows, cache.weights, lse[rows], cache.block_table, lens, sm_scale=ex.SM_SCALE,
                                 page_size=ex.PAGE, rms_offset=ex.QK, qrows=4)
    # softmax weights over all visible tokens: one per query row and head
    assert (cache.weights.sum(dim=1) - 4 * ex.HEADS).abs().max() < 4 * ex.HEADS * 1e-4
    assert not cache.weights[:, 104:].any()


def test_library_ops_match_the_functions(cuda_device):
    import qwen_mla_vllm_b200.ops  # noqa: F401
    from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights, evict_cache
    from qwen_mla_vllm_b200.rotary import rope_kv_cache_update, rotary_steps
    from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks
    from tree_util import SM, build_case
    c, q, bt, ctx, _ = build_case(cuda_device, 2, 4, 12, 384, 116, 16, [100, 37])
    mask = tree_masks(torch.tensor([-1, 0, 0, 1], device=cuda_device))
    outs = []
    for lib in (False, True):
        o, lse = torch.empty(8, 12, 384, dtype=torch.bfloat16, device=cuda_device), torch.empty(8, 12, device=cuda_device)
        cc, w = c.clone(), torch.zeros(2, 120, device=cuda_device)
        lens = (ctx[:, None] + torch.arange(1, 5, device=cuda_device)).reshape(-1).to(torch.int32)
        pos = torch.arange(120, dtype=torch.int32, device=cuda_device).repeat(2, 1)
        steps, _ = rotary_steps(58, device=cuda_device)
        qp, kp = q[..., 384:].clone(), torch.rand(8, 128, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1)).to(torch.bfloat16)
        lat = kp[:, :1].expand(8, 384).contiguous()
        slot = torch.arange(8, device=cuda_device)
        rp = torch.arange(8, device=cuda_device)
        nw, npos, nl = torch.empty(2, 30, device=cuda_device), torch.empty(2, 30, dtype=torch.int32, device=cuda_device), torch.empty(2, dtype=torch.int32, device=cuda_device)
        qo = torch.empty_like(qp)
        new = (ctx + 4).to(torch.int32)
        if lib:
            t = torch.ops.qmla
            t.tree_attention(q, cc, o, lse, bt, ctx, mask, 384, SM, 16, 500, False, False, 0.0, None)
            t.accumulate_attention_weights(q, cc, w, lse, bt, lens, SM, 16, 500, False, False, 0.0, None, 4, 0.9)
            t.evict_cache(cc, w, pos, bt, new, nw, npos, nl, 30, 16, 2, None)
            t.rope_kv_cache_update(qp, kp, lat, rp, slot, steps, cc, qo, 116, 12, False, 1.0, None, "native")
        else:
            tree_attention(q, cc, o, lse, bt, ctx, mask, rank=384, sm_scale=SM, page_size=16, rms_offset=500)
            accumulate_attention_weights(q, cc, w, lse, bt, lens, sm_scale=SM, page_size=16, rms_offset=500, qrows=4, decay=0.9)
            evict_cache(cc, w, pos, bt, new, 30, page_size=16, sinks=2, out=(nw, npos, nl))
            rope_kv_cache_update(qp, kp, lat, rp, slot, steps, cc, packed_rope=116, local_heads=12, q_out=qo)
        outs.append((o, lse, w, cc, nw, npos, nl, qo))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
