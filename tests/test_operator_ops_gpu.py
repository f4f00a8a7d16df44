"""The torch.library ops describe every call of the functions: queries in two parts, a row width with padding
and no divisors, a budget per request."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200 import ops  # noqa: F401
from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights, evict_cache
from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks
from test_eviction_gpu import evict_case
from tree_util import SM, build_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rms_offset", [500, -1])
def test_split_queries_and_qk_dim(cuda_device, rms_offset):
    c, q, bt, ctx, _ = build_case(cuda_device, 2, 3, 12, 384, 116, 16, [200, 33])
    assert c.shape[3] > 500  # without divisors the row width is not the attention's
    lat, pe = q[..., :384].contiguous(), q[..., 384:].contiguous()
    mask = tree_masks(torch.tensor([-1, 0, 0], device=cuda_device))
    o, o2 = (torch.zeros(6, 12, 384, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    l1, l2 = torch.zeros(6, 12, device=cuda_device), torch.zeros(6, 12, device=cuda_device)
    tree_attention(lat, c, o, l1, bt, ctx, mask, rank=384, sm_scale=SM, page_size=16, rms_offset=rms_offset, q_pe=pe, qk_dim=500)
    torch.ops.qmla.tree_attention(lat, c, o2, l2, bt, ctx, mask, 384, SM, 16, rms_offset, False, False, 0.0, None, q_pe=pe, qk_dim=500)
    assert torch.equal(o, o2) and torch.equal(l1, l2) and o.any()
    lens = (ctx[:, None] + torch.arange(1, 4, dtype=torch.int32, device=cuda_device)).flatten().contiguous()
    w, w2 = torch.ones(2, 210, device=cuda_device), torch.ones(2, 210, device=cuda_device)
    accumulate_attention_weights(lat, c, w, l1, bt, lens, sm_scale=SM, page_size=16, rank=384, rms_offset=rms_offset, q_pe=pe, qk_dim=500, qrows=3)
    torch.ops.qmla.accumulate_attention_weights(lat, c, w2, l1, bt, lens, SM, 16, rms_offset, False, False, 0.0, None, 3, 1.0, q_pe=pe,
                                                rank=384, qk_dim=500)
    assert torch.equal(w, w2) and (w > 1).any()


def test_budgets(cuda_device):
    cache, w, pos, bt, lens = evict_case(cuda_device, 3, [200, 90, 150], 16)
    budgets = torch.tensor([20, 1000, 0], dtype=torch.int32, device=cuda_device)
    a, b = cache.clone(), cache.clone()
    want = evict_cache(a, w, pos, bt, lens, 50, page_size=16, budgets=budgets)
    new = tuple(torch.zeros_like(t) for t in want)
    torch.ops.qmla.evict_cache(b, w, pos, bt, lens, *new, 50, 16, 0, None, budgets=budgets)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(want, new)) and new[2].tolist() == [20, 50, 0]
