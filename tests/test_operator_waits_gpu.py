"""How the tensor-core operators end: nothing of a call is in flight when its blocks leave."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights
from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks
from tree_util import SM, build_case

pytestmark = pytest.mark.gpu


def test_short_calls_back_to_back_repeat_themselves(cuda_device):
    """Blocks of one call take over the shared memory of the call before within microseconds: an arrival
    or a copy that outlived its block would land in theirs."""
    c, q, bt, ctx, _ = build_case(cuda_device, 40, 3, 12, 384, 116, 16, [17 * i % 300 for i in range(40)])
    mask = tree_masks(torch.tensor([-1, 0, 0], device=cuda_device))
    o = torch.empty(120, 12, 384, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.empty(120, 12, device=cuda_device)
    w = torch.zeros(40, 320, device=cuda_device)
    lens = (ctx[:, None] + torch.arange(1, 4, dtype=torch.int32, device=cuda_device)).flatten().contiguous()

    def both():
        tree_attention(q, c, o, lse, bt, ctx, mask, rank=384, sm_scale=SM, page_size=16, rms_offset=500)
        w.zero_()
        accumulate_attention_weights(q, c, w, lse, bt, lens, sm_scale=SM, page_size=16, rms_offset=500, qrows=3)

    both()
    first = o.clone(), lse.clone(), w.clone()
    for _ in range(10):
        for _ in range(20):
            both()
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1]) and torch.equal(w, first[2])
