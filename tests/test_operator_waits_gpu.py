"""How the tensor-core operators end: nothing of a call is in flight when its blocks leave, and a wait that
gives up is told."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200 import _lib
from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights
from qwen_mla_vllm_b200.tree_attention import operator_status, tree_attention, tree_masks
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


@pytest.mark.parametrize("fp8", [False, True])
def test_a_wait_that_gives_up_is_reported(cuda_device, monkeypatch, fp8):
    """With no patience at all, the first unfinished copy ends the call: NaN from the tree, old or new weights
    and nothing else from the accumulation, the bit set until it is cleared; the next call is sound."""
    c, q, bt, ctx, ks = build_case(cuda_device, 6, 5, 12, 384, 116, 16, [900, 0, 77, 3000, 128, 5], mode="log8" if fp8 else "native", fp8=fp8)
    kw = dict(sm_scale=SM, page_size=16, rms_offset=500, rms_log8=fp8, k_scale=torch.tensor(ks, device=cuda_device) if fp8 else None)
    mask = tree_masks((torch.arange(5) - 1).to(cuda_device))
    o = torch.empty(30, 12, 384, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.empty(30, 12, device=cuda_device)
    lens = (ctx[:, None] + torch.arange(1, 6, dtype=torch.int32, device=cuda_device)).flatten().contiguous()
    old = torch.rand(6, 3100, device=cuda_device)
    w = old.clone()
    tree = lambda: tree_attention(q, c, o, lse, bt, ctx, mask, rank=384, **kw)  # noqa: E731
    weights = lambda: accumulate_attention_weights(q, c, w, good[1], bt, lens, qrows=5, decay=0.5, **kw)  # noqa: E731
    operator_status()
    tree()
    good = o.clone(), lse.clone()
    weights()
    new = w.clone()
    assert operator_status() == 0
    monkeypatch.setenv("QMLA_WAIT_US", "0")
    tree()
    assert operator_status(clear=False) == _lib.DEV_ERR_TIMEOUT and operator_status() == _lib.DEV_ERR_TIMEOUT
    assert o.isnan().all() and lse.isnan().all()
    assert operator_status() == 0
    w.copy_(old)
    weights()
    assert operator_status(cuda_device) == _lib.DEV_ERR_TIMEOUT and operator_status(0) == 0
    assert ((w == old) | (w == new)).all()
    monkeypatch.delenv("QMLA_WAIT_US")
    tree()
    w.copy_(old)
    weights()
    assert torch.equal(o, good[0]) and torch.equal(lse, good[1]) and torch.equal(w, new)
    assert operator_status() == 0
