"""The status word of the gather and of the fused update, first used inside a capture."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200 import _lib, mla_gather
from qwen_mla_vllm_b200.rotary import rope_kv_cache_update, rotary_steps

pytestmark = pytest.mark.gpu


def test_a_capture_neither_makes_nor_clears_the_word(cuda_device, monkeypatch):
    bf = torch.bfloat16
    q, k, lat = torch.randn(3, 2, 58, device=cuda_device).to(bf), torch.rand(3, 60, device=cuda_device).to(bf), torch.randn(3, 64, device=cuda_device).to(bf)
    cache = torch.zeros(4, 16, 1, 128, dtype=bf, device=cuda_device)
    pos, steps = torch.arange(3, device=cuda_device), rotary_steps(58, device=cuda_device)[0]
    good, bad = torch.tensor([0, 5, 63], device=cuda_device), torch.tensor([0, 64, 1], device=cuda_device)
    out = torch.empty_like(q)
    call = lambda slots: rope_kv_cache_update(q, k, lat, pos, slots, steps, cache, packed_rope=58, local_heads=2, q_out=out)  # noqa: E731
    call(good)  # the module is loaded
    torch.cuda.synchronize()
    monkeypatch.setattr(mla_gather, "_status", {})
    g, gb, gb2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(good)
    with torch.cuda.graph(gb):
        call(bad)
    torch.cuda.synchronize()
    assert mla_gather.gather_status(cuda_device) == 0  # nothing has run
    cache.zero_()
    gb.replay()  # captured while there was no word: the bad slot is skipped all the same
    torch.cuda.synchronize()
    assert mla_gather.gather_status(cuda_device) == 0 and (cache.view(64, 128).abs().amax(1) > 0).nonzero().flatten().tolist() == [0, 1]
    call(bad)
    g.replay()  # a sound replay does not clear what another call reported
    assert mla_gather.gather_status(cuda_device) == _lib.DEV_ERR_INDEX
    with torch.cuda.graph(gb2):
        call(bad)  # there is a word now
    gb2.replay()
    call(good)
    g.replay()
    assert mla_gather.gather_status(cuda_device, clear=False) == _lib.DEV_ERR_INDEX
    assert mla_gather.gather_status(cuda_device) == _lib.DEV_ERR_INDEX and mla_gather.gather_status(cuda_device) == 0
