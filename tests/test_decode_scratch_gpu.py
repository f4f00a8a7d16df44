"""A captured decode does not hold the scratch that later, larger decodes replace."""
from __future__ import annotations

import pytest
import torch

from gpu_util import make_bf16_case
from qwen_mla_vllm_b200 import mla_decode_attention as m

pytestmark = pytest.mark.gpu


def test_a_graph_outlives_a_larger_decode(cuda_device):
    def call(rows, length, seed):
        cache, q, bt, sl = make_bf16_case(rows, 24, 768, 232, 16, [length] * rows, seed=seed, device=cuda_device)
        o = torch.zeros(rows, 24, 768, dtype=torch.bfloat16, device=cuda_device)
        lse = torch.zeros(rows, 24, device=cuda_device)
        p = m.build_params(q, cache, o, lse, bt, sl, rank=768, qk_dim=1000, rms_offset=1000, rms_mode=1, page_size=16, sm_scale=1 / 16)
        return p, o, lse, (cache, q, bt, sl)

    p, o, lse, keep = call(3, 500, 1)
    m.run_params(p, cuda_device)
    want = o.clone(), lse.clone()
    held = m._ws_cache[0]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        m.run_params(p, cuda_device)
    assert m._ws_cache[0] is held
    size = held.numel()
    m._ws_cache[0] = held = None  # what a larger call does
    big, *_, keep2 = call(64, 9000, 2)
    m.run_params(big, cuda_device)
    others = [torch.full((size,), 77, dtype=torch.uint8, device=cuda_device) for _ in range(8)]
    for _ in range(3):
        o.zero_(), lse.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert all((t == 77).all() for t in others)
