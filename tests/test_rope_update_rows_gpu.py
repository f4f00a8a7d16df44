"""The fused update on a step without queries of its own (a cache filled ahead of them)."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200.rotary import rope_kv_cache_update, rotary_steps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 700])
def test_rows_are_written_without_heads(cuda_device, n, fp8):
    g = torch.Generator().manual_seed(n)
    bf = torch.bfloat16
    q = torch.randn(n, 12, 116, generator=g).to(bf).to(cuda_device)
    k = torch.cat([torch.randn(n, 116, generator=g), torch.rand(n, 12, generator=g) + 0.5], 1).to(bf).to(cuda_device)
    lat = torch.randn(n, 384, generator=g).to(bf).to(cuda_device)
    pos = torch.randint(0, 10000, (n,), generator=g).to(cuda_device)
    slots = torch.randperm(720, generator=g)[:n].to(cuda_device)
    steps = rotary_steps(58, device=cuda_device)[0]
    kw = dict(packed_rope=116, local_heads=12, k_scale=torch.tensor(0.02, device=cuda_device) if fp8 else None,
              rms_mode="log8" if fp8 else "native")
    a, b = (torch.zeros(45, 16, 1, 512, dtype=torch.uint8 if fp8 else bf, device=cuda_device) for _ in range(2))
    rope_kv_cache_update(q, k, lat, pos, slots, steps, a, **kw)
    out = rope_kv_cache_update(q[:, :0], k, lat, pos, slots, steps, b, **kw)
    assert out.shape == (n, 0, 116) and torch.equal(a, b) and a.any()
