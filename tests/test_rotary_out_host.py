"""An out= that autograd would have to follow is refused before anything is asked of the GPU."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200.rotary import rotary_embed, rotary_steps


def test_out_of_a_tensor_that_needs_a_gradient():
    x = torch.zeros(1, 1, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="automatic differentiation"):
        rotary_embed(x, torch.zeros(1, dtype=torch.int32), rotary_steps(8)[0], out=x)
    with torch.no_grad(), pytest.raises(ValueError):  # the CPU tensor
        rotary_embed(x, torch.zeros(1, dtype=torch.int32), rotary_steps(8)[0], out=x)
