"""The operators' torch.library schemas and fake kernels, and refusals that need no GPU."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import qwen_mla_vllm_b200.ops  # noqa: F401
from qwen_mla_vllm_b200 import _lib
from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights, evict_cache
from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks


def test_ops_trace_without_the_library():
    with FakeTensorMode():
        e = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        x = e(5, 3, 64, dt=torch.bfloat16)
        y = torch.ops.qmla.rotary(x, e(5, dt=torch.int64), e(29, dt=torch.int64), 0, 1, False, 1.0, False)
        assert y.shape == x.shape and y.dtype == x.dtype
        c, q = e(8, 16, 1, 512, dt=torch.bfloat16), e(6, 12, 500, dt=torch.bfloat16)
        o, lse, bt, n = e(6, 12, 384, dt=torch.bfloat16), e(6, 12), e(2, 4, dt=torch.int32), e(2, dt=torch.int32)
        t = torch.ops.qmla
        assert t.tree_attention(q, c, o, lse, bt, n, e(2, 3, dt=torch.int64), 384, 0.1, 16, 500, False, False, 0.0, None) is None
        assert t.accumulate_attention_weights(q, c, e(2, 64), lse, bt, e(6, dt=torch.int32), 0.1, 16, 500, False, False, 0.0, None, 3, 1.0) is None
        assert t.evict_cache(c, e(2, 64), e(2, 64, dt=torch.int32), bt, n, e(2, 9), e(2, 9, dt=torch.int32), n, 9, 16, 0, None) is None


@pytest.mark.parametrize("op,written", [("tree_attention", {"o", "lse"}), ("accumulate_attention_weights", {"weights"}),
                                        ("evict_cache", {"kv_cache", "new_weights", "new_positions", "new_lens"}),
                                        ("rope_kv_cache_update", {"kv_cache", "q_out"}), ("rotary", set())])
def test_schemas_name_what_they_write(op, written):
    schema = getattr(torch.ops.qmla, op).default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written


def test_tree_masks_on_the_host():
    assert tree_masks(torch.tensor([-1, 0, 1, 0])).tolist() == [1, 3, 7, 9]
    with pytest.raises(ValueError):
        tree_masks(torch.zeros(65, dtype=torch.int64))


def test_host_tensors_are_refused():
    z = torch.zeros
    i = torch.int32
    with pytest.raises(ValueError):
        tree_attention(z(1, 1, 8), z(1, 16, 1, 8), z(1, 1, 8), None, z(1, 1, dtype=i), z(1, dtype=i), z(1, 1, dtype=torch.int64),
                       rank=8, sm_scale=1.0, page_size=16)
    with pytest.raises(ValueError):
        accumulate_attention_weights(z(1, 1, 8), z(1, 16, 1, 8), z(1, 4), z(1, 1), z(1, 1, dtype=i), z(1, dtype=i), sm_scale=1.0,
                                     page_size=16)
    with pytest.raises(ValueError):
        evict_cache(z(1, 16, 1, 8), z(1, 4), z(1, 4, dtype=i), z(1, 1, dtype=i), z(1, dtype=i), 2, page_size=16)


@pytest.mark.parametrize("cls", [_lib.RotaryParams, _lib.RopeCacheParams, _lib.TreeParams, _lib.WeightsParams, _lib.EvictParams])
def test_packed_parameters_are_the_structures(cls):
    vals = [(k + 1.5 if t is _lib.ctypes.c_float else k + 1) for k, (_, t) in enumerate(cls._fields_)]
    raw = _lib.packer(cls).pack(*vals)
    back = cls.from_buffer_copy(raw)
    assert [getattr(back, n) for n, _ in cls._fields_] == vals


def test_null_parameters_are_errors():
    lib = _lib.load()
    need = _lib.ctypes.c_int64(0)
    for name in ("qmla_rotary", "qmla_rope_cache_write", "qmla_tree_attention", "qmla_accumulate_weights", "qmla_evict"):
        assert getattr(lib, name)(None, None) == -1
    for name in ("qmla_tree_workspace_bytes", "qmla_weights_workspace_bytes", "qmla_evict_workspace_bytes"):
        assert getattr(lib, name)(None, _lib.ctypes.byref(need)) == -1
