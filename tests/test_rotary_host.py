"""Rotary frequencies and steps (host arithmetic), and the new parameter structs' layout."""
from __future__ import annotations

import math

import pytest
import torch

from qwen_mla_vllm_b200 import _lib
from qwen_mla_vllm_b200.rotary import rotary_embed, rotary_frequencies, rotary_steps
from test_abi import test_params_struct_layout_matches_header as check_layout
from test_abi import shutil


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("cname,pystruct", [("qmla_rotary_params", _lib.RotaryParams),
                                            ("qmla_rope_cache_params", _lib.RopeCacheParams),
                                            ("qmla_tree_params", _lib.TreeParams),
                                            ("qmla_weights_params", _lib.WeightsParams),
                                            ("qmla_evict_params", _lib.EvictParams)])
def test_struct_layout(tmp_path, cname, pystruct):
    check_layout(tmp_path, cname, pystruct)


def test_plain_frequencies_and_steps():
    freq, scale = rotary_frequencies(58, 1e6)
    assert scale == 1.0 and len(freq) == 29 and freq[0] == 1.0
    assert freq[7] == pytest.approx(1e6 ** (-14 / 58), rel=1e-15)
    steps, _ = rotary_steps(58, 1e6)
    assert steps.dtype == torch.int64
    # the phase of a far position against the angle itself, in exact arithmetic
    p = 1_000_003
    for w, s in zip(freq, steps.tolist()):
        frac = (p * s) % 2**64 / 2**64
        want = (p * w / (2 * math.pi)) % 1.0
        assert min(abs(frac - want), 1 - abs(frac - want)) < 1e-9


def test_scalings():
    plain, _ = rotary_frequencies(64, 1e4)
    lin, s = rotary_frequencies(64, 1e4, {"type": "linear", "factor": 4})
    assert s == 1.0 and all(a == b / 4 for a, b in zip(lin, plain))
    ntk, _ = rotary_frequencies(64, 1e4, {"type": "ntk", "factor": 8})
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 8, rel=1e-12)
    cfg = {"type": "banded", "factor": 8, "low_freq_factor": 1, "high_freq_factor": 4, "original_max_position": 8192}
    l3, _ = rotary_frequencies(64, 5e5, cfg)
    base, _ = rotary_frequencies(64, 5e5)
    for a, w in zip(l3, base):
        turns = 8192 * w / (2 * math.pi)
        if turns > 4:
            assert a == w
        elif turns < 1:
            assert a == pytest.approx(w / 8, rel=1e-15)
        else:
            assert w / 8 < a < w
    y, s = rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 16, "original_max_position": 4096})
    assert s == pytest.approx(0.1 * math.log(16) + 1)
    assert y[0] == plain[0] and y[-1] == pytest.approx(plain[-1] / 16, rel=1e-12)
    assert all(p / 16 * (1 - 1e-12) <= v <= p for v, p in zip(y, plain))
    _, s = rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 16, "original_max_position": 4096, "attention_factor": 1.0})
    assert s == 1.0


@pytest.mark.parametrize("rot,scaling", [(7, None), (0, None), (8, {"type": "what"}), (8, {"type": "linear", "factor": 0}),
                                         (2, {"type": "ntk", "factor": 2}),
                                         (8, {"type": "banded", "factor": 2, "original_max_position": 10,
                                              "low_freq_factor": 4, "high_freq_factor": 4})])
def test_bad_frequencies(rot, scaling):
    with pytest.raises(ValueError):
        rotary_frequencies(rot, 1e4, scaling)


def test_needs_a_gpu_tensor():
    with pytest.raises(ValueError):
        rotary_embed(torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int32), rotary_steps(8)[0])
