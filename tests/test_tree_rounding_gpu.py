"""What the rounding of the softmax weights costs tree_attention, seen through 32-bit outputs.

The weights p_i are rounded to 8 significant bits (9 over an FP8 cache): p_i (1 + d_i), |d_i| <= 2^-9.  The
output is their mean of the values, so its error is sum p_i d_i (v_i - o) / (1 + sum p_i d_i).  Where a request is
worked on in pieces, each piece is such a mean about its own o, which at most doubles the bound:
    |error| <= 2^-8 * 1.01 * sum p_i |v_i - o|.
A score is off by at most ds (tree_util), which moves a weight by a factor e^ds; O is summed in 32 bits, at most
64 + 2 steps of 2^-23 each for the lengths used here.  FP8: weights below 2^-19 of the row's largest may lose
all their bits.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen_mla_vllm_b200.tree_attention import tree_masks
from test_tree_gpu import run
from tree_util import SM, build_case, keys_of, random_parents, scores64, visible

pytestmark = pytest.mark.gpu


def mean_ref(q, cache, bt, ctx, mask, *, rank, qk, page, mode, fp8, k_scale):
    """(o, bound on |o - o32|) for every row."""
    nodes, H = mask.shape[-1], q.shape[1]
    q64, btn, ctxn, m2 = q.double().cpu().numpy(), bt.cpu().numpy(), ctx.cpu().tolist(), mask.cpu().tolist()
    o, lim = np.zeros((q.shape[0], H, rank)), np.zeros((q.shape[0], H, rank))
    for r, c in enumerate(ctxn):
        for i in range(nodes):
            row = r * nodes + i
            toks = visible(c, m2[r][i] & (2**64 - 1), nodes, btn.shape[1] * page)
            k, div = keys_of(cache, btn[r], toks, page, qk, H, qk, mode, fp8, k_scale)
            s, mag = scores64(q64[row, :, :qk], k, div, SM, 0.0)
            w = np.exp(s - s.max(axis=0))
            p = w / w.sum(axis=0)
            ds = mag.max(axis=0) * 2.0**-19 + 1e-6 * (1 + np.abs(s).max(axis=0))
            v = k[:, :rank]
            o[row] = p.T @ v
            for h in range(H):
                off = p[:, h] @ np.abs(v - o[row, h])
                lim[row, h] = (2.0**-8 * 1.01 + 2 * ds[h]) * off + 66 * 2.0**-23 * (p[:, h] @ np.abs(v))
                if fp8:
                    lim[row, h] += np.where(w[:, h] < 2.0**-19, p[:, h], 0.0) @ np.abs(v)
    return o, lim


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,rank,rope", [(24, 768, 232), (12, 384, 116)])
@pytest.mark.parametrize("spread", [4.0, 64.0])  # many tokens count; a few do
def test_rounded_weights_average_the_values(cuda_device, spread, heads, rank, rope, fp8):
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 3, 4, heads, rank, rope, 16, [1000, 40, 333], mode=mode, fp8=fp8, q_scale=spread)
    mask = tree_masks(random_parents(3, 4).to(cuda_device))
    kw = dict(rank=rank, rope=rope, page=16, mode=mode, fp8=fp8, ks=ks)
    o, _ = run(c, q, bt, ctx, mask, o_dtype=torch.float32, **kw)
    ref, lim = mean_ref(q, c, bt, ctx, mask, rank=rank, qk=rank + rope, page=16, mode=mode, fp8=fp8, k_scale=ks)
    d = np.abs(o.double().cpu().numpy() - ref)
    assert (d <= lim).all(), f"off by {d.max():.3e}, {(d / lim).max():.2f} of the bound"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rank,rope", [(768, 232), (384, 116)])
def test_equal_values_come_back_as_they_are(cuda_device, rank, rope, fp8):
    """With one value in every row the mean is that value, whatever the weights' rounding did."""
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 2, 3, 12, rank, rope, 16, [700, 90], mode=mode, fp8=fp8, q_scale=64.0)
    if fp8:
        c.view(torch.uint8)[..., :rank] = c.view(torch.uint8)[0, 0, 0, :rank]
    else:
        c[..., :rank] = c[0, 0, 0, :rank]
    v = c[0, 0, 0, :rank].float() * ks
    mask = tree_masks(torch.tensor([[-1, 0, 0], [-1, 0, 1]], device=cuda_device))
    o, _ = run(c, q, bt, ctx, mask, o_dtype=torch.float32, rank=rank, rope=rope, page=16, mode=mode, fp8=fp8, ks=ks)
    lost = 793 * 2.0**-19 if fp8 else 0.0  # the weights below 2^-19 of the largest, all of them lost at worst
    assert ((o - v).abs() <= (66 * 2.0**-23 + lost) * v.abs()).all()
