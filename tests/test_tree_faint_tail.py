"""One token with a weight of 1 and 30,000 faint ones that together hold a sixth of the mass, and that agree on
some output dims: losing or coarsening their weights moves those dims.

What the kernel does to a weight w of a row whose largest is 1.  bf16 cache: one rounding to 8 significant bits,
2^-9 w.  FP8 cache: f16 (2^-11 w), then 9 significant bits (2^-9 w), then three e5m2 terms of 3 bits, which stop at
2^-29; below 2^-19, where the last bits reach that, up to 2^-29 is cut off, or the whole weight where it is less.
The output is divided by the sum of the rounded weights (test_tree_rounding_gpu has the rest of the bound; 150 steps
of 2^-23 for sums over a range of tiles and the join of 74 pieces)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen_mla_vllm_b200.tree_attention import tree_masks
from tree_util import SM, build_case, keys_of, scores64

N, HEADS, RANK, ROPE = 30000, 6, 256, 58
QK = RANK + ROPE
SAME = slice(10, 40)  # dims on which the faint tokens agree


def case(dev, fp8):
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(dev, 1, 2, HEADS, RANK, ROPE, 16, [N], mode=mode, fp8=fp8, q_scale=0.0)
    g = torch.Generator().manual_seed(9)
    q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16) * 1e-3)
    raw = c.view(torch.uint8) if fp8 else c
    raw[..., 0] = 0
    raw[..., SAME] = 0x50 if fp8 else 2.0  # e4m3 8.0 (times k_scale)
    raw[..., QK:QK + HEADS] = 128 if fp8 else 1.0  # divisors about 1
    heavy = raw[int(bt[0, 0]), 0, 0]
    heavy[0] = 0x7E if fp8 else 24.0  # 448 k_scale, or 24
    heavy[SAME] = 0
    q[..., SAME] = 0
    q[..., 0] = 12 * 16 / (448 * ks if fp8 else 24.0)  # a score of 12 over scores about 0
    return c, q, bt, ctx, ks, mode


def parts(c, q, bt, fp8, ks, mode, row):
    """Weights (the largest 1) [tokens, heads], values, and the bound on a score's error."""
    k, div = keys_of(c, bt[0].cpu().numpy(), np.arange(N + 1 + row), 16, QK, HEADS, QK, mode, fp8, ks)
    s, mag = scores64(q[row].double().cpu().numpy()[:, :QK], k, div, SM, 0.0)
    return np.exp(s - s.max(axis=0)), k[:, :RANK], mag.max(axis=0) * 2.0**-19 + 1e-6 * (1 + np.abs(s).max(axis=0))


def outputs(w, v, ds, fp8):
    p = w / w.sum(axis=0)
    o, lim = p.T @ v, np.zeros((HEADS, RANK))
    for h in range(HEADS):
        lim[h] = ((2.5 if fp8 else 2.0) * 2.0**-9 * 1.01 + 2 * ds[h]) * (p[:, h] @ np.abs(v - o[h])) + 150 * 2.0**-23 * (p[:, h] @ np.abs(v))
        if fp8:
            cut = np.where(w[:, h] < 2.0**-19, np.minimum(w[:, h], 2.0**-29), 0.0) / w[:, h].sum()
            lim[h] += cut @ np.abs(v)
    return o, lim


def bits(x, n):
    """x rounded to n significant bits."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 2.0**n), e - n)


@pytest.mark.parametrize("fp8", [False, True])
def test_the_bound_sees_a_lost_or_coarse_tail(fp8):
    """Planted in the formula: weights under 2^-15 of the largest dropped, or kept to 3 bits, are out of the
    bound on the dims where the faint tokens agree; 8 bits are within it everywhere."""
    c, q, bt, ctx, ks, mode = case(torch.device("cpu"), fp8)
    w, v, ds = parts(c, q, bt, fp8, ks, mode, 1)
    assert 0.1 < 1 - 1 / w.sum(axis=0).max() < 0.2 and (w[1:] < 2.0**-15).all() and (w[1:] > 2.0**-19).all()
    o, lim = outputs(w, v, ds, fp8)
    off = lambda x: np.abs(x.T @ v / x.sum(axis=0)[:, None] - o)  # noqa: E731
    assert (off(bits(w, 8)) <= lim).all()
    assert (off(np.where(w < 2.0**-15, 0.0, w))[:, SAME] > lim[:, SAME]).all()
    assert (off(np.where(w < 2.0**-15, bits(w, 3), w))[:, SAME] > lim[:, SAME]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_a_faint_tail_counts_in_full(cuda_device, fp8):
    from test_tree_gpu import run
    c, q, bt, ctx, ks, mode = case(cuda_device, fp8)
    mask = tree_masks(torch.tensor([[-1, 0]], device=cuda_device))
    o, lse = run(c, q, bt, ctx, mask, rank=RANK, rope=ROPE, page=16, mode=mode, fp8=fp8, ks=ks, o_dtype=torch.float32)
    for row in range(2):
        ref, lim = outputs(*parts(c, q, bt, fp8, ks, mode, row), fp8)
        d = np.abs(o[row].double().cpu().numpy() - ref)
        assert (d <= lim).all(), f"off by {d.max():.3e}, {(d / lim).max():.2f} of the bound"
