"""Masks and scores at the edge of what a node sees, on both kernels of tree_attention."""
from __future__ import annotations

import pytest
import torch

from test_tree_gpu import run, verify
from tree_util import build_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 3])  # tensor cores, CUDA cores
def test_bits_past_the_nodes(cuda_device, page, fp8):
    """They name no token.  A node that has no other bit is not padding: it sees the committed tokens."""
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 3, 5, 12, 384, 116, page, [200, 0, 127], mode=mode, fp8=fp8)
    top = -2**63
    mask = torch.tensor([[1, 1 << 5, 0, top, 1 << 40 | 9], [1 << 63 - 1, 3, top | 4, 0, 1 << 6],
                         [top, top | 1, 1 << 5 | 6, 8, 0]], dtype=torch.int64, device=cuda_device)
    kw = dict(rank=384, rope=116, page=page, mode=mode, fp8=fp8, ks=ks)
    o, lse = run(c, q, bt, ctx, mask, **kw)
    verify(o, lse, c, q, bt, ctx, mask, **kw)
    assert lse[[1, 3, 10]].isfinite().all()  # committed tokens alone
    for row in (2, 8, 14):  # padding
        assert not o[row].any() and (lse[row] == float("-inf")).all()
    for row in (5, 9):  # nothing committed, and only bits that name nothing
        assert not o[row].any() and (lse[row] == float("-inf")).all()


@pytest.mark.parametrize("page", [16, 3])
def test_scores_of_minus_infinity(cuda_device, page):
    """Tokens that score -inf with every query (an infinite rope element) weigh nothing, at the start of a
    row as anywhere: as if their pages were absent.  A row that sees nothing else is an empty one."""
    c, q, bt, ctx, _ = build_case(cuda_device, 3, 2, 12, 384, 116, page, [20001, 300, 40])
    mask = torch.tensor([[1, 3], [1, 3], [1, 3]], dtype=torch.int64, device=cuda_device)
    q[..., 400] = q[..., 400].abs() + 1
    gone = bt.clone()
    for r, n in ((0, 400), (1, 150), (2, bt.shape[1] * page)):
        pages = bt[r, :n // page].long()
        c[pages, :, :, 400] = -float("inf")
        gone[r, :n // page] = -1
    kw = dict(rank=384, rope=116, page=page)
    o, lse = run(c, q, bt, ctx, mask, **kw)
    o2, lse2 = run(c, q, gone, ctx, mask, **kw)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    assert lse[:4].isfinite().all() and o[:4].isfinite().all()
    assert not o[4:].any() and (lse[4:] == float("-inf")).all()
