"""Query rows whose lse is not finite add nothing to the weights, whatever their scores are."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights
from test_eviction_gpu import go, weights_case
from tree_util import SM

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 3])  # tensor cores, CUDA cores
@pytest.mark.parametrize("qrows,heads", [(1, 24), (2, 12), (3, 12), (4, 6)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_a_bad_query_beside_good_ones(cuda_device, bad, qrows, heads, page, fp8):
    """The lse of a query that holds NaN is NaN; of one that holds an infinity, NaN or an infinity."""
    mode = "log8" if fp8 else "native"
    case = weights_case(cuda_device, 3, qrows, heads, 384, 116, page, [400, 61, 200], mode=mode, fp8=fp8)
    _, q, _, _, w, lse, _ = case
    q[qrows - 1, 2, 17], lse[qrows - 1, 2] = bad, NAN  # one head of a row
    q[2 * qrows, :, 3], lse[2 * qrows] = bad, torch.tensor([NAN, INF, -INF], device=cuda_device).repeat(heads)[:heads]  # a row
    go(case, qrows, 384, 116, page, mode=mode, fp8=fp8)
    assert w.isfinite().all()


@pytest.mark.parametrize("page", [16, 3])
def test_infinite_keys(cuda_device, page):
    """A key that scores -inf with every query draws nothing: padded query columns must not add a NaN."""
    case = weights_case(cuda_device, 2, 1, 12, 384, 116, page, [300, 40])
    cache, q, bt, lens, w, lse, _ = case
    q[..., 5] = q[..., 5].abs() + 1
    for t in (7, 250):
        cache[bt[0, t // page].long(), t % page, 0, 5] = -INF
    w0 = w.clone()
    accumulate_attention_weights(q, cache, w, lse, bt, lens, sm_scale=SM, page_size=page, rms_offset=500, decay=0.5)
    assert w.isfinite().all() and torch.equal(w[0, [7, 250]], 0.5 * w0[0, [7, 250]])


@pytest.mark.parametrize("page", [16, 3])
def test_nothing_counts_when_no_row_has_an_lse(cuda_device, page):
    cache, q, bt, lens, w, lse, _ = weights_case(cuda_device, 2, 2, 12, 384, 116, page, [300, 40])
    q.fill_(NAN)
    lse.copy_(torch.from_numpy(np.resize(np.array([NAN, -INF, INF], np.float32), tuple(lse.shape))))
    w0 = w.clone()
    accumulate_attention_weights(q, cache, w, lse, bt, lens, sm_scale=SM, page_size=page, rms_offset=500, qrows=2, decay=0.5)
    n = lens.view(2, 2).amax(1).tolist()
    for r in range(2):
        assert torch.equal(w[r, :n[r]], 0.5 * w0[r, :n[r]]) and torch.equal(w[r, n[r]:], w0[r, n[r]:])
