"""Where evict_cache may write: beside its inputs in one storage, not over them."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200.cache_eviction import evict_cache
from test_eviction_gpu import evict_case

pytestmark = pytest.mark.gpu
I32 = torch.int32


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_out_in_the_storage_of_the_inputs(cuda_device):
    """Two halves of a buffer that take turns, and columns of one row side by side."""
    cache, w, pos, bt, lens = evict_case(cuda_device, 4, [100, 0, 60, 77], 16)
    R, n = w.shape
    kw = dict(page_size=16, sinks=2)
    first = cache.clone()
    want = evict_cache(first, w, pos, bt, lens, 40, **kw)
    wb, pb, lb = torch.zeros(2, R, n, device=cuda_device), torch.zeros(2, R, n, dtype=I32, device=cuda_device), torch.zeros(2, R, dtype=I32, device=cuda_device)
    wb[0], pb[0], lb[0] = w, pos, lens
    c = cache.clone()
    got = evict_cache(c, wb[0], pb[0], bt, lb[0], 40, out=(wb[1], pb[1], lb[1]), **kw)
    assert torch.equal(c, first) and equal([got[0][:, :40], got[1][:, :40], got[2]], want)
    assert torch.equal(wb[0], w) and torch.equal(pb[0], pos)
    wide, pwide = torch.zeros(R, n + 40, device=cuda_device), torch.zeros(R, n + 40, dtype=I32, device=cuda_device)
    wide[:, :n], pwide[:, :n] = w, pos
    c = cache.clone()
    got = evict_cache(c, wide[:, :n], pwide[:, :n], bt, lens, 40, out=(wide[:, n:], pwide[:, n:], torch.empty(R, dtype=I32, device=cuda_device)), **kw)
    assert torch.equal(c, first) and equal(got, want) and torch.equal(wide[:, :n], w)


def test_out_over_an_input_is_refused(cuda_device):
    cache, w, pos, bt, lens = evict_case(cuda_device, 3, [100, 60, 77], 16)
    R, n = w.shape
    nw, npos, nl = torch.empty(R, 40, device=cuda_device), torch.empty(R, 40, dtype=I32, device=cuda_device), torch.empty(R, dtype=I32, device=cuda_device)
    budgets = torch.full((R,), 30, dtype=I32, device=cuda_device)
    both = torch.empty(R, 80, dtype=I32, device=cuda_device)
    like = torch.empty(R, n, dtype=I32, device=cuda_device)
    before = cache.clone()
    for out in ((w[:, n - 40:], like[:, :40], nl), (like.view(torch.float32)[:, :40], pos[:, :40], nl), (nw, npos, lens), (nw, npos, budgets), (nw, npos, nw.view(I32)[0, :R]),
                (both.view(torch.float32)[:, 1:41], both[:, 40:], nl), (nw, npos, bt.view(-1)[:R])):
        with pytest.raises(ValueError, match="share memory"):
            evict_cache(cache, w, pos, bt, lens, 40, page_size=16, budgets=budgets, out=out)
    assert torch.equal(cache, before)
    evict_cache(cache, w, pos, bt, lens, 40, page_size=16, budgets=budgets, out=(both.view(torch.float32)[:, :40], both[:, 40:], nl))
