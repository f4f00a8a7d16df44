"""Accumulated attention weights and eviction on the GPU, against 64-bit and exact restatements.

Bounds of a weight: a score is off by at most 2^-19 of the sum of its terms' magnitudes (32-bit sums;
FP8 queries in two 8-bit terms) plus a few roundings of s and lse (1e-6 of 1 + |s| + |lse|), and
exp turns that into a relative error of each term of the sum.  Eviction moves numbers: all of it is exact.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen_mla_vllm_b200 import _lib
from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights, evict_cache
from tree_util import SM, build_case, keys_of, scores64

pytestmark = pytest.mark.gpu


def weights_ref(w, q, lse, cache, bt, lens, qrows, *, qk, page, rms_offset, mode, fp8, k_scale, cap, decay):
    w64, tol = w.double().cpu().numpy().copy(), np.zeros(w.shape)
    H = q.shape[1]
    q64, l64, btn, ln = q.double().cpu().numpy(), lse.double().cpu().numpy(), bt.cpu().numpy(), lens.cpu().tolist()
    for r in range(w.shape[0]):
        rows = range(r * qrows, (r + 1) * qrows)
        n = min(max(max(ln[x], 0) for x in rows), w.shape[1], btn.shape[1] * page)
        w64[r, :n] *= decay
        tol[r, :n] = 2e-7 * w64[r, :n]
        if n == 0:
            continue
        k, div = keys_of(cache, btn[r], np.arange(n), page, qk, H, rms_offset, mode, fp8, k_scale)
        for x in rows:
            m = min(max(ln[x], 0), n)
            s, mag = scores64(q64[x, :, :qk], k[:m], div[:m], SM, cap)
            fin = np.isfinite(l64[x])
            p = np.exp(s[:, fin] - l64[x][fin])
            w64[r, :m] += p.sum(axis=1)
            tol[r, :m] += (p * (2.0**-19 * mag[:, fin] + 1.2e-6 * (1 + np.abs(s[:, fin]) + np.abs(l64[x][fin])))).sum(axis=1)
    return w64, tol


def weights_case(dev, reqs, qrows, heads, rank, rope, page, lens, *, mode="native", fp8=False, seed=0):
    cache, q, bt, last, ks = build_case(dev, reqs, qrows, heads, rank, rope, page, lens, mode=mode, fp8=fp8, seed=seed)
    cols = max(lens) + qrows + 3
    row_lens = (last[:, None] + torch.arange(1, qrows + 1, dtype=torch.int32, device=dev)).flatten().contiguous()
    g = torch.Generator().manual_seed(seed + 5)
    w = torch.rand(reqs, cols, generator=g).to(dev)
    # an lse near the rows' own: weights of ordinary size
    lse = (torch.rand(reqs * qrows, heads, generator=g) * 2 + 6).to(dev)
    return cache, q, bt, row_lens, w, lse, ks


def go(case, qrows, rank, rope, page, *, mode="native", fp8=False, cap=0.0, decay=0.9, **kw):
    cache, q, bt, lens, w, lse, ks = case
    qk = rank + rope
    w64, tol = weights_ref(w, q, lse, cache, bt, lens, qrows, qk=qk, page=page, rms_offset=qk, mode=mode, fp8=fp8, k_scale=ks,
                           cap=cap, decay=decay)
    accumulate_attention_weights(q, cache, w, lse, bt, lens, sm_scale=SM, page_size=page, rms_offset=-1 if mode == "none" else qk,
                                 qk_dim=qk, rms_log8=mode == "log8", rms_bf16=mode == "bf16", logit_cap=cap,
                                 k_scale=torch.tensor(ks, device=q.device) if fp8 else None, qrows=qrows, decay=decay, **kw)
    d = np.abs(w.double().cpu().numpy() - w64)
    assert (d <= tol * 1.1).all(), f"off by {d.max():.3e}, {np.nanmax(d / np.maximum(tol, 1e-30)):.2f} of the bound"


@pytest.mark.parametrize("fp8,mode", [(False, "native"), (False, "none"), (True, "log8"), (True, "bf16"), (True, "native"), (True, "none")])
@pytest.mark.parametrize("qrows,heads,rank,rope", [(1, 24, 768, 232), (4, 24, 768, 232), (2, 12, 384, 116), (3, 6, 512, 58),
                                                   (1, 1, 256, 0), (1, 48, 1792, 232), (2, 48, 256, 58), (1, 24, 1792, 232)])
def test_weights_shapes_and_row_formats(cuda_device, qrows, heads, rank, rope, fp8, mode):
    cm = "e4m3" if fp8 and mode == "native" else ("log8" if fp8 and mode == "none" else mode)
    case = weights_case(cuda_device, 4, qrows, heads, rank, rope, 16, [130, 0, 61, 400], mode=cm, fp8=fp8)
    go(case, qrows, rank, rope, 16, mode=mode, fp8=fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [1, 3, 16, 24, 32, 64, 128, 256])
def test_weights_page_sizes(cuda_device, page, fp8):
    mode = "log8" if fp8 else "native"
    case = weights_case(cuda_device, 3, 2, 12, 384, 116, page, [383, 40, 255], mode=mode, fp8=fp8)
    go(case, 2, 384, 116, page, mode=mode, fp8=fp8, cap=4.0)


@pytest.mark.parametrize("fp8", [False, True])
def test_weights_many_and_long_rows(cuda_device, fp8):
    mode = "log8" if fp8 else "native"
    for lens in ([20000, 9001], [1, 127, 128, 129, 255, 256] + [37 * i % 300 for i in range(170)]):
        case = weights_case(cuda_device, len(lens), 1, 24, 768, 232, 16, lens, mode=mode, fp8=fp8)
        go(case, 1, 768, 232, 16, mode=mode, fp8=fp8, decay=1.0)


def test_weights_rows_without_tokens_or_lse(cuda_device):
    cache, q, bt, lens, w, lse, ks = weights_case(cuda_device, 4, 2, 12, 384, 116, 16, [50, 60, 0, 70])
    lens[:] = torch.tensor([0, 0, -4, 30, 5, 2, 71, 10**9], dtype=torch.int32)  # not in order, beyond the tables
    lse[3], lse[4, 2], lse[5, 1], lse[6, 0] = -float("inf"), float("nan"), float("inf"), -float("inf")
    go((cache, q, bt, lens, w, lse, ks), 2, 384, 116, 16)
    assert w.isfinite().all()


def test_weights_nan_keys_and_absent_pages(cuda_device):
    cache, q, bt, lens, w, lse, ks = weights_case(cuda_device, 2, 1, 12, 384, 116, 16, [50, 40])
    w0 = w.clone()
    cache[bt[0, 1].long(), 3] = float("nan")  # token 19 of request 0
    for r, n in ((0, 51), (1, 41)):  # and everything past the ends
        for t in range(n, bt.shape[1] * 16):
            cache[bt[r, t // 16].long(), t % 16] = float("nan")
    bt[1, 0], bt[1, 1] = -1, 10**6
    accumulate_attention_weights(q, cache, w, lse, bt, lens, sm_scale=SM, page_size=16, rms_offset=500, decay=0.5)
    assert w[0, 19].isnan() and w[0].isnan().sum() == 1 and w[1].isfinite().all()
    assert torch.equal(w[1, :32], 0.5 * w0[1, :32]) and torch.equal(w[0, 51:], w0[0, 51:]) and torch.equal(w[1, 41:], w0[1, 41:])


def test_weights_strides_and_f16_queries(cuda_device):
    cache, q, bt, lens, w, lse, ks = weights_case(cuda_device, 2, 3, 24, 768, 232, 16, [200, 77])
    q = q.half()
    qn = torch.zeros(6, 24, 800, dtype=q.dtype, device=cuda_device)
    qn[..., 3:771] = q[..., :768]
    qp = torch.zeros(6, 30, 300, dtype=q.dtype, device=cuda_device)
    qp[:, 4:28, 5:237] = q[..., 768:]
    wide = torch.full((2, w.shape[1] + 9), 7.0, device=cuda_device)
    wide[:, 4:-5] = w
    lw = torch.zeros(6, 40, device=cuda_device)
    lw[:, 1:25] = lse
    big = torch.zeros(cache.shape[0], 20, 1, cache.shape[3] + 16, dtype=cache.dtype, device=cuda_device)
    big[:, :16, :, :cache.shape[3]] = cache
    w64, tol = weights_ref(w, q, lse, cache, bt, lens, 3, qk=1000, page=16, rms_offset=1000, mode="native", fp8=False, k_scale=1.0,
                           cap=0.0, decay=1.0)
    accumulate_attention_weights(qn[..., 3:771], big[:, :16, :, :cache.shape[3]], wide[:, 4:-5], lw[:, 1:25], bt, lens, sm_scale=SM,
                                 page_size=16, rank=768, rms_offset=1000, q_pe=qp[:, 4:28, 5:237], qrows=3)
    assert (np.abs(wide[:, 4:-5].double().cpu().numpy() - w64) <= tol * 1.1).all()
    assert (wide[:, :4] == 7).all() and (wide[:, -5:] == 7).all()


def test_weights_of_a_decode_add_up_to_its_heads(cuda_device):
    """With the decode's own lse, a row's weights sum to one per head."""
    from qwen_mla_vllm_b200.mla_decode_attention import build_params, run_params
    cache, q, bt, lens, w, _, _ = weights_case(cuda_device, 3, 1, 24, 768, 232, 16, [3000, 17, 700])
    o = torch.empty(3, 24, 768, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.empty(3, 24, device=cuda_device)
    run_params(build_params(q, cache, o, lse, bt, lens, rank=768, qk_dim=1000, rms_offset=1000, rms_mode=_lib.RMS_NATIVE,
                            page_size=16, sm_scale=SM), q.device)
    w.zero_()
    accumulate_attention_weights(q, cache, w, lse, bt, lens, sm_scale=SM, page_size=16, rms_offset=1000)
    assert (w.sum(dim=1) - 24).abs().max() < 24 * 1e-4


def test_weights_graph_and_stream(cuda_device):
    cache, q, bt, lens, w, lse, _ = weights_case(cuda_device, 3, 1, 24, 768, 232, 16, [3000, 17, 700])
    call = lambda x: accumulate_attention_weights(q, cache, x, lse, bt, lens, sm_scale=SM, page_size=16, rms_offset=1000, decay=0.5)  # noqa: E731
    a, b = w.clone(), w.clone()
    call(a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        call(b)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call(b)
        g.replay()
    st.synchronize()
    call(a)
    assert torch.equal(a, b)


def test_weights_refusals(cuda_device):
    cache, q, bt, lens, w, lse, _ = weights_case(cuda_device, 2, 2, 12, 384, 116, 16, [20, 5])
    ok = dict(q=q, kv_cache=cache, weights=w, lse=lse, block_table=bt, seq_lens=lens, sm_scale=SM, page_size=16, rms_offset=500, qrows=2)
    for bad, err in ((dict(qrows=3), ValueError), (dict(qrows=0), ValueError), (dict(weights=w.double()), TypeError), (dict(lse=lse[:3]), ValueError),
                     (dict(lse=lse.half()), TypeError), (dict(seq_lens=lens.long()), TypeError), (dict(block_table=bt[:1]), ValueError),
                     (dict(q=q[..., :400]), ValueError), (dict(page_size=8), ValueError), (dict(kv_cache=cache.half()), TypeError),
                     (dict(q_pe=q), ValueError), (dict(weights=w.t()), ValueError), (dict(rms_offset=511, qk_dim=500), _lib.QmlaError),
                     (dict(q=q.float()), _lib.QmlaError), (dict(kv_cache=cache[..., 1:]), _lib.QmlaError), (dict(q=q.cpu()), ValueError)):
        with pytest.raises(err):
            accumulate_attention_weights(**dict(ok, **bad))


# ------------------------------------------------------------------ eviction
def evict_ref(cache, w, pos, bt, lens, budget, page, sinks, recent, budgets):
    c, w, pos, bt = cache.clone(), w.cpu().numpy(), pos.cpu().numpy(), bt.cpu().numpy()
    R, cols = w.shape
    keep = min(budget, cols)
    nw, npos, nl = np.zeros((R, keep), np.float32), np.full((R, keep), -1, np.int32), np.zeros(R, np.int32)
    at = lambda r, t: (int(bt[r, t // page]), t % page)  # noqa: E731
    for r in range(R):
        n = min(max(int(lens[r]), 0), cols, bt.shape[1] * page)
        K = min(n, budget if budgets is None else min(budget, max(int(budgets[r]), 0)))
        held = (pos[r, :n] < sinks) | (pos[r, :n] >= (int(recent[r]) if recent is not None else 2**31))
        rank = lambda t: (0 if held[t] else 1 if not np.isnan(w[r, t]) else 2, 0.0 if held[t] or np.isnan(w[r, t]) else -w[r, t], t)  # noqa: E731
        stay = set(sorted(range(n), key=rank)[:K])
        nw[r, :K], npos[r, :K], nl[r] = w[r, :K], pos[r, :K], K
        holes, movers = [t for t in range(K) if t not in stay], [t for t in range(K, n) if t in stay]
        assert len(holes) == len(movers)
        for d, s in zip(holes, movers):
            c[at(r, d)] = cache[at(r, s)]
            nw[r, d], npos[r, d] = w[r, s], pos[r, s]
    return c, nw, npos, nl


def evict_case(dev, reqs, lens, page, width=64, dtype=torch.bfloat16, seed=0, kind="random"):
    g = torch.Generator().manual_seed(seed)
    cols = max(max(lens), 1) + 5
    pps = -(-cols // page)
    cache = torch.randint(0, 255, (reqs * pps, page, 1, width), generator=g).to(torch.uint8 if dtype == torch.uint8 else dtype).to(dev)
    bt = torch.randperm(reqs * pps, generator=g).reshape(reqs, pps).to(torch.int32).to(dev)
    w = torch.exp(torch.randn(reqs, cols, generator=g) * 2)
    if kind == "ties":
        w = torch.randint(0, 4, (reqs, cols), generator=g).float()
    elif kind == "equal":
        w = torch.ones(reqs, cols)
    elif kind == "odd":
        w = torch.randn(reqs, cols, generator=g)
        w[:, ::7], w[:, 1::11], w[:, 2::13], w[:, 3::5], w[:, 4::17] = float("nan"), float("inf"), -float("inf"), 0.0, -0.0
    pos = torch.stack([torch.randperm(cols, generator=g) for _ in range(reqs)]).to(torch.int32)
    return cache, w.to(dev), pos.to(dev), bt, torch.tensor(lens, dtype=torch.int32, device=dev)


def both(case, budget, page, *, sinks=0, recent=None, budgets=None):
    cache, w, pos, bt, lens = case
    c, nw, npos, nl = evict_ref(cache, w, pos, bt, lens, budget, page, sinks, recent, budgets)
    w0, p0 = w.clone(), pos.clone()
    gw, gp, gl = evict_cache(cache, w, pos, bt, lens, budget, page_size=page, sinks=sinks, recent_from=recent, budgets=budgets)
    assert np.array_equal(gl.cpu().numpy(), nl)
    assert np.array_equal(gp.cpu().numpy(), npos)
    assert np.array_equal(gw.cpu().numpy(), nw, equal_nan=True)
    assert torch.equal(cache.view(torch.uint8), c.view(torch.uint8))
    assert torch.equal(w.view(torch.int32), w0.view(torch.int32)) and torch.equal(pos, p0)


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("budget", [0, 1, 31, 64, 100, 255, 5000])
def test_evict_budgets_and_orders(cuda_device, budget, kind):
    case = evict_case(cuda_device, 7, [300, 0, 1, 64, 65, 255, 129], 16, kind=kind)
    both(case, budget, 16)


@pytest.mark.parametrize("page,width,dtype", [(1, 8, torch.bfloat16), (3, 40, torch.uint8), (16, 1024, torch.bfloat16),
                                              (64, 1024, torch.uint8), (24, 77, torch.uint8)])
def test_evict_rows_of_any_kind(cuda_device, page, width, dtype):
    both(evict_case(cuda_device, 3, [200, 33, 150], page, width, dtype), 60, page)


def test_evict_protects_sinks_and_recent(cuda_device):
    case = evict_case(cuda_device, 3, [200, 90, 150], 16)
    recent = torch.tensor([180, 60, 1 << 30], dtype=torch.int32, device=cuda_device)
    both(case, 40, 16, sinks=4, recent=recent)
    case = evict_case(cuda_device, 3, [200, 90, 150], 16, seed=1)
    both(case, 10, 16, sinks=100, recent=recent)  # more protected tokens than fit


def test_evict_budgets_per_request_and_bad_lengths(cuda_device):
    case = evict_case(cuda_device, 5, [200, 90, 150, 40, 77], 16)
    case[4][3], case[4][4] = -5, 10**9
    both(case, 100, 16, budgets=torch.tensor([50, 1000, 0, 10, -3], dtype=torch.int32, device=cuda_device))


@pytest.mark.parametrize("n,budget,kind", [(9000, 3000, "random"), (30000, 100, "ties"), (70000, 65000, "odd"), (70000, 20000, "equal")])
def test_evict_long_requests(cuda_device, n, budget, kind):
    both(evict_case(cuda_device, 2, [n, n // 3], 16, 16, kind=kind), budget, 16, sinks=4)


def test_evict_more_keys_than_shared_memory(cuda_device):
    both(evict_case(cuda_device, 1, [400000], 64, 8), 150000, 64)


def test_evict_absent_pages_strided_cache_and_out(cuda_device):
    cache, w, pos, bt, lens = evict_case(cuda_device, 2, [100, 80], 16, 64)
    big = torch.zeros(cache.shape[0], 20, 1, 96, dtype=cache.dtype, device=cuda_device)
    big[:, :16, :, 16:80] = cache
    view = big[:, :16, :, 16:80]
    ref, nw, npos, nl = evict_ref(cache, w, pos, bt, lens, 30, 16, 0, None, None)
    ow = torch.full((2, 50), 9.0, device=cuda_device)
    op = torch.full((2, 50), 9, dtype=torch.int32, device=cuda_device)
    ol = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    got = evict_cache(view, w, pos, bt, lens, 30, page_size=16, out=(ow, op, ol))
    assert got[0] is ow and torch.equal(view, ref)
    assert np.array_equal(ow[:, :30].cpu().numpy(), nw) and not ow[:, 30:].any() and (op[:, 30:] == -1).all()
    assert not big[:, 16:].any() and not big[..., :16].any() and not big[..., 80:].any()
    bt[0, 0], bt[0, 3] = -1, 10**6  # tokens of absent pages have no row to move
    evict_cache(view, w, pos, bt, lens, 30, page_size=16)


def test_evict_refusals_and_empty(cuda_device):
    cache, w, pos, bt, lens = evict_case(cuda_device, 2, [100, 80], 16)
    ok = dict(kv_cache=cache, weights=w, positions=pos, block_table=bt, seq_lens=lens, budget=10, page_size=16)
    o = lambda n: (torch.empty(2, n, device=cuda_device), torch.empty(2, n, dtype=torch.int32, device=cuda_device), torch.empty(2, dtype=torch.int32, device=cuda_device))  # noqa: E731
    for bad, err in ((dict(budget=-1), ValueError), (dict(weights=w.double()), TypeError), (dict(positions=pos.long()), TypeError),
                     (dict(positions=pos[:, 1:]), ValueError), (dict(seq_lens=lens[:1]), ValueError), (dict(block_table=bt[:1]), ValueError),
                     (dict(page_size=8), ValueError), (dict(recent_from=lens[:1]), ValueError), (dict(budgets=lens.long()), TypeError),
                     (dict(out=o(9)), ValueError), (dict(out=(w, pos, lens)), ValueError), (dict(weights=w.cpu()), ValueError),
                     (dict(workspace=torch.empty(64, dtype=torch.uint8, device=cuda_device)), _lib.QmlaError)):
        with pytest.raises(err):
            evict_cache(**dict(ok, **bad))
    a, b, c = evict_cache(**dict(ok, weights=w[:, :0], positions=pos[:, :0]))
    assert a.shape == (2, 0) and b.shape == (2, 0) and not c.any()
    assert evict_cache(cache, w[:0], pos[:0], bt, lens[:0], 3, page_size=16)[0].shape == (0, 3)
