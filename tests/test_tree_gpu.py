"""Attention of a drafted token tree on the GPU against its 64-bit formula.

Bounds (tree_util.tree_ref): scores are products accumulated in 32 bits (FP8 queries are split in two
8-bit terms that keep 2^-19 of the largest element), so a score is off by at most 2^-19 of the sum of
its terms' magnitudes; each softmax weight is rounded once to 8 bits before it meets the values
(2^-8 of sum p |v|; FP8: 3 bits for weights under 2^-15 of the row's largest); lse takes no part in
that rounding; o is rounded once to its own type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen_mla_vllm_b200 import _lib
from qwen_mla_vllm_b200.tree_attention import tree_attention, tree_masks
from tree_util import SM, build_case, random_parents, tree_ref

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}


def run(c, q, bt, ctx, mask, *, rank, rope, page, mode="native", fp8=False, ks=1.0, cap=0.0, o_dtype=torch.bfloat16, **kw):
    qk = rank + rope
    n, H = q.shape[:2]
    o = torch.full((n, H, rank), float("nan"), dtype=o_dtype, device=q.device)
    lse = torch.full((n, H), float("nan"), dtype=torch.float32, device=q.device)
    k_scale = torch.tensor(ks, dtype=torch.float32, device=q.device) if fp8 else None
    tree_attention(q, c, o, lse, bt, ctx, mask, rank=rank, sm_scale=SM, page_size=page,
                   rms_offset=-1 if mode == "none" else qk, qk_dim=qk, rms_log8=mode == "log8", rms_bf16=mode == "bf16",
                   logit_cap=cap, k_scale=k_scale, **kw)
    return o, lse


def verify(o, lse, c, q, bt, ctx, mask, *, rank, rope, page, mode="native", fp8=False, ks=1.0, cap=0.0):
    ro, rl, tol, ltol = tree_ref(q, c, bt, ctx, mask, rank=rank, qk=rank + rope, page=page, rms_offset=rank + rope,
                                 mode=mode, fp8=fp8, k_scale=ks, cap=cap)
    d = np.abs(o.double().cpu().numpy() - ro)
    lim = tol + U[o.dtype] * np.abs(ro) * 1.01 + 1e-7
    assert (d <= lim).all(), f"o off by {d.max():.3e}, {np.nanmax(d / lim):.2f} of its bound"
    l = lse.double().cpu().numpy()
    fin = np.isfinite(rl)
    assert np.array_equal(l == -np.inf, ~fin)
    assert (np.abs(l[fin] - rl[fin]) <= ltol[fin]).all(), f"lse off by {np.abs(l[fin] - rl[fin]).max():.3e}"


SHAPES = [  # heads, rank, rope
    (24, 768, 232), (12, 384, 116), (24, 256, 232), (6, 512, 58), (1, 256, 0), (24, 1792, 232), (48, 256, 58), (5, 768, 58)]


@pytest.mark.parametrize("fp8,mode", [(False, "native"), (False, "none"), (True, "log8"), (True, "bf16"), (True, "native"), (True, "none")])
@pytest.mark.parametrize("heads,rank,rope", SHAPES)
def test_shapes_and_row_formats(cuda_device, heads, rank, rope, fp8, mode):
    nodes, ctxs, page = 5, [130, 0, 61, 257], 16
    cm = "e4m3" if fp8 and mode == "native" else ("log8" if fp8 and mode == "none" else mode)
    c, q, bt, ctx, ks = build_case(cuda_device, 4, nodes, heads, rank, rope, page, ctxs, mode=cm, fp8=fp8)
    mask = tree_masks(random_parents(4, nodes).to(cuda_device))
    kw = dict(rank=rank, rope=rope, page=page, mode=mode, fp8=fp8, ks=ks)
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx, mask, **kw)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("nodes", [1, 2, 3, 7, 16, 33, 64])
@pytest.mark.parametrize("heads,rank,rope", [(24, 768, 232), (12, 384, 116)])
def test_tree_sizes(cuda_device, heads, rank, rope, nodes, fp8):
    ctxs, page, mode = [0, 1, 127, 128, 500], 16, "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 5, nodes, heads, rank, rope, page, ctxs, mode=mode, fp8=fp8, seed=nodes)
    mask = tree_masks(random_parents(5, nodes, nodes).to(cuda_device))
    kw = dict(rank=rank, rope=rope, page=page, mode=mode, fp8=fp8, ks=ks)
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx, mask, **kw)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [1, 3, 16, 24, 32, 48, 64, 128, 256])
def test_page_sizes(cuda_device, page, fp8):
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 3, 4, 12, 384, 116, page, [383, 40, 255], mode=mode, fp8=fp8)
    mask = tree_masks(torch.tensor([-1, 0, 0, 1], device=cuda_device))  # one tree for all
    kw = dict(rank=384, rope=116, page=page, mode=mode, fp8=fp8, ks=ks)
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx, mask, **kw)


@pytest.mark.parametrize("fp8", [False, True])
def test_long_rows_split_over_blocks(cuda_device, fp8):
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 2, 3, 24, 768, 232, 16, [9000, 20001], mode=mode, fp8=fp8)
    mask = tree_masks(random_parents(2, 3).to(cuda_device))
    kw = dict(rank=768, rope=232, page=16, mode=mode, fp8=fp8, ks=ks)
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx, mask, **kw)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_sink_and_a_long_faint_tail(cuda_device, fp8):
    """One token takes a weight of 1, tens of thousands a tiny weight each: together they count."""
    mode = "log8" if fp8 else "native"
    c, q, bt, ctx, ks = build_case(cuda_device, 1, 2, 6, 256, 58, 16, [30000], mode=mode, fp8=fp8, q_scale=0.0)
    g = torch.Generator().manual_seed(9)
    q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16) * 1e-3)
    raw = c.view(torch.uint8) if fp8 else c
    raw[..., 0] = 0
    raw[..., 314:320] = 128 if fp8 else 1.0  # divisors about 1
    raw[int(bt[0, 0]), 0, 0, 0] = 0x7E if fp8 else 24.0  # 448 k_scale, or 24
    q[..., 0] = 12 * 16 / (448 * ks if fp8 else 24.0)  # a score of 12 over scores about 0
    mask = tree_masks(torch.tensor([[-1, 0]], device=cuda_device))
    kw = dict(rank=256, rope=58, page=16, mode=mode, fp8=fp8, ks=ks)
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx, mask, **kw)


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("o_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_types_strides_and_cap(cuda_device, o_dtype, cap):
    """f16 queries with the rope part apart, padded rows, pages with gaps, strided outputs."""
    c, q, bt, ctx, _ = build_case(cuda_device, 2, 6, 24, 768, 232, 16, [200, 77])
    q = q.to(torch.float16)
    big = torch.zeros(c.shape[0], 20, 1, c.shape[3] + 16, dtype=c.dtype, device=cuda_device)
    big[:, :16, :, :c.shape[3]] = c
    cv = big[:, :16, :, :c.shape[3]]
    qn = torch.zeros(12, 24, 800, dtype=q.dtype, device=cuda_device)
    qn[..., 3:771] = q[..., :768]
    qp = torch.zeros(12, 24, 300, dtype=q.dtype, device=cuda_device)
    qp[..., 5:237] = q[..., 768:]
    ob = torch.zeros(12, 30, 900, dtype=o_dtype, device=cuda_device)
    lb = torch.zeros(12, 40, device=cuda_device)
    o, lse = ob[:, 2:26, 7:775], lb[:, 3:27]
    mask = tree_masks(random_parents(2, 6).to(cuda_device))
    tree_attention(qn[..., 3:771], cv, o, lse, bt, ctx, mask, rank=768, sm_scale=SM, page_size=16, rms_offset=1000,
                   q_pe=qp[..., 5:237], logit_cap=cap)
    verify(o, lse, c, q, bt, ctx, mask, rank=768, rope=232, page=16, cap=cap)
    ob[:, 2:26, 7:775] = 0
    lb[:, 3:27] = 0
    assert not ob.any() and not lb.any()


@pytest.mark.parametrize("heads,rank,rope,page", [(24, 768, 232, 16), (12, 384, 116, 3), (24, 1792, 232, 16)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_hidden_rows_do_not_matter(cuda_device, heads, rank, rope, page, poison):
    """Rows past the drafts, and a sibling's row, hold NaN or inf: only the nodes that see it do too."""
    c, q, bt, ctx, _ = build_case(cuda_device, 2, 4, heads, rank, rope, page, [30, 130])
    mask = tree_masks(torch.tensor([[-1, 0, 0, 2], [-1, 0, 1, 1]], device=cuda_device))
    kw = dict(rank=rank, rope=rope, page=page)
    clean_o, clean_lse = run(c, q, bt, ctx, mask, **kw)
    verify(clean_o, clean_lse, c, q, bt, ctx, mask, **kw)
    ends = [30 + 4, 130 + 4]
    for r in range(2):
        for t in list(range(ends[r], bt.shape[1] * page)) + [ends[r] - 3]:  # and node 1 of each request
            c[bt[r, t // page].long(), t % page] = poison
    o, lse = run(c, q, bt, ctx, mask, **kw)
    sees = (mask >> 1 & 1).bool().flatten()
    assert torch.equal(o[~sees], clean_o[~sees]) and torch.equal(lse[~sees], clean_lse[~sees])
    assert o[sees].isnan().all() and not lse[sees].isfinite().any()


def test_rows_that_see_nothing(cuda_device):
    """Padding nodes, empty contexts, negative lengths, drafts beyond the block table, absent pages."""
    c, q, bt, ctx, _ = build_case(cuda_device, 4, 3, 12, 384, 116, 16, [20, 0, -7, 33])
    mask = torch.tensor([[1, 0, 5], [1, 2, 0], [0, 2, 4], [1, 2, 4]], dtype=torch.int64, device=cuda_device)
    kw = dict(rank=384, rope=116, page=16)
    o, lse = run(c, q, bt, ctx, mask, **kw)
    verify(o, lse, c, q, bt, ctx, mask, **kw)
    for row in (1, 5, 6):
        assert not o[row].any() and (lse[row] == float("-inf")).all()
    ctx[3] = bt.shape[1] * 16 - 1  # node 0 is the table's last token; nodes 1 and 2 lie beyond
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx, mask, **kw)
    ctx[3] = 10**9
    verify(*run(c, q, bt, ctx, mask, **kw), c, q, bt, ctx.clamp(max=bt.shape[1] * 16), mask, **kw)
    bt2 = bt.clone()
    bt2[0] = 10**6
    bt2[1] = -3
    o, lse = run(c, q, bt2, ctx, mask, **kw)
    assert not o[:6].any() and (lse[:6] == float("-inf")).all()


def test_far_pages(cuda_device):
    """Pages more than 2^32 bytes (and 2^31 elements) into the cache."""
    c, q, bt, ctx, _ = build_case(cuda_device, 1, 2, 12, 384, 116, 16, [40])
    step = (1 << 30) // 16 * 16
    big = torch.empty(step * (c.shape[0] - 1) + c[0].numel(), dtype=torch.bfloat16, device=cuda_device)
    far = big.as_strided((c.shape[0], 16, 1, c.shape[3]), (step, c.shape[3], c.shape[3], 1))
    far.copy_(c)
    mask = tree_masks(torch.tensor([[-1, 0]], device=cuda_device))
    a, b = run(far, q, bt, ctx, mask, rank=384, rope=116, page=16)
    x, y = run(c, q, bt, ctx, mask, rank=384, rope=116, page=16)
    assert torch.equal(a, x) and torch.equal(b, y)


def test_chain_agrees_with_the_flattened_decode(cuda_device):
    """A chain of drafts is the plugin's causal verify: the decode of rows of growing length."""
    from qwen_mla_vllm_b200.mla_decode_attention import build_params, run_params
    c, q, bt, ctx, _ = build_case(cuda_device, 3, 4, 24, 768, 232, 16, [100, 900, 3])
    mask = tree_masks(torch.tensor([-1, 0, 1, 2], device=cuda_device))
    o, lse = run(c, q, bt, ctx, mask, rank=768, rope=232, page=16)
    lens = (ctx[:, None] + torch.arange(1, 5, dtype=torch.int32, device=cuda_device)).flatten().contiguous()
    o2, l2 = torch.empty_like(o), torch.empty_like(lse)
    p = build_params(q, c, o2, l2, bt.repeat_interleave(4, 0).contiguous(), lens, rank=768, qk_dim=1000, rms_offset=1000,
                     rms_mode=_lib.RMS_NATIVE, page_size=16, sm_scale=SM, qrows=4)
    run_params(p, q.device)
    assert (o.float() - o2.float()).abs().max() < 2e-2 and (lse - l2).abs().max() < 1e-4


def test_repeats_streams_and_graphs_agree(cuda_device):
    c, q, bt, ctx, _ = build_case(cuda_device, 4, 8, 24, 768, 232, 16, [1000, 50, 3000, 129])
    mask = tree_masks(random_parents(4, 8).to(cuda_device))
    kw = dict(rank=768, rope=232, page=16)
    o, lse = run(c, q, bt, ctx, mask, **kw)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o2, l2 = run(c, q, bt, ctx, mask, **kw)
        st.synchronize()
        assert torch.equal(o, o2) and torch.equal(lse, l2)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            tree_attention(q, c, o2, l2, bt, ctx, mask, rank=768, sm_scale=SM, page_size=16, rms_offset=1000)
        ctx.copy_(torch.tensor([7, 2000, 0, 640], dtype=torch.int32))
        g.replay()
    st.synchronize()
    o, lse = run(c, q, bt, ctx, mask, **kw)
    assert torch.equal(o, o2) and torch.equal(lse, l2)


def test_tree_masks():
    got = tree_masks(torch.tensor([[-1, 0, 1, 0, 3, 4], [2, 2, -1, 9, 0, 4]]))
    assert got.tolist() == [[1, 3, 7, 9, 25, 57], [5, 6, 4, 8, 21, 53]]
    chain = tree_masks(torch.arange(64) - 1)
    assert [m & (2**64 - 1) for m in chain.tolist()] == [2**(i + 1) - 1 for i in range(64)]


def test_refusals(cuda_device):
    c, q, bt, ctx, _ = build_case(cuda_device, 2, 3, 12, 384, 116, 16, [20, 5])
    mask = tree_masks(torch.tensor([-1, 0, 0], device=cuda_device))
    o, lse = torch.empty(6, 12, 384, dtype=torch.bfloat16, device=cuda_device), torch.empty(6, 12, device=cuda_device)
    ok = dict(q=q, kv_cache=c, o=o, lse=lse, block_table=bt, ctx_lens=ctx, tree_mask=mask, rank=384, sm_scale=SM,
              page_size=16, rms_offset=500)
    tree_attention(**ok)
    tree_attention(**dict(ok, lse=None))
    for bad, err in ((dict(q=q[:5]), ValueError), (dict(q=q[..., :400]), ValueError), (dict(o=o[:, :, :100]), ValueError),
                     (dict(lse=lse[:3]), ValueError), (dict(tree_mask=mask.int()), TypeError),
                     (dict(tree_mask=mask.expand(3, 3)), ValueError), (dict(ctx_lens=ctx.long()), TypeError),
                     (dict(block_table=bt[:1]), ValueError), (dict(page_size=8), ValueError), (dict(kv_cache=c.half()), TypeError),
                     (dict(q=q.float()), _lib.QmlaError), (dict(rms_offset=300, qk_dim=500), _lib.QmlaError),
                     (dict(rms_offset=2000, qk_dim=500), _lib.QmlaError), (dict(q=q.cpu()), ValueError),
                     (dict(tree_mask=torch.zeros(65, dtype=torch.int64, device=cuda_device)), ValueError),
                     (dict(workspace=torch.empty(16, dtype=torch.uint8, device=cuda_device)), _lib.QmlaError),
                     (dict(kv_cache=c[..., 1:]), _lib.QmlaError)):
        with pytest.raises(err):
            tree_attention(**dict(ok, **bad))
    tree_attention(**dict(ok, q=q[:0], o=o[:0], lse=lse[:0], ctx_lens=ctx[:0]))
