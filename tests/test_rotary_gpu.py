"""Rotary positions and the fused rotate-and-write on the GPU, against 64-bit formulas.

Tolerances: the kernel works in 32 bits and rounds once.  An angle is off by at most 2^-25 turns
(1.9e-7 rad), sin and cos by 2 ulp, the two products and the sum by 3 roundings: under 1e-6 of
(|a| + |b|) together; then one rounding to the output type, u |y| with u = 2^-8 (bf16), 2^-11 (f16).
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import oracle
from qwen_mla_vllm_b200.mla_gather import gather_status
from qwen_mla_vllm_b200.rotary import rope_kv_cache_update, rotary_embed, rotary_steps

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def rotate64(x, pos, steps, interleaved, sign=1.0, scale=1.0):
    """x [n, heads, rot] float64, every block of rot dims turned by its own pairs' phases."""
    n, rot = x.shape[0], 2 * len(steps)
    ang = np.array([[((int(p) * int(s)) % 2**64) / 2**64 * 2 * math.pi for s in steps] for p in pos])
    c, s = scale * np.cos(ang)[:, None, :], scale * sign * np.sin(ang)[:, None, :]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:])
    ra, rb = a * c - b * s, b * c + a * s
    y, mag = np.empty_like(x), np.empty_like(x)
    m = np.abs(a) + np.abs(b)
    if interleaved:
        y[..., 0::2], y[..., 1::2], mag[..., 0::2], mag[..., 1::2] = ra, rb, m, m
    else:
        y = np.concatenate([ra, rb], -1)
        mag = np.concatenate([m, m], -1)
    return y, mag * scale


def expect(x, pos, steps, start, blocks, interleaved, adjoint=False, scale=1.0):
    x64 = x.detach().double().cpu().numpy()
    y, mag = x64.copy(), np.zeros_like(x64)
    rot = 2 * len(steps)
    for b in range(blocks):
        d = slice(start + b * rot, start + (b + 1) * rot)
        y[..., d], mag[..., d] = rotate64(x64[..., d], pos.tolist(), steps.tolist(), interleaved,
                                          -1.0 if adjoint else 1.0, scale)
    return y, mag


def check(got, y, mag, dtype, half_step=0.0):
    g = got.double().cpu().numpy()
    tol = U[dtype] * np.abs(y) * 1.0001 + 1e-6 * mag + half_step
    bad = np.abs(g - y) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.abs(g - y).max():.3e}"


SHAPES = [  # tokens, heads, dim, rot, start, blocks
    (1, 1, 2, 2, 0, 1), (1, 24, 256, 58, 198, 1), (7, 3, 58, 58, 0, 1), (5, 2, 61, 30, 31, 1), (129, 12, 64, 64, 0, 1),
    (33, 24, 232, 58, 0, 4), (3, 1, 128, 32, 7, 3), (300, 1, 58, 58, 0, 1), (2, 5, 1024, 512, 0, 2),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary_matches_the_formula(cuda_device, shape, interleaved, dtype):
    n, heads, dim, rot, start, blocks = shape
    g = torch.Generator().manual_seed(n + dim)
    x = torch.randn(n, heads, dim, generator=g).to(dtype).to(cuda_device)
    pos = torch.randint(0, 1 << 20, (n,), generator=g)
    pos[0] = 0
    steps, _ = rotary_steps(rot, 1e6, device=cuda_device)
    for adjoint in (False, True):
        y, mag = expect(x, pos, steps.cpu(), start, blocks, interleaved, adjoint, 1.25)
        got = rotary_embed(x, pos.to(cuda_device), steps, start=start, blocks=blocks, interleaved=interleaved,
                           scale=1.25, adjoint=adjoint)
        check(got, y, mag, dtype)
        assert torch.equal(got[..., :start], x[..., :start])
        assert torch.equal(got[..., start + blocks * rot:], x[..., start + blocks * rot:])


@pytest.mark.parametrize("case", ["in_place", "view_in", "view_out", "odd_offset", "two_dim", "broadcast_heads"])
def test_rotary_strides(cuda_device, case):
    g = torch.Generator().manual_seed(4)
    n, heads, dim, rot = 37, 6, 232, 58
    pos = torch.arange(100, 100 + n, dtype=torch.int32, device=cuda_device)
    steps, _ = rotary_steps(rot, 1e4, device=cuda_device)
    big = torch.randn(n, heads, 1000, generator=g).to(torch.bfloat16).to(cuda_device)
    x, out = big[..., 768:], None
    if case == "odd_offset":
        x = big[..., 701:701 + dim]
    elif case == "two_dim":
        x = big[:, 2, 768:]
    elif case == "broadcast_heads":
        x = big[:, :1, 768:].expand(n, heads, dim)
    x0 = x.clone()
    if case == "in_place":
        out = x
    elif case == "view_out":
        out = torch.zeros(n, heads, 500, dtype=torch.bfloat16, device=cuda_device)[..., 8:8 + dim]
    before = big.clone()
    got = rotary_embed(x, pos, steps, blocks=4, out=out)
    x64 = x0 if x0.dim() == 3 else x0[:, None]
    y, mag = expect(x64, pos.cpu(), steps.cpu(), 0, 4, False)
    check(got if got.dim() == 3 else got[:, None], y, mag, torch.bfloat16)
    if case == "in_place":
        assert got.data_ptr() == x.data_ptr()
        assert torch.equal(big[..., :768], before[..., :768])
    else:
        assert torch.equal(big, before)


def test_rotary_in_place_touches_the_window_only(cuda_device):
    x = torch.full((3, 2, 64), float("nan"), device=cuda_device)
    x[..., 20:52] = 1.0
    steps, _ = rotary_steps(32, device=cuda_device)
    rotary_embed(x, torch.zeros(3, dtype=torch.int64, device=cuda_device), steps, start=20, out=x)
    assert torch.equal(x[..., 20:52], torch.ones_like(x[..., 20:52]))
    assert x[..., :20].isnan().all() and x[..., 52:].isnan().all()


@pytest.mark.parametrize("p", [0, 1, -5, 2**20, 2**31 - 1, 2**40])
def test_rotary_far_positions(cuda_device, p):
    x = torch.randn(1, 2, 128, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    steps, _ = rotary_steps(128, 1e6, device=cuda_device)
    pos = torch.tensor([p], dtype=torch.int64)
    y, mag = expect(x, pos, steps.cpu(), 0, 1, True)
    check(rotary_embed(x, pos.to(cuda_device), steps, interleaved=True), y, mag, torch.float32)


def test_rotary_nan_and_inf_stay_in_their_pair(cuda_device):
    x = torch.ones(1, 1, 8, device=cuda_device)
    x[0, 0, 2] = float("nan")
    x[0, 0, 5] = float("inf")
    steps, _ = rotary_steps(8, device=cuda_device)
    y = rotary_embed(x, torch.tensor([3], device=cuda_device), steps, interleaved=True)[0, 0]
    assert y[2:4].isnan().all() and not y[4:6].isfinite().any() and y[[0, 1, 6, 7]].isfinite().all()


def test_rotary_empty(cuda_device):
    steps, _ = rotary_steps(8, device=cuda_device)
    y = rotary_embed(torch.empty(0, 4, 8, device=cuda_device), torch.empty(0, dtype=torch.int32, device=cuda_device), steps)
    assert y.shape == (0, 4, 8)


def test_rotary_gradient(cuda_device):
    """Autograd's gradient is the adjoint, and agrees with differences of the loss."""
    import qwen_mla_vllm_b200.ops  # noqa: F401
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 3, 40, generator=g).to(cuda_device).requires_grad_()
    w = torch.randn(5, 3, 40, generator=g).to(cuda_device)
    pos = torch.tensor([0, 3, 1000, 70000, 5], device=cuda_device)
    steps, _ = rotary_steps(30, 1e4, device=cuda_device)
    f = lambda t: torch.ops.qmla.rotary(t, pos, steps, 6, 1, False, 1.5, False)  # noqa: E731
    (f(x) * w).sum().backward()
    y, mag = expect(w, pos.cpu(), steps.cpu(), 6, 1, False, True, 1.5)
    check(x.grad, y, mag, torch.float32)
    # the map is linear, so a difference over a large step is exact up to rounding (2e-6 of |x||w|)
    d = torch.randn(5, 3, 40, generator=g).to(cuda_device)
    with torch.no_grad():
        diff = ((f(x + 4 * d) - f(x - 4 * d)).double() * w.double()).sum() / 8
    dot = (x.grad.double() * d.double()).sum()
    assert abs(float(diff - dot)) < 2e-6 * float(d.norm() * w.norm()) * 8
    torch.library.opcheck(torch.ops.qmla.rotary.default, (x.detach(), pos, steps, 6, 1, False, 1.5, False),
                          test_utils=("test_schema", "test_faketensor"))


def test_rotary_other_stream(cuda_device):
    x = torch.randn(4096, 24, 64, device=cuda_device)
    pos = torch.arange(4096, device=cuda_device)
    steps, _ = rotary_steps(64, device=cuda_device)
    want = rotary_embed(x, pos, steps)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = rotary_embed(x, pos, steps)
    st.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------------------ the fused cache write
def update_case(dev, n, heads, rank, groups, fp8, mode, page, *, seed=0, pad=0, gap=0):
    g = torch.Generator().manual_seed(seed)
    win = 58 * groups
    tail = {"none": 0, "bf16": 2 * heads}.get(mode, heads)
    W = rank + win + tail + pad
    W += (-W) % 16
    pages = -(-n // page) + 1
    es = torch.uint8 if fp8 else torch.bfloat16
    full = torch.randint(0, 120, (pages, page + gap, 1, W), generator=g).to(es).to(dev)
    cache = full[:, :page]
    t = dict(
        q_pe=torch.randn(n, heads, win, generator=g).to(torch.bfloat16).to(dev),
        kv_c_normed=(torch.randn(n, rank, generator=g) * 3).to(torch.bfloat16).to(dev),
        k_pe=torch.cat([torch.randn(n, win, generator=g), torch.exp(torch.randn(n, heads, generator=g) * 0.8)], 1)
        .to(torch.bfloat16).to(dev),
        positions=torch.randint(0, 300000, (n,), generator=g).to(dev),
        slot_mapping=torch.randperm(pages * page, generator=g)[:n].to(dev))
    scale = torch.tensor(0.011, device=dev) if fp8 else None
    return t, full, cache, scale, win, W


def check_rows(t, before, cache, scale, win, rank, heads, mode, steps, page, interleaved):
    n = t["q_pe"].shape[0]
    k64, mag = rotate64(t["k_pe"][:, :win].double().cpu().numpy().reshape(n, -1, 2 * len(steps)),
                        t["positions"].tolist(), steps.tolist(), interleaved)
    k64, mag = k64.reshape(n, win), mag.reshape(n, win)
    rows = cache.reshape(-1, cache.shape[-1])
    written = t["slot_mapping"].clamp(min=0)
    got = rows[written].cpu()
    if scale is None:
        assert torch.equal(got[:, :rank], t["kv_c_normed"].cpu())
        kr = got[:, rank:rank + win].double().numpy()
        assert (np.abs(kr - k64) <= 2.0**-8 * np.abs(k64) * 1.0001 + 1e-6 * mag).all()
        if mode != "none":
            assert torch.equal(got[:, rank + win:rank + win + heads], t["k_pe"][:, win:].cpu())
        used = rank + win + (0 if mode == "none" else heads)
    else:
        b = got.numpy()
        inv = np.float32(1.0) / np.float32(scale.cpu().numpy())
        lat = t["kv_c_normed"].float().cpu().numpy() * inv
        assert np.array_equal(b[:, :rank], oracle.e4m3_encode(np.clip(lat, -448, 448)))
        y = np.clip(k64 * float(inv), -448, 448)
        kr = oracle.e4m3_decode(b[:, rank:rank + win]).astype(np.float64)
        # one rounding to e4m3 (4-bit significand, subnormal step 2^-9)
        assert (np.abs(kr - y) <= np.maximum(2.0**-4 * np.abs(y), 2.0**-10) * 1.0001 + 2e-6 * mag * float(inv)).all()
        r = t["k_pe"][:, win:]
        if mode == "log8":
            assert np.array_equal(b[:, rank + win:rank + win + heads], oracle.log8_encode(r.float().cpu().numpy()))
        elif mode == "bf16":
            assert np.array_equal(b[:, rank + win:rank + win + 2 * heads],
                                  np.ascontiguousarray(r.contiguous().cpu().view(torch.int16).numpy()).view(np.uint8).reshape(n, -1))
        used = rank + win + {"none": 0, "bf16": 2 * heads, "log8": heads}[mode]
    # nothing else of the cache changed
    keep = torch.ones(rows.shape[0], dtype=torch.bool)
    keep[written.cpu()] = False
    b0 = before.reshape(-1, before.shape[-1]).cpu()
    assert torch.equal(rows.cpu()[keep], b0[keep])
    assert torch.equal(got[:, used:], b0[written.cpu()][:, used:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fp8,mode", [(False, "native"), (False, "none"), (True, "log8"), (True, "bf16"), (True, "none")])
@pytest.mark.parametrize("n,heads,rank,groups,page,gap", [
    (1, 24, 768, 4, 16, 0), (5, 12, 384, 2, 16, 2), (67, 6, 512, 1, 3, 0), (9, 24, 1792, 4, 64, 1), (3, 1, 20, 1, 1, 0)])
def test_rope_update_rows(cuda_device, n, heads, rank, groups, page, gap, fp8, mode, interleaved):
    t, full, cache, scale, win, W = update_case(cuda_device, n, heads, rank, groups, fp8, mode, page, gap=gap)
    steps, _ = rotary_steps(58, 1e6, device=cuda_device)
    before, gap_before = cache.clone(), full[:, page:].clone()
    q = rope_kv_cache_update(**t, steps=steps, kv_cache=cache, packed_rope=win, local_heads=heads,
                             q_out=torch.empty_like(t["q_pe"]), interleaved=interleaved, k_scale=scale, rms_mode=mode)
    y, mag = expect(t["q_pe"], t["positions"], steps.cpu(), 0, groups, interleaved)
    check(q, y, mag, torch.bfloat16)
    check_rows(t, before, cache, scale, win, rank, heads, mode, steps.cpu(), page, interleaved)
    assert torch.equal(full[:, page:], gap_before)


def test_rope_update_agrees_with_the_row_writer_at_position_zero(cuda_device):
    """Position 0 turns nothing: an FP8 row is then byte for byte fp8_kv_cache_update's."""
    from qwen_mla_vllm_b200.kv_cache import fp8_kv_cache_update
    t, _, cache, scale, win, _ = update_case(cuda_device, 50, 24, 768, 4, True, "log8", 16)
    t["positions"].zero_()
    steps, _ = rotary_steps(58, 1e6, device=cuda_device)
    other = cache.clone()
    fp8_kv_cache_update(t["kv_c_normed"], t["k_pe"], other, t["slot_mapping"], scale, win, 24, "log8")
    q = t["q_pe"].clone()
    rope_kv_cache_update(**t, steps=steps, kv_cache=cache, packed_rope=win, local_heads=24, k_scale=scale, rms_mode="log8")
    assert torch.equal(cache, other) and torch.equal(t["q_pe"], q)


def test_rope_update_bad_and_padding_slots(cuda_device):
    t, _, cache, _, win, _ = update_case(cuda_device, 6, 4, 256, 1, False, "native", 16)
    before = cache.clone()
    steps, _ = rotary_steps(58, device=cuda_device)
    gather_status(cuda_device)
    t["slot_mapping"][:] = torch.tensor([-1, cache.shape[0] * 16, 3, -(1 << 40), 1 << 40, 5], device=cuda_device)
    q = rope_kv_cache_update(**t, steps=steps, kv_cache=cache, packed_rope=win, local_heads=4, q_out=torch.empty_like(t["q_pe"]))
    y, mag = expect(t["q_pe"], t["positions"], steps.cpu(), 0, 1, False)
    check(q, y, mag, torch.bfloat16)  # q turns whatever the slot
    rows, b0 = cache.reshape(-1, cache.shape[-1]), before.reshape(-1, cache.shape[-1])
    changed = (rows != b0).any(dim=1).nonzero().flatten().tolist()
    assert changed == [3, 5]
    assert gather_status(cuda_device) == 2


def test_rope_update_q_view_in_place_and_saturation(cuda_device):
    t, _, cache, scale, win, _ = update_case(cuda_device, 8, 24, 768, 4, True, "log8", 16)
    full_q = torch.randn(8, 24, 1000, device=cuda_device).to(torch.bfloat16)
    t["q_pe"] = full_q[..., 768:]
    q0 = t["q_pe"].clone()
    t["kv_c_normed"][0, :3] = torch.tensor([1e30, -1e30, float("nan")])
    steps, _ = rotary_steps(58, 1e6, device=cuda_device)
    nope = full_q[..., :768].clone()
    rope_kv_cache_update(**t, steps=steps, kv_cache=cache, packed_rope=win, local_heads=24, k_scale=scale, rms_mode="log8")
    y, mag = expect(q0, t["positions"], steps.cpu(), 0, 4, False)
    check(t["q_pe"], y, mag, torch.bfloat16)
    assert torch.equal(full_q[..., :768], nope)
    row = cache.reshape(-1, cache.shape[-1])[t["slot_mapping"][0]]
    assert row[:3].tolist() == [0x7E, 0xFE, 0x7F]


def test_refusals(cuda_device):
    steps, _ = rotary_steps(8, device=cuda_device)
    x = torch.zeros(2, 3, 16, device=cuda_device)
    pos = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for kw in (dict(start=9), dict(blocks=3), dict(start=-1), dict(blocks=0)):
        with pytest.raises(ValueError):
            rotary_embed(x, pos, steps, **kw)
    with pytest.raises(ValueError):
        rotary_embed(x, pos[:1], steps)
    with pytest.raises(TypeError):
        rotary_embed(x, pos.float(), steps)
    with pytest.raises(TypeError):
        rotary_embed(x.double(), pos, steps)
    with pytest.raises(TypeError):
        rotary_embed(x, pos, steps.int())
    with pytest.raises(ValueError):
        rotary_embed(x, pos, steps, out=torch.zeros(2, 3, 8, device=cuda_device))
    with pytest.raises(ValueError):
        rotary_embed(x.transpose(1, 2), pos, steps)
    with pytest.raises(ValueError):
        rotary_embed(x, pos.cpu(), steps)
    t, _, cache, scale, win, _ = update_case(cuda_device, 4, 4, 256, 1, True, "log8", 16)
    s58, _ = rotary_steps(58, device=cuda_device)
    ok = dict(t, steps=s58, kv_cache=cache, packed_rope=win, local_heads=4, k_scale=scale, rms_mode="log8")
    for bad, err in ((dict(k_scale=None), TypeError), (dict(rms_mode="native"), ValueError), (dict(rms_mode="x"), ValueError),
                     (dict(steps=steps), ValueError), (dict(packed_rope=116), ValueError), (dict(local_heads=40), ValueError),
                     (dict(slot_mapping=t["slot_mapping"].int()), TypeError), (dict(k_pe=t["k_pe"].float()), TypeError),
                     (dict(kv_cache=cache[:, :, 0]), ValueError)):
        with pytest.raises(err):
            rope_kv_cache_update(**dict(ok, **bad))


# Widest segments (two stages of 16 KB and the sines pass 48 KB of shared memory) and calls long enough
# for a block to walk several token groups, the last one ragged.
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,shape", [
    (torch.float32, (3, 2, 4096, 512, 0, 8)), (torch.bfloat16, (2, 1, 8192, 512, 0, 16)),
    (torch.bfloat16, (8193, 12, 58, 58, 0, 1)), (torch.bfloat16, (4099, 5, 234, 58, 2, 4)),
    (torch.float16, (40001, 1, 64, 64, 0, 1)),
])
def test_rotary_wide_and_long(cuda_device, dtype, shape, interleaved):
    n, heads, dim, rot, start, blocks = shape
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, heads, dim, generator=g).to(dtype).to(cuda_device)
    pos = torch.randint(0, 1 << 20, (n,), generator=g)
    steps, _ = rotary_steps(rot, 1e6, device=cuda_device)
    y, mag = expect(x, pos, steps.cpu(), start, blocks, interleaved)
    # two million values reach f16's subnormals, spaced 2^-24: there even the exact value rounds by 2^-25
    check(rotary_embed(x, pos.to(cuda_device), steps, start=start, blocks=blocks, interleaved=interleaved), y, mag, dtype,
          half_step=2.0**-25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fp8,mode", [(False, "native"), (True, "log8")])
def test_rope_update_long(cuda_device, fp8, mode, interleaved):
    n, heads, rank, groups, page = 8199, 9, 256, 2, 64
    t, _, cache, scale, win, _ = update_case(cuda_device, n, heads, rank, groups, fp8, mode, page)
    steps, _ = rotary_steps(58, 1e6, device=cuda_device)
    before = cache.clone()
    q = rope_kv_cache_update(**t, steps=steps, kv_cache=cache, packed_rope=win, local_heads=heads,
                             q_out=torch.empty_like(t["q_pe"]), interleaved=interleaved, k_scale=scale, rms_mode=mode)
    y, mag = expect(t["q_pe"], t["positions"], steps.cpu(), 0, groups, interleaved)
    check(q, y, mag, torch.bfloat16)
    check_rows(t, before, cache, scale, win, rank, heads, mode, steps.cpu(), page, interleaved)
