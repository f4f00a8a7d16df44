"""64-bit restatement of the tree attention and of the accumulated attention weights, with the
magnitudes their error bounds are made of."""
from __future__ import annotations

import math

import numpy as np
import torch

import oracle
from gpu_util import make_bf16_case, make_fp8_case

SM = 1 / 16


def keys_of(cache, bt_row, toks, page, qk, heads, rms_offset, mode, fp8, k_scale):
    """Rows of tokens ``toks`` of one request: keys [n, qk] and divisors [n, heads] in float64."""
    toks = np.asarray(toks, dtype=np.int64)
    pages = torch.from_numpy(np.asarray(bt_row)[toks // page].astype(np.int64)).to(cache.device)
    rows = cache[pages, torch.from_numpy(toks % page).to(cache.device), 0].contiguous().cpu()
    if fp8:
        raw = rows.view(torch.uint8).numpy()
        k = oracle.e4m3_decode(raw[:, :qk]).astype(np.float64) * k_scale
    else:
        raw = rows.view(torch.int16).numpy().view(np.uint16)
        k = oracle.bf16_bits_to_f32(raw[:, :qk]).astype(np.float64)
    if mode == "none":
        return k, np.ones((len(toks), heads))
    if mode == "log8":
        rms = 2.0 ** (raw[:, rms_offset:rms_offset + heads].astype(np.float64) * 6 / 255 - 3)
    elif mode == "bf16":
        b = raw[:, rms_offset:rms_offset + 2 * heads].astype(np.uint16)
        rms = oracle.bf16_bits_to_f32(b[:, 0::2] | (b[:, 1::2] << 8)).astype(np.float64)
    elif fp8:
        rms = oracle.e4m3_decode(raw[:, rms_offset:rms_offset + heads]).astype(np.float64) * k_scale
    else:
        rms = oracle.bf16_bits_to_f32(raw[:, rms_offset:rms_offset + heads]).astype(np.float64)
    return k, np.where(rms > 0, rms, 1.0)


def scores64(q, k, div, sm_scale, cap):
    """Scores [n, heads] and the sum of their terms' magnitudes."""
    s = (k @ q.T) / div * sm_scale
    mag = (np.abs(k) @ np.abs(q).T) / div * sm_scale
    if cap > 0:
        s = cap * np.tanh(s / cap)
    return s, mag


def visible(ctx, mask, nodes, room):
    toks = list(range(min(ctx, room))) + [ctx + j for j in range(nodes) if mask >> j & 1]
    return [t for t in toks if t < room] if mask else []


def tree_ref(q, cache, bt, ctx, mask, *, rank, qk, page, rms_offset, mode, fp8, k_scale=1.0, cap=0.0, sm_scale=SM):
    """(o, lse, tol of o in f32, tol of lse): see the bounds in test_tree_gpu.py."""
    nodes = mask.shape[-1]
    rows, H = q.shape[0], q.shape[1]
    q64 = q.double().cpu().numpy()
    btn, ctxn = bt.cpu().numpy(), ctx.cpu().tolist()
    m2 = (mask if mask.dim() == 2 else mask.expand(len(ctxn), nodes)).cpu().tolist()
    o, lse = np.zeros((rows, H, rank)), np.full((rows, H), -np.inf)
    tol, ltol = np.zeros((rows, H, rank)), np.zeros((rows, H))
    for r, c in enumerate(ctxn):
        c = max(c, 0)
        for i in range(nodes):
            toks = visible(c, m2[r][i] & (2**64 - 1), nodes, btn.shape[1] * page)
            if not toks:
                continue
            k, div = keys_of(cache, btn[r], toks, page, qk, H, rms_offset, mode, fp8, k_scale)
            s, mag = scores64(q64[r * nodes + i, :, :qk], k, div, sm_scale, cap)
            m = s.max(axis=0)
            p = np.exp(s - m)
            den = p.sum(axis=0)
            p /= den
            v = k[:, :rank]
            row = r * nodes + i
            o[row] = p.T @ v
            lse[row] = m + np.log(den)
            ds = mag.max(axis=0) * 2.0**-19 + 1e-6 * (1 + np.abs(s).max(axis=0))  # error of a score
            vm = p.T @ np.abs(v)
            tol[row] = (2.0**-8 + 2 * ds[:, None]) * vm + 1e-6 * vm
            if fp8:  # weights under 2^-15 of the largest keep 3 bits; under 2^-24 none
                w = p * den
                small = np.where(w < 2.0**-15, p, 0.0).T @ np.abs(v)
                lost = np.where(w < 2.0**-23, p, 0.0).T @ np.abs(v)
                tol[row] += 2.0**-4 * small + lost
            ltol[row] = ds + 2e-6 * (1 + np.abs(lse[row]))
    return o, lse, tol, ltol


def fp8_cache(reqs, heads, rank, rope, page, lens, mode, seed, dev):
    """gpu_util.make_fp8_case's cache; without rope columns (which it does not take) the same recipe."""
    if rope:
        cache, _, bt, _, ks = make_fp8_case(reqs, heads, rank, rope, page, lens, mode=mode, seed=seed, device=dev)
        return cache, bt, ks
    g = torch.Generator().manual_seed(seed)
    pps = max(1, max(-(-x // page) for x in lens))
    n = (reqs * pps + 3) * page
    lat = oracle.bf16_round((torch.randn(n, rank, generator=g) * 2.0).numpy())
    rms = oracle.bf16_round(torch.exp(torch.randn(n, heads, generator=g) * 0.6).numpy())
    ks = float(np.abs(lat).max()) / 448
    rows = oracle.fp8_cache_rows(lat, rms, ks, 0, heads, "log8" if mode == "e4m3" else mode)
    if mode == "e4m3":
        rows = np.concatenate([rows[:, :rank], oracle.e4m3_encode(np.clip(rms / np.float32(ks), -448, 448))], axis=1)
    buf = np.zeros((n, rows.shape[1] + (-rows.shape[1]) % 16), np.uint8)
    buf[:, :rows.shape[1]] = rows
    cache = torch.from_numpy(buf.reshape(-1, page, 1, buf.shape[1])).to(dev).view(torch.float8_e4m3fn)
    return cache, torch.randperm(reqs * pps, generator=g).reshape(reqs, pps).to(torch.int32).to(dev), ks


def build_case(dev, reqs, nodes, heads, rank, rope, page, ctxs, *, mode="native", fp8=False, seed=0, q_scale=16.0):
    """A cache with the committed and drafted rows of every request, and queries whose scores spread over several units."""
    lens = [max(c, 0) + nodes for c in ctxs]
    if fp8:
        cache, bt, ks = fp8_cache(reqs, heads, rank, rope, page, lens, mode, seed, dev)
    else:
        cache, _, bt, _ = make_bf16_case(reqs, heads, rank, rope, page, lens, seed=seed, device=dev)
        ks = 1.0
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(reqs * nodes, heads, rank + rope, generator=g) * q_scale / math.sqrt(rank + rope)).to(torch.bfloat16).to(dev)
    return cache, q, bt, torch.tensor(ctxs, dtype=torch.int32, device=dev), ks


def random_parents(reqs, nodes, seed=0):
    g = np.random.RandomState(seed)
    return torch.tensor([[-1 if i == 0 or g.rand() < 0.1 else int(g.randint(max(0, i - 5), i)) for i in range(nodes)] for _ in range(reqs)])
