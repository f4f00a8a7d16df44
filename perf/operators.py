"""Cases and plain forms of the operators around speculative decoding over a bounded latent cache.

Five operators of one serving loop over the paged MLA / GLA latent cache
(row = [latent | rope | rms tail], bf16 or FP8 e4m3):

  rotary       rotary positions applied to (part of) each head, and their adjoint (the gradient)
  rope_update  a step's new tokens: rotate q and the packed rope keys, write the paged cache rows
  tree         attention of a tree of drafted tokens over the cache
  weights      accumulated attention weight of every cached token
  evict        keep each request's heaviest tokens, close the holes in the cache

``run`` computes them with elementary torch operations in 32 bits, or (``own``) through
``qwen_mla_vllm_b200``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
SM_SCALE = 1.0 / 16.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SINKS = 4


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one verify step of 8 requests x 8 drafted tokens: rotate one 58-wide group of every head
        {"name": "rotary decode", "op": "rotary", "tokens": 64, "heads": 24, "dim": 256, "rot": 58, "start": 198,
         "interleaved": False, "adjoint": False, "dtype": "bf16", "maxpos": 131072},
        # a long prefill's queries, whole heads, pairs side by side, and the gradient's direction
        {"name": "rotary prefill adjoint", "op": "rotary", "tokens": 32768, "heads": 24, "dim": 128, "rot": 128,
         "start": 0, "interleaved": True, "adjoint": True, "dtype": "bf16", "maxpos": 262144},
        # one token of each of 64 requests, bf16 cache (the plugin's tp1 row)
        {"name": "rope update decode bf16", "op": "rope_update", "tokens": 64, "heads": 24, "rank": 768, "groups": 4,
         "rot": 58, "interleaved": False, "page": 16, "fp8": False, "maxpos": 32768},
        # a prefill chunk into an FP8 cache with log2-coded score divisors
        {"name": "rope update prefill fp8", "op": "rope_update", "tokens": 16384, "heads": 24, "rank": 768, "groups": 4,
         "rot": 58, "interleaved": False, "page": 16, "fp8": True, "maxpos": 262144},
        # a single chat request: a chain of 4 drafts over a short context (latency)
        {"name": "tree one request", "op": "tree", "reqs": 1, "nodes": 4, "lo": 517, "hi": 517, "lens_seed": 1,
         "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": False},
        # ordinary serving: 16 requests, 8 drafted nodes each, mixed contexts
        {"name": "tree 16x8 bf16", "op": "tree", "reqs": 16, "nodes": 8, "lo": 1024, "hi": 32768, "lens_seed": 2,
         "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": False},
        # wide trees over an FP8 cache
        {"name": "tree 8x16 fp8", "op": "tree", "reqs": 8, "nodes": 16, "lo": 8192, "hi": 32768, "lens_seed": 3,
         "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": True},
        # one GLA head group (12 heads, rank 384) of a batch with long contexts
        {"name": "tree gla 16x4", "op": "tree", "reqs": 16, "nodes": 4, "lo": 4096, "hi": 65536, "lens_seed": 4,
         "heads": 12, "rank": 384, "rope": 116, "page": 16, "fp8": False},
        # every decoded token adds its attention weights: the decode benchmark's batch
        {"name": "weights 64 bf16", "op": "weights", "reqs": 64, "qrows": 1, "lo": 1024, "hi": 32768, "lens_seed": 1,
         "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": False, "decay": 0.95},
        # four verified tokens at once over an FP8 cache
        {"name": "weights 16x4 fp8", "op": "weights", "reqs": 16, "qrows": 4, "lo": 8192, "hi": 8192, "lens_seed": 5,
         "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": True, "decay": 1.0},
        # a small batch that passed its budget a little
        {"name": "evict 4 small", "op": "evict", "reqs": 4, "lo": 1100, "hi": 2048, "lens_seed": 6, "budget": 1024,
         "recent": 64, "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": False},
        # long contexts cut back to a quarter
        {"name": "evict 16 long", "op": "evict", "reqs": 16, "lo": 16384, "hi": 65536, "lens_seed": 7, "budget": 12288,
         "recent": 1024, "heads": 24, "rank": 768, "rope": 232, "page": 16, "fp8": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rope_update", "tree", "weights", "evict"])
    if op == "rotary":
        heads = rng.choice([1, 3, 8, 12, 24, 32])
        dim = rng.choice([58, 64, 96, 128, 192, 256])
        rot = min(dim, rng.choice([32, 58, 64, 128]))
        tokens = max(1, min(_log(rng, 1, 60000), 32768 * 24 * 128 // (heads * dim)))
        return {"op": op, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot,
                "start": 2 * rng.randint(0, (dim - rot) // 2), "interleaved": rng.random() < 0.5,
                "adjoint": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "maxpos": rng.choice([4096, 131072, 1048576])}
    heads, rank, groups = rng.choice([(24, 768, 4), (12, 768, 2), (24, 256, 4), (12, 384, 2), (6, 512, 1)])
    fp8 = rng.random() < 0.5
    if op == "rope_update":
        return {"op": op, "tokens": _log(rng, 1, 16000), "heads": heads, "rank": rank, "groups": groups, "rot": 58,
                "interleaved": rng.random() < 0.5, "page": rng.choice([16, 32, 64]), "fp8": fp8,
                "maxpos": rng.choice([4096, 262144])}
    base = {"lens_seed": rng.randint(1, 10**6), "heads": heads, "rank": rank, "rope": 58 * groups,
            "page": rng.choice([16, 32, 64]), "fp8": fp8}
    if op == "tree":
        nodes = rng.choice([1, 2, 3, 5, 7, 8, 13, 16, 24, 32])
        hi = _log(rng, 40, 32768)
        # rows x tokens no more than those of the 8 x 16 case
        reqs = max(1, min(_log(rng, 1, 48), 8 * 16 * 24 * 20480 // (nodes * heads * hi)))
        nodes = max(1, min(nodes, 8 * 16 * 24 * 20480 // (reqs * heads * hi)))
        return {"op": op, "reqs": reqs, "nodes": nodes, "lo": max(1, hi // rng.choice([1, 2, 8])), "hi": hi, **base}
    hi = _log(rng, 60, 65536)
    reqs = max(1, min(_log(rng, 1, 64), 64 * 16384 // hi))
    lo = max(1, hi // rng.choice([1, 2, 8]))
    if op == "weights":
        return {"op": op, "reqs": reqs, "qrows": rng.choice([1, 1, 2, 3, 4]), "lo": max(lo, 8), "hi": hi,
                "decay": rng.choice([1.0, 0.9]), **base}
    reqs = max(1, min(reqs, 16 * 40000 // hi))
    return {"op": op, "reqs": reqs, "lo": lo, "hi": hi, "budget": max(1, int(hi * rng.choice([0.1, 0.25, 0.5, 0.9]))),
            "recent": rng.choice([0, 16, 32]), **base}


# ------------------------------------------------------------------ what a case holds
def _lens(c):
    r = random.Random(c["lens_seed"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["reqs"])]


def _row(c):
    """(elements of the QK part, elements a row uses, row width) of a cache row."""
    qk = c["rank"] + (c["rope"] if "rope" in c else c["groups"] * c["rot"])
    used = qk + c["heads"]
    return qk, used, used + (-used) % 16


def work(case):
    c = case
    op = c["op"]
    if op == "rotary":
        es = 4 if c["dtype"] == "f32" else 2
        n = c["tokens"] * c["heads"]
        # in place would leave the other dims alone; a new output holds all of them
        return {"bytes": 2 * es * n * c["dim"] + 8 * c["tokens"], "flops": 3 * n * c["rot"]}
    es = 1 if c["fp8"] else 2
    qk, used, width = _row(c)
    if op == "rope_update":
        win = c["groups"] * c["rot"]
        n = c["tokens"]
        return {"bytes": n * (2 * 2 * c["heads"] * win + 2 * used + es * used + 16),
                "flops": 3 * n * win * (c["heads"] + 1)}
    lens = _lens(c)
    if op == "tree":
        rows = c["nodes"] * c["heads"]
        toks = sum(x + c["nodes"] for x in lens)
        return {"bytes": toks * used * es + len(lens) * rows * 2 * (qk + c["rank"] + 2) + 4 * toks // c["page"],
                "flops": 2 * toks * rows * (qk + c["rank"])}
    if op == "weights":
        rows = c["qrows"] * c["heads"]
        toks = sum(lens)
        return {"bytes": toks * (used * es + 8) + len(lens) * rows * (2 * qk + 4), "flops": 2 * toks * rows * qk}
    moved = sum(k * (x - k) // x for x, k in ((x, min(x, c["budget"])) for x in lens))
    kept = sum(min(x, c["budget"]) for x in lens)
    return {"bytes": 2 * moved * width * es + 4 * sum(lens) * 2 + 8 * kept, "flops": sum(lens)}


def _steps(rot, base=1.0e6):
    """Turns a position advances each pair by, in units of 2^-64 (as signed 64-bit numbers)."""
    out = []
    for i in range(rot // 2):
        v = int(round(base ** (-2.0 * i / rot) / (2.0 * math.pi) * 2.0**64))
        out.append(v - 2**64 if v >= 2**63 else v)
    return out


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _positions(n, maxpos, g):
    start = torch.randint(0, max(1, maxpos - 1), (max(1, -(-n // 4096)),), generator=g, device=DEV)
    pos = (start[:, None] + torch.arange(4096, device=DEV)[None, :]).reshape(-1)[:n]
    return (pos % maxpos).contiguous()


def _cache(c, toks, g):
    """A paged cache with room for toks tokens per request, its block table and k_scale."""
    qk, used, width = _row(c)
    page, R = c["page"], c["reqs"]
    pps = -(-toks // page)
    P = R * pps
    if c["fp8"]:
        scale = 4.5 * 2.0 / 448.0
        cache = torch.zeros(P, page, 1, width, dtype=torch.uint8, device=DEV)
        for p0 in range(0, P, 4096):
            n = min(4096, P - p0)
            x = torch.randn(n, page, qk, generator=g, device=DEV) * 2.0
            cache[p0:p0 + n, :, 0, :qk] = (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            code = ((torch.randn(n, page, c["heads"], generator=g, device=DEV) * 0.6 / math.log(2) + 3) * 255 / 6)
            cache[p0:p0 + n, :, 0, qk:used] = code.round().clamp(0, 255).to(torch.uint8)
        cache = cache.view(torch.float8_e4m3fn)
        k_scale = torch.full((), scale, dtype=F32, device=DEV)
    else:
        cache = torch.empty(P, page, 1, width, dtype=torch.bfloat16, device=DEV)
        cache.normal_(generator=g)
        cache[..., qk:] = (torch.rand(P, page, 1, width - qk, generator=g, device=DEV) * 1.5 + 0.5).to(torch.bfloat16)
        k_scale = None
    bt = torch.randperm(P, generator=g, device=DEV).reshape(R, pps).to(torch.int32)
    return cache, bt, k_scale


def _parents(n, r):
    """A drafted tree in depth order: node 0 is the root, later nodes hang from earlier ones."""
    return [-1] + [r.randint(max(0, i - 4), i - 1) for i in range(1, n)]


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    op = c["op"]
    s = {"c": c}
    if op == "rotary":
        s["x"] = torch.randn(c["tokens"], c["heads"], c["dim"], generator=g, device=DEV).to(DTYPES[c["dtype"]])
        s["pos"] = _positions(c["tokens"], c["maxpos"], g)
        s["steps"] = torch.tensor(_steps(c["rot"]), dtype=torch.int64, device=DEV)
        return s
    qk, used, width = _row(c)
    if op == "rope_update":
        n, page, win = c["tokens"], c["page"], c["groups"] * c["rot"]
        P = -(-n // page)
        s["q_pe"] = torch.randn(n, c["heads"], win, generator=g, device=DEV).to(torch.bfloat16)
        s["latent"] = torch.randn(n, c["rank"], generator=g, device=DEV).to(torch.bfloat16)
        rms = torch.exp(torch.randn(n, c["heads"], generator=g, device=DEV) * 0.4)
        s["k_pe"] = torch.cat([torch.randn(n, win, generator=g, device=DEV), rms], dim=1).to(torch.bfloat16)
        s["pos"] = _positions(n, c["maxpos"], g)
        s["slots"] = torch.randperm(P * page, generator=g, device=DEV)[:n].contiguous()
        s["steps"] = torch.tensor(_steps(c["rot"]), dtype=torch.int64, device=DEV)
        s["cache"] = torch.zeros(P, page, 1, width, dtype=torch.uint8 if c["fp8"] else torch.bfloat16, device=DEV)
        s["k_scale"] = torch.full((), 4.5 / 448.0, dtype=F32, device=DEV) if c["fp8"] else None
        s["q_out"] = torch.empty_like(s["q_pe"])
        return s
    lens = _lens(c)
    extra = c.get("nodes", 0)
    toks = max(lens) + extra
    s["cache"], s["bt"], s["k_scale"] = _cache(c, toks, g)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    R = c["reqs"]
    if op == "evict":
        # attention mass falls off steeply: most of it sits on a few tokens
        w = torch.exp(torch.randn(R, toks, generator=g, device=DEV) * 2.0)
        live = torch.arange(toks, device=DEV)[None, :] < s["lens"][:, None]
        s["weights"] = torch.where(live, w, torch.zeros_like(w))
        s["positions"] = torch.arange(toks, dtype=torch.int32, device=DEV).repeat(R, 1)
        s["recent_from"] = (s["lens"] - c["recent"]).to(torch.int32)
        return s
    rows = c["nodes"] if op == "tree" else c["qrows"]
    s["q"] = torch.randn(R * rows, c["heads"], qk, generator=g, device=DEV).to(torch.bfloat16)
    if op == "tree":
        r = random.Random(seed)
        mask = []
        for _ in range(R):
            m = []
            for i, p in enumerate(_parents(c["nodes"], r)):
                m.append((m[p] if p >= 0 else 0) | (1 << i))
            mask.append([v - 2**64 if v >= 2**63 else v for v in m])
        s["mask"] = torch.tensor(mask, dtype=torch.int64, device=DEV)
        s["o"] = torch.empty(R * rows, c["heads"], c["rank"], dtype=torch.bfloat16, device=DEV)
        s["lse"] = torch.empty(R * rows, c["heads"], dtype=F32, device=DEV)
        return s
    # verified tokens are causal: row j of a request sees len - (qrows - 1 - j) tokens
    back = torch.arange(1 - rows, 1, dtype=torch.int32, device=DEV)
    s["row_lens"] = (s["lens"][:, None] + back[None, :]).reshape(-1).contiguous()
    s["weights"] = torch.rand(R, toks, generator=g, device=DEV)
    s["weights"] *= (torch.arange(toks, device=DEV)[None, :] < s["lens"][:, None])
    # the log-sum-exp that the decode of these rows returned
    lse = [torch.logsumexp(_scores(c, s, F32, slice(i, i + 1)), dim=-1) for i in range(R)]
    s["lse"] = torch.cat(lse).reshape(R * rows, c["heads"]).contiguous()
    return s


# ------------------------------------------------------------------ plain forms (32 bits)
def _rotate(x, pos, steps, interleaved, adjoint, start, rot):
    """x [tokens, heads, dim] in 32 bits with dims [start, start + rot) rotated by pos."""
    turns = ((pos[:, None] * steps[None, :]) >> 32).to(F32) * 2.0**-32
    ang = turns * (2.0 * math.pi)
    cos, sin = torch.cos(ang)[:, None, :], torch.sin(ang)[:, None, :]
    if adjoint:
        sin = -sin
    w = x[..., start:start + rot]
    a, b = (w[..., 0::2], w[..., 1::2]) if interleaved else (w[..., :rot // 2], w[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    w = torch.stack([ra, rb], dim=-1).flatten(-2) if interleaved else torch.cat([ra, rb], dim=-1)
    return torch.cat([x[..., :start], w, x[..., start + rot:]], dim=-1)


def _log8(x):
    return ((torch.log2(x) + 3.0) * (255.0 / 6.0)).round().clamp(0, 255).to(torch.uint8)


def _rows(c, s, dt, reqs):
    """The cached rows of some requests: keys [n, T, qk], score divisors [n, T, heads] in dt."""
    qk, used, _ = _row(c)
    raw = s["cache"][s["bt"][reqs].long()]  # [n, pages, page, 1, width]
    raw = raw.reshape(raw.shape[0], -1, raw.shape[-1])
    if c["fp8"]:
        k = raw[..., :qk].to(dt) * s["k_scale"].to(dt)
        rms = torch.exp2(raw[..., qk:used].view(torch.uint8).to(dt) * (6.0 / 255.0) - 3.0)
    else:
        k, rms = raw[..., :qk].to(dt), raw[..., qk:used].to(dt)
    return k, rms


def _scores(c, s, dt, reqs, keys=None):
    """Scaled scores [n, rows, heads, T] with -inf where a row does not see a token."""
    k, rms = _rows(c, s, dt, reqs) if keys is None else keys
    n, T = k.shape[0], k.shape[1]
    rows = s["q"].shape[0] // c["reqs"]
    q = s["q"].reshape(c["reqs"], rows * c["heads"], -1)[reqs].to(dt)
    x = torch.matmul(q, k.transpose(1, 2)).reshape(n, rows, c["heads"], T)
    x = x / rms.transpose(1, 2)[:, None] * SM_SCALE
    t = torch.arange(T, device=DEV)
    if c["op"] == "tree":
        j = t[None, :] - s["lens"][reqs][:, None].long()  # drafted token's number, or negative
        bit = (s["mask"][reqs][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
        see = (j < 0)[:, None, :] | ((j < c["nodes"])[:, None, :] & (bit == 1))
    else:
        see = t[None, None, :] < s["row_lens"].reshape(c["reqs"], rows)[reqs][:, :, None]
    return torch.where(see[:, :, None, :], x, torch.full_like(x, float("-inf")))


def _plain(s):
    c = s["c"]
    op = c["op"]
    if op == "rotary":
        return _rotate(s["x"].to(F32), s["pos"], s["steps"], c["interleaved"], c["adjoint"], c["start"],
                       c["rot"]).to(s["x"].dtype)
    if op == "rope_update":
        qk, used, width = _row(c)
        win, rank = c["groups"] * c["rot"], c["rank"]
        n = c["tokens"]

        def window(x):  # [n, heads, groups * rot]: every group's rot dims turn alike
            y = x.to(F32).reshape(n, -1, c["rot"])
            return _rotate(y, s["pos"], s["steps"], c["interleaved"], False, 0, c["rot"]).reshape(x.shape)

        s["q_out"].copy_(window(s["q_pe"]))
        kr = window(s["k_pe"][:, None, :win])[:, 0]
        flat = s["cache"].view(-1, width)
        if c["fp8"]:
            x = torch.cat([s["latent"].to(F32), kr], dim=1) * (1.0 / s["k_scale"])
            b = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            flat[s["slots"], :used] = torch.cat([b, _log8(s["k_pe"][:, win:].to(F32))], dim=1)
        else:
            flat[s["slots"], :used] = torch.cat([s["latent"], kr.to(torch.bfloat16), s["k_pe"][:, win:]], dim=1)
        return _update_out(s)
    if op == "tree":
        keys = _rows(c, s, F32, slice(None))
        x = _scores(c, s, F32, slice(None), keys)
        n, rows, H, T = x.shape
        x = x.reshape(n, rows * H, T)
        m = x.amax(dim=-1, keepdim=True)
        p = torch.exp(x - m)
        den = p.sum(dim=-1, keepdim=True)
        o = torch.matmul(p, keys[0][..., :c["rank"]]) / den
        s["o"].copy_(o.reshape(s["o"].shape))
        s["lse"].copy_((m + torch.log(den)).reshape(s["lse"].shape))
        return {"o": s["o"], "lse": s["lse"]}
    if op == "weights":
        x = _scores(c, s, F32, slice(None))
        p = torch.exp(x - s["lse"].reshape(c["reqs"], c["qrows"], c["heads"], 1)).sum(dim=(1, 2))
        n = s["weights"].shape[1]
        s["weights"].copy_(s["weights"] * c["decay"] + p[:, :n])
        return s["weights"]
    return _evict_plain(s)


def _evict_plain(s):
    c = s["c"]
    R, n = s["weights"].shape
    K = c["budget"]
    t = torch.arange(n, device=DEV)
    lens = s["lens"].long()
    live = t[None, :] < lens[:, None]
    new_lens = torch.clamp(lens, max=K)
    held = (s["positions"] < SINKS) | (s["positions"] >= s["recent_from"][:, None])
    score = torch.where(held, torch.full_like(s["weights"], float("inf")), s["weights"])
    score = torch.where(live, score, torch.full_like(score, float("-inf")))
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    keep = torch.zeros(R, n, dtype=torch.bool, device=DEV)
    keep.scatter_(1, order, t[None, :].expand(R, n) < new_lens[:, None])
    front = t[None, :] < new_lens[:, None]
    hole, mover = front & ~keep, keep & ~front
    src = t[None, :].expand(R, n).clone()  # the token that ends up in each place
    at = torch.nonzero(hole)
    frm = torch.nonzero(mover)  # as many in each request, both ascending
    src[at[:, 0], at[:, 1]] = frm[:, 1]
    m = min(K, n)
    keepm = front[:, :m]
    new_w = torch.where(keepm, torch.gather(s["weights"], 1, src)[:, :m], torch.zeros_like(s["weights"][:, :m]))
    new_p = torch.where(keepm, torch.gather(s["positions"], 1, src)[:, :m], torch.full_like(s["positions"][:, :m], -1))
    page = c["page"]
    flat = s["cache"].view(torch.uint8).view(-1, s["cache"].view(torch.uint8).shape[-1])
    slot = lambda i: s["bt"][i[:, 0], i[:, 1] // page].long() * page + i[:, 1] % page  # noqa: E731
    flat[slot(at)] = flat[slot(frm)]
    return _evict_out(s, new_w, new_p, new_lens.to(torch.int32))


def _evict_out(s, w, p, lens):
    c = s["cache"] if not s["c"]["fp8"] else s["cache"].view(torch.uint8)
    return {"cache": c, "weights": w, "positions": p, "lens": lens}


def _update_out(s):
    c = s["c"]
    qk, used, _ = _row(c)
    if c["fp8"]:
        return {"q": s["q_out"], "kv": s["cache"][..., :qk].view(torch.float8_e4m3fn), "rms": s["cache"][..., qk:used]}
    return {"q": s["q_out"], "kv": s["cache"][..., :used]}


# ------------------------------------------------------------------ the framework's operators
def _own(s):
    c = s["c"]
    op = c["op"]
    if op == "rotary":
        from qwen_mla_vllm_b200.rotary import rotary_embed
        return rotary_embed(s["x"], s["pos"], s["steps"], start=c["start"], interleaved=c["interleaved"],
                            adjoint=c["adjoint"])
    qk, _, _ = _row(c)
    if op == "rope_update":
        from qwen_mla_vllm_b200.rotary import rope_kv_cache_update
        rope_kv_cache_update(s["q_pe"], s["k_pe"], s["latent"], s["pos"], s["slots"], s["steps"], s["cache"],
                             packed_rope=c["groups"] * c["rot"], local_heads=c["heads"], q_out=s["q_out"],
                             interleaved=c["interleaved"], k_scale=s["k_scale"],
                             rms_mode="log8" if c["fp8"] else "native")
        return _update_out(s)
    kind = {"rms_offset": qk, "rms_log8": c["fp8"], "page_size": c["page"]}
    if op == "tree":
        from qwen_mla_vllm_b200.tree_attention import tree_attention
        tree_attention(s["q"], s["cache"], s["o"], s["lse"], s["bt"], s["lens"], s["mask"], rank=c["rank"],
                       sm_scale=SM_SCALE, k_scale=s["k_scale"], **kind)
        return {"o": s["o"], "lse": s["lse"]}
    if op == "weights":
        from qwen_mla_vllm_b200.cache_eviction import accumulate_attention_weights
        accumulate_attention_weights(s["q"], s["cache"], s["weights"], s["lse"], s["bt"], s["row_lens"],
                                     sm_scale=SM_SCALE, k_scale=s["k_scale"], decay=c["decay"], qrows=c["qrows"], **kind)
        return s["weights"]
    from qwen_mla_vllm_b200.cache_eviction import evict_cache
    w, p, lens = evict_cache(s["cache"], s["weights"], s["positions"], s["bt"], s["lens"], min(c["budget"], s["weights"].shape[1]),
                             page_size=c["page"], sinks=SINKS, recent_from=s["recent_from"])
    return _evict_out(s, w, p, lens)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ 64 bits
def _turn64(x, pos, rot, interleaved, sign):
    """Rotary of x [n, ..., rot] straight from its definition: pair i turns by pos * base^(-2i/rot)."""
    i = torch.arange(rot // 2, dtype=F64, device=DEV)
    ang = pos.to(F64)[:, None] * torch.pow(torch.full_like(i, 1.0e6), -2.0 * i / rot)
    z = torch.polar(torch.ones_like(ang), sign * ang)
    z = z.reshape(z.shape[0], *([1] * (x.dim() - 2)), z.shape[1])
    x = x.to(F64)
    pairs = x.unflatten(-1, (rot // 2, 2)) if interleaved else x.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    return (y if interleaved else y.transpose(-1, -2)).reshape(x.shape)


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    op = c["op"]
    if op == "rotary":
        y = s["x"].to(F64)
        a, b = c["start"], c["start"] + c["rot"]
        y[..., a:b] = _turn64(s["x"][..., a:b], s["pos"], c["rot"], c["interleaved"], -1.0 if c["adjoint"] else 1.0)
        return y
    qk, used, width = _row(c)
    if op == "rope_update":
        win, n = c["groups"] * c["rot"], c["tokens"]
        turn = lambda x: _turn64(x.unflatten(-1, (c["groups"], c["rot"])), s["pos"], c["rot"],  # noqa: E731
                                 c["interleaved"], 1.0).flatten(-2)
        q, k = turn(s["q_pe"]), turn(s["k_pe"][:, :win])
        total = s["cache"].shape[0] * c["page"]
        tail = [] if c["fp8"] else [s["k_pe"][:, win:].to(F64)]
        rows = torch.cat([s["latent"].to(F64), k] + tail, dim=1)
        kv = torch.zeros(total, rows.shape[1], dtype=F64, device=DEV)
        kv[s["slots"]] = rows / s["k_scale"].to(F64) if c["fp8"] else rows
        kv = kv.reshape(-1, c["page"], 1, rows.shape[1])
        return {"q": q, "kv": kv, "rms": None} if c["fp8"] else {"q": q, "kv": kv}
    if op == "evict":
        return None  # rows are moved, not computed
    lens = _lens(c)
    H, T = c["heads"], s["bt"].shape[1] * c["page"]
    rows = c["nodes"] if op == "tree" else c["qrows"]
    outs, lses = [], []
    w = s["weights"].to(F64) * c["decay"] if op == "weights" else None
    for r, L in enumerate(lens):
        n = L + c.get("nodes", 0)
        t = torch.arange(n, device=DEV)
        raw = s["cache"][s["bt"][r].long()[t // c["page"]], t % c["page"], 0]
        if c["fp8"]:
            k = raw[:, :qk].to(F64) * float(s["k_scale"])
            div = 2.0 ** (raw[:, qk:used].view(torch.uint8).to(F64) * 6.0 / 255.0 - 3.0)
        else:
            k, div = raw[:, :qk].to(F64), raw[:, qk:used].to(F64)
        for j in range(rows):
            q = s["q"][r * rows + j].to(F64)  # [H, qk]
            if op == "tree":
                m = int(s["mask"][r, j]) & (2**64 - 1)
                seen = torch.cat([torch.arange(L, device=DEV),
                                  torch.tensor([L + b for b in range(c["nodes"]) if m >> b & 1], device=DEV).long()])
            else:
                seen = torch.arange(max(0, L - (rows - 1 - j)), device=DEV)
            ks = k if len(seen) == n else k[seen]
            x = (ks @ q.T) / (div if len(seen) == n else div[seen]) * SM_SCALE  # [seen, H]
            if op == "tree":
                lse = torch.logsumexp(x, dim=0)
                outs.append(torch.exp(x - lse).T @ ks[:, :c["rank"]])
                lses.append(lse)
            else:
                w[r, seen] += torch.exp(x - s["lse"][r * rows + j].to(F64)).sum(dim=1)
    if op == "tree":
        return {"o": torch.stack(outs), "lse": torch.stack(lses)}
    return w
