"""A bounded latent cache: accumulated attention weight of every cached token, and eviction by it.

``accumulate_attention_weights`` adds, after a decode, what each cached token drew of the step's
attention; ``evict_cache`` keeps a request's heaviest tokens (with its first and its most recent ones)
and closes up its pages.  The plugin has no counterpart: its cache only grows
(``qwen_mla/mla_impl.py:309-342`` writes rows, nothing removes them).
"""
from __future__ import annotations

import torch

from . import _lib
from .mla_decode_attention import _FP8_TYPES, _dt, rms_mode_for
from .tree_attention import run_with_workspace, workspace_bytes

_PACK_WEIGHTS = _lib.packer(_lib.WeightsParams)
_PACK_EVICT = _lib.packer(_lib.EvictParams)


def accumulate_attention_weights(q: torch.Tensor, kv_cache: torch.Tensor, weights: torch.Tensor, lse: torch.Tensor,
                                 block_table: torch.Tensor, seq_lens: torch.Tensor, *, sm_scale: float, page_size: int,
                                 rank: int | None = None, rms_offset: int = -1, rms_bf16: bool = False,
                                 rms_log8: bool = False, qk_dim: int | None = None, logit_cap: float = 0.0,
                                 k_scale: torch.Tensor | None = None, q_pe: torch.Tensor | None = None, qrows: int = 1,
                                 decay: float = 1.0, workspace: torch.Tensor | None = None) -> None:
    """``weights[r, t] = decay * weights[r, t] + sum of request r's softmax weights on token t``, in place.

    q [reqs * qrows, heads, >= qk_dim] bf16 or f16 and seq_lens [reqs * qrows] int32 are the decode's
    flattened rows (``qrows`` of one request side by side), lse [reqs * qrows, heads] fp32 what it
    returned for them; block_table [reqs, cols] int32.  weights [reqs, columns] fp32: columns at or
    past a request's longest row are left alone.  ``rank`` is needed with a separate ``q_pe`` only
    (the width of q's latent part).  The row format flags are ``decode_attention_fwd``'s; ``workspace`` is
    as ``tree_attention``'s (``accumulate_attention_weights_workspace_bytes``).
    """
    args = _weights_args(q, kv_cache, weights, lse, block_table, seq_lens, sm_scale=sm_scale, page_size=page_size,
                         rank=rank, rms_offset=rms_offset, rms_bf16=rms_bf16, rms_log8=rms_log8, qk_dim=qk_dim,
                         logit_cap=logit_cap, k_scale=k_scale, q_pe=q_pe, qrows=qrows, decay=decay)
    if args is not None:
        run_with_workspace("qmla_accumulate_weights", _PACK_WEIGHTS.pack, args, q.device, workspace)


def accumulate_attention_weights_workspace_bytes(q: torch.Tensor, kv_cache: torch.Tensor, weights: torch.Tensor,
                                                 lse: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                                                 page_size: int, **how) -> int:
    """Bytes of ``workspace`` that ``accumulate_attention_weights`` of these arguments needs (shapes and
    types count, not what the tensors hold)."""
    how.setdefault("sm_scale", 1.0)
    args = _weights_args(q, kv_cache, weights, lse, block_table, seq_lens, page_size=page_size, **how)
    return 0 if args is None else workspace_bytes("qmla_accumulate_weights", _PACK_WEIGHTS.pack, args, q.device)


def _weights_args(q, kv_cache, weights, lse, block_table, seq_lens, *, sm_scale, page_size, rank=None, rms_offset=-1,
                  rms_bf16=False, rms_log8=False, qk_dim=None, logit_cap=0.0, k_scale=None, q_pe=None, qrows=1,
                  decay=1.0) -> tuple | None:
    """The checked call as qmla_weights_params' fields up to the workspace; None when there is nothing to do."""
    if not all(t.is_cuda for t in (q, kv_cache, weights, lse, block_table, seq_lens)):
        raise ValueError("accumulate_attention_weights: all tensors must be CUDA tensors")
    if any(t is not None and t.device != q.device for t in (kv_cache, weights, lse, block_table, seq_lens, k_scale, q_pe)):
        raise ValueError("accumulate_attention_weights: all tensors must be on one device")
    fp8 = kv_cache.dtype in _FP8_TYPES or kv_cache.dtype == torch.uint8
    if not fp8 and kv_cache.dtype != torch.bfloat16:
        raise TypeError(f"cache dtype {kv_cache.dtype} not supported (bf16 or float8_e4m3fn)")
    if kv_cache.dim() != 4 or kv_cache.shape[2] != 1 or kv_cache.shape[1] != page_size or kv_cache.stride(3) != 1:
        raise ValueError(f"kv_cache must be [pages, {page_size}, 1, width], got {tuple(kv_cache.shape)}")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_table and seq_lens must be int32")
    if weights.dtype != torch.float32 or lse.dtype != torch.float32:
        raise TypeError("weights and lse must be fp32")
    if qrows < 1 or q.dim() != 3 or q.shape[0] % qrows or weights.dim() != 2 or weights.shape[0] * qrows != q.shape[0]:
        raise ValueError(f"q must have {qrows} rows for each of weights' {weights.shape[0]} requests, got {tuple(q.shape)}")
    reqs, heads, width = weights.shape[0], q.shape[1], kv_cache.shape[3]
    qk = qk_dim if qk_dim is not None else (rms_offset if rms_offset >= 0 else width)
    if q_pe is not None and rank is None:
        raise ValueError("a separate q_pe needs rank")
    lat = rank if q_pe is not None else qk
    if q.shape[2] < lat or q_pe is not None and (q_pe.shape[:2] != q.shape[:2] or q_pe.shape[2] < qk - lat or q_pe.dtype != q.dtype):
        raise ValueError(f"q (and q_pe) do not hold {qk} dims")
    if lse.shape != (q.shape[0], heads) or seq_lens.shape != (q.shape[0],):
        raise ValueError(f"lse must be [{q.shape[0]}, {heads}] and seq_lens [{q.shape[0]}]")
    if block_table.dim() != 2 or block_table.shape[0] < reqs:
        raise ValueError(f"block_table must have {reqs} rows, got {tuple(block_table.shape)}")
    if any(t is not None and t.numel() and t.stride(-1) != 1 for t in (q, q_pe, weights, lse, block_table, seq_lens)):
        raise ValueError("q, q_pe, weights, lse, block_table and seq_lens need a unit stride on the last dim")
    if k_scale is not None and k_scale.dtype != torch.float32:
        raise TypeError("k_scale must be an fp32 device scalar")
    if reqs == 0 or heads == 0:
        return None
    pe = q_pe if q_pe is not None else q
    mode = rms_mode_for(kv_cache.dtype, rms_offset, rms_bf16, rms_log8)
    return (
        q.data_ptr(), q.stride(0), q.stride(1),
        pe.data_ptr() if q_pe is not None else q.data_ptr() + lat * q.element_size(), pe.stride(0), pe.stride(1),
        _dt(q), kv_cache.data_ptr(), kv_cache.stride(0), kv_cache.stride(1), kv_cache.shape[0], width,
        _lib.DT_FP8E4M3 if fp8 else _lib.DT_BF16, page_size, block_table.data_ptr(), block_table.stride(0),
        block_table.shape[1], seq_lens.data_ptr(), reqs, qrows, heads, lat, qk, rms_offset, mode, sm_scale,
        logit_cap or 0.0, decay, k_scale.data_ptr() if k_scale is not None else 0, lse.data_ptr(), lse.stride(0),
        weights.data_ptr(), weights.stride(0), weights.shape[1])


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two vectors or matrices with dense rows have a byte in common (True where rows of different
    strides mingle: that is not looked into)."""
    if a.numel() == 0 or b.numel() == 0:
        return False

    def rows(t):  # first byte, bytes of a row, bytes between rows, one past the last byte
        es, many = t.element_size(), t.dim() == 2 and t.shape[0] > 1
        w, step = t.shape[-1] * es, t.stride(0) * es if many else 0
        return t.data_ptr(), w, step, t.data_ptr() + (t.shape[0] - 1 if many else 0) * step + w

    pa, wa, sa, ea = rows(a)
    pb, wb, sb, eb = rows(b)
    if ea <= pb or eb <= pa:
        return False
    step = sa or sb
    if step == 0 or sa and sb and sa != sb or max(wa, wb) > step:
        return True
    apart = (pb - pa) % step  # rows of one grid: they meet in every step or never
    return apart < wa or apart + wb > step


def evict_cache(kv_cache: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, budget: int, *, page_size: int, sinks: int = 0,
                recent_from: torch.Tensor | None = None, budgets: torch.Tensor | None = None,
                out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keep each request's ``budget`` heaviest tokens and close up its pages; (weights, positions, lengths).

    kv_cache [pages, page_size, 1, width] of any type is changed in place: request r's kept tokens are
    its first ``lengths[r] = min(seq_lens[r], budget)`` ones afterwards (``budgets`` [reqs] int32 may
    lower it per request).  Tokens whose ``positions`` [reqs, columns] int32 is below ``sinks``, or at
    or past ``recent_from`` [reqs] int32, stay before all others; then the larger ``weights``
    [reqs, columns] fp32 stay (NaN goes first), ties in favour of the lower index.  Kept tokens past
    the new length move into the places given up below it, both in ascending order; the rest stay put.
    Returns new weights and positions [reqs, min(budget, columns)] (0 and -1 past the length) and int32
    lengths, in ``out`` when given; they must not share memory with the inputs.  The requests' pages
    must not be shared; pages past a new length are free.  ``workspace`` is as ``tree_attention``'s
    (``evict_cache_workspace_bytes``).
    """
    ts = (kv_cache, weights, positions, block_table, seq_lens)
    if not all(t.is_cuda for t in ts):
        raise ValueError("evict_cache: all tensors must be CUDA tensors")
    dev = kv_cache.device
    if any(t is not None and t.device != dev for t in (*ts, recent_from, budgets)):
        raise ValueError("evict_cache: all tensors must be on one device")
    if kv_cache.dim() != 4 or kv_cache.shape[2] != 1 or kv_cache.shape[1] != page_size or kv_cache.stride(3) != 1:
        raise ValueError(f"kv_cache must be [pages, {page_size}, 1, width], got {tuple(kv_cache.shape)}")
    if weights.dtype != torch.float32 or any(t is not None and t.dtype != torch.int32 for t in (positions, block_table, seq_lens, recent_from, budgets)):
        raise TypeError("weights must be fp32; positions, block_table, seq_lens, recent_from and budgets int32")
    reqs = seq_lens.shape[0]
    if weights.dim() != 2 or weights.shape[0] != reqs or positions.shape != weights.shape:
        raise ValueError(f"weights and positions must be [{reqs}, columns], got {tuple(weights.shape)}, {tuple(positions.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] < reqs or any(t is not None and t.shape != (reqs,) for t in (seq_lens, recent_from, budgets)):
        raise ValueError(f"block_table must have {reqs} rows; seq_lens, recent_from and budgets [{reqs}]")
    if any(t is not None and t.numel() and t.stride(-1) != 1 for t in (weights, positions, block_table, seq_lens, recent_from, budgets)):
        raise ValueError("weights, positions, block_table, seq_lens, recent_from and budgets need a unit stride on the last dim")
    if budget < 0:
        raise ValueError(f"budget {budget}: expected a number of tokens")
    cols = weights.shape[1]
    keep = min(budget, cols)
    if out is None:
        new_w = torch.empty(reqs, keep, dtype=torch.float32, device=dev)
        new_p = torch.empty(reqs, keep, dtype=torch.int32, device=dev)
        new_l = torch.empty(reqs, dtype=torch.int32, device=dev)
    else:
        new_w, new_p, new_l = out
        if new_w.dtype != torch.float32 or new_p.dtype != torch.int32 or new_l.dtype != torch.int32 or \
                new_w.dim() != 2 or new_w.shape[0] != reqs or new_w.shape[1] < keep or new_p.shape != new_w.shape or \
                new_l.shape != (reqs,) or new_p.stride() != new_w.stride() or new_w.stride(1) != 1 or new_l.stride(0) != 1 or \
                any(t.device != dev for t in out):
            raise ValueError(f"out must be fp32 and int32 [{reqs}, >= {keep}] of one layout and int32 [{reqs}]")
        read = [t for t in (weights, positions, seq_lens, block_table, recent_from, budgets) if t is not None]
        if any(_overlap(a, b) for i, a in enumerate(out) for b in (*read, *out[i + 1:])):
            raise ValueError("out must not share memory with the inputs, nor its parts with each other")
    if reqs == 0:
        return new_w, new_p, new_l
    es = kv_cache.element_size()
    run_with_workspace("qmla_evict", _PACK_EVICT.pack, (
        kv_cache.data_ptr(), kv_cache.stride(0) * es, kv_cache.stride(1) * es, kv_cache.shape[3] * es, kv_cache.shape[0],
        page_size, block_table.data_ptr(), block_table.stride(0), block_table.shape[1], weights.data_ptr(),
        weights.stride(0), positions.data_ptr(), positions.stride(0), cols, seq_lens.data_ptr(),
        budgets.data_ptr() if budgets is not None else 0, min(budget, 2**31 - 1), sinks,
        recent_from.data_ptr() if recent_from is not None else 0, new_w.data_ptr(), new_p.data_ptr(), new_w.stride(0),
        new_w.shape[1], new_l.data_ptr(), reqs), dev, workspace)
    return new_w, new_p, new_l


def evict_cache_workspace_bytes(reqs: int, columns: int, budget: int) -> int:
    """Bytes of ``workspace`` that ``evict_cache`` of ``reqs`` requests and ``columns`` weights each needs."""
    if reqs < 0 or columns < 0 or budget < 0:
        raise ValueError(f"{reqs} requests, {columns} columns, budget {budget}: expected no negative number")
    budget = min(budget, 2**31 - 1)
    return workspace_bytes("qmla_evict", _PACK_EVICT.pack, (
        0, 1, 1, 1, 0, 1, 0, 0, 0, 0, 0, 0, 0, columns, 0, 0, budget, 0, 0, 0, 0, 0, min(budget, columns), 0, reqs),
        torch.device("cuda", 0))
