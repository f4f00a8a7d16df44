"""Attention of a drafted token tree over the paged latent cache (speculative verify).

The plugin verifies a chain of drafts by flattening it into decode rows of growing length
(``qwen_mla/mla_impl.py:628-662``).  A tree of drafts is not a chain: siblings sit side by side in
the cache and must not see each other.  Here every node brings a 64-bit mask of the drafted tokens it
sees, and all nodes of a request read its cache together.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .mla_decode_attention import _FP8_TYPES, _dt, capturing, rms_mode_for

_ws: dict[tuple[int, int], torch.Tensor] = {}
_raw_stream = torch._C._cuda_getCurrentRawStream  # (device index) -> the current stream's handle
_PACK = _lib.packer(_lib.TreeParams)


def device_index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def workspace_bytes(name: str, pack, args: tuple, device: torch.device) -> int:
    """Bytes of workspace the call ``qmla_<name>`` with ``args`` asks for."""
    need = ctypes.c_int64(0)
    sizer = _SIZER[name]
    _lib.check(sizer, getattr(_lib.load(), sizer)(pack(*args, 0, 0, device_index(device)), ctypes.byref(need)))
    return need.value


def run_with_workspace(name: str, pack, args: tuple, device: torch.device, workspace: torch.Tensor | None) -> None:
    """Call ``qmla_<name>`` on the current stream with ``args``, its workspace and the device.

    Without a ``workspace``, scratch is kept for the stream (calls on two streams never share it) and
    grown when the library asks for more; it refuses a small one before it launches anything.  A call
    that is captured into a CUDA graph gets scratch of its own from the graph's memory pool, as torch's
    own temporaries do: the graph keeps the address, so what is kept for the stream must not be in it.
    """
    idx = device_index(device)
    stream = _raw_stream(idx)
    lib = _lib.load()
    if workspace is not None:
        if workspace.device.type != "cuda" or device_index(workspace.device) != idx or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on cuda:{idx}")
        ws = workspace
    elif capturing(idx):
        need = workspace_bytes(name, pack, args, device)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    else:
        ws = _ws.get((idx, stream))
        if ws is None:
            ws = _ws[(idx, stream)] = torch.empty(1 << 20, dtype=torch.uint8, device=device)
    ptr, size = (ws.data_ptr(), ws.numel() * ws.element_size()) if ws is not None else (0, 0)
    rc = getattr(lib, name)(pack(*args, ptr, size, idx), stream)
    if rc == _E_WORKSPACE and workspace is None:
        ws = _ws[(idx, stream)] = torch.empty(workspace_bytes(name, pack, args, device), dtype=torch.uint8, device=device)
        rc = getattr(lib, name)(pack(*args, ws.data_ptr(), ws.numel(), idx), stream)
    _lib.check(name, rc)


def operator_status(device: torch.device | int | None = None, clear: bool = True) -> int:
    """Status bits of the ``tree_attention`` and ``accumulate_attention_weights`` calls on a device since the
    last clear (1: a wait inside a kernel gave up; such a tree attention returned NaN, such an accumulation
    left some weights as they were).  Synchronises the current stream."""
    dev = torch.device("cuda", device) if isinstance(device, int) else (device or torch.device("cuda"))
    idx = device_index(dev)
    bits = ctypes.c_int32(0)
    _lib.check("qmla_operator_status", _lib.load().qmla_operator_status(idx, clear, _raw_stream(idx), ctypes.byref(bits)))
    return bits.value


_E_WORKSPACE = -4
_SIZER = {"qmla_tree_attention": "qmla_tree_workspace_bytes", "qmla_accumulate_weights": "qmla_weights_workspace_bytes",
          "qmla_evict": "qmla_evict_workspace_bytes"}


def tree_masks(parents: torch.Tensor) -> torch.Tensor:
    """Masks of the trees ``parents`` [..., nodes] describes (the parent's number, negative: a root).

    int64 [..., nodes] on the same device: bit j of entry i is set when j is i or an ancestor of i.
    Nodes may be numbered in any order; at most 64 of them.
    """
    n = parents.shape[-1]
    if n > 64:
        raise ValueError(f"{n} nodes: a tree has at most 64")
    p = parents.long()
    bits = torch.ones((), dtype=torch.int64, device=p.device) << torch.arange(n, device=p.device)
    mask = bits.expand(p.shape).clone()
    up = torch.where((p >= 0) & (p < n), p, torch.full_like(p, n))  # n: past the root
    steps = 1
    while steps < n:  # pointer doubling: mask covers `steps` generations, up jumps as far
        padded = torch.cat([mask, torch.zeros_like(mask[..., :1])], -1)
        mask = mask | torch.gather(padded, -1, up)
        up = torch.gather(torch.cat([up, torch.full_like(up[..., :1], n)], -1), -1, up)
        steps *= 2
    return mask


def tree_attention(q: torch.Tensor, kv_cache: torch.Tensor, o: torch.Tensor, lse: torch.Tensor | None,
                   block_table: torch.Tensor, ctx_lens: torch.Tensor, tree_mask: torch.Tensor, *, rank: int,
                   sm_scale: float, page_size: int, rms_offset: int = -1, rms_bf16: bool = False,
                   rms_log8: bool = False, qk_dim: int | None = None, logit_cap: float = 0.0,
                   k_scale: torch.Tensor | None = None, q_pe: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> None:
    """Every node's attention over its request's committed tokens and its own ancestors, into ``o``, ``lse``.

    q [reqs * nodes, heads, >= qk_dim] bf16 or f16, request-major (the rope part may be a separate
    ``q_pe``); kv_cache [pages, page_size, 1, width] bf16 or FP8 (``k_scale``: fp32 device scalar);
    o [reqs * nodes, heads, rank] bf16, f16 or f32; lse [reqs * nodes, heads] or None.
    block_table [reqs, cols] int32; ctx_lens [reqs] int32 committed tokens.  The drafted tokens' rows
    are already in the cache, node j of request r as token ctx_lens[r] + j.
    tree_mask int64 [reqs, nodes], or [nodes] for one tree shared by all (``tree_masks``); a node
    whose mask is 0 is padding (o = 0, lse = -inf).
    ``qk_dim`` defaults to ``rms_offset``, or the row width without rms; the rms flags are
    ``decode_attention_fwd``'s.  Scratch is kept per stream, or is ``workspace``, a contiguous tensor of at
    least ``tree_attention_workspace_bytes`` bytes, 256-byte aligned.  In a CUDA graph captured with
    ``torch.cuda.graph`` it comes from the graph's pool; any other capture needs a ``workspace``.
    """
    args = _tree_args(q, kv_cache, o, lse, block_table, ctx_lens, tree_mask, rank=rank, sm_scale=sm_scale,
                      page_size=page_size, rms_offset=rms_offset, rms_bf16=rms_bf16, rms_log8=rms_log8, qk_dim=qk_dim,
                      logit_cap=logit_cap, k_scale=k_scale, q_pe=q_pe)
    if args is not None:
        run_with_workspace("qmla_tree_attention", _PACK.pack, args, q.device, workspace)


def tree_attention_workspace_bytes(q: torch.Tensor, kv_cache: torch.Tensor, o: torch.Tensor, lse: torch.Tensor | None,
                                   block_table: torch.Tensor, ctx_lens: torch.Tensor, tree_mask: torch.Tensor, *,
                                   rank: int, page_size: int, **how) -> int:
    """Bytes of ``workspace`` that ``tree_attention`` of these arguments needs (shapes and types count, not
    what the tensors hold)."""
    how.setdefault("sm_scale", 1.0)
    args = _tree_args(q, kv_cache, o, lse, block_table, ctx_lens, tree_mask, rank=rank, page_size=page_size, **how)
    return 0 if args is None else workspace_bytes("qmla_tree_attention", _PACK.pack, args, q.device)


def _tree_args(q, kv_cache, o, lse, block_table, ctx_lens, tree_mask, *, rank, sm_scale, page_size, rms_offset=-1,
               rms_bf16=False, rms_log8=False, qk_dim=None, logit_cap=0.0, k_scale=None, q_pe=None) -> tuple | None:
    """The checked call as qmla_tree_params' fields up to the workspace; None when there is nothing to do."""
    if not all(t.is_cuda for t in (q, kv_cache, o, block_table, ctx_lens, tree_mask)):
        raise ValueError("tree_attention: all tensors must be CUDA tensors")
    if any(t is not None and t.device != q.device for t in (kv_cache, o, lse, block_table, ctx_lens, tree_mask, k_scale, q_pe)):
        raise ValueError("tree_attention: all tensors must be on one device")
    fp8 = kv_cache.dtype in _FP8_TYPES or kv_cache.dtype == torch.uint8
    if not fp8 and kv_cache.dtype != torch.bfloat16:
        raise TypeError(f"cache dtype {kv_cache.dtype} not supported (bf16 or float8_e4m3fn)")
    if kv_cache.dim() != 4 or kv_cache.shape[2] != 1 or kv_cache.shape[1] != page_size or kv_cache.stride(3) != 1:
        raise ValueError(f"kv_cache must be [pages, {page_size}, 1, width], got {tuple(kv_cache.shape)}")
    if block_table.dtype != torch.int32 or ctx_lens.dtype != torch.int32 or tree_mask.dtype != torch.int64:
        raise TypeError("block_table and ctx_lens must be int32, tree_mask int64")
    reqs, nodes = ctx_lens.shape[0], tree_mask.shape[-1]
    if tree_mask.dim() not in (1, 2) or tree_mask.dim() == 2 and tree_mask.shape[0] != reqs:
        raise ValueError(f"tree_mask must be [{reqs}, nodes] or [nodes], got {tuple(tree_mask.shape)}")
    if nodes > 64:
        raise ValueError(f"{nodes} nodes: a tree has at most 64")
    if q.dim() != 3 or q.shape[0] != reqs * nodes:
        raise ValueError(f"q must have {reqs} * {nodes} rows, got {tuple(q.shape)}")
    width, heads = kv_cache.shape[3], q.shape[1]
    qk = qk_dim if qk_dim is not None else (rms_offset if rms_offset >= 0 else width)
    if q.shape[2] < (rank if q_pe is not None else qk) or \
            q_pe is not None and (q_pe.shape[:2] != q.shape[:2] or q_pe.shape[2] < qk - rank or q_pe.dtype != q.dtype):
        raise ValueError(f"q (and q_pe) do not hold {qk} dims")
    if o.shape != (q.shape[0], heads, rank) or lse is not None and lse.shape != (q.shape[0], heads):
        raise ValueError(f"o must be [{q.shape[0]}, {heads}, {rank}] and lse [{q.shape[0]}, {heads}]")
    if any(t is not None and t.numel() and t.stride(-1) != 1 for t in (q, q_pe, o, lse, block_table, ctx_lens, tree_mask)):
        raise ValueError("q, q_pe, o, lse, block_table, ctx_lens and tree_mask need a unit stride on the last dim")
    if block_table.dim() != 2 or block_table.shape[0] < reqs:
        raise ValueError(f"block_table must have {reqs} rows, got {tuple(block_table.shape)}")
    if k_scale is not None and k_scale.dtype != torch.float32:
        raise TypeError("k_scale must be an fp32 device scalar")
    if reqs * nodes == 0:
        return None
    pe = q_pe if q_pe is not None else q
    mode = rms_mode_for(kv_cache.dtype, rms_offset, rms_bf16, rms_log8)
    return (
        q.data_ptr(), q.stride(0), q.stride(1),
        pe.data_ptr() if q_pe is not None else q.data_ptr() + rank * q.element_size(), pe.stride(0), pe.stride(1),
        _dt(q), kv_cache.data_ptr(), kv_cache.stride(0), kv_cache.stride(1), kv_cache.shape[0], width,
        _lib.DT_FP8E4M3 if fp8 else _lib.DT_BF16, page_size, block_table.data_ptr(), block_table.stride(0),
        block_table.shape[1], ctx_lens.data_ptr(), tree_mask.data_ptr(),
        tree_mask.stride(0) if tree_mask.dim() == 2 else 0, reqs, nodes, heads, rank, qk, rms_offset, mode, sm_scale,
        logit_cap or 0.0, k_scale.data_ptr() if k_scale is not None else 0, o.data_ptr(), o.stride(0), o.stride(1), _dt(o),
        lse.data_ptr() if lse is not None else 0, lse.stride(0) if lse is not None else 0,
        _dt(lse) if lse is not None else _lib.DT_F32)
