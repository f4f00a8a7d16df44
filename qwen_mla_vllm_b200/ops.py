"""``torch.library`` custom ops over libqmla: ``torch.ops.qmla.mla_decode``, ``gather_cache``,
``rotary``, ``rope_kv_cache_update``, ``tree_attention``, ``accumulate_attention_weights`` and
``evict_cache``.

vLLM compiles its model with torch.compile and captures CUDA graphs around it. A ctypes call
inside a compiled region would break the graph. These ops are opaque to the compiler: each
declares which arguments it writes (``o`` / ``lse``, ``dst``) and has a fake kernel that does
nothing, so tracing never touches the library. The real kernels run the same entry points as
``mla_decode_attention.decode_attention_fwd``, ``mla_gather.gather_cache_torch`` and the functions
of ``rotary``, ``tree_attention`` and ``cache_eviction``.

    qmla::mla_decode(Tensor q, Tensor kv_cache, Tensor(a!) o, Tensor(b!) lse, Tensor block_table,
                     Tensor seq_lens, Tensor workspace, int rank, int qk_dim, int rms_offset,
                     int rms_mode, int page_size, float sm_scale, float logit_cap,
                     Tensor? k_scale, int qrows) -> ()
    qmla::gather_cache(Tensor src_cache, Tensor(a!) dst, Tensor block_table, Tensor cu_seq_lens,
                       Tensor token_to_seq, int num_tokens, str kv_cache_dtype, Tensor scale,
                       Tensor? seq_starts, int rms_offset, int rms_heads, str rms_mode) -> ()
    qmla::rotary(Tensor x, Tensor positions, Tensor steps, int start, int blocks, bool interleaved,
                 float scale, bool adjoint) -> Tensor                       (differentiable in x)
    qmla::rope_kv_cache_update(Tensor q_pe, Tensor k_pe, Tensor kv_c_normed, Tensor positions,
                 Tensor slot_mapping, Tensor steps, Tensor(a!) kv_cache, Tensor(b!) q_out,
                 int packed_rope, int local_heads, bool interleaved, float scale, Tensor? k_scale,
                 str rms_mode) -> ()
    qmla::tree_attention(Tensor q, Tensor kv_cache, Tensor(a!) o, Tensor(b!) lse, Tensor block_table,
                 Tensor ctx_lens, Tensor tree_mask, int rank, float sm_scale, int page_size,
                 int rms_offset, bool rms_bf16, bool rms_log8, float logit_cap, Tensor? k_scale,
                 Tensor? workspace=None, Tensor? q_pe=None, int? qk_dim=None) -> ()
    qmla::accumulate_attention_weights(Tensor q, Tensor kv_cache, Tensor(a!) weights, Tensor lse,
                 Tensor block_table, Tensor seq_lens, float sm_scale, int page_size, int rms_offset,
                 bool rms_bf16, bool rms_log8, float logit_cap, Tensor? k_scale, int qrows, float decay,
                 Tensor? workspace=None, Tensor? q_pe=None, int? rank=None, int? qk_dim=None) -> ()
    qmla::evict_cache(Tensor(a!) kv_cache, Tensor weights, Tensor positions, Tensor block_table,
                 Tensor seq_lens, Tensor(b!) new_weights, Tensor(c!) new_positions, Tensor(d!) new_lens,
                 int budget, int page_size, int sinks, Tensor? recent_from, Tensor? workspace=None,
                 Tensor? budgets=None) -> ()

``rms_mode`` of mla_decode is a ``QMLA_RMS_*`` code (0 none, 1 native, 2 bf16 bytes, 3 log8).
Set ``rms_offset`` < 0 in gather_cache for a 2-byte cache (no rms layout).  ``workspace`` is scratch (the
functions' ``workspace``); without one a captured call takes its scratch from the graph's pool.
"""
from __future__ import annotations

from typing import Optional

import torch

from .cache_eviction import accumulate_attention_weights as _accumulate_attention_weights
from .cache_eviction import evict_cache as _evict_cache
from .mla_decode_attention import build_params, run_params
from .mla_gather import gather_cache_torch
from .rotary import rope_kv_cache_update as _rope_kv_cache_update
from .rotary import rotate
from .tree_attention import tree_attention as _tree_attention


@torch.library.custom_op("qmla::mla_decode", mutates_args=("o", "lse"), device_types="cuda")
def mla_decode(q: torch.Tensor, kv_cache: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
               block_table: torch.Tensor, seq_lens: torch.Tensor, workspace: torch.Tensor, rank: int,
               qk_dim: int, rms_offset: int, rms_mode: int, page_size: int, sm_scale: float,
               logit_cap: float, k_scale: Optional[torch.Tensor], qrows: int) -> None:
    """Paged latent decode into ``o`` / ``lse`` (``qmla_mla_decode``).  ``workspace`` backs the
    kernel's split scratch when it is large enough (vLLM's ``attn_logits`` qualifies)."""
    p = build_params(q, kv_cache, o, lse, block_table, seq_lens, rank=rank, qk_dim=qk_dim,
                     rms_offset=rms_offset, rms_mode=rms_mode, page_size=page_size, sm_scale=sm_scale,
                     logit_cap=logit_cap, k_scale=k_scale, qrows=qrows)
    run_params(p, q.device, scratch=workspace)


@mla_decode.register_fake
def _mla_decode_fake(q, kv_cache, o, lse, block_table, seq_lens, workspace, rank, qk_dim, rms_offset,
                     rms_mode, page_size, sm_scale, logit_cap, k_scale, qrows) -> None:
    return None


@torch.library.custom_op("qmla::gather_cache", mutates_args=("dst",), device_types="cuda")
def gather_cache(src_cache: torch.Tensor, dst: torch.Tensor, block_table: torch.Tensor,
                 cu_seq_lens: torch.Tensor, token_to_seq: torch.Tensor, num_tokens: int,
                 kv_cache_dtype: str, scale: torch.Tensor, seq_starts: Optional[torch.Tensor],
                 rms_offset: int, rms_heads: int, rms_mode: str) -> None:
    """Chunked-prefill context gather into ``dst`` (``qmla_gather_cache``)."""
    gather_cache_torch(src_cache=src_cache, dst=dst, block_table=block_table, cu_seq_lens=cu_seq_lens,
                       token_to_seq=token_to_seq, num_tokens=num_tokens, kv_cache_dtype=kv_cache_dtype,
                       scale=scale, seq_starts=seq_starts,
                       mla_rms=(rms_offset, rms_heads, rms_mode) if rms_offset >= 0 else None)


@gather_cache.register_fake
def _gather_cache_fake(src_cache, dst, block_table, cu_seq_lens, token_to_seq, num_tokens, kv_cache_dtype,
                       scale, seq_starts, rms_offset, rms_heads, rms_mode) -> None:
    return None


@torch.library.custom_op("qmla::rotary", mutates_args=(), device_types="cuda")
def rotary(x: torch.Tensor, positions: torch.Tensor, steps: torch.Tensor, start: int, blocks: int,
           interleaved: bool, scale: float, adjoint: bool) -> torch.Tensor:
    """Rotary positions into a new tensor (``qmla_rotary``); differentiable in ``x``."""
    return rotate(x, positions, steps, start, blocks, interleaved, scale, adjoint)


@rotary.register_fake
def _rotary_fake(x, positions, steps, start, blocks, interleaved, scale, adjoint):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _rotary_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[1], inputs[2])
    ctx.how = inputs[3:]


def _rotary_backward(ctx, grad):
    positions, steps = ctx.saved_tensors
    start, blocks, interleaved, scale, adjoint = ctx.how
    # the map is linear in x: its gradient is the transposed map of the incoming gradient
    gx = torch.ops.qmla.rotary(grad if grad.stride(-1) == 1 else grad.contiguous(), positions, steps, start, blocks,
                               interleaved, scale, not adjoint)
    return gx, None, None, None, None, None, None, None


rotary.register_autograd(_rotary_backward, setup_context=_rotary_setup)


@torch.library.custom_op("qmla::rope_kv_cache_update", mutates_args=("kv_cache", "q_out"), device_types="cuda")
def rope_kv_cache_update(q_pe: torch.Tensor, k_pe: torch.Tensor, kv_c_normed: torch.Tensor, positions: torch.Tensor,
                         slot_mapping: torch.Tensor, steps: torch.Tensor, kv_cache: torch.Tensor, q_out: torch.Tensor,
                         packed_rope: int, local_heads: int, interleaved: bool, scale: float,
                         k_scale: Optional[torch.Tensor], rms_mode: str) -> None:
    """Rotated queries into ``q_out`` and a step's rows into ``kv_cache`` (``qmla_rope_cache_write``)."""
    _rope_kv_cache_update(q_pe, k_pe, kv_c_normed, positions, slot_mapping, steps, kv_cache, packed_rope=packed_rope,
                          local_heads=local_heads, q_out=q_out, interleaved=interleaved, scale=scale, k_scale=k_scale,
                          rms_mode=rms_mode)


@rope_kv_cache_update.register_fake
def _rope_kv_cache_update_fake(q_pe, k_pe, kv_c_normed, positions, slot_mapping, steps, kv_cache, q_out, packed_rope,
                               local_heads, interleaved, scale, k_scale, rms_mode) -> None:
    return None


@torch.library.custom_op("qmla::tree_attention", mutates_args=("o", "lse"), device_types="cuda")
def tree_attention(q: torch.Tensor, kv_cache: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                   block_table: torch.Tensor, ctx_lens: torch.Tensor, tree_mask: torch.Tensor, rank: int,
                   sm_scale: float, page_size: int, rms_offset: int, rms_bf16: bool, rms_log8: bool,
                   logit_cap: float, k_scale: Optional[torch.Tensor],
                   workspace: Optional[torch.Tensor] = None, q_pe: Optional[torch.Tensor] = None,
                   qk_dim: Optional[int] = None) -> None:
    """Attention of a drafted token tree into ``o`` / ``lse`` (``qmla_tree_attention``)."""
    _tree_attention(q, kv_cache, o, lse, block_table, ctx_lens, tree_mask, rank=rank, sm_scale=sm_scale,
                    page_size=page_size, rms_offset=rms_offset, rms_bf16=rms_bf16, rms_log8=rms_log8,
                    logit_cap=logit_cap, k_scale=k_scale, workspace=workspace, q_pe=q_pe, qk_dim=qk_dim)


@tree_attention.register_fake
def _tree_attention_fake(q, kv_cache, o, lse, block_table, ctx_lens, tree_mask, rank, sm_scale, page_size, rms_offset,
                         rms_bf16, rms_log8, logit_cap, k_scale, workspace=None, q_pe=None, qk_dim=None) -> None:
    return None


@torch.library.custom_op("qmla::accumulate_attention_weights", mutates_args=("weights",), device_types="cuda")
def accumulate_attention_weights(q: torch.Tensor, kv_cache: torch.Tensor, weights: torch.Tensor, lse: torch.Tensor,
                                 block_table: torch.Tensor, seq_lens: torch.Tensor, sm_scale: float, page_size: int,
                                 rms_offset: int, rms_bf16: bool, rms_log8: bool, logit_cap: float,
                                 k_scale: Optional[torch.Tensor], qrows: int, decay: float,
                                 workspace: Optional[torch.Tensor] = None, q_pe: Optional[torch.Tensor] = None,
                                 rank: Optional[int] = None, qk_dim: Optional[int] = None) -> None:
    """A step's softmax weights added to ``weights`` (``qmla_accumulate_weights``)."""
    _accumulate_attention_weights(q, kv_cache, weights, lse, block_table, seq_lens, sm_scale=sm_scale,
                                  page_size=page_size, rms_offset=rms_offset, rms_bf16=rms_bf16, rms_log8=rms_log8,
                                  logit_cap=logit_cap, k_scale=k_scale, qrows=qrows, decay=decay,
                                  workspace=workspace, q_pe=q_pe, rank=rank, qk_dim=qk_dim)


@accumulate_attention_weights.register_fake
def _accumulate_attention_weights_fake(q, kv_cache, weights, lse, block_table, seq_lens, sm_scale, page_size,
                                       rms_offset, rms_bf16, rms_log8, logit_cap, k_scale, qrows, decay,
                                       workspace=None, q_pe=None, rank=None, qk_dim=None) -> None:
    return None


@torch.library.custom_op("qmla::evict_cache", mutates_args=("kv_cache", "new_weights", "new_positions", "new_lens"),
                         device_types="cuda")
def evict_cache(kv_cache: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, new_weights: torch.Tensor, new_positions: torch.Tensor, new_lens: torch.Tensor,
                budget: int, page_size: int, sinks: int, recent_from: Optional[torch.Tensor],
                workspace: Optional[torch.Tensor] = None, budgets: Optional[torch.Tensor] = None) -> None:
    """Keep each request's heaviest tokens and close up its pages (``qmla_evict``)."""
    _evict_cache(kv_cache, weights, positions, block_table, seq_lens, budget, page_size=page_size, sinks=sinks,
                 recent_from=recent_from, out=(new_weights, new_positions, new_lens), workspace=workspace, budgets=budgets)


@evict_cache.register_fake
def _evict_cache_fake(kv_cache, weights, positions, block_table, seq_lens, new_weights, new_positions, new_lens, budget,
                      page_size, sinks, recent_from, workspace=None, budgets=None) -> None:
    return None
