"""``torch.library`` custom ops over libqmla: ``torch.ops.qmla.mla_decode``, ``gather_cache``,
``rotary`` and ``rope_kv_cache_update``.

vLLM compiles its model with torch.compile and captures CUDA graphs around it. A ctypes call
inside a compiled region would break the graph. These ops are opaque to the compiler: each
declares which arguments it writes (``o`` / ``lse``, ``dst``) and has a fake kernel that does
nothing, so tracing never touches the library. The real kernels run the same entry points as
``mla_decode_attention.decode_attention_fwd``, ``mla_gather.gather_cache_torch`` and the functions
of ``rotary``.

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

``rms_mode`` of mla_decode is a ``QMLA_RMS_*`` code (0 none, 1 native, 2 bf16 bytes, 3 log8).
Set ``rms_offset`` < 0 in gather_cache for a 2-byte cache (no rms layout).
"""
from __future__ import annotations

from typing import Optional

import torch

from .mla_decode_attention import build_params, run_params
from .mla_gather import gather_cache_torch
from .rotary import rope_kv_cache_update as _rope_kv_cache_update
from .rotary import rotary_embed


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
    return rotary_embed(x, positions, steps, start=start, blocks=blocks, interleaved=interleaved, scale=scale,
                        adjoint=adjoint)


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
