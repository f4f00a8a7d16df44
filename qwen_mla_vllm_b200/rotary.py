"""Rotary positions: the frequencies of the usual long-context scalings, the rotation of (part of)
each head with its adjoint, and the fused write of a step's rotated keys into the latent cache.

The layout semantics are the plugin's partial rope (``qwen_mla/partial_rope.py:28-91``): a packed
window of 58-dim groups, each rotated as one block; q holds a head's group in its slot of the window
and zeros elsewhere, k_pe holds every group followed by the per-head rms.

A pair's frequency is given as ``steps``: its turns per position as a 64-bit binary fraction
(``rotary_steps``).  ``position * step`` modulo 2^64 is then the exact phase, at a position of a
million as at one, with no table of sines and nothing to rebuild when contexts grow.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .mla_gather import status_pointer
from .tree_attention import _raw_stream

_DT = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}
_FP8 = (torch.float8_e4m3fn, torch.uint8)
_PACK_ROTARY = _lib.packer(_lib.RotaryParams)
_PACK_UPDATE = _lib.packer(_lib.RopeCacheParams)
_RMS = {"native": _lib.RMS_NATIVE, "log8": _lib.RMS_LOG8, "bf16": _lib.RMS_BF16, "none": _lib.RMS_NONE}


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[list[float], float]:
    """(radians per position of each of the rot_dim / 2 pairs, the scale of cos and sin).

    ``scaling`` (None: the plain ``base ** (-2i / rot_dim)``) is one of
      {"type": "linear", "factor": f}   every frequency divided by f;
      {"type": "ntk", "factor": f}      the base raised so that the last pair is slowed by f;
      {"type": "banded", "factor": f, "low_freq_factor": a, "high_freq_factor": b,
       "original_max_position": n}      pairs slower than n / a turns are divided by f, faster than
                                        n / b kept, those between blended linearly in turns;
      {"type": "yarn", "factor": f, "original_max_position": n, "beta_fast": 32, "beta_slow": 1,
       "attention_factor": None}        a ramp over the pair index between the pairs that make
                                        beta_fast and beta_slow turns in n positions (the slow end
                                        may lie past the last pair, up to rot_dim - 1); the scale is
                                        attention_factor, by default 0.1 ln f + 1.
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim}: expected an even number of dims")
    half = rot_dim // 2
    plain = [base ** (-2.0 * i / rot_dim) for i in range(half)]
    if scaling is None:
        return plain, 1.0
    kind, f = scaling.get("type"), float(scaling.get("factor", 1.0))
    if f <= 0:
        raise ValueError(f"scaling factor {f}: expected a positive number")
    if kind == "linear":
        return [w / f for w in plain], 1.0
    if kind == "ntk":
        if rot_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        b = base * f ** (rot_dim / (rot_dim - 2.0))
        return [b ** (-2.0 * i / rot_dim) for i in range(half)], 1.0
    if kind == "banded":
        n = float(scaling["original_max_position"])
        lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if hi <= lo:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        out = []
        for w in plain:
            turns = n * w / (2.0 * math.pi)
            t = min(1.0, max(0.0, (turns - lo) / (hi - lo)))
            out.append(w * (t + (1.0 - t) / f))
        return out, 1.0
    if kind == "yarn":
        n = float(scaling["original_max_position"])

        def index(turns):  # the (fractional) pair that makes this many turns in n positions
            return rot_dim * math.log(n / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        lo = max(0.0, math.floor(index(float(scaling.get("beta_fast", 32.0)))))
        hi = min(rot_dim - 1.0, math.ceil(index(float(scaling.get("beta_slow", 1.0)))))
        out = []
        for i, w in enumerate(plain):
            t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            out.append(w * ((1.0 - t) + t / f))
        att = scaling.get("attention_factor")
        return out, float(att) if att is not None else (0.1 * math.log(f) + 1.0 if f > 1 else 1.0)
    raise ValueError(f"scaling type {kind!r}: expected linear, ntk, banded or yarn")


def rotary_steps(rot_dim: int, base: float = 10000.0, scaling: dict | None = None, *,
                 device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """(``steps`` int64 [rot_dim / 2] on ``device``, the scale) for the entry points below."""
    freq, scale = rotary_frequencies(rot_dim, base, scaling)
    vals = [int(round(w / (2.0 * math.pi) * 2.0**64)) % 2**64 for w in freq]
    return torch.tensor([v - 2**64 if v >= 2**63 else v for v in vals], dtype=torch.int64, device=device), scale


def _check_positions(positions: torch.Tensor, steps: torch.Tensor, n: int, device: torch.device) -> None:
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions dtype {positions.dtype}: expected int32 or int64")
    if positions.dim() != 1 or positions.shape[0] != n or positions.stride(0) != 1 and n > 1:
        raise ValueError(f"positions must be [{n}] contiguous, got {tuple(positions.shape)}")
    if steps.dtype != torch.int64 or steps.dim() != 1 or not steps.is_contiguous():
        raise TypeError("steps must be a contiguous int64 vector (rotary_steps)")
    if positions.device != device or steps.device != device:
        raise ValueError("positions and steps must be on the device of the data")


def _index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def rotary_embed(x: torch.Tensor, positions: torch.Tensor, steps: torch.Tensor, *, start: int = 0, blocks: int = 1,
                 interleaved: bool = False, scale: float = 1.0, adjoint: bool = False,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate dims [start, start + blocks * rot_dim) of every head; rot_dim = 2 * steps.numel().

    x [tokens, heads, dim] (or [tokens, dim]) bf16, f16 or f32 with any token / head strides.
    ``interleaved`` pairs dims (2i, 2i + 1), otherwise (i, i + rot_dim / 2) of each block.
    ``adjoint`` applies the transpose: the gradient with respect to x of a loss whose gradient with
    respect to the output is given.  ``out=x`` works in place; None allocates a contiguous output.
    Differentiable in x; an ``out`` takes no part in autograd and is refused where x needs a gradient.
    """
    how = (start, blocks, interleaved, scale, adjoint)
    if not (x.requires_grad and torch.is_grad_enabled()):
        return rotate(x, positions, steps, *how, out)
    if out is not None:
        raise RuntimeError("rotary_embed: out= does not support automatic differentiation, but x requires a gradient")
    return _Rotary.apply(x, positions, steps, *how)


class _Rotary(torch.autograd.Function):
    """The map is linear in x: its gradient is the transposed map of the incoming one, which is the same
    operator again (and so has a gradient itself)."""

    @staticmethod
    def forward(ctx, x, positions, steps, *how):
        ctx.save_for_backward(positions, steps)
        ctx.how = how
        return rotate(x, positions, steps, *how)

    @staticmethod
    def backward(ctx, grad):
        *how, adjoint = ctx.how
        grad = grad if grad.stride(-1) == 1 else grad.contiguous()
        return (rotary_embed(grad, *ctx.saved_tensors, **dict(zip(("start", "blocks", "interleaved", "scale"), how)),
                             adjoint=not adjoint), *[None] * 7)


def rotate(x: torch.Tensor, positions: torch.Tensor, steps: torch.Tensor, start: int, blocks: int, interleaved: bool,
           scale: float, adjoint: bool, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rotary_embed`` outside of autograd."""
    if not x.is_cuda:
        raise ValueError("rotary_embed: x must be a CUDA tensor")
    if x.dtype not in _DT:
        raise TypeError(f"x dtype {x.dtype}: expected bf16, f16 or f32")
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be [tokens, heads, dim] or [tokens, dim], got {tuple(x.shape)}")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError("out must have x's shape, dtype and device")
    n, heads, dim = x.shape[0], x.shape[1] if x.dim() == 3 else 1, x.shape[-1]
    if (x.stride(-1) != 1 or out.stride(-1) != 1) and dim > 1:
        raise ValueError("x and out need a unit stride on the last dim")
    _check_positions(positions, steps, n, x.device)
    rot = 2 * steps.shape[0]
    if rot < 2 or blocks < 1 or start < 0 or start + blocks * rot > dim:
        raise ValueError(f"dims [{start}, {start} + {blocks} * {rot}) lie outside a head of {dim}")
    if n == 0 or heads == 0:
        return out
    idx = _index(x.device)
    p = _PACK_ROTARY.pack(
        x.data_ptr(), x.stride(0), x.stride(1) if x.dim() == 3 else dim, out.data_ptr(), out.stride(0),
        out.stride(1) if x.dim() == 3 else dim, n, heads, dim, _DT[x.dtype], start, rot, blocks, interleaved, adjoint,
        scale, positions.data_ptr(), positions.dtype == torch.int64, steps.data_ptr(), idx)
    _lib.check("qmla_rotary", _lib.load().qmla_rotary(p, _raw_stream(idx)))
    return out


def rope_kv_cache_update(q_pe: torch.Tensor, k_pe: torch.Tensor, kv_c_normed: torch.Tensor, positions: torch.Tensor,
                         slot_mapping: torch.Tensor, steps: torch.Tensor, kv_cache: torch.Tensor, *, packed_rope: int,
                         local_heads: int, q_out: torch.Tensor | None = None, interleaved: bool = False,
                         scale: float = 1.0, k_scale: torch.Tensor | None = None, rms_mode: str = "native") -> torch.Tensor:
    """Rotate a step's queries and write its rows into the paged cache, in one launch.

    q_pe [n, heads, packed_rope] bf16 (any strides) is rotated into ``q_out`` (in place when None).
    Row ``slot_mapping[i]`` of ``kv_cache`` [pages, page_size, 1, width] becomes [latent | rotated
    rope | rms tail] from kv_c_normed [n, rank] and k_pe [n, packed_rope + local_heads] (bf16,
    ``[rope | rms]``, un-rotated).  A bf16 cache takes rms_mode "native"; an FP8 cache needs
    ``k_scale`` (fp32 device scalar) and "log8" or "bf16", and holds what ``fp8_kv_cache_update``
    would write for keys rotated in fp32.  "none" writes no tail.  A negative slot writes no row; a
    slot outside the cache is skipped and reported by ``mla_gather.gather_status`` (bit 2).
    """
    if rms_mode not in _RMS:
        raise ValueError(f"rms_mode {rms_mode!r}: expected native, log8, bf16 or none")
    if q_out is None:
        q_out = q_pe
    bf = torch.bfloat16
    if q_pe.dtype != bf or k_pe.dtype != bf or kv_c_normed.dtype != bf or q_out.dtype != bf:
        raise TypeError("q_pe, q_out, k_pe and kv_c_normed must be bf16")
    if not kv_cache.is_cuda or any(t.device != kv_cache.device for t in (q_pe, q_out, k_pe, kv_c_normed, slot_mapping)):
        raise ValueError("rope_kv_cache_update: all tensors must be on the cache's CUDA device")
    fp8 = kv_cache.dtype in _FP8
    if not fp8 and kv_cache.dtype != bf:
        raise TypeError(f"cache dtype {kv_cache.dtype} not supported (bf16 or float8_e4m3fn)")
    if (rms_mode in ("log8", "bf16")) != fp8 and rms_mode != "none":
        raise ValueError(f"rms_mode {rms_mode!r} does not fit a {'FP8' if fp8 else 'bf16'} cache")
    if kv_cache.dim() != 4 or kv_cache.shape[2] != 1 or kv_cache.stride(-1) != 1:
        raise ValueError(f"kv_cache must be [pages, page_size, 1, width], got {tuple(kv_cache.shape)}")
    n, rank = kv_c_normed.shape
    tail = 0 if rms_mode == "none" else local_heads
    if q_pe.dim() != 3 or q_pe.shape[0] != n or q_pe.shape[2] != packed_rope or q_out.shape != q_pe.shape:
        raise ValueError(f"q_pe and q_out must be [{n}, heads, {packed_rope}], got {tuple(q_pe.shape)}, {tuple(q_out.shape)}")
    if k_pe.dim() != 2 or k_pe.shape[0] != n or k_pe.shape[1] < packed_rope + tail:
        raise ValueError(f"k_pe must be [{n}, >= {packed_rope + tail}], got {tuple(k_pe.shape)}")
    if any(t.stride(-1) != 1 for t in (q_pe, q_out, k_pe, kv_c_normed)):
        raise ValueError("q_pe, q_out, k_pe and kv_c_normed need a unit stride on the last dim")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (n,) or not slot_mapping.is_contiguous():
        raise TypeError(f"slot_mapping must be a contiguous int64 [{n}]")
    _check_positions(positions, steps, n, kv_cache.device)
    rot = 2 * steps.shape[0]
    if rot < 2 or packed_rope % rot:
        raise ValueError(f"packed_rope {packed_rope} is not a whole number of {rot}-dim blocks")
    width = kv_cache.shape[3]
    if width < rank + packed_rope + (2 * tail if rms_mode == "bf16" else tail):
        raise ValueError(f"cache rows of {width} do not hold {rank} + {packed_rope} and the rms of {tail} heads")
    if fp8 and (k_scale is None or k_scale.dtype != torch.float32 or k_scale.device != kv_cache.device):
        raise TypeError("an FP8 cache needs k_scale, an fp32 scalar on the device")
    if n == 0:
        return q_out
    idx = _index(kv_cache.device)
    p = _PACK_UPDATE.pack(
        q_pe.data_ptr(), q_pe.stride(0), q_pe.stride(1), q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
        kv_c_normed.data_ptr(), kv_c_normed.stride(0), k_pe.data_ptr(), k_pe.stride(0), positions.data_ptr(),
        slot_mapping.data_ptr(), steps.data_ptr(), kv_cache.data_ptr(), kv_cache.stride(0), kv_cache.stride(1), n,
        kv_cache.shape[0], kv_cache.shape[1], width, _lib.DT_FP8E4M3 if fp8 else _lib.DT_BF16, q_pe.shape[1], rank,
        packed_rope, rot, local_heads, _RMS[rms_mode], interleaved, positions.dtype == torch.int64, scale,
        k_scale.data_ptr() if fp8 else 0, status_pointer(kv_cache.device), idx)
    _lib.check("qmla_rope_cache_write", _lib.load().qmla_rope_cache_write(p, _raw_stream(idx)))
    return q_out
