"""Rotary positions on q and k, alone or while a fused projection is split into q, k, v.

Pair p of a head turns by t = position * freqs[p]: (a, b) -> (a cos t - b sin t, a sin t + b cos t), in half layout
(elements p and p + R) or interleaved (2p and 2p + 1), on the first 2 R dimensions of the head. Frequencies are 64-bit and
position * frequency is reduced modulo a turn exactly in the kernel, so far positions lose nothing. Images and videos
give one position per axis: `freqs` [axes, R / axes] with `positions` [..., axes]. The gradient is the same rotation
backwards. The operator has no counterpart in the reference, whose attention (`novadit/modules/dit_attention.py:10-80`)
has no positions.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import require_cuda_extension
from .qkv_pack import qkv_pack_ref


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, axes: int = 1, scaling: str | None = None,
                       factor: float = 1.0, original_length: int = 8192, fast_turns: float = 32.0,
                       slow_turns: float = 1.0, device=None):
    """(freqs, attention_factor) for `rotary_dim` rotated dimensions: freqs float64 [rotary_dim / 2], or
    [axes, rotary_dim / (2 axes)] when axes > 1, freqs[i] = base^(-2 i / d) with d the dimensions of one axis.

    `scaling` stretches a context by `factor`: "linear" divides every frequency by it (positions interpolated), "ntk"
    multiplies the base by factor^(d / (d - 2)), so that the slowest pair is interpolated and the fastest kept, "yarn"
    divides only the pairs that make less than `slow_turns` turns over `original_length` positions, keeps those that
    make more than `fast_turns`, blends linearly between, and returns attention_factor = 0.1 ln(factor) + 1 (1 otherwise)."""
    if axes < 1 or rotary_dim < 2 * axes or rotary_dim % (2 * axes) != 0:
        raise ValueError(f"rotary_dim must be a positive multiple of 2 * axes, got {rotary_dim} and {axes}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"Unsupported scaling: {scaling}")
    if not (base > 0 and factor >= 1):
        raise ValueError(f"base must be positive and factor at least 1, got {base} and {factor}")
    d = rotary_dim // axes
    if scaling == "ntk":
        if d <= 2:
            raise ValueError("ntk scaling needs more than one pair per axis")
        base = base * factor ** (d / (d - 2))
    i = torch.arange(d // 2, dtype=torch.float64)
    freqs = torch.tensor(base, dtype=torch.float64) ** (-2.0 * i / d)
    attention_factor = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if base <= 1 or not fast_turns > slow_turns > 0 or original_length <= 0:
            raise ValueError("yarn scaling needs base > 1, fast_turns > slow_turns > 0 and a positive original_length")
        fast, slow = (d * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
                      for turns in (fast_turns, slow_turns))
        low, high = max(math.floor(fast), 0), min(math.ceil(slow), d - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freqs = freqs / factor * ramp + freqs * (1 - ramp)
        attention_factor = 0.1 * math.log(factor) + 1.0
    if axes > 1:
        freqs = freqs.expand(axes, d // 2).contiguous()
    return freqs.to(device), attention_factor


def rotary_ref(x, positions, freqs, interleaved: bool = False, attention_factor: float = 1.0):
    """PyTorch definition on x [B, S, heads, D]: angles in float64, the rotation in x's dtype but at least float32."""
    pairs = freqs.numel()
    angle = positions.double()[..., None] * freqs.double()
    if freqs.dim() == 2:
        angle = angle.flatten(-2)
    angle = angle.unsqueeze(-2)  # one table for all heads
    t = torch.promote_types(x.dtype, torch.float32)
    cos, sin = (angle.cos() * attention_factor).to(t), (angle.sin() * attention_factor).to(t)
    rot, rest = x[..., :2 * pairs].to(t), x[..., 2 * pairs:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = rot[..., :pairs], rot[..., pairs:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([rot.to(x.dtype), rest], dim=-1)


def qkv_pack_rotary_ref(qkv, num_heads: int, head_dim: int, positions, freqs, interleaved: bool = False,
                        attention_factor: float = 1.0):
    q, k, v = qkv_pack_ref(qkv, num_heads, head_dim)
    return (rotary_ref(q, positions, freqs, interleaved, attention_factor),
            rotary_ref(k, positions, freqs, interleaved, attention_factor), v)


class _FusedRotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, freqs, interleaved, attention_factor):
        ext = require_cuda_extension("fused_rotary", x, "rotary_ref")
        ctx.save_for_backward(positions, freqs)
        ctx.interleaved, ctx.attention_factor = interleaved, attention_factor
        return ext.fused_rotary_apply(x, positions, freqs, interleaved, attention_factor, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ext = require_cuda_extension("fused_rotary", dy, "rotary_ref")
        positions, freqs = ctx.saved_tensors
        return ext.fused_rotary_apply(dy, positions, freqs, ctx.interleaved, ctx.attention_factor, True), None, None, None, None


def fused_rotary(x, positions, freqs, interleaved: bool = False, attention_factor: float = 1.0):
    """x [B, S, heads, D] (fp32 / fp16 / bf16, CUDA, head dimensions contiguous, any other strides) -> rotated, contiguous.

    positions int32 / int64 [S] or [B, S] with freqs float64 [R]; [S, axes] or [B, S, axes] with freqs [axes, R / axes]
    (`rotary_frequencies`). 2 R <= D: the dimensions behind are copied. The rotated part is multiplied by
    `attention_factor`. Interleaved pairs need an even D. Differentiable in x, once."""
    require_cuda_extension("fused_rotary", x, "rotary_ref")
    _check_even(x.shape[-1], interleaved)
    if not (torch.is_grad_enabled() and x.requires_grad):  # nothing to record
        ext = require_cuda_extension("fused_rotary", x, "rotary_ref")
        return ext.fused_rotary_apply(x, positions, freqs, bool(interleaved), float(attention_factor), False)
    return _FusedRotaryFunction.apply(x, positions, freqs, bool(interleaved), float(attention_factor))


class _FusedQkvPackRotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, num_heads, head_dim, positions, freqs, interleaved, attention_factor):
        ext = require_cuda_extension("fused_qkv_pack_rotary", qkv, "qkv_pack_rotary_ref")
        ctx.save_for_backward(positions, freqs)
        ctx.interleaved, ctx.attention_factor = interleaved, attention_factor
        return tuple(ext.fused_qkv_pack_rotary_forward(qkv, num_heads, head_dim, positions, freqs, interleaved,
                                                       attention_factor))

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv):
        ext = require_cuda_extension("fused_qkv_pack_rotary", dq, "qkv_pack_rotary_ref")
        positions, freqs = ctx.saved_tensors
        dqkv = ext.fused_qkv_pack_rotary_backward(dq, dk, dv, positions, freqs, ctx.interleaved, ctx.attention_factor)
        return dqkv, None, None, None, None, None, None


def fused_qkv_pack_rotary(qkv, num_heads: int, head_dim: int, positions, freqs, interleaved: bool = False,
                          attention_factor: float = 1.0):
    """`fused_qkv_pack` with `fused_rotary` of q and k in the same pass over qkv [B, S, 3 * heads * head_dim]: (q, k, v),
    each [B, S, heads, head_dim] and contiguous. The other arguments as in `fused_rotary`. Differentiable in qkv, once."""
    if qkv.dim() != 3 or qkv.shape[-1] != 3 * num_heads * head_dim:
        raise ValueError(f"Expected last dim {3 * num_heads * head_dim}, got {tuple(qkv.shape)}")
    require_cuda_extension("fused_qkv_pack_rotary", qkv, "qkv_pack_rotary_ref")
    _check_even(head_dim, interleaved)
    if not (torch.is_grad_enabled() and qkv.requires_grad):  # nothing to record
        ext = require_cuda_extension("fused_qkv_pack_rotary", qkv, "qkv_pack_rotary_ref")
        return tuple(ext.fused_qkv_pack_rotary_forward(qkv, num_heads, head_dim, positions, freqs, bool(interleaved),
                                                       float(attention_factor)))
    return _FusedQkvPackRotaryFunction.apply(qkv, num_heads, head_dim, positions, freqs, bool(interleaved),
                                             float(attention_factor))


def _check_even(head_dim: int, interleaved: bool) -> None:
    if interleaved and head_dim % 2 != 0:
        raise ValueError(f"interleaved rotary pairs need an even head_dim, got {head_dim}")
