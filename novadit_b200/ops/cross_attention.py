"""Attention of one sequence to the keys and values of another: out = softmax(scale q k^T) v.

A text-conditioned DiT block reads its prompt's states with it; with queries and keys of one sequence it is the block's
self attention. One pass over the keys with the running maximum and sum of the softmax, products on tcgen05, fp32
scores, sums and accumulators; the backward pass recomputes the weights from the saved log-sum-exp and uses no atomics.
The reference calls a library here (`novadit/modules/dit_attention.py:10-80`).
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import require_cuda_extension


def cross_attention_ref(q, k, v, key_mask=None, kv_lens=None, scale: float | None = None):
    """PyTorch definition in at least float32. Keys that take no part are left out whatever they hold; a sample without
    keys gives zeros."""
    b, n, h, d = q.shape
    m, hk = k.shape[1], k.shape[2]
    t = torch.promote_types(q.dtype, torch.float32)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    keep = key_mask
    if kv_lens is not None:
        keep = torch.arange(m, device=q.device)[None] < kv_lens[:, None]
    qf, kf, vf = q.to(t), k.to(t), v.to(t)
    if keep is not None:
        kf = torch.where(keep[:, :, None, None], kf, torch.zeros((), dtype=t, device=q.device))
        vf = torch.where(keep[:, :, None, None], vf, torch.zeros((), dtype=t, device=q.device))
    kf, vf = kf.repeat_interleave(h // hk, dim=2), vf.repeat_interleave(h // hk, dim=2)
    s = torch.einsum("bnhd,bmhd->bhnm", qf, kf) * scale
    if keep is not None:
        s = s.masked_fill(~keep[:, None, None], -math.inf)
        none = ~keep.any(1)
        s = s.masked_fill(none[:, None, None, None], 0.0)  # softmax of nothing: weights replaced below
    p = torch.softmax(s, dim=-1)
    if keep is not None:
        p = p.masked_fill(~keep[:, None, None], 0.0)
    return torch.einsum("bhnm,bmhd->bnhd", p, vf).to(q.dtype)


class _FusedCrossAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, kv_lens, scale):
        ext = require_cuda_extension("fused_cross_attention", q, "cross_attention_ref")
        out, lse = ext.fused_cross_attention_forward(q, k, v, key_mask, kv_lens, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, key_mask, kv_lens)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        ext = require_cuda_extension("fused_cross_attention", dout, "cross_attention_ref")
        q, k, v, out, lse, key_mask, kv_lens = ctx.saved_tensors
        dq, dk, dv = ext.fused_cross_attention_backward(dout, q, k, v, out, lse, key_mask, kv_lens, ctx.scale)
        return dq, dk, dv, None, None, None


def fused_cross_attention(q, k, v, key_mask=None, kv_lens=None, scale: float | None = None):
    """q [B, Sq, heads, D], k and v [B, Sk, kv_heads, D] (CUDA, one dtype of fp16 / bf16, D a multiple of 8 up to 128,
    heads a multiple of kv_heads: query head h reads key head h // (heads // kv_heads)) -> [B, Sq, heads, D], contiguous.

    Views whose head dimensions are contiguous and whose other strides are multiples of 8 elements are read in place
    (the halves of a fused key/value projection, a transposed [B, heads, S, D]); others are copied. key_mask [B, Sk] bool
    (True: the key takes part) or kv_lens [B] int32 / int64 (the first kv_lens[b] keys, clamped to 0 .. Sk), not both;
    keys that take no part are never looked at. A sample without keys gives zeros and zero gradients. scale: 1 / sqrt(D)
    by default, positive. B and heads up to 65535. Differentiable in q, k and v, once."""
    require_cuda_extension("fused_cross_attention", q, "cross_attention_ref")
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.shape[-1] > 0 else 1.0
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _FusedCrossAttentionFunction.apply(q, k, v, key_mask, kv_lens, float(scale))
    ext = require_cuda_extension("fused_cross_attention", q, "cross_attention_ref")
    return ext.fused_cross_attention_forward(q, k, v, key_mask, kv_lens, float(scale), False)[0]
