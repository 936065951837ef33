"""Cross attention without a GPU: argument checks of the C ABI, workspace sizes, the PyTorch definition, refusals."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import novadit_b200.ops as ops
from novadit_b200 import capi


def fwd(dtype=1, b=1, sq=4, sk=5, hq=4, hkv=2, d=16, scale=0.25, ptr=None, mask=None, lens=None, strides=None):
    p = ctypes.c_void_p(ptr)
    return capi.lib().nd_attn_fwd(dtype, p, p, p, p, None, mask, lens, b, sq, sk, hq, hkv, d, strides, scale, None, 0, None)


def bwd(dtype=1, b=1, sq=4, sk=5, hq=4, hkv=2, d=16, scale=0.25):
    return capi.lib().nd_attn_bwd(dtype, *[None] * 11, b, sq, sk, hq, hkv, d, None, scale, None, 0, None)


@pytest.mark.parametrize("call", [fwd, bwd])
def test_arguments_are_checked_before_any_cuda_call(call):
    assert call() == -1  # null pointers
    assert call(b=0) == 0 and (call is bwd or call(sq=0) == 0)
    for kw in (dict(b=-1), dict(sq=-1), dict(sk=-1), dict(hq=3), dict(hq=0), dict(hkv=0), dict(d=0), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=math.nan), dict(scale=math.inf)):
        assert call(**kw) == -1, kw
    for kw in (dict(dtype=2), dict(dtype=3), dict(d=12), dict(d=136), dict(b=1 << 17), dict(hq=1 << 17, hkv=1), dict(sq=1 << 26),
               dict(sk=1 << 31)):
        assert call(**kw) == -2, kw


def test_addresses_strides_and_workspace_are_checked():
    nine = (ctypes.c_int64 * 9)(*[8] * 9)
    odd = (ctypes.c_int64 * 9)(*[8] * 8, 12)
    down = (ctypes.c_int64 * 9)(*[8] * 8, -8)
    at = 1 << 20  # never looked at
    assert fwd(ptr=at, strides=None) == -1
    assert fwd(ptr=at + 2, strides=nine) == -2
    assert fwd(ptr=at, strides=odd) == -2 and fwd(ptr=at, strides=down) == -2
    assert fwd(ptr=at, strides=nine, mask=at, lens=at) == -1
    assert fwd(ptr=at, strides=nine, sq=1, hq=2, sk=100000) == -4  # split keys without a workspace
    assert fwd(ptr=at, strides=nine, sq=100, sk=100000) == -4


@pytest.mark.parametrize("tensor", [0, 1, 2, 3])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_broadcast_strides_are_refused_at_the_c_boundary(tensor, dim):
    at = 1 << 20  # never looked at
    L, p = capi.lib(), ctypes.c_void_p(1 << 20)
    values = [8] * 12
    values[3 * tensor + dim] = 0
    twelve = (ctypes.c_int64 * 12)(*values)
    many, one = (2, 100000, 100000, 4, 2), [2, 100000, 100000, 4, 2]  # b, sq, sk, hq, hkv
    for i in {0: (0,), 1: (1, 2), 2: (3, 4)}[dim]:
        one[i] = 1
    if tensor < 3:
        assert fwd(ptr=at, strides=twelve, b=many[0], sq=many[1], sk=many[2], hq=many[3], hkv=many[4]) == -2
    for sizes, code in ((many, -2), (one, -4)):  # an extent of one has no stride; then the missing workspace is next
        assert L.nd_attn_bwd(1, p, p, p, p, p, p, p, p, p, None, None, *sizes, 16, twelve, 0.25, None, 0, None) == code


def test_workspace_sizes():
    L = capi.lib()
    assert L.nd_attn_lse_floats(2, 100, 8, 2) == 2 * 2 * 512  # blocks of four heads: 400 rows, padded to four tiles
    assert L.nd_attn_lse_floats(2, 100, 6, 2) == 2 * 6 * 128  # groups of three are not packed
    assert L.nd_attn_lse_floats(0, 100, 6, 2) == 0 and L.nd_attn_lse_floats(1, 1, 3, 2) == 0
    assert L.nd_attn_fwd_ws_bytes(64, 4096, 4096, 16, 16, 64) == 0  # more than enough work without splitting
    assert L.nd_attn_fwd_ws_bytes(1, 128, 100000, 1, 1, 64) > 0
    assert L.nd_attn_fwd_ws_bytes(1, 128, 100000, 1, 1, 63) == 0  # a refused call needs nothing
    stats = 2 * 4 * 2 * 2 * 512
    assert L.nd_attn_bwd_ws_bytes(2, 100, 100000, 8, 2, 64) == stats
    assert L.nd_attn_bwd_ws_bytes(2, 100, 10, 8, 2, 64) > stats  # queries split
    assert L.nd_attn_bwd_ws_bytes(2, 0, 10, 8, 2, 64) == 0


@pytest.mark.parametrize("kind", ["none", "mask", "lens"])
def test_definition(kind):
    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 5, 4, 8, generator=g, dtype=torch.float64)
    k, v = (torch.randn(3, 6, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    lens = torch.tensor([6, 0, 3])
    keep = torch.arange(6)[None] < lens[:, None]
    if kind == "none":
        keep = torch.ones_like(keep)
    out = ops.cross_attention_ref(q, k, v, key_mask=keep if kind == "mask" else None, kv_lens=lens if kind == "lens" else None)
    for b in range(3):
        for h in range(4):
            kk, vv = k[b, keep[b], h // 2], v[b, keep[b], h // 2]
            want = torch.softmax(q[b, :, h] @ kk.T / math.sqrt(8), -1) @ vv if len(kk) else torch.zeros(5, 8, dtype=torch.float64)
            assert torch.allclose(out[b, :, h], want, rtol=1e-12, atol=1e-12)


def test_definition_ignores_what_masked_keys_hold():
    q, k, v = (torch.ones(1, 2, 1, 8) for _ in range(3))
    k[0, 1], v[0, 1] = math.nan, math.inf
    assert torch.equal(ops.cross_attention_ref(q, k, v, kv_lens=torch.tensor([1])), torch.ones(1, 2, 1, 8))


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 1, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fused_cross_attention(q, q, q)
