"""Rotary positions: kernels against a 64-bit evaluation of the definition, gradients against the inverse rotation and
against differences, layouts, strides, far positions."""
from __future__ import annotations

import math

import pytest
import torch

import novadit_b200.ops as ops
from novadit_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def exact(x, positions, freqs, interleaved, factor, sign=1.0):
    """(y, |a| + |b| per element) in 64 bits on the CPU."""
    x, positions, freqs = x.detach().cpu().double(), positions.cpu(), freqs.cpu()
    pairs = freqs.numel()
    angle = sign * positions.double()[..., None] * freqs
    if freqs.dim() == 2:
        angle = angle.flatten(-2)
    angle = angle.unsqueeze(-2)
    c, s = angle.cos() * factor, angle.sin() * factor
    y, mag = x.clone(), torch.zeros_like(x)
    ia = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    ib = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * factor
    return y, mag


def check(got, want, mag, what):
    """One rounding to the type (half a step of the value, half the smallest number near zero) and the 32-bit arithmetic
    before it: the angle as a 24-bit fraction of a half turn (pi 2^-24), sincospi (2 steps of 2^-23 at most), the factor
    and the two products (3 x 2^-24), together below 12 x 2^-24 of |a| + |b|."""
    info = torch.finfo(got.dtype)
    err = (got.detach().cpu().double() - want).abs()
    bar = info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2 + 12 * 2.0 ** -24 * (1 + info.eps) * mag
    assert bool((err <= bar).all()), f"{what}: {float((err - bar).max()):.3e} over the bar"


def inputs(shape, dtype, seed, axes, reach, shared=False, pos_type=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(dtype)
    lead = (shape[1],) if shared else (shape[0], shape[1])
    pos = torch.randint(0, reach, lead + ((axes,) if axes > 1 else ()), generator=g).to(pos_type)
    return x, pos


SHAPES = [  # B, S, heads, D, rotated dimensions, axes
    (1, 1, 1, 2, 2, 1), (2, 5, 3, 72, 72, 1), (2, 9, 16, 72, 72, 2), (1, 130, 2, 64, 32, 1), (3, 7, 5, 96, 96, 3),
    (2, 6, 4, 80, 20, 1), (1, 33, 1, 128, 128, 1), (2, 3, 7, 24, 6, 3), (4, 1, 32, 128, 64, 1), (1, 4, 2, 50, 50, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,h,d,rot,axes", SHAPES)
def test_rotary_matches_the_definition(dtype, interleaved, b, s, h, d, rot, axes):
    freqs, _ = ops.rotary_frequencies(rot, axes=axes)
    x, pos = inputs((b, s, h, d), dtype, 1, axes, 5000)
    y = ops.fused_rotary(x.to(DEV), pos.to(DEV), freqs.to(DEV), interleaved=interleaved, attention_factor=1.25)
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    want, mag = exact(x, pos, freqs, interleaved, 1.25)
    check(y, want, mag, "y")
    assert torch.equal(y[..., rot:].cpu(), x[..., rot:])  # the rest of the head is untouched


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pos_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("reach", [2 ** 20, 2 ** 31 - 1])
def test_far_and_negative_positions(dtype, pos_type, reach):
    freqs, factor = ops.rotary_frequencies(64, scaling="yarn", factor=16.0, original_length=4096)
    x, pos = inputs((2, 64, 2, 64), dtype, 2, 1, reach, pos_type=pos_type)
    pos[0, ::2] *= -1
    y = ops.fused_rotary(x.to(DEV), pos.to(DEV), freqs.to(DEV), attention_factor=factor)
    # the definition's own angle in 64 bits is off by reach * 2^-53 radians: nothing beside the bar
    want, mag = exact(x, pos, freqs, False, factor)
    check(y, want, mag, "y")


def test_positions_past_32_bits():
    # position p and p + 2^33 differ by whole turns for frequencies that are multiples of 2 pi 2^-33
    freqs = torch.tensor([2 * math.pi * k / 2 ** 33 for k in (1, 3, 2 ** 20 + 1)], dtype=torch.float64)
    x, pos = inputs((1, 50, 2, 6), torch.float32, 3, 1, 2 ** 33)
    near = ops.fused_rotary(x.to(DEV), pos.to(DEV), freqs.to(DEV))
    far = ops.fused_rotary(x.to(DEV), (pos + 5 * 2 ** 33).to(DEV), freqs.to(DEV))
    # freqs / (2 pi) is off by 2^-52 relative at most: 6 * 2^33 * 2^-12 * 2^-52 of a turn
    assert float((near - far).abs().max()) < 1e-5
    want, mag = exact(x, pos, freqs, False, 1.0)
    check(near, want, mag, "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_views_and_shared_positions(dtype, interleaved):
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(3, 11, 2, 4, 40, generator=g).to(dtype)
    freqs, _ = ops.rotary_frequencies(40)
    pos = torch.arange(11) * 37
    k = wide.to(DEV)[:, :, 1]                       # the key half of a fused projection
    y = ops.fused_rotary(k, pos.to(DEV), freqs.to(DEV), interleaved=interleaved)
    want, mag = exact(wide[:, :, 1], pos.expand(3, 11), freqs, interleaved, 1.0)
    check(y, want, mag, "strided")
    by_head = k.transpose(1, 2).contiguous().transpose(1, 2)  # [B, heads, S, D] memory
    assert torch.equal(ops.fused_rotary(by_head, pos.to(DEV), freqs.to(DEV), interleaved=interleaved), y)
    one = k[:1].expand(3, -1, -1, -1)               # a broadcast batch
    assert torch.equal(ops.fused_rotary(one, pos.to(DEV), freqs.to(DEV), interleaved=interleaved)[2], y[0])
    flat = torch.empty(1 + k.numel(), dtype=dtype, device=DEV)[1:].view(k.shape)  # off the vector boundary
    flat.copy_(k)
    assert torch.equal(ops.fused_rotary(flat, pos.to(DEV), freqs.to(DEV), interleaved=interleaved), y)
    turned = k.transpose(2, 3).contiguous().transpose(2, 3)  # head dimensions not contiguous: copied first
    assert torch.equal(ops.fused_rotary(turned, pos.to(DEV), freqs.to(DEV), interleaved=interleaved), y)


def test_odd_head_dim_in_half_layout():
    freqs = torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64)
    x, pos = inputs((2, 3, 5, 7), torch.bfloat16, 5, 1, 100)
    y = ops.fused_rotary(x.to(DEV), pos.to(DEV), freqs.to(DEV))
    want, mag = exact(x, pos, freqs, False, 1.0)
    check(y, want, mag, "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,h,d,rot,axes", [(2, 5, 3, 72, 72, 2), (1, 1, 1, 8, 4, 1), (3, 33, 16, 72, 72, 1), (1, 9, 5, 128, 32, 2)])
def test_pack_forward_and_backward(dtype, interleaved, b, s, h, d, rot, axes):
    freqs, _ = ops.rotary_frequencies(rot, axes=axes)
    qkv, pos = inputs((b, s, 3 * h * d), dtype, 6, axes, 300)
    qd, pd, fd = qkv.to(DEV).requires_grad_(True), pos.to(DEV), freqs.to(DEV)
    out = ops.fused_qkv_pack_rotary(qd, h, d, pd, fd, interleaved=interleaved, attention_factor=1.5)
    parts = ops.qkv_pack_ref(qkv, h, d)
    for i, (g, p) in enumerate(zip(out, parts)):
        assert g.shape == (b, s, h, d) and g.is_contiguous()
        if i == 2:
            assert torch.equal(g.detach().cpu(), p)
        else:
            want, mag = exact(p, pos, freqs, interleaved, 1.5)
            check(g, want, mag, "qk"[i])
            assert torch.equal(g, ops.fused_rotary(p.to(DEV), pd, fd, interleaved=interleaved, attention_factor=1.5))
    gen = torch.Generator().manual_seed(7)
    grads = [torch.randn(b, s, h, d, generator=gen).to(dtype) for _ in range(3)]
    (dqkv,) = torch.autograd.grad(out, (qd,), [g.to(DEV) for g in grads])
    dq, dk, dv = dqkv.cpu().view(b, s, 3, h, d).unbind(2)
    for got, g in ((dq, grads[0]), (dk, grads[1])):
        want, mag = exact(g, pos, freqs, interleaved, 1.5, sign=-1.0)
        check(got, want, mag, "gradient")
    assert torch.equal(dv, grads[2])
    # one output alone: the others' gradients are zero
    only = torch.autograd.grad(ops.fused_qkv_pack_rotary(qd, h, d, pd, fd, interleaved=interleaved)[2], (qd,), grads[2].to(DEV))[0]
    assert torch.equal(only.cpu().view(b, s, 3, h, d)[:, :, 2], grads[2]) and not bool(only.view(b, s, 3, h, d)[:, :, :2].any())


def test_gradient_against_differences():
    freqs, _ = ops.rotary_frequencies(16)
    x, pos = inputs((1, 4, 2, 20), torch.float32, 8, 1, 50)
    xd, pd, fd = x.to(DEV).requires_grad_(True), pos.to(DEV), freqs.to(DEV)
    w = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(DEV)
    (dx,) = torch.autograd.grad(ops.fused_rotary(xd, pd, fd), (xd,), w)
    step = 0.5  # the rotation is linear: any step gives the derivative, up to the rounding of 32-bit sums
    for at in ((0, 0, 0, 0), (0, 3, 1, 9), (0, 2, 0, 15), (0, 1, 1, 17)):
        e = torch.zeros_like(xd)
        e[at] = step
        with torch.no_grad():
            up = (ops.fused_rotary(xd + e, pd, fd).double() * w.double()).sum()
            down = (ops.fused_rotary(xd - e, pd, fd).double() * w.double()).sum()
        # 160 values of magnitude below 8 and weight below 5, each within 14 * 2^-24 * 8
        assert abs(float((up - down) / (2 * step) - dx[at])) < 160 * 5 * 8 * 28 * 2.0 ** -24


def test_empty_and_refusals():
    f = torch.ones(4, dtype=torch.float64, device=DEV)
    x = torch.randn(2, 3, 2, 8, device=DEV)
    pos = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    assert ops.fused_rotary(x[:, :0], pos[:, :0], f).shape == (2, 0, 2, 8)
    assert ops.fused_rotary(x[:0], pos[:0], f).shape == (0, 3, 2, 8)
    bad = [
        (x, pos.float(), f), (x, pos, f.float()), (x, pos[:, :2], f), (x, pos[:1], f), (x, pos, torch.ones(5, dtype=torch.float64, device=DEV)),
        (x, pos, f[:0]), (x, pos.cpu(), f), (x, pos, f.cpu()), (x.double(), pos, f), (x[0], pos, f),
        (x, pos, f.view(2, 2)), (x, pos, f.view(1, 2, 2)), (x, pos, f.clone().requires_grad_(True)),
    ]
    for args in bad:
        with pytest.raises(RuntimeError):
            ops.fused_rotary(*args)
    with pytest.raises(RuntimeError, match="rotary_ref"):
        ops.fused_rotary(x.cpu(), pos, f)
    with pytest.raises(ValueError, match="even head_dim"):
        ops.fused_rotary(torch.randn(1, 3, 2, 7, device=DEV), pos[:1], f[:3], interleaved=True)
    with pytest.raises(ValueError, match="Expected last dim"):
        ops.fused_qkv_pack_rotary(torch.zeros(2, 3, 50, device=DEV), 2, 8, pos, f)


def test_other_stream_and_graph():
    freqs, _ = ops.rotary_frequencies(72, device=DEV)
    x, pos = inputs((2, 40, 4, 72), torch.bfloat16, 10, 1, 900)
    x, pos = x.to(DEV), pos.to(DEV)
    want = ops.fused_rotary(x, pos, freqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.fused_rotary(x, pos, freqs)
    side.synchronize()
    assert torch.equal(got, want)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.fused_rotary(static, pos, freqs)
    static.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.fused_rotary(x.flip(0), pos, freqs))


def test_c_abi_helper():
    freqs, _ = ops.rotary_frequencies(32, device=DEV)
    x, pos = inputs((2, 6, 3, 32), torch.float32, 11, 1, 77)
    y = capi.rotary(x.to(DEV), pos.to(DEV), freqs)
    assert torch.equal(y, ops.fused_rotary(x.to(DEV), pos.to(DEV), freqs))
    back = capi.rotary(y, pos.to(DEV), freqs, inverse=True)
    # there and back: two rotations, each within 12 x 2^-24 of |a| + |b| plus its rounding
    assert float((back.cpu() - x).abs().max()) < 2 * 14 * 2.0 ** -24 * 2 * float(x.abs().max()) * 2
