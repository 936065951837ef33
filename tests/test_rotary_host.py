"""Rotary frequencies, the PyTorch definition and the argument checks of the C ABI: no GPU."""
from __future__ import annotations

import math

import pytest
import torch

import novadit_b200.ops as ops
from novadit_b200 import capi


def test_frequencies_of_each_scaling():
    plain, one = ops.rotary_frequencies(64)
    assert plain.dtype == torch.float64 and plain.shape == (32,) and one == 1.0
    assert float(plain[0]) == 1.0 and math.isclose(float(plain[16]), 10000.0 ** -0.5, rel_tol=1e-14)
    linear, _ = ops.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.allclose(linear * 4, plain, rtol=1e-15, atol=0)
    ntk, _ = ops.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]) * 4, float(plain[-1]), rel_tol=1e-12)
    yarn, att = ops.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])       # often turning pairs keep their frequency
    assert torch.allclose(yarn[turns < 0.7] * 4, plain[turns < 0.7], rtol=1e-15, atol=0)  # slow ones are interpolated
    assert bool((yarn <= plain).all()) and bool((yarn * 4 >= plain * (1 - 1e-15)).all())
    assert math.isclose(att, 0.1 * math.log(4.0) + 1.0)
    grid, _ = ops.rotary_frequencies(72, axes=2)
    assert grid.shape == (2, 18) and torch.equal(grid[0], grid[1]) and torch.equal(grid[0], ops.rotary_frequencies(36)[0])


def test_frequency_refusals():
    for args in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, axes=3), dict(rotary_dim=8, axes=0),
                 dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, base=0.0),
                 dict(rotary_dim=2, scaling="ntk", factor=2.0),
                 dict(rotary_dim=8, scaling="yarn", factor=2.0, fast_turns=1.0, slow_turns=1.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**args)


@pytest.mark.parametrize("interleaved", [False, True])
def test_definition_is_a_rotation_of_relative_positions(interleaved):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(1, 1, 1, 16, dtype=torch.float64, generator=g) for _ in range(2))
    freqs, _ = ops.rotary_frequencies(16)

    def dot(m, n):
        a = ops.rotary_ref(q, torch.tensor([m]), freqs, interleaved)
        b = ops.rotary_ref(k, torch.tensor([n]), freqs, interleaved)
        return float((a * b).sum())

    assert math.isclose(dot(5, 2), dot(1005, 1002), rel_tol=1e-9)
    assert math.isclose(dot(0, 0), float((q * k).sum()), rel_tol=1e-12)


def test_c_abi_checks_arguments_before_any_cuda_call():
    L = capi.lib()

    def call(dtype=1, batch=1, seq=1, heads=1, dim=8, sb=8, ss=8, sh=8, pos_bytes=8, pos_b=0, pairs=4, axes=1):
        return L.nd_rotary(dtype, None, None, batch, seq, heads, dim, sb, ss, sh, None, pos_bytes, pos_b, None, pairs, axes,
                           0, 1.0, 0, None)

    assert call() == -1                     # null pointers
    assert call(batch=0) == 0 and call(seq=0) == 0
    assert call(dtype=3) == -2
    for kw in (dict(pairs=5), dict(pairs=0), dict(axes=3), dict(pos_bytes=2), dict(heads=0), dict(dim=0), dict(batch=-1),
               dict(sb=-1), dict(pos_b=-1), dict(axes=0)):
        assert call(**kw) == -1
    assert call(dim=1 << 17) == -2
    assert L.nd_qkv_pack_rotary_fwd(1, None, None, None, None, 1, 1, 1, 8, None, 8, 0, None, 4, 1, 0, 1.0, None) == -1
    assert L.nd_qkv_pack_rotary_bwd(1, None, None, None, None, 0, 1, 1, 8, None, 8, 0, None, 4, 1, 0, 1.0, None) == 0
    assert L.nd_qkv_pack_rotary_bwd(3, None, None, None, None, 1, 1, 1, 8, None, 8, 0, None, 4, 1, 0, 1.0, None) == -2


def test_cpu_tensors_are_refused():
    x, pos, f = torch.zeros(1, 2, 1, 8), torch.zeros(2, dtype=torch.int64), torch.ones(4, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fused_rotary(x, pos, f)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fused_qkv_pack_rotary(torch.zeros(1, 2, 24), 1, 8, pos, f)


def test_attention_module_keeps_its_frequencies():
    from novadit_b200.modules import RotaryAttention

    want = ops.rotary_frequencies(16, 10000.0, 2)[0]
    moved = RotaryAttention(64, 4, axes=2).to(torch.bfloat16)
    placed = RotaryAttention(64, 4, axes=2, device="meta").to_empty(device="cpu")
    for module in (moved, placed, placed.half()):
        assert module.freqs.dtype == torch.float64 and torch.equal(module.freqs, want)
    assert moved.qkv.weight.dtype == torch.bfloat16 and "freqs" not in moved.state_dict()
