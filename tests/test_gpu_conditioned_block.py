"""Rotary self attention and cross attention to a prompt as a block uses them: the modules on the fused operators against
the same modules in 64 bits, and the adaLN-Zero block and stack around them. The reference's own block is not needed: a
stand-in with its interface gives the norm, the MLP and an attention."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F
from torch import nn

import novadit_b200.ops as ops
from novadit_b200 import modules

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel_l2(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


def no_worse(fused, plain, exact, what):
    """The fused path rounds where the PyTorch definitions round, or less often, and once more inside (the weights before
    the second product of attention): independent roundings add up in the square, so half as much again covers it."""
    f, p = rel_l2(fused, exact), rel_l2(plain, exact)
    assert f <= 1.5 * p + 1e-6, f"{what}: {f:.2e} against {p:.2e}"


def grid(side):
    at = torch.arange(side * side, device=DEV)
    return torch.stack([at // side, at % side], dim=-1)


def twins(make, dtype):
    """(fused, plain, exact) modules of the same weights."""
    torch.manual_seed(3)
    fused = make(True).to(DEV, dtype)
    plain, exact = make(False).to(DEV, dtype), make(False).to(DEV, torch.float64)
    plain.load_state_dict(fused.state_dict())
    exact.load_state_dict({k: v.double() for k, v in fused.state_dict().items()})
    return fused, plain, exact


def compare(mods, inputs, extra, dy, names):
    outs = []
    for m in mods:
        t = torch.float64 if next(m.parameters()).dtype == torch.float64 else dy.dtype
        leaves = [x.detach().to(t).requires_grad_(True) for x in inputs]
        y = m(*leaves, **extra)
        params = [p for n, p in m.named_parameters() if ".body.attn." not in n]
        outs.append((y, *torch.autograd.grad(y, (*leaves, *params), dy.to(t))))
    for what, f, p, e in zip(names + ["parameter"] * 99, *outs):
        no_worse(f, p, e, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,hidden,side", [(4, 288, 9), (2, 256, 12)])
def test_rotary_attention(dtype, heads, hidden, side):
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(2, side * side, hidden, generator=g).to(DEV, dtype) for _ in range(2))
    mods = twins(lambda fused: modules.RotaryAttention(hidden, heads, use_fused=fused), dtype)
    assert mods[0].freqs.dtype == torch.float64  # through .to(dtype)
    compare(mods, [x], {"positions": grid(side)}, dy, ["y", "dx"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv_heads", [4, 2])
def test_cross_attention_module(dtype, kv_heads):
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(3, 150, 288, generator=g).to(DEV, dtype) for _ in range(2))
    ctx = torch.randn(3, 77, 128, generator=g).to(DEV, dtype)
    lens = torch.tensor([77, 0, 13], device=DEV)
    mods = twins(lambda fused: modules.CrossAttention(288, 128, 4, kv_heads, use_fused=fused), dtype)
    compare(mods, [x, ctx], {"context_lens": lens}, dy, ["y", "dx", "dcontext"])
    y = mods[0](x, ctx, context_lens=lens)
    assert torch.equal(y[1], mods[0].proj.bias.expand_as(y[1]))  # an empty prompt
    keep = torch.arange(77, device=DEV)[None] < lens[:, None]
    assert torch.equal(y, mods[0](x, ctx, context_mask=keep))


class _Mlp(nn.Module):
    def __init__(self, hidden, inter, device, dtype):
        super().__init__()
        self.fc1 = nn.Linear(hidden, inter, device=device, dtype=dtype)
        self.fc2 = nn.Linear(inter, hidden, device=device, dtype=dtype)
        self.activation = "gelu"

    def forward(self, x):
        return self.fc2(F.gelu(self.fc1(x), approximate="tanh"))


class _Block(nn.Module):
    """The parts of the reference's block that the adaLN-Zero block drives."""

    def __init__(self, hidden_size, num_heads, mlp_ratio, use_fused_adaln, device=None, dtype=None, **_):
        super().__init__()
        self.fused = use_fused_adaln
        self.attn = nn.Linear(hidden_size, hidden_size, device=device, dtype=dtype)
        self.mlp = _Mlp(hidden_size, int(mlp_ratio * hidden_size), device, dtype)

    def _adaln(self, x, scale, shift):
        return ops.fused_adaln(x, scale, shift, eps=1e-5) if self.fused else ops.adaln_ref(x, scale, shift, eps=1e-5)


@pytest.fixture
def stand_in(monkeypatch):
    monkeypatch.setattr(modules, "reference_modules", lambda: type("Ref", (), {"NovaDiTBlock": _Block}))


def stack(fused, depth=2, **kw):
    st = modules.DiTStack(288, 4, depth, use_fused=fused, use_fused_fc1_bias_act=False, zero_init=False, **kw)
    for p in st.parameters():
        nn.init.normal_(p, std=0.05)
    return st


@pytest.mark.parametrize("rotary,prompt", [(2, 96), (2, None), (0, 96)])
def test_conditioned_stack(stand_in, rotary, prompt):
    g = torch.Generator().manual_seed(4)
    dtype = torch.bfloat16
    x, dy = (torch.randn(2, 100, 288, generator=g).to(DEV, dtype) for _ in range(2))
    cond = torch.randn(2, 288, generator=g).to(DEV, dtype)
    mods = twins(lambda fused: stack(fused, rotary_axes=rotary, context_size=prompt), dtype)
    inputs, extra, names = [x, cond], {"positions": grid(10) if rotary else None}, ["y", "dx", "dcond"]
    if prompt:
        context = torch.randn(2, 40, prompt, generator=g).to(DEV, dtype)
        extra |= {"context_lens": torch.tensor([40, 17], device=DEV)}
        outs = []
        for m in mods:
            t = torch.float64 if next(m.parameters()).dtype == torch.float64 else dtype
            leaves = [v.detach().to(t).requires_grad_(True) for v in (x, cond, context)]
            y = m(leaves[0], leaves[1], context=leaves[2], **extra)
            outs.append((y, *torch.autograd.grad(y, leaves, dy.to(t))))
        for what, f, p, e in zip(names + ["dcontext"], *outs):
            no_worse(f, p, e, what)
    else:
        compare(mods, inputs, extra, dy, names)


def test_captured_step_beside_an_eager_one(stand_in):
    """Forward and backward of a conditioned stack captured into a graph and replayed on new inputs."""
    g = torch.Generator().manual_seed(5)
    st = stack(True, depth=1, rotary_axes=2, context_size=64).to(DEV, torch.bfloat16)
    x = torch.randn(2, 64, 288, generator=g).to(DEV, torch.bfloat16)
    cond, ctx = torch.randn(2, 288, generator=g).to(DEV, torch.bfloat16), torch.randn(2, 33, 64, generator=g).to(DEV, torch.bfloat16)
    dy, lens = torch.randn(x.shape, generator=g).to(DEV, torch.bfloat16), torch.tensor([33, 5], dtype=torch.int32, device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (x, cond, ctx)]

    def step():
        y = st(leaves[0], leaves[1], positions=grid8, context=leaves[2], context_lens=lens)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    grid8 = grid(8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        leaves[0].copy_(x.flip(1))
        lens.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert rel_l2(a, b) < 1e-3  # (library products may choose other kernels while captured)


FIRST_CALL = """
import torch
import novadit_b200.ops as ops
qkv = torch.randn(2, 50, 3 * 288, device="cuda").bfloat16().requires_grad_(True)
ctx = torch.randn(2, 20, 4, 72, device="cuda").bfloat16()
pos, (freqs, _) = torch.arange(50, device="cuda"), ops.rotary_frequencies(72, device="cuda")
dy = torch.randn(2, 50, 4, 72, device="cuda").bfloat16()
def step():
    q, k, v = ops.fused_qkv_pack_rotary(qkv, 4, 72, pos, freqs)
    y = ops.fused_cross_attention(ops.fused_cross_attention(q, k, v), ctx, ctx)
    return y.detach(), torch.autograd.grad(y, qkv, dy)[0]
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("same")
"""


def test_first_calls_of_a_process_may_be_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]
