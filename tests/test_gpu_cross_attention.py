"""Cross attention: forward and gradients against the definition in 64 bits at the sizes, masks, layouts and types where
it can go wrong.

Bars. With e = finfo.eps / 2 (one rounding to the type), W the weights, |.| elementwise:
  out   e |out| for its rounding, and e W|V| because every weight is rounded once before the second product
  dV    the same with W^T |dO|
  dS    e |dS| for its rounding; the row's delta is taken from the ROUNDED out, whose error is the one above:
        W (sum |dO| (e |out| + e W|V|)) ; dQ and dK take that through |K| and |Q|, and a rounding of their own
and on each product 2^-13 of the sum of its magnitudes for the 32-bit part (scores: up to 128 products, exponential,
sums). 16-bit floats that are not bf16 also have a smallest number: half of it for each rounded weight or dS."""
from __future__ import annotations

import math

import pytest
import torch

import novadit_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
FINE = 2.0 ** -13


def make(b, n, m, h, hk, d, dtype, seed, fused=True):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, n, h, d, generator=g).to(dtype)
    kv = torch.randn(b, m, 2, hk, d, generator=g).to(dtype)
    dout = torch.randn(b, n, h, d, generator=g).to(dtype)
    q, kv, dout = q.to(DEV), kv.to(DEV), dout.to(DEV)
    k, v = kv.unbind(2)
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    return q, k, v, dout


def exact(q, k, v, dout, keep, scale, tiny_s=None, tiny_p=None):
    """(out, dq, dk, dv) in 64 bits and their bars."""
    t = torch.finfo(q.dtype)
    e = t.eps / 2
    tiny = 0.0 if q.dtype == torch.bfloat16 else t.smallest_normal * t.eps / 2
    tiny_s, tiny_p = (tiny if x is None else x for x in (tiny_s, tiny_p))
    b, n, h, d = q.shape
    m, hk = k.shape[1], k.shape[2]
    Q = q.detach().double().view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    K = k.detach().double().permute(0, 2, 1, 3)[:, :, None]
    V = v.detach().double().permute(0, 2, 1, 3)[:, :, None]
    G = dout.double().view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    if keep is not None:
        K = torch.where(keep[:, None, None, :, None], K, 0.0)
        V = torch.where(keep[:, None, None, :, None], V, 0.0)
    S = Q @ K.transpose(-1, -2) * scale
    if keep is not None:
        S = S.masked_fill(~keep[:, None, None, None], -math.inf)
        S = S.masked_fill(~keep.any(1)[:, None, None, None, None], 0.0)
    W = torch.softmax(S, -1) if m > 0 else S
    if keep is not None:
        W = W.masked_fill(~keep[:, None, None, None], 0.0)
    O = W @ V
    WV = W @ V.abs()
    ones = torch.ones_like(W)
    bar_o = e * O.abs() + (e + FINE) * WV + tiny * (ones @ V.abs()) + tiny
    dV = W.transpose(-1, -2) @ G
    bar_v = (e + FINE) * (W.transpose(-1, -2) @ G.abs()) + tiny_p * (ones.transpose(-1, -2) @ G.abs())
    dP = G @ V.transpose(-1, -2)
    delta = (G * O).sum(-1, keepdim=True)
    dS = W * (dP - delta)
    off = (G.abs() * (e * O.abs() + e * WV)).sum(-1, keepdim=True)  # delta's error
    mag = G.abs() @ V.abs().transpose(-1, -2) + (G.abs() * O.abs()).sum(-1, keepdim=True)
    bar_s = e * dS.abs() + W * (off + FINE * mag) + tiny_s
    dQ, dK = scale * (dS @ K), scale * (dS.transpose(-1, -2) @ Q)
    bar_q = scale * (bar_s @ K.abs())
    bar_k = scale * (bar_s.transpose(-1, -2) @ Q.abs())

    def rows(x):
        return x.permute(0, 3, 1, 2, 4).reshape(b, n, h, d)

    def cols(x):
        return x.sum(2).permute(0, 2, 1, 3)

    want = (rows(O), rows(dQ), cols(dK), cols(dV))
    bars = (rows(bar_o), rows(bar_q) + e * want[1].abs() + tiny, cols(bar_k) + e * want[2].abs() + tiny,
            cols(bar_v) + e * want[3].abs() + tiny)
    return want, bars


def check(got, want, bars):
    for name, g, w, bar in zip(("out", "dq", "dk", "dv"), got, want, bars):
        assert g.shape == w.shape, f"{name}: shape {tuple(g.shape)}"
        assert torch.isfinite(g).all(), f"{name}: not finite"
        over = (g.detach().double() - w).abs() - bar * (1 + 1e-9)
        assert g.numel() == 0 or float(over.max()) <= 0, f"{name}: {float(over.max()):.3e} over the bar"


def run(q, k, v, dout, key_mask=None, kv_lens=None, scale=None):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = ops.fused_cross_attention(q, k, v, key_mask=key_mask, kv_lens=kv_lens, scale=scale)
    assert out.dtype == q.dtype and out.is_contiguous()
    with torch.no_grad():  # the inference path gives the same bits
        assert torch.equal(ops.fused_cross_attention(q, k, v, key_mask=key_mask, kv_lens=kv_lens, scale=scale), out)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


SHAPES = [  # B, queries, keys, heads, key heads, D
    (1, 1, 1, 1, 1, 8), (2, 1, 77, 16, 16, 72), (1, 128, 128, 2, 2, 64), (2, 129, 127, 3, 3, 64), (1, 256, 256, 1, 1, 128),
    (2, 300, 77, 4, 4, 72), (1, 257, 129, 4, 2, 80), (3, 70, 333, 6, 2, 40), (1, 33, 1000, 8, 1, 128), (2, 1, 2049, 8, 2, 64),
    (1, 1000, 3, 2, 1, 96), (1, 5, 17, 12, 1, 16), (2, 640, 500, 2, 2, 120), (1, 64, 64, 48, 3, 24), (9, 400, 130, 16, 16, 56),
    (1, 1, 700, 64, 1, 128), (40, 3, 40, 5, 5, 88),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,n,m,h,hk,d", SHAPES)
def test_forward_and_gradients(dtype, b, n, m, h, hk, d):
    q, k, v, dout = make(b, n, m, h, hk, d, dtype, 1)
    want, bars = exact(q, k, v, dout, None, 1 / math.sqrt(d))
    check(run(q, k, v, dout), want, bars)


def masks(kind, b, m, seed=3):
    """(key_mask, kv_lens, keep): an empty sample, a full one and ragged ones."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, m + 1, (b,), generator=g)
    lens[0] = 0
    lens[-1] = m
    at = torch.arange(m)[None]
    if kind.startswith("lens"):
        given = lens.to(torch.int32 if kind == "lens32" else torch.int64).to(DEV)
        return None, given, (at < lens[:, None]).to(DEV)
    if kind == "right":
        keep = at < lens[:, None]
    elif kind == "left":
        keep = at >= m - lens[:, None]
    else:  # holes, one whole tile among them where there are several
        keep = (torch.rand(b, m, generator=g) < 0.4) & (lens[:, None] > 0)
        keep[:, 128:256] = False
        keep[1 % b, min(3, m - 1)] = True
    keep = keep.to(DEV)
    return keep, None, keep


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["lens32", "lens64", "right", "left", "holes"])
@pytest.mark.parametrize("b,n,m,h,hk,d", [(4, 200, 300, 4, 2, 72), (3, 1, 77, 16, 16, 64), (3, 40, 1, 2, 1, 128), (5, 130, 1100, 2, 2, 64),
                                          (2, 2, 3000, 4, 1, 128)])
@pytest.mark.parametrize("poison", [False, True])
def test_keys_that_take_no_part(dtype, kind, b, n, m, h, hk, d, poison):
    q, k, v, dout = make(b, n, m, h, hk, d, dtype, 2)
    key_mask, kv_lens, keep = masks(kind, b, m)
    want, bars = exact(q, k, v, dout, keep, 1 / math.sqrt(d))
    if poison:  # whatever lies in the masked places
        g = torch.Generator().manual_seed(4)
        bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min])[torch.randint(0, 4, (b, m), generator=g)].to(dtype).to(DEV)
        k = torch.where(keep[:, :, None, None], k, bad[:, :, None, None])
        v = torch.where(keep[:, :, None, None], v, bad.flip(1)[:, :, None, None])
    got = run(q, k, v, dout, key_mask=key_mask, kv_lens=kv_lens)
    check(got, want, bars)
    empty = ~keep.any(1)
    assert not bool(got[0][empty].any()) and not bool(got[1][empty].any())
    assert not bool(got[2][~keep].any()) and not bool(got[3][~keep].any())


def test_lengths_outside_the_range_are_clamped():
    q, k, v, dout = make(4, 30, 50, 2, 2, 32, torch.bfloat16, 5)
    for t in (torch.int32, torch.int64):
        lens = torch.tensor([-7, 2 ** 31 - 1, 50, 10]).to(t).to(DEV)
        want = run(q, k, v, dout, kv_lens=torch.tensor([0, 50, 50, 10], dtype=t, device=DEV))
        for a, b in zip(run(q, k, v, dout, kv_lens=lens), want):
            assert torch.equal(a, b)
    far = torch.tensor([2 ** 40, -2 ** 40, 50, 10], device=DEV)
    assert torch.equal(run(q, k, v, dout, kv_lens=far)[0][0], run(q, k, v, dout)[0][0])
    assert not bool(run(q, k, v, dout, kv_lens=far)[0][1].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,scale", [(12.0, None), (1.0, 3.0), (0.02, 1.0)])
def test_score_ranges(dtype, size, scale):
    """Scores up to several hundred (one key takes all the weight, the maximum moves from tile to tile), and tiny ones."""
    q, k, v, dout = make(2, 150, 700, 2, 2, 64, dtype, 6, fused=False)
    q = (q.float() * size).to(dtype)
    ramp = torch.linspace(0.2, 1.0, 700, device=DEV)[None, :, None, None]  # later keys score higher
    k = (k.float() * ramp).to(dtype)
    s = 0.125 if scale is None else scale
    want, bars = exact(q, k, v, dout, None, s)
    # the scores' own 32-bit error grows with them: 64 products and their sum, 66 x 2^-24 of |q||k| scale, in the exponent
    room = 66 * 2.0 ** -24 * s * float((q.detach().double().abs().sum(-1).max()) * k.detach().double().abs().max())
    grow = 1 + 4 * room / FINE
    check(run(q, k, v, dout, scale=scale), want, [b * grow for b in bars])


def test_strides_and_copies():
    q, k, v, dout = make(2, 100, 90, 4, 4, 64, torch.bfloat16, 7)
    base = run(q, k, v, dout)
    def same(got):
        for a, b in zip(got, base):
            assert torch.equal(a, b)
    by_head = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731  [B, heads, S, D] memory
    same(run(by_head(q), by_head(k), by_head(v), by_head(dout)))
    inner = lambda x: x.transpose(1, 3).contiguous().transpose(1, 3)  # noqa: E731  head dimensions not contiguous
    same(run(inner(q), inner(k), inner(v), inner(dout)))
    def odd(x):  # rows 65 elements apart, base off by one element
        flat = torch.empty(x.numel() // 64 * 65 + 1, dtype=x.dtype, device=DEV)[1:].view(*x.shape[:3], 65)[..., :64]
        return flat.copy_(x)
    same(run(odd(q), odd(k), odd(v), odd(dout)))
    def wide(x):  # rows 72 elements apart: read in place
        return torch.empty(*x.shape[:3], 72, dtype=x.dtype, device=DEV)[..., :64].copy_(x)
    same(run(wide(q), wide(k), wide(v), wide(dout)))
    # one set of keys for the whole batch, and gradients of the broadcast
    k1, v1 = (x[:1].contiguous().requires_grad_(True) for x in (k, v))
    out = ops.fused_cross_attention(q, k1.expand(2, -1, -1, -1), v1.expand(2, -1, -1, -1))
    gk, gv = torch.autograd.grad(out, (k1, v1), dout)
    full = run(q, k[:1].repeat(2, 1, 1, 1), v[:1].repeat(2, 1, 1, 1), dout)
    assert torch.equal(out, full[0])
    assert torch.equal(gk, full[2].sum(0, keepdim=True)) and torch.equal(gv, full[3].sum(0, keepdim=True))
    # a gradient that is one number broadcast
    qd = q.detach().requires_grad_(True)
    (g1,) = torch.autograd.grad(ops.fused_cross_attention(qd, k, v).sum(), (qd,))
    assert torch.equal(g1, run(q, k, v, torch.ones_like(dout))[1])


def test_no_keys_no_queries_no_samples():
    q, k, v, dout = make(2, 5, 7, 4, 2, 16, torch.float16, 8)
    out, dq, dk, dv = run(q, k[:, :0], v[:, :0], dout)
    assert not bool(out.any()) and not bool(dq.any()) and dk.shape == (2, 0, 2, 16) and dv.shape == (2, 0, 2, 16)
    out, dq, dk, dv = run(q[:, :0], k, v, dout[:, :0])
    assert out.shape == (2, 0, 4, 16) and not bool(dk.any()) and not bool(dv.any()) and dk.shape == k.shape
    out, dq, dk, dv = run(q[:0], k[:0], v[:0], dout[:0])
    assert out.shape == (0, 5, 4, 16) and dk.shape == (0, 7, 2, 16)
    out, dq, dk, dv = run(q[:, :0], k[:, :0], v[:, :0], dout[:, :0])
    assert out.numel() == 0 and dk.numel() == 0


@pytest.mark.parametrize("b,n,m,h,hk,d", [(2, 300, 400, 4, 2, 72), (1, 4, 2000, 8, 1, 128), (1, 2000, 40, 2, 1, 64)])
def test_same_bits_every_time(b, n, m, h, hk, d):
    q, k, v, dout = make(b, n, m, h, hk, d, torch.bfloat16, 9)
    first = run(q, k, v, dout)
    for _ in range(3):
        for a, c in zip(run(q, k, v, dout), first):
            assert torch.equal(a, c)
    # a sample's results do not depend on its neighbours
    one = run(q[-1:], k[-1:], v[-1:], dout[-1:])
    if b > 1:
        want, bars = exact(q[-1:], k[-1:], v[-1:], dout[-1:], None, 1 / math.sqrt(d))
        check(one, want, bars)


def test_gradients_against_differences():
    q, k, v, dout = make(1, 40, 150, 2, 1, 32, torch.float16, 10, fused=False)
    lens = torch.tensor([140], device=DEV)
    got = run(q, k, v, dout, kv_lens=lens)
    def loss(q, k, v):
        return (ops.cross_attention_ref(q.double(), k.double(), v.double(), kv_lens=lens) * dout.double()).sum()
    g = torch.Generator().manual_seed(11)
    want, bars = exact(q, k, v, dout, torch.arange(150, device=DEV)[None] < lens[:, None], 1 / math.sqrt(32))
    for i, x in enumerate((q, k, v)):
        step = torch.randn(x.shape, generator=g).double().to(DEV) * 1e-4
        args = [[a.double() for a in (q, k, v)] for _ in range(2)]
        args[0][i] = args[0][i] + step
        args[1][i] = args[1][i] - step
        diff = float(loss(*args[0]) - loss(*args[1])) / 2
        # the difference itself is exact to second order in 1e-4 (third derivatives of order 1): 1e-8 beside 1e-4
        assert abs(diff - float((got[i + 1].double() * step).sum())) <= float((bars[i + 1] * step.abs()).sum()) + 1e-6 * float(step.abs().sum())


def test_partial_gradients_and_inference_mode():
    q, k, v, dout = make(2, 60, 50, 2, 2, 64, torch.bfloat16, 12)
    full = run(q, k, v, dout)
    qd = q.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.fused_cross_attention(qd, k, v), qd, dout)[0], full[1])
    vd = v.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.fused_cross_attention(q, k, vd), vd, dout)[0], full[3])
    with torch.inference_mode():
        assert torch.equal(ops.fused_cross_attention(q, k, v), full[0])


def test_streams_and_captured_graphs():
    q, k, v, dout = make(1, 3, 1500, 4, 4, 64, torch.bfloat16, 13)  # few rows: keys split, workspace in use
    q2, k2, v2, _ = make(1, 3, 1500, 4, 4, 64, torch.bfloat16, 14)
    want, want2 = ops.fused_cross_attention(q, k, v), ops.fused_cross_attention(q2, k2, v2)
    sides = [torch.cuda.Stream() for _ in range(2)]
    for st in sides:
        st.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for i, (st, args) in enumerate(zip(sides, ((q, k, v), (q2, k2, v2)))):
        with torch.cuda.stream(st):
            for _ in range(5):
                got[i] = ops.fused_cross_attention(*args)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want2)
    # two captured graphs replayed at the same time
    graphs, outs = [], []
    for args in ((q, k, v), (q2, k2, v2)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.fused_cross_attention(*args))
        graphs.append(graph)
    for _ in range(3):
        for st, graph in zip(sides, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_training_step_captured():
    q, k, v, dout = (x.clone() for x in make(2, 200, 90, 2, 2, 72, torch.bfloat16, 15))
    lens = torch.tensor([40, 90], dtype=torch.int32, device=DEV)
    want = run(q, k, v, dout, kv_lens=lens)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.fused_cross_attention(*leaves, kv_lens=lens)
        grads = torch.autograd.grad(out, leaves, dout)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((out.detach(), *grads), want):
        assert torch.equal(a, b)
    lens.fill_(0)  # the same graph on other lengths
    graph.replay()
    torch.cuda.synchronize()
    assert not bool(out.any()) and not any(bool(g.any()) for g in grads)


def test_one_key_takes_all_the_weight():
    """Nothing a query does changes the result: its gradient, and the key's, are exactly zero; v's is the sum."""
    for d, dtype in ((72, torch.bfloat16), (128, torch.float16)):
        q, k, v, dout = make(3, 200, 9, 4, 2, d, dtype, 17)
        out, dq, dk, dv = run(q, k, v, dout, kv_lens=torch.tensor([1, 1, 1], device=DEV))
        assert torch.equal(out, v[:, :1].repeat_interleave(2, dim=2).expand(3, 200, 4, d))
        assert not bool(dq.any()) and not bool(dk.any())


@pytest.mark.parametrize("kind", ["lens32", "holes"])
@pytest.mark.parametrize("b,n,m,h,hk,d", [(300, 20, 30, 2, 1, 64), (2, 9, 40000, 2, 2, 64), (300, 1, 30, 2, 2, 64), (70, 6, 1000, 2, 2, 72)])
def test_many_samples_and_long_masks(kind, b, n, m, h, hk, d):
    """More samples, or more mask, than the kernels keep key counts of."""
    q, k, v, dout = make(b, n, m, h, hk, d, torch.bfloat16, 18)
    key_mask, kv_lens, keep = masks(kind, b, m)
    want, bars = exact(q, k, v, dout, keep, 1 / math.sqrt(d))
    check(run(q, k, v, dout, key_mask=key_mask, kv_lens=kv_lens), want, bars)


@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** 11])
@pytest.mark.parametrize("n,m", [(150, 90), (64, 700)])
def test_gradients_of_other_magnitudes_in_fp16(size, n, m):
    """dS of these would leave fp16's range (its normal numbers end at 6e-5, its largest at 65504) without the kernels' powers
    of two: P is rounded times 2^floor(log2 m), dS times a power of two that brings the largest |dO| to 2^-4 or a little
    below 2^-3, so half of fp16's smallest number, 2^-25, becomes 2^-25 / 2^floor(log2 m) and at most 2^-21 of that |dO|."""
    q, k, v, dout = make(1, n, m, 2, 1, 64, torch.float16, 19)
    dout = (dout.float() / 8 * size).half()
    v = (v.float() * (8 if size > 1 else 1)).half()
    want, bars = exact(q, k, v, dout, None, 0.125, 2.0 ** -21 * float(dout.abs().max()), 2.0 ** -25 / 2 ** int(math.log2(m)))
    got = run(q, k, v, dout)
    check(got, want, bars)
    if size > 1:
        assert float((want[1].abs().max())) < 6e4  # the gradients themselves fit


def test_c_abi_helpers():
    from novadit_b200 import capi

    q, k, v, dout = make(2, 70, 90, 4, 2, 64, torch.float16, 20, fused=False)
    lens = torch.tensor([90, 31], dtype=torch.int32, device=DEV)
    want = run(q, k, v, dout, kv_lens=lens)
    out, lse = capi.attn_fwd(q, k, v, kv_lens=lens, with_lse=True)
    for a, b in zip((out, *capi.attn_bwd(dout, q, k, v, out, lse, kv_lens=lens)), want):
        assert torch.equal(a, b)
    keep = torch.arange(90, device=DEV)[None] < lens[:, None]
    assert torch.equal(capi.attn_fwd(q, k, v, key_mask=keep)[0], out)


def test_second_derivatives_are_refused():
    q, k, v, dout = make(1, 8, 8, 1, 1, 16, torch.bfloat16, 21)
    qd = q.detach().requires_grad_(True)
    (dq,) = torch.autograd.grad(ops.fused_cross_attention(qd, k, v), qd, dout, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), qd)


def test_refusals():
    q, k, v, dout = make(2, 6, 5, 4, 2, 16, torch.bfloat16, 16)
    keep = torch.ones(2, 5, dtype=torch.bool, device=DEV)
    lens = torch.tensor([5, 5], device=DEV)
    bad = [
        dict(q=q.float(), k=k.float(), v=v.float()), dict(q=q.half()), dict(k=k[:1]), dict(v=v[:, :4]), dict(k=k[..., :8]),
        dict(q=q[:, :, :3]), dict(q=q[0]), dict(key_mask=keep.int()), dict(key_mask=keep[:1]), dict(key_mask=keep[:, :4]),
        dict(key_mask=keep.cpu()), dict(kv_lens=lens.float()), dict(kv_lens=lens[:1]), dict(kv_lens=lens.cpu()),
        dict(key_mask=keep, kv_lens=lens), dict(scale=-1.0), dict(scale=0.0), dict(scale=1e-60), dict(scale=math.nan), dict(scale=math.inf), dict(k=k.cpu()),
        dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]),
        dict(q=torch.zeros(1, 2, 1, 136, dtype=q.dtype, device=DEV), k=torch.zeros(1, 2, 1, 136, dtype=q.dtype, device=DEV),
             v=torch.zeros(1, 2, 1, 136, dtype=q.dtype, device=DEV)),
    ]
    for kw in bad:
        args = dict(q=q, k=k, v=v) | kw
        with pytest.raises(RuntimeError):
            ops.fused_cross_attention(**args)
        with pytest.raises(RuntimeError):
            ops.fused_cross_attention(**(args | dict(q=args["q"].detach().requires_grad_(True))))
    with pytest.raises(RuntimeError, match="cross_attention_ref"):
        ops.fused_cross_attention(q.cpu(), k, v)
    from novadit_b200 import capi
    assert capi.lib().nd_device_error(0) == 0


@pytest.mark.parametrize("kind", ["none", "holes", "lens32"])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("n,h,hk", [(1, 2, 2), (1, 4, 2), (2, 2, 2), (1, 6, 2), (3, 1, 1), (1, 4, 1)])
def test_few_rows_of_every_head_size(kind, d, n, h, hk):
    """One to four query rows per key head, heads of three sharing among them; later keys score higher, so that the maximum
    moves all along."""
    b, m = 3, 1100
    dtype = torch.bfloat16 if n * h % 3 else torch.float16
    q, k, v, dout = make(b, n, m, h, hk, d, dtype, 21)
    k = (k.float() * torch.linspace(0.2, 2.0, m, device=DEV)[None, :, None, None]).to(dtype)
    key_mask, kv_lens, keep = masks(kind, b, m) if kind != "none" else (None, None, None)
    # fp16: most weights are small here and eight products hide little, so the rounding of dS below fp16's normal numbers
    # shows. The largest |dO| of the rows goes to 2^-4 or a little below 2^-3 (see above): half of fp16's smallest number,
    # 2^-25, is at most 2^-21 of that |dO| before the power of two is taken back.
    tiny_s = 2.0 ** -21 * float(dout.abs().max()) if dtype == torch.float16 else None
    want, bars = exact(q, k, v, dout, keep, 1 / math.sqrt(d), tiny_s)
    check(run(q, k, v, dout, key_mask=key_mask, kv_lens=kv_lens), want, bars)
