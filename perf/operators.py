"""Rotary positions and cross attention: the calls a diffusion transformer makes around its attention, in their plain
form (elementary torch operations in 32 bits, angles in 64, rounded once at the end) and, with `own` true, through this
framework's operators. Cases are dicts of plain values; `op` says which call a case is.

  rotary       y = a R(p f) x on [B, S, heads, D]: half or interleaved pairs, the first 2 R dimensions of a head
  pack_rotary  a fused projection [B, S, 3 heads D] split into q, k, v with q and k rotated; `train` adds its backward
  attention    softmax(scale q k^T) v over the keys of another sequence, padded keys masked; `train` adds its backward
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decoding step of a long conversation: eight sequences, one token each, far positions, context extended
        # by frequency bands; what counts is latency
        {"name": "rotary_token", "op": "rotary", "type": "fp16", "batch": 8, "seq": 1, "heads": 16, "dim": 128,
         "pairs": 64, "axes": 1, "interleaved": False, "scaling": "yarn", "reach": 131072, "train": False},
        # keys of a long document in 32 bits: a quarter of an odd batch, half of each head rotated in adjacent pairs,
        # positions interpolated
        {"name": "rotary_document", "op": "rotary", "type": "fp32", "batch": 3, "seq": 10007, "heads": 12, "dim": 64,
         "pairs": 16, "axes": 1, "interleaved": True, "scaling": "linear", "reach": 40000, "train": False},
        # the DiT-XL/2 block at 256 tokens (16 heads of 72, batch 32): row and column positions of the patches
        {"name": "pack_image", "op": "pack_rotary", "type": "bf16", "batch": 32, "seq": 256, "heads": 16, "dim": 72,
         "pairs": 36, "axes": 2, "interleaved": False, "scaling": "none", "reach": 64, "train": False},
        # a training step of the same block on a higher resolution (64 x 64 patches), forward and backward
        {"name": "pack_image_train", "op": "pack_rotary", "type": "bf16", "batch": 8, "seq": 4096, "heads": 16,
         "dim": 72, "pairs": 36, "axes": 2, "interleaved": False, "scaling": "ntk", "reach": 64, "train": True},
        # one query against one key: the smallest call there is
        {"name": "attention_one", "op": "attention", "type": "bf16", "batch": 1, "queries": 1, "keys": 1, "heads": 4,
         "kv_heads": 4, "dim": 64, "mask": "none", "fused_kv": True, "train": False},
        # one new token of each of 32 sequences reads its encoder's states, padded to a common length
        {"name": "attention_token", "op": "attention", "type": "bf16", "batch": 32, "queries": 1, "keys": 1500,
         "heads": 20, "kv_heads": 20, "dim": 64, "mask": "lens", "fused_kv": True, "train": False},
        # one token of two sequences against a very long memory, query heads sharing key heads
        {"name": "attention_memory", "op": "attention", "type": "fp16", "batch": 2, "queries": 1, "keys": 50021,
         "heads": 32, "kv_heads": 8, "dim": 128, "mask": "none", "fused_kv": False, "train": False},
        # the DiT-XL/2 block reads a prompt of 77 tokens, some of the prompts empty: sampling
        {"name": "attention_prompt", "op": "attention", "type": "bf16", "batch": 32, "queries": 256, "keys": 77,
         "heads": 16, "kv_heads": 16, "dim": 72, "mask": "mask", "fused_kv": True, "train": False},
        # the same while training, with a longer prompt and more patches
        {"name": "attention_prompt_train", "op": "attention", "type": "bf16", "batch": 16, "queries": 1024,
         "keys": 300, "heads": 16, "kv_heads": 16, "dim": 72, "mask": "lens", "fused_kv": True, "train": True},
        # ragged sizes, shared key heads and the other 16-bit type, forward and backward
        {"name": "attention_shared_train", "op": "attention", "type": "fp16", "batch": 3, "queries": 777, "keys": 1301,
         "heads": 12, "kv_heads": 4, "dim": 128, "mask": "mask", "fused_kv": False, "train": True},
        # the patches of a large image read one another, all 4096 of them: the largest forward pass
        {"name": "attention_image", "op": "attention", "type": "bf16", "batch": 4, "queries": 4096, "keys": 4096,
         "heads": 16, "kv_heads": 16, "dim": 72, "mask": "none", "fused_kv": False, "train": False},
        # and a training step of such an image with heads of 64
        {"name": "attention_image_train", "op": "attention", "type": "bf16", "batch": 2, "queries": 4096,
         "keys": 4096, "heads": 16, "kv_heads": 16, "dim": 64, "mask": "none", "fused_kv": False, "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "pack_rotary", "attention", "attention"])
    train = rng.random() < 0.5
    if op == "attention":
        dim = 8 * rng.randint(2, 16)
        kv_heads = rng.randint(1, 20)
        heads = kv_heads * rng.choice([1, 1, 1, 2, 3, 4])
        few = not train and rng.random() < 0.4  # serving: one or a few new tokens
        queries = rng.randint(1, 4) if few else _spread(rng, 1, 4096)
        keys = _spread(rng, 1, 50000 if few else 4096)
        most = 4 * 4096 * 4096 * 16 * 72  # no more than the largest listed case, in products and in elements
        batch = max(1, min(_spread(rng, 1, 64), most // (queries * keys * heads * max(dim, 64) * (4 if train else 1)),
                           160_000_000 // (keys * kv_heads * dim), 60_000_000 // (queries * heads * dim)))
        return {"op": op, "type": rng.choice(["bf16", "fp16"]), "batch": batch, "queries": queries, "keys": keys,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "mask": rng.choice(["none", "lens", "mask"]),
                "fused_kv": rng.random() < 0.5, "train": train}
    axes = rng.choice([1, 1, 2, 3])
    dim = rng.choice([32, 48, 64, 72, 80, 96, 120, 128])
    part = rng.choice([1, 1, 2, 4])
    pairs = max(1, dim // (2 * part * axes)) * axes
    heads = rng.randint(1, 24)
    seq = 1 if rng.random() < 0.2 else _spread(rng, 2, 16000)
    wide = heads * dim * (3 if op == "pack_rotary" else 1)
    batch = max(1, min(_spread(rng, 1, 64), 110_000_000 // (seq * wide)))
    return {"op": op, "type": rng.choice(["bf16", "fp16", "fp32"]), "batch": batch, "seq": seq, "heads": heads,
            "dim": dim, "pairs": pairs, "axes": axes, "interleaved": rng.random() < 0.5,
            "scaling": rng.choice(["none", "linear", "ntk", "yarn"]) if axes == 1 else "none",
            "reach": _spread(rng, 16, 1_000_000), "train": train}


def _frequencies(case):
    """([axes, pairs / axes] radians per position in 64 bits, the factor on cosine and sine) of a case."""
    r = case["pairs"] // case["axes"]
    base, factor, original = 10000.0, 8.0, 8192.0
    rot = 2 * r
    if case["scaling"] == "ntk":
        base *= factor ** (rot / max(rot - 2, 1))
    i = torch.arange(r, dtype=torch.float64)
    f = base ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "yarn":  # bands that turn often keep their frequency, slow ones are interpolated
        at = [rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        return f.expand(case["axes"], r).contiguous(), 0.1 * math.log(factor) + 1.0
    return f.expand(case["axes"], r).contiguous(), 1.0


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(t)

    if case["op"] == "attention":
        b, n, m, h, hk, d = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        s = {"case": case, "q": normal(b, n, h, d), "lens": None, "mask": None}
        if case["fused_kv"]:  # one projection gives keys and values side by side: two strided views
            s["k"], s["v"] = normal(b, m, 2, hk, d).unbind(2)
        else:
            s["k"], s["v"] = normal(b, m, hk, d), normal(b, m, hk, d)
        if case["mask"] != "none":  # lengths of a padded batch, one empty prompt among several
            lens = torch.randint(1, m + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            if b >= 3:
                lens[seed % b] = 0
            if case["mask"] == "lens":
                s["lens"] = lens
            else:
                s["mask"] = torch.arange(m, device="cuda")[None] < lens[:, None]
        if case["train"]:
            s["q"].requires_grad_(True)
            s["k"] = s["k"].detach().requires_grad_(True)
            s["v"] = s["v"].detach().requires_grad_(True)
            s["dout"] = normal(b, n, h, d)
        return s
    b, n, h, d = (case[x] for x in ("batch", "seq", "heads", "dim"))
    freqs, factor = _frequencies(case)
    pos = torch.randint(0, case["reach"], (b, n, case["axes"]), generator=g, device="cuda", dtype=torch.int64)
    s = {"case": case, "freqs": freqs.cuda(), "factor": factor, "pos": pos}
    if case["op"] == "rotary":
        s["x"] = normal(b, n, h, d).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = normal(b, n, h, d)
    else:
        s["x"] = normal(b, n, 3 * h * d).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = [normal(b, n, h, d) for _ in range(3)]
    return s


def _tables(s):
    """Cosine and sine of position times frequency, [B, S, 1, pairs]: the angle and both in 64 bits, then 32."""
    angle = (s["pos"].double()[..., None] * s["freqs"]).flatten(2)[:, :, None]
    return (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()


def _turned(x, cos, sin, pairs, interleaved):
    """The first 2 * pairs dimensions of each head turned, the others as they are; in 32 bits."""
    x = x.float()
    rot, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = rot[..., :pairs], rot[..., pairs:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([rot, rest], dim=-1)


def _plain_rotary(s):
    c, t = s["case"], s["x"].dtype
    cos, sin = _tables(s)
    x = s["x"].detach()
    if c["op"] == "rotary":
        y = _turned(x, cos, sin, c["pairs"], c["interleaved"]).to(t)
        if not c["train"]:
            return y
        return y, _turned(s["dy"], cos, -sin, c["pairs"], c["interleaved"]).to(t)
    q, k, v = x.view(c["batch"], c["seq"], 3, c["heads"], c["dim"]).unbind(2)
    out = [_turned(q, cos, sin, c["pairs"], c["interleaved"]).to(t),
           _turned(k, cos, sin, c["pairs"], c["interleaved"]).to(t), v.contiguous()]
    if c["train"]:
        dq, dk, dv = s["dy"]
        out.append(torch.cat([_turned(dq, cos, -sin, c["pairs"], c["interleaved"]).to(t).flatten(2),
                              _turned(dk, cos, -sin, c["pairs"], c["interleaved"]).to(t).flatten(2), dv.flatten(2)], dim=-1))
    return out


def _plain_attention(s):
    c, t = s["case"], s["q"].dtype
    b, n, m, h, hk, d = (c[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    scale = 1.0 / math.sqrt(d)
    q = s["q"].detach().float().view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4)  # [B, kv heads, group, n, d]
    k = s["k"].detach().float().permute(0, 2, 1, 3)[:, :, None]
    v = s["v"].detach().float().permute(0, 2, 1, 3)[:, :, None]
    keep = s["mask"]
    if s["lens"] is not None:
        keep = torch.arange(m, device="cuda")[None] < s["lens"][:, None]
    w = (q @ k.transpose(-1, -2)) * scale
    if keep is not None:
        w = w.masked_fill(~keep[:, None, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)  # a row without keys: weights of zero
    w = (w - top).exp()
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    o = w @ v
    out = o.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(t)
    if not c["train"]:
        return out
    do = s["dout"].float().view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    dv = (w.transpose(-1, -2) @ do).sum(2)
    ds = (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * w * scale
    dq = (ds @ k).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return out, dq.to(t), dk.permute(0, 2, 1, 3).contiguous().to(t), dv.permute(0, 2, 1, 3).contiguous().to(t)


def run(s):
    c = s["case"]
    if not own:
        return _plain_attention(s) if c["op"] == "attention" else _plain_rotary(s)
    from novadit_b200 import ops

    if c["op"] == "attention":
        out = ops.fused_cross_attention(s["q"], s["k"], s["v"], key_mask=s["mask"], kv_lens=s["lens"])
        if not c["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    if c["op"] == "rotary":
        y = ops.fused_rotary(s["x"], s["pos"], s["freqs"], interleaved=c["interleaved"], attention_factor=s["factor"])
        if not c["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
    q, k, v = ops.fused_qkv_pack_rotary(s["x"], c["heads"], c["dim"], s["pos"], s["freqs"],
                                        interleaved=c["interleaved"], attention_factor=s["factor"])
    if not c["train"]:
        return [q, k, v]
    return [q.detach(), k.detach(), v.detach(), torch.autograd.grad((q, k, v), s["x"], s["dy"])[0]]


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "attention":
        b, n, m, h, hk, d = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        if case["mask"] != "none":  # lengths are drawn from 1..keys: half of the keys on average
            m = (m + 1) / 2
        one = 2.0 * b * h * n * m * d  # one of the products
        rows, cols = b * n * h * d * size, b * m * hk * d * size
        if not case["train"]:
            return {"bytes": 2 * rows + 2 * cols, "flops": 2 * one}
        # forward: q, k, v in, out written; backward: q, k, v, out, dout in, three gradients written; 2 + 5 products
        return {"bytes": 2 * rows + 2 * cols + 4 * rows + 4 * cols, "flops": 7 * one}
    wide = case["batch"] * case["seq"] * case["heads"] * case["dim"] * (3 if case["op"] == "pack_rotary" else 1)
    turned = case["batch"] * case["seq"] * case["heads"] * case["pairs"] * (2 if case["op"] == "pack_rotary" else 1)
    passes = 2 if case["train"] else 1
    return {"bytes": passes * (2 * wide * size + 8 * case["batch"] * case["seq"] * case["axes"]), "flops": passes * 6 * turned}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    # every pair as a complex number, turned by e^(i angle)
    f = s["freqs"]
    angle = torch.einsum("bsa,ar->bsar", s["pos"].double(), f).reshape(case["batch"], case["seq"], 1, case["pairs"])
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)

    def turned(x, by):
        y = x.detach().double().clone()
        r = case["pairs"]
        if case["interleaved"]:
            z = torch.complex(y[..., 0:2 * r:2].contiguous(), y[..., 1:2 * r:2].contiguous()) * by
            y[..., 0:2 * r:2], y[..., 1:2 * r:2] = z.real, z.imag
        else:
            z = torch.complex(y[..., :r].contiguous(), y[..., r:2 * r].contiguous()) * by
            y[..., :r], y[..., r:2 * r] = z.real, z.imag
        return y

    if case["op"] == "rotary":
        y = turned(s["x"], turn)
        return (y, turned(s["dy"], turn.conj())) if case["train"] else y
    shape = (case["batch"], case["seq"], 3, case["heads"], case["dim"])
    x = s["x"].detach().reshape(shape)
    out = [turned(x[:, :, 0], turn), turned(x[:, :, 1], turn), x[:, :, 2].double()]
    if case["train"]:
        dq, dk, dv = s["dy"]
        out.append(torch.stack([turned(dq, turn.conj()), turned(dk, turn.conj()), dv.double()], dim=2).reshape(*shape[:2], -1))
    return out


def _exact_attention(case, s):
    """One sample and one key head after the other, in 64 bits, over the keys that take part alone."""
    b, hk, group, d = case["batch"], case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    q, k, v = (s[x].detach() for x in "qkv")
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    if case["train"]:
        dq = torch.zeros_like(out)
        dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device=k.device) for _ in range(2))
    for i in range(b):
        here = slice(0, case["keys"])
        if s["lens"] is not None:
            here = slice(0, int(s["lens"][i]))
        if s["mask"] is not None:
            here = s["mask"][i].nonzero()[:, 0]
        for j in range(hk):
            heads = slice(j * group, (j + 1) * group)
            qi, ki, vi = q[i, :, heads].double(), k[i, here, j].double(), v[i, here, j].double()
            if not ki.shape[0]:
                continue
            w = torch.softmax(torch.einsum("nhd,md->hnm", qi, ki) / math.sqrt(d), dim=-1)
            out[i, :, heads] = torch.einsum("hnm,md->nhd", w, vi)
            if case["train"]:
                gi = s["dout"][i, :, heads].double()
                dv[i, here, j] = torch.einsum("hnm,nhd->md", w, gi)
                dw = torch.einsum("nhd,md->hnm", gi, vi)
                ds = w * (dw - (w * dw).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i, :, heads] = torch.einsum("hnm,md->nhd", ds, ki)
                dk[i, here, j] = torch.einsum("hnm,nhd->md", ds, qi)
    return (out, dq, dk, dv) if case["train"] else out
