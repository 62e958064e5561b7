"""Timing cases of the conditioning operators: a prompt or an image encoder's states on their way into the DiT stream.

``k2b.ops.w4_linear``       a few rows times INT4 weights with group-128 scales (timestep MLP, modulation, encoder K/V)
``k2b.ops.qk_norm_rope``    RMSNorm of every query and key head with the position rotation, in one pass
``k2b.ops.cross_attention`` attention of one sequence to the states of another, with per-latent lengths, masks and biases

``listed`` and ``draw`` give the cases, ``prepare`` their inputs, ``run`` one call (plain torch in 32 bits, or with
``own`` the library's operators), ``exact`` the same from the definitions in 64 bits and ``work`` the bytes and
operations that one call cannot do without.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def listed():
    return [
        # the timestep MLP's first layer at one latent: the smallest product, its launch is its cost
        dict(name="w4-timestep", op="w4", rows=1, n=6144, k=256, dtype="bf16", bias=True, act="gelu", rotate=False),
        # the six modulation vectors of one latent (tproj): 113 MB of weights for one row
        dict(name="w4-modulation-1", op="w4", rows=1, n=36864, k=6144, dtype="bf16", bias=True, act="none", rotate=True),
        # the same for a batch of eight latents
        dict(name="w4-modulation-8", op="w4", rows=8, n=36864, k=6144, dtype="bf16", bias=True, act="none", rotate=True),
        # an odd number of encoder tokens to the keys of 12 heads
        dict(name="w4-encoder-keys", op="w4", rows=77, n=1536, k=2560, dtype="fp16", bias=False, act="none", rotate=True),
        # one query and one key token
        dict(name="norm-token", op="norm", batch=1, lq=1, lk=1, heads=48, kvheads=12, dim=128, dtype="bf16", rope="both"),
        # self-attention's queries and keys of one latent at 4050 tokens, views of the fused projection
        dict(name="norm-stream", op="norm", batch=1, lq=4050, lk=4050, heads=48, kvheads=12, dim=128, dtype="bf16", rope="both"),
        # queries of eight latents at 4224 tokens, keys of a short prompt that carry no positions
        dict(name="norm-cross", op="norm", batch=8, lq=4224, lk=154, heads=48, kvheads=12, dim=128, dtype="fp16", rope="q"),
        # a single token against a long encoder sequence
        dict(name="attn-token", op="attn", batch=1, heads=48, kvheads=12, lq=1, lk=4096, dim=128, dtype="bf16",
             lengths="full", regions=0, bias=False, shared=False),
        # sixteen learned queries against ragged image-encoder states, one latent's encoder sequence empty
        dict(name="attn-queries", op="attn", batch=4, heads=20, kvheads=20, lq=16, lk=729, dim=64, dtype="fp16",
             lengths="ragged0", regions=0, bias=False, shared=False),
        # image tokens against two prompts of different length with per-token emphasis
        dict(name="attn-prompt", op="attn", batch=2, heads=48, kvheads=12, lq=4050, lk=154, dim=128, dtype="bf16",
             lengths="ragged", regions=0, bias=True, shared=False),
        # regional prompts: each image token sees its region's part of the prompt, some tokens see none
        dict(name="attn-regions", op="attn", batch=1, heads=48, kvheads=12, lq=4096, lk=1000, dim=128, dtype="fp16",
             lengths="full", regions=4, bias=False, shared=False),
        # eight latents of one long prompt: the largest
        dict(name="attn-long", op="attn", batch=8, heads=48, kvheads=12, lq=4224, lk=2048, dim=128, dtype="bf16",
             lengths="full", regions=0, bias=False, shared=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["w4", "norm", "attn", "attn"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "w4":
        k = 128 * _log(rng, 1, 128)
        return dict(op=op, rows=_log(rng, 1, 96), n=_log(rng, 1, min(36864, 36864 * 6144 // k)), k=k, dtype=dtype,
                    bias=rng.random() < 0.5, act=rng.choice(["none", "gelu", "silu"]), rotate=rng.random() < 0.7)
    heads, kvheads = rng.choice([(48, 12), (24, 6), (20, 20), (8, 2), (6, 2), (5, 5)])
    dim = rng.choice([64, 128, 128])
    batch = _log(rng, 1, 8)
    if op == "norm":
        lq = _log(rng, 1, 4224)
        same = rng.random() < 0.5
        return dict(op=op, batch=batch, lq=lq, lk=lq if same else _log(rng, 1, 4224), heads=heads, kvheads=kvheads,
                    dim=dim, dtype=dtype, rope=rng.choice(["both", "both", "q", "none"]))
    return dict(op=op, batch=batch, heads=heads, kvheads=kvheads, lq=_log(rng, 1, 4224), lk=_log(rng, 1, 2048),
                dim=dim, dtype=dtype, lengths=rng.choice(["full", "ragged", "ragged0"]), regions=rng.choice([0, 0, 0, 3, 5]),
                bias=rng.random() < 0.3, shared=rng.random() < 0.25)


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """The keys that each latent attends to, by the case alone."""
    b, lk = case["batch"], case["lk"]
    if case["lengths"] == "full":
        return [lk] * b
    some = [max(1, lk * (b - i) // b - (i % 2)) for i in range(b)]
    if case["lengths"] == "ragged0":
        some[-1] = 0
    return some


def _region_mask(case, gen):
    """bool [1, 1, lq, lk]: token i sees a prompt head of lk/8 keys and its region's share of the rest; one token in
    32 sees nothing."""
    lq, lk, r = case["lq"], case["lk"], case["regions"]
    head = lk // 8
    token = torch.arange(lq, device="cuda") * r // lq
    key = (torch.arange(lk, device="cuda") - head).clamp(min=0) * r // max(1, lk - head)
    see = (token[:, None] == key[None, :]) | (torch.arange(lk, device="cuda") < head)[None, :]
    none = torch.rand(lq, generator=gen, device="cuda") < 1 / 32
    return (see & ~none[:, None]).view(1, 1, lq, lk)


def _table(length, dim):
    """The rotation table of a 64-wide token grid, fp32 [length, dim/2, 2, 2]: half of the dimensions turn with the
    row, half with the column."""
    i = torch.arange(length, device="cuda", dtype=torch.float64)
    pos = torch.stack([i // 64, i % 64], 1)
    q = dim // 4
    omega = 10000.0 ** (-torch.arange(q, device="cuda", dtype=torch.float64) / q)
    a = (pos[:, :, None] * omega).reshape(length, 2 * q)
    return torch.stack([a.cos(), -a.sin(), a.sin(), a.cos()], -1).view(length, dim // 2, 2, 2).float().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "w4":
        rows, n, k = case["rows"], case["n"], case["k"]
        w = (randn(n, k) * 0.02).view(n, k // 128, 128)
        scales = (w.abs().amax(-1) / 7).half()
        codes = torch.round(w / scales[..., None].float()).clamp_(-8, 7).to(torch.int8).view(n, k)
        packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).view(torch.uint8)
        x = randn(rows, k)
        x[:, :: 97] *= 8.0  # a few loud channels
        return dict(case=case, x=x.to(dt), packed=packed.contiguous(), scales=scales.contiguous(),
                    bias=(randn(n) * 0.02).to(dt) if case["bias"] else None)
    h, hk, d, b, lq, lk = (case[x] for x in ("heads", "kvheads", "dim", "batch", "lq", "lk"))
    if case["op"] == "norm":
        if lq == lk:
            fused = randn(b, lq, h + 2 * hk, d).to(dt)  # one projection's queries, keys and values
            q, k = fused[:, :, :h], fused[:, :, h:h + hk]
        else:
            q, k = randn(b, lq, h, d).to(dt), randn(b, lk, 2 * hk, d).to(dt)[:, :, :hk]
        return dict(case=case, q=q.transpose(1, 2), k=k.transpose(1, 2),
                    wq=torch.rand(d, generator=gen, device="cuda") * 0.2 - 0.1,
                    wk=torch.rand(d, generator=gen, device="cuda") * 0.2 - 0.1,
                    fq=_table(lq, d) if case["rope"] in ("both", "q") else None,
                    fk=_table(lk, d) if case["rope"] == "both" else None)
    bk = 1 if case["shared"] else b

    def unit(t):  # what the head norms leave
        return (t * torch.rsqrt(t.square().mean(-1, keepdim=True))).to(dt).transpose(1, 2)

    bias = None
    if case["bias"]:  # the logarithm of prompt weights between 0.8 and 1.5
        bias = torch.log(0.8 + 0.7 * torch.rand(b, lk, generator=gen, device="cuda"))
    return dict(case=case, q=unit(randn(b, lq, h, d)), k=unit(randn(bk, lk, hk, d)),
                v=randn(bk, lk, hk, d).to(dt).transpose(1, 2), bias=bias,
                lengths=None if case["lengths"] == "full" else torch.tensor(_lengths(case), dtype=torch.int32, device="cuda"),
                mask=_region_mask(case, gen) if case["regions"] else None)


# --------------------------------------------------------------- one call

def _ops():
    sub = os.path.join(ROOT, "comfyui-k2-precompile_b200")
    if sub not in sys.path:
        sys.path.insert(0, sub)
    from k2b import ops

    return ops


def run(state):
    op = state["case"]["op"]
    if own:
        ops = _ops()
        if op == "w4":
            return ops.w4_linear(state["x"], state["packed"], state["scales"], state["bias"],
                                 rotate=state["case"]["rotate"], act=state["case"]["act"])
        if op == "norm":
            return ops.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"], state["fq"], state["fk"])
        return ops.cross_attention(state["q"], state["k"], state["v"], lengths=state["lengths"], mask=state["mask"],
                                   bias=state["bias"])
    return {"w4": _plain_w4, "norm": _plain_norm, "attn": _plain_attn}[op](state)


def _hadamard():
    i = torch.arange(128, device="cuda")
    bits = i[:, None] & i[None, :]
    odd = bits ^ (bits >> 4)
    odd = odd ^ (odd >> 2)
    odd = (odd ^ (odd >> 1)) & 1
    return (1.0 - 2.0 * odd.float()) / math.sqrt(128.0)


def _plain_w4(s):
    x, packed, case = s["x"], s["packed"], s["case"]
    n, k = packed.shape[0], 2 * packed.shape[1]
    low, high = (packed & 15).float(), (packed >> 4).float()
    codes = torch.stack([low - 16 * (low > 7), high - 16 * (high > 7)], -1).view(n, k // 128, 128)
    w = (codes * s["scales"].float()[..., None]).view(n, k)
    y = x.float()
    if case["rotate"]:
        y = (y.view(-1, k // 128, 128) @ _hadamard()).view(-1, k)
    y = y @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    return y.to(x.dtype)


def _plain_norm(s):
    def one(t, w, f):
        y = t.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (w + 1)
        if f is not None:
            p = y.unflatten(-1, (-1, 2))
            y = (f[..., 0] * p[..., 0:1] + f[..., 1] * p[..., 1:2]).flatten(-2)
        return y.to(t.dtype)

    return one(s["q"], s["wq"], s["fq"]), one(s["k"], s["wk"], s["fk"])


def _plain_attn(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, h, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    g = h // hk
    scores = (q.float().reshape(b, hk, g * lq, d) @ k.float().transpose(-1, -2)).view(b, hk, g, lq, lk) / math.sqrt(d)
    if s["bias"] is not None:
        scores = scores + s["bias"].view(b, 1, 1, 1, lk)
    if s["lengths"] is not None:
        out = torch.arange(lk, device=q.device) >= s["lengths"][:, None]
        scores = scores.masked_fill(out.view(b, 1, 1, 1, lk), -math.inf)
    if s["mask"] is not None:
        scores = scores.masked_fill(~s["mask"].unsqueeze(2), -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    o = e.view(b, hk, g * lq, lk) @ v.float()
    total = e.sum(-1).view(b, hk, g * lq, 1)
    o = torch.where(total > 0, o / total, 0.0)  # a row that sees no key is zero
    return o.view(b, h, lq, d).transpose(1, 2).reshape(b, lq, h * d).to(q.dtype)


# ------------------------------------------------------------- definitions

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "w4":
        x = s["x"].to(f64)
        rows, k = x.shape
        if case["rotate"]:  # butterflies over the seven index bits of each group of 128
            x = x.view(rows, k // 128, *([2] * 7))
            for bit in range(2, 9):
                a, b = x.select(bit, 0), x.select(bit, 1)
                x = torch.stack([a + b, a - b], bit)
            x = x.reshape(rows, k) * 128.0 ** -0.5
        out = torch.empty((rows, case["n"]), dtype=f64, device="cuda")
        for at in range(0, case["n"], 4096):
            p = s["packed"][at:at + 4096].to(torch.int16)
            c = torch.stack([((p & 15) ^ 8) - 8, ((p >> 4) ^ 8) - 8], -1).reshape(p.shape[0], k).to(f64)
            c *= s["scales"][at:at + 4096].to(f64).repeat_interleave(128, 1)
            out[:, at:at + 4096] = x @ c.t()
        if s["bias"] is not None:
            out += s["bias"].to(f64)
        if case["act"] == "gelu":
            out = out / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (out + 0.044715 * out ** 3)))
        elif case["act"] == "silu":
            out = out / (1 + torch.exp(-out))
        return out
    if case["op"] == "norm":
        res = []
        for t, w, f in ((s["q"], s["wq"], s["fq"]), (s["k"], s["wk"], s["fk"])):
            y = t.to(f64)
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["dim"] + 1e-6) * (1 + w.to(f64))
            if f is not None:
                m = f.to(f64)
                y = torch.einsum("lpij,bhlpj->bhlpi", m, y.unflatten(-1, (-1, 2))).flatten(-2)
            res.append(y)
        return tuple(res)
    b, h, hk, lq, d = case["batch"], case["heads"], case["kvheads"], case["lq"], case["dim"]
    out = torch.zeros((b, lq, h, d), dtype=f64, device="cuda")
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        for j in range(h):
            kk, vv = (s[x][0 if case["shared"] else i, j * hk // h, :n].to(f64) for x in ("k", "v"))
            t = s["q"][i, j].to(f64) @ kk.t() * d ** -0.5
            if s["bias"] is not None:
                t = t + s["bias"][i, :n].to(f64)
            if s["mask"] is not None:
                t = torch.where(s["mask"][0, 0, :, :n], t, -math.inf)
            out[i, :, j] = torch.nan_to_num(torch.softmax(t, -1), nan=0.0) @ vv
    return out.view(b, lq, h * d)


def work(case):
    """Each input read once and each output written once; of the attention's keys those within the lengths and, for
    regions, the share of pairs that the mask leaves."""
    if case["op"] == "w4":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k // 2 + n * k // 64 + 2 * rows * (k + n) + (2 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    b, h, hk, lq, lk, d = (case[x] for x in ("batch", "heads", "kvheads", "lq", "lk", "dim"))
    if case["op"] == "norm":
        tables = (lq if case["rope"] in ("both", "q") else 0) + (lk if case["rope"] == "both" else 0)
        values = b * (lq * h + lk * hk) * d
        return {"bytes": 4 * values + 8 * d * tables, "flops": 8 * values}
    keys = _lengths(case)
    read = max(keys) if case["shared"] else sum(keys)
    pairs = sum(keys) * lq
    bytes_ = 4 * b * lq * h * d + 4 * read * hk * d + (4 * sum(keys) if case["bias"] else 0)
    if case["regions"]:
        pairs = int(pairs * (1 / 8 + 7 / 8 / case["regions"]))
        bytes_ += lq * lk
    return {"bytes": bytes_, "flops": 4 * pairs * h * d}
