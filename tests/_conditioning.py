"""The conditioning operators' definitions in 64 bits, for the GPU tests, and the bounds that their arithmetic allows."""
import math

import torch

F64 = torch.float64
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # unit roundoff


def codes_of(packed):
    p = packed.to(torch.int16)
    return torch.stack([((p & 15) ^ 8) - 8, ((p >> 4) ^ 8) - 8], -1).flatten(1)


def random_w4(n, k, gen, device):
    """A weight whose every code, the whole nibble range, occurs."""
    packed = torch.randint(0, 256, (n, k // 2), generator=gen, device=device, dtype=torch.uint8)
    scales = (torch.rand(n, k // 128, generator=gen, device=device) * 0.02 + 1e-3).half()
    return packed, scales


def hadamard(device):
    h = torch.ones(1, 1, dtype=F64, device=device)
    for _ in range(7):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(128.0)


def w4_linear(x, packed, scales, bias, rotate, act):
    """(y, bound): the exact product and what |got - y| may be.

    The output is rounded once (u |y|).  A rotated row's values are rounded to fp16 relative to themselves (2^-11 each,
    and 2^-25 of the group's largest value where they are smaller than 2^-14 of the fp16 range), a sum of k fp32
    products errs by less than 2^-17 of the sum of magnitudes at these k, and gelu and silu stretch an error by at
    most 1.13."""
    n, k = packed.shape[0], packed.shape[1] * 2
    w = codes_of(packed).to(F64).view(n, k // 128, 128) * scales.to(F64)[..., None]
    w = w.view(n, k)
    xr = x.to(F64).reshape(-1, k)
    if rotate:
        xr = (xr.view(-1, k // 128, 128) @ hadamard(x.device)).view(-1, k)
    y = xr @ w.t()
    mag = xr.abs() @ w.abs().t()
    if bias is not None:
        y = y + bias.to(F64)
        mag = mag + bias.to(F64).abs()
    err = mag * ((2.0 ** -11 if rotate else 0.0) + 2.0 ** -17)
    if act == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    elif act == "silu":
        y = y * torch.sigmoid(y)
    u = UNIT[x.dtype]
    return y.view(*x.shape[:-1], n), (u * y.abs() + 1.13 * err + 2.0 ** -24).view(*x.shape[:-1], n)


def norm_rope(x, w, freqs, eps):
    """(y, bound) of one side, x [B, H, L, D]: one rounding of the output and some twenty fp32 steps on values of at
    most sqrt(D) (w + 1)."""
    D = x.shape[-1]
    y = x.to(F64)
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (w.to(F64) + 1)
    mag = y.abs()
    if freqs is not None:
        f = freqs.to(F64).view(-1, 1, x.shape[2], D // 2, 2, 2)
        pair = y.unflatten(-1, (-1, 2)).unsqueeze(-2)
        mag = (f.abs() * pair.abs()).sum(-1).flatten(-2)
        y = (f * pair).sum(-1).flatten(-2)
    return y, UNIT[x.dtype] * y.abs() + 2.0 ** -19 * mag + 2.0 ** -25


def keep_mask(B, H, Lq, Lk, lengths, mask, bias, device):
    keep = torch.ones(B, H, Lq, Lk, dtype=torch.bool, device=device)
    if lengths is not None:
        keep &= (torch.arange(Lk, device=device) < lengths.clamp(0, Lk).view(B, 1).long()).view(B, 1, 1, Lk)
    if mask is not None:
        keep &= mask if mask.dim() == 4 else mask[:, None, None, :]
    if bias is not None:
        keep &= (bias != -math.inf)[:, None, None, :]
    return keep


def cross_attention(q, k, v, lengths=None, mask=None, bias=None, scale=None):
    """(o, bound).  P is rounded to the type of V (u of each probability, and 2^-25 below fp16's normal range), the
    output once more; fp32 scores of magnitude s err by 2^-17 s, which changes a probability by as much."""
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    keep = keep_mask(B, H, Lq, Lk, lengths, mask, bias, q.device)
    any_row = keep.any(2, keepdim=True)  # [B, H, 1, Lk]
    kk = k.to(F64).expand(B, -1, -1, -1).repeat_interleave(H // Hk, 1)
    vv = v.to(F64).expand(B, -1, -1, -1).repeat_interleave(H // Hk, 1)
    kk = torch.where(any_row.transpose(-1, -2), kk, 0.0)  # what a key nobody sees holds does not count
    vv = torch.where(any_row.transpose(-1, -2), vv, 0.0)
    s = q.to(F64) @ kk.transpose(-1, -2) * scale
    smag = q.to(F64).abs() @ kk.abs().transpose(-1, -2) * abs(scale)
    if bias is not None:
        bb = torch.where(bias == -math.inf, 0.0, bias.to(F64))[:, None, None, :]
        s, smag = s + bb, smag + bb.abs()
    s = torch.where(keep, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = torch.where(keep, p, 0.0)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = p @ vv
    u = UNIT[q.dtype]
    worst = torch.where(keep, smag, 0.0).amax(-1, keepdim=True) if Lk else torch.zeros_like(total)
    pmag = p @ vv.abs()
    tiny = 2.0 ** -24 * vv.abs().sum(2, keepdim=True) if q.dtype == torch.float16 else 0.0
    bound = u * o.abs() + (u + 2 * 2.0 ** -17 * worst + 2.0 ** -18) * pmag + tiny + 2.0 ** -24
    flat = lambda t: t.transpose(1, 2).reshape(B, Lq, H * D)  # noqa: E731
    return flat(o), flat(bound)


def check(got, want, bound, what=""):
    g = got.to(F64)
    assert torch.isfinite(g).all(), f"{what}: not finite"
    over = (g - want).abs() / bound
    assert float(over.max() if over.numel() else 0.0) <= 1.0, f"{what}: {float(over.max()):.3f} of the bound"
