"""The conditioning path run together: the image-prompt adapter against its formula in 64 bits, and the DiT forward with
INT4 conditioning weights and an image prompt."""
import numpy as np
import pytest
import torch

import _conditioning as R
from _helpers import TOL_COS, cosine

pytestmark = pytest.mark.gpu


def _dequant(w):
    """The plain weight that a W4Linear stands for, fp64."""
    n, k = w.packed.shape[0], 2 * w.packed.shape[1]
    full = (R.codes_of(w.packed).double().view(n, k // 128, 128) * w.scales.double()[..., None])
    if w.rotate:
        full = full @ R.hadamard(full.device)
    return full.reshape(n, k)


def test_adapter_matches_its_formula(cuda):
    from k2b import ops
    from k2b.adapter import synthetic_adapter
    from k2b.model import ModelConfig, rope_positions, rope_table

    cfg = ModelConfig(hidden=512, heads=8, kvheads=2, mlp=1024, blocks=1)
    a = synthetic_adapter(cfg, width=640, seed=1, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(2)
    B, L, E = 2, 150, 77
    x = torch.randn(B, L, 512, generator=gen, device=cuda).to(torch.bfloat16)
    states = torch.randn(B, E, 640, generator=gen, device=cuda).to(torch.bfloat16)
    lengths = torch.tensor([77, 20], dtype=torch.int32, device=cuda)
    emphasis = torch.rand(B, E, generator=gen, device=cuda) + 0.5
    freqs = rope_table(rope_positions(6, 12, 12), (64, 64), cfg.theta).to(cuda)
    kept = a.keys(states, lengths, emphasis)
    got = a.attend(x, kept, freqs)
    # the same in 64 bits from the plain weights; the query projection is the W4A4 GEMM's own (tested elsewhere)
    heads = lambda t, h: t.view(B, -1, h, 128).transpose(1, 2)  # noqa: E731
    k = heads(states.double() @ _dequant(a.wk).t(), 2)
    v = heads(states.double() @ _dequant(a.wv).t(), 2)
    k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + cfg.qk_eps) * (a.knorm.double() + 1)
    q = ops.gemm_bf16(*ops.rotate_quant(x.view(B * L, 512)), a.wq)
    q, _ = R.norm_rope(heads(q, 8), a.qnorm, freqs, cfg.qk_eps)
    s = q @ k.repeat_interleave(4, 1).transpose(-1, -2) / 128 ** 0.5 + torch.log(emphasis.double())[:, None, None]
    s = s.masked_fill(torch.arange(E, device=cuda) >= lengths.view(B, 1, 1, 1), -torch.inf)
    want = (torch.softmax(s, -1) @ v.repeat_interleave(4, 1)).transpose(1, 2).reshape(B, L, 1024)
    # bf16 queries, keys, values, probabilities and output: five roundings of 2^-9 rms/sqrt(3) each, and scores of
    # unit size carry theirs into the probabilities
    rel = float((got.double() - want).norm() / want.norm())
    assert rel < 5 * 2.0 ** -9, rel
    # strength 0 leaves the stream, and the output is the residual plus the projection
    assert torch.equal(a.add(x, kept, freqs=freqs, strength=0.0), x)
    full = a.add(x, kept, freqs=freqs, strength=1.0)
    oq, os_ = ops.rotate_quant(got.view(B * L, 1024))
    step = ops.gemm_f32(oq, os_, a.wo).view(B, L, 512)
    assert cosine((full.float() - x.float()).cpu().numpy(), step.cpu().numpy()) > TOL_COS


def test_dit_with_w4_conditioning_and_image_prompt(cuda):
    from k2b.dit import DiTConfig, Krea2DiT, synthetic_dit
    from k2b.adapter import W4Linear
    from k2b.model import ModelConfig

    core = ModelConfig(hidden=512, heads=4, kvheads=2, mlp=1024, blocks=2)
    cfg = DiTConfig(core=core, channels=4, patch=2, tdim=256, txtdim=512, txt_heads=4, txt_kvheads=4, txt_mlp=1024,
                    txt_layers=1)
    B = 2
    gen = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(B, 4, 16, 12, generator=gen, device=cuda).to(torch.bfloat16)
    ts = torch.tensor([0.3, 0.9], device=cuda)
    ctx = torch.randn(B, 7, 512, generator=gen, device=cuda).to(torch.bfloat16)
    w4 = synthetic_dit(cfg, batch=B, seed=5, device=cuda, w4_conditioning=True, adapter_width=640)
    assert all(isinstance(getattr(w4, n), W4Linear) for n in ("tmlp1", "tmlp2", "tproj", "txtmlp"))
    plain = synthetic_dit(cfg, batch=B, seed=5, device=cuda)
    for n in ("tmlp1", "tmlp2", "tproj", "txtmlp"):  # the plain linears that the INT4 ones stand for
        w = getattr(w4, n)
        setattr(plain, n, (_dequant(w).to(torch.bfloat16), w.bias))
    t4, tp = {}, {}
    y4 = Krea2DiT(cfg, w4).forward(x, ts, ctx, trace=t4)
    yp = Krea2DiT(cfg, plain).forward(x, ts, ctx, trace=tp)
    for stage in ("t", "tvec"):
        assert cosine(t4[stage].float().cpu().numpy(), tp[stage].float().cpu().numpy()) > 0.9999, stage
    assert cosine(y4.float().cpu().numpy(), yp.float().cpu().numpy()) > TOL_COS
    states = torch.randn(1, 50, 640, generator=gen, device=cuda).to(torch.bfloat16)  # one image prompt for both latents
    kept = w4.adapter.keys(states, torch.tensor([50, 33], dtype=torch.int32, device=cuda))
    tr = {}
    yi = Krea2DiT(cfg, w4).forward(x, ts, ctx, trace=tr, image_prompt=kept, strength=0.5)
    assert torch.isfinite(yi.float()).all() and not torch.equal(yi, y4)
    assert not torch.equal(tr["adapted"], tr["combined"])
    assert torch.equal(Krea2DiT(cfg, w4).forward(x, ts, ctx, image_prompt=kept, strength=0.0), y4)
    with pytest.raises(ValueError, match="adapter"):
        Krea2DiT(cfg, plain).forward(x, ts, ctx, image_prompt=kept)
    assert np.isfinite(yp.float().cpu().numpy()).all()
