"""W4Linear in the places of a model's linears: sequences taken out of longer ones."""
import pytest
import torch

import _conditioning as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def linear_of(cuda, n, k, seed):
    from k2b.adapter import W4Linear

    gen = torch.Generator(device=cuda).manual_seed(seed)
    w = (torch.randn(n, k, generator=gen, device=cuda) * 0.02).to(BF)
    return W4Linear.of(w, torch.randn(n, generator=gen, device=cuda).to(BF)), gen


@pytest.mark.parametrize("k", [512, 640])
def test_slices_of_a_batch(cuda, k):
    """A batch of sequences without their first token: the rows are not evenly spaced."""
    w, gen = linear_of(cuda, 96, k, 1)
    states = torch.randn(3, 20, k, generator=gen, device=cuda).to(BF)
    for x in (states[:, 1:], states[:, 4:5], states[1, 3:], states[:, :, None].transpose(1, 2)[:, 0, 2:]):
        got = w(x)
        assert got.shape == (*x.shape[:-1], 96)
        R.check(got, *R.w4_linear(x.contiguous(), w.packed, w.scales, w.bias, w.rotate, "none"))
    assert w(states[:0]).shape == (0, 20, 96)


def test_adapter_keys_of_a_slice(cuda):
    from k2b.adapter import synthetic_adapter
    from k2b.model import ModelConfig

    a = synthetic_adapter(ModelConfig(hidden=512, heads=8, kvheads=2, mlp=1024, blocks=1), width=640, seed=1, device=cuda)
    states = torch.randn(2, 33, 640, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).to(BF)
    got, want = a.keys(states[:, 1:]), a.keys(states[:, 1:].contiguous())
    assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v)


def small_dit(cuda, **options):
    from k2b.dit import DiTConfig, synthetic_dit
    from k2b.model import ModelConfig

    core = ModelConfig(hidden=512, heads=4, kvheads=2, mlp=1024, blocks=1)
    cfg = DiTConfig(core=core, channels=4, patch=2, tdim=256, txtdim=512, txt_heads=4, txt_kvheads=4, txt_mlp=1024,
                    txt_layers=1)
    return cfg, synthetic_dit(cfg, batch=2, seed=5, device=cuda, **options)


def forward(cuda, cfg, weights, tokens, trace=None):
    from k2b.dit import Krea2DiT

    gen = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(2, 4, 16, 12, generator=gen, device=cuda).to(BF)
    ctx = torch.randn(2, tokens, 512, generator=gen, device=cuda).to(BF)
    return Krea2DiT(cfg, weights).forward(x, torch.tensor([0.3, 0.9], device=cuda), ctx, trace=trace)


def test_last_linear(cuda):
    """The projection behind the blocks, whose rows are a slice of the stream, as INT4."""
    from k2b.adapter import W4Linear
    from k2b.dit import unpatchify

    cfg, w = small_dit(cuda)
    w.last = W4Linear.of(*w.last)
    trace = {}
    got = forward(cuda, cfg, w, 7, trace)
    rows = trace["normed"].view(2, -1, 512)[:, 7:].contiguous()
    want, bound = R.w4_linear(rows, w.last.packed, w.last.scales, w.last.bias, w.last.rotate, "none")
    h, wd = 8, 6
    R.check(got, unpatchify(want, h, wd, cfg.patch, cfg.channels), unpatchify(bound, h, wd, cfg.patch, cfg.channels))


@pytest.mark.parametrize("tokens", [8, 9, 60])
def test_prompts_of_many_rows(cuda, monkeypatch, tokens):
    """The few-row product is not asked for more rows than it reads its weight once for, and the plain linear that
    takes them has the same weight."""
    import torch.nn.functional as F

    from k2b import ops

    cfg, w = small_dit(cuda, w4_conditioning=True)
    rows, few = [], ops.w4_linear
    monkeypatch.setattr(ops, "w4_linear", lambda x, *a, **k: (rows.append(x.numel() // x.shape[-1]), few(x, *a, **k))[1])
    trace = {}
    forward(cuda, cfg, w, tokens, trace)
    assert max(rows) <= 16 and (2 * tokens in rows) == (2 * tokens <= 16)
    ctx, got = trace["txt0"].view(2, tokens, 512), trace["combined"][:, :tokens]
    if 2 * tokens > 16:
        assert torch.equal(got, F.linear(ctx, w.txtmlp.dense, w.txtmlp.bias))
    want, bound = R.w4_linear(ctx, w.txtmlp.packed, w.txtmlp.scales, w.txtmlp.bias, w.txtmlp.rotate, "none")
    # and the dense form rounds each weight to bf16, relative to itself
    mag = ctx.double().abs() @ w.txtmlp.dense.double().abs().t()
    R.check(got, want, bound + 2.0 ** -7 * mag)


@pytest.mark.parametrize("k", [512, 640])
def test_expanded_weight(cuda, k):
    """The bf16 form is the packed one, rounded once: 128 fp32 terms of a row of H / sqrt(128) before it."""
    w, _ = linear_of(cuda, 96, k, 3)
    want = R.codes_of(w.packed).double().view(96, k // 128, 128) * w.scales.double()[..., None]
    mag = want.abs()
    if w.rotate:
        h = R.hadamard(cuda)
        want, mag = want @ h, mag @ h.abs()
    want, mag = want.reshape(96, k), mag.reshape(96, k)
    # (compared, not divided: a code of zero has a bound of zero)
    assert ((w.expand().double() - want).abs() <= R.UNIT[BF] * want.abs() + 2.0 ** -16 * mag).all()
