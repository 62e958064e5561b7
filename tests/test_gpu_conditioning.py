"""w4_linear, qk_norm_rope and cross_attention against their definitions in 64 bits, at the sizes, strides and masks
where they can go wrong."""
import math

import pytest
import torch

import _conditioning as R
from k2b import ops

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def gen_of(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


# ------------------------------------------------------------- w4_linear

@pytest.mark.parametrize("m,n,k,dtype,rotate,bias,act", [
    (1, 1, 128, BF, True, False, "none"),        # one output
    (1, 6144, 256, BF, False, True, "gelu"),     # the timestep MLP's first layer
    (2, 15, 384, FP, True, True, "none"),        # three groups, a part of a row tile
    (3, 130, 640, BF, True, True, "silu"),
    (7, 33, 1024, FP, False, False, "none"),
    (8, 2000, 6144, BF, True, True, "none"),
    (9, 257, 896, FP, True, False, "gelu"),      # a second block of rows, seven groups
    (16, 48, 1152, BF, False, True, "silu"),     # nine groups for eight warps
    (17, 1000, 2560, BF, True, True, "none"),
    (32, 17, 128, FP, True, False, "none"),
    (33, 300, 512, BF, True, False, "none"),     # a second launch row
    (77, 1536, 2560, FP, True, True, "none"),
    (1, 100, 16384, BF, True, False, "none"),    # the longest K of the framework's weights
    (96, 40000, 128, BF, True, False, "none"),
    (1, 300, 2048, FP, True, True, "none"),      # the widest that one launch does
    (4, 300, 2048, BF, True, False, "none"),
    (5, 300, 2048, BF, True, False, "none"),     # and the first that takes two
    (8, 129, 1024, BF, False, False, "none"),
])
def test_w4_linear(cuda, m, n, k, dtype, rotate, bias, act):
    gen = gen_of(cuda, m * 1000 + n)
    packed, scales = R.random_w4(n, k, gen, cuda)
    x = torch.randn(m, k, generator=gen, device=cuda)
    x[:, ::37] *= 20.0
    x = x.to(dtype)
    b = torch.randn(n, generator=gen, device=cuda).to(dtype) if bias else None
    got = ops.w4_linear(x, packed, scales, b, rotate=rotate, act=act)
    assert got.dtype == dtype and tuple(got.shape) == (m, n)
    R.check(got, *R.w4_linear(x, packed, scales, b, rotate, act))
    assert torch.equal(got, ops.w4_linear(x, packed, scales, b, rotate=rotate, act=act))


def test_w4_linear_takes_quantize_weight(cuda):
    """The framework's own packed weights: y is close to the unquantised product."""
    from k2b.model import quantize_weight

    gen = gen_of(cuda, 3)
    w = (torch.randn(512, 1024, generator=gen, device=cuda) * 0.02).to(BF)
    x = torch.randn(4, 1024, generator=gen, device=cuda).to(BF)
    packed, scales = quantize_weight(w)
    got = ops.w4_linear(x, packed, scales)
    R.check(got, *R.w4_linear(x, packed, scales, None, True, "none"))
    want = x.double() @ w.double().t()
    # a step of absmax/7 over Gaussian groups (absmax ~ 2.8 sigma) leaves an error of 0.4/sqrt(12) sigma
    assert float((got.double() - want).norm() / want.norm()) < 0.2


def test_w4_linear_layouts(cuda):
    """Leading dimensions, rows taken out of a wider buffer, no rows, no outputs, another stream."""
    gen = gen_of(cuda, 5)
    packed, scales = R.random_w4(96, 256, gen, cuda)
    wide = torch.randn(6, 5, 512, generator=gen, device=cuda).to(BF)
    x = wide[:, 2, 128:384]
    assert x.stride(0) == 5 * 512
    R.check(ops.w4_linear(x, packed, scales), *R.w4_linear(x, packed, scales, None, True, "none"))
    one = wide[3, 1, 4:260]  # 8-byte aligned only
    R.check(ops.w4_linear(one, packed, scales), *R.w4_linear(one, packed, scales, None, True, "none"))
    x3 = wide[..., :256].contiguous()
    got = ops.w4_linear(x3, packed, scales)
    assert tuple(got.shape) == (6, 5, 96)
    R.check(got, *R.w4_linear(x3, packed, scales, None, True, "none"))
    assert tuple(ops.w4_linear(x3[:0], packed, scales).shape) == (0, 5, 96)
    assert tuple(ops.w4_linear(x3, packed[:0], scales[:0]).shape) == (6, 5, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.w4_linear(x3, packed, scales)
    side.synchronize()
    assert torch.equal(other, got)


def test_w4_linear_extreme_rows(cuda):
    """Zero rows give the bias; a row of tiny or of large values keeps its accuracy; an infinity or a NaN stays in
    its row."""
    gen = gen_of(cuda, 7)
    packed, scales = R.random_w4(64, 512, gen, cuda)
    b = torch.randn(64, generator=gen, device=cuda).to(BF)
    base = torch.randn(10, 512, generator=gen, device=cuda)
    x = base.clone()
    x[1] = 0
    x[2] *= 1e-30
    x[3] *= 1e30
    x[4, :256] *= 1e-20  # groups of different size in one row
    x = x.to(BF)
    for rotate in (False, True):
        got = ops.w4_linear(x, packed, scales, b, rotate=rotate)
        R.check(got, *R.w4_linear(x, packed, scales, b, rotate, "none"))
        assert torch.equal(got[1], b)
        bad = x.clone()
        bad[5, 7] = math.inf
        bad[6, 300] = math.nan
        hit = ops.w4_linear(bad, packed, scales, b, rotate=rotate)
        assert not torch.isfinite(hit[5:7]).any() if rotate else torch.isnan(hit[6]).all()
        rest = [0, 1, 2, 3, 4, 7, 8, 9]
        assert torch.equal(hit[rest], got[rest])


# ---------------------------------------------------------- qk_norm_rope

def table(L, D, cuda, seed, batch=None):
    a = torch.rand((L,) if batch is None else (batch, L), generator=gen_of(cuda, seed), device=cuda)[..., None]
    a = a * 100.0 * torch.rand(D // 2, generator=gen_of(cuda, seed + 1), device=cuda)
    return torch.stack([a.cos(), -a.sin(), a.sin(), a.cos()], -1).unflatten(-1, (2, 2)).contiguous()


@pytest.mark.parametrize("B,H,Hk,Lq,Lk,D,dtype,rope", [
    (1, 48, 12, 1, 1, 128, BF, "both"),
    (2, 3, 1, 7, 5, 64, FP, "both"),
    (1, 9, 9, 33, 1, 128, FP, "q"),
    (3, 20, 5, 2, 300, 64, BF, "none"),
    (2, 48, 12, 130, 130, 128, BF, "batched"),
    (5, 1, 1, 1, 1000, 128, FP, "k"),
])
def test_qk_norm_rope(cuda, B, H, Hk, Lq, Lk, D, dtype, rope):
    gen = gen_of(cuda, B * 100 + H)
    # views of joint projections
    q = torch.randn(B, Lq, H + 2, D, generator=gen, device=cuda).to(dtype)[:, :, 1:H + 1].transpose(1, 2)
    k = torch.randn(B, Lk, 2 * Hk, D, generator=gen, device=cuda).to(dtype)[:, :, Hk:].transpose(1, 2)
    wq, wk = (torch.rand(D, generator=gen, device=cuda) * 0.4 - 0.2 for _ in range(2))
    fb = B if rope == "batched" else None
    fq = table(Lq, D, cuda, 1, fb) if rope in ("both", "q", "batched") else None
    fk = table(Lk, D, cuda, 2, fb) if rope in ("both", "k", "batched") else None
    qo, ko = ops.qk_norm_rope(q, k, wq, wk, fq, fk, eps_q=1e-6, eps_k=1e-5)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == dtype
    R.check(qo, *R.norm_rope(q, wq, fq, 1e-6), "q")
    R.check(ko, *R.norm_rope(k, wk, fk, 1e-5), "k")


def test_qk_norm_rope_edges(cuda):
    """Zero heads give zeros, fp16's largest values do not overflow, the queries alone, no tokens, head-major
    memory, a NaN that stays in its head."""
    gen = gen_of(cuda, 11)
    q = torch.randn(2, 4, 6, 128, generator=gen, device=cuda).to(FP)  # head-major
    q[0, 1, 2] = 0
    q[0, 2, 3] = 65504.0
    q[1, 3, 5, 17] = math.nan
    w = torch.zeros(128, device=cuda)
    qo, none = ops.qk_norm_rope(q, None, w, None)
    assert none is None
    assert torch.isnan(qo[1, 3, 5]).all()
    want, bound = R.norm_rope(q, w, None, 1e-6)
    fine = torch.ones(2, 4, 6, dtype=torch.bool, device=cuda)
    fine[1, 3, 5] = False
    R.check(qo[fine], want[fine], bound[fine])
    assert not qo[0, 1, 2].any()
    empty, ko = ops.qk_norm_rope(q[:, :, :0], q, w, w)
    assert tuple(empty.shape) == (2, 4, 0, 128) and torch.equal(ko[fine], qo[fine])


# ------------------------------------------------------- cross_attention

def states(cuda, B, H, L, D, dtype, seed, scale=1.0):
    return (torch.randn(B, L, H, D, generator=gen_of(cuda, seed), device=cuda) * scale).to(dtype).transpose(1, 2)


SHAPES = [  # B, H, Hk, Lq, Lk, D, dtype
    (1, 1, 1, 1, 1, 64, BF),
    (1, 48, 12, 1, 1000, 128, BF),
    (2, 4, 1, 3, 17, 128, FP),
    (3, 6, 2, 16, 129, 64, FP),
    (1, 5, 5, 17, 300, 128, BF),
    (2, 8, 2, 127, 128, 128, BF),
    (1, 20, 20, 130, 77, 64, BF),
    (2, 12, 4, 257, 255, 128, FP),
    (1, 7, 7, 300, 640, 128, BF),
    (1, 48, 12, 520, 154, 128, BF),
    (4, 2, 2, 1000, 33, 64, FP),
]


@pytest.mark.parametrize("B,H,Hk,Lq,Lk,D,dtype", SHAPES)
@pytest.mark.parametrize("kind", ["plain", "lengths", "keys", "rows", "heads", "bias", "all"])
def test_cross_attention(cuda, B, H, Hk, Lq, Lk, D, dtype, kind):
    gen = gen_of(cuda, Lq * 7 + Lk)
    q, k, v = (states(cuda, B, h, n, D, dtype, s) for h, n, s in ((H, Lq, 1), (Hk, Lk, 2), (Hk, Lk, 3)))
    lengths = mask = bias = None
    if kind in ("lengths", "all"):
        lengths = torch.randint(0, Lk + 1, (B,), generator=gen, device=cuda, dtype=torch.int32)
        lengths[0] = max(1, Lk - 1)
        if B > 1:
            lengths[-1] = 0
    if kind == "keys":
        mask = torch.rand(B, Lk, generator=gen, device=cuda) < 0.6
        mask[0, :Lk // 2] = False  # whole tiles that nobody sees
    if kind in ("rows", "all"):
        mask = torch.rand(1, 1, Lq, Lk, generator=gen, device=cuda) < 0.5
        mask[:, :, ::3] = False    # rows that see nothing
    if kind == "heads":
        mask = torch.rand(B, H, Lq, Lk, generator=gen, device=cuda) < 0.3
    if kind in ("bias", "all"):
        bias = torch.randn(B, Lk, generator=gen, device=cuda) * 2
        bias[:, ::5] = -math.inf
    got = ops.cross_attention(q, k, v, lengths=lengths, mask=mask, bias=bias)
    assert got.dtype == dtype and tuple(got.shape) == (B, Lq, H * D)
    want, bound = R.cross_attention(q, k, v, lengths, mask, bias)
    R.check(got, want, bound)
    gone = ~R.keep_mask(B, H, Lq, Lk, lengths, mask, bias, cuda).any(-1)
    assert not got.view(B, Lq, H, D).transpose(1, 2)[gone].any()
    assert torch.equal(got, ops.cross_attention(q, k, v, lengths=lengths, mask=mask, bias=bias))


@pytest.mark.parametrize("Lq", [1, 5, 200])
def test_cross_attention_excluded_keys_hold_anything(cuda, Lq):
    """NaN and infinities in K and V at keys that lengths, a key mask or a bias of -inf leave out."""
    B, H, Hk, Lk, D = 3, 8, 2, 300, 128
    q, k, v = (states(cuda, B, h, n, D, BF, s) for h, n, s in ((H, Lq, 1), (Hk, Lk, 2), (Hk, Lk, 3)))
    lengths = torch.tensor([300, 130, 0], dtype=torch.int32, device=cuda)
    mask = torch.ones(B, Lk, dtype=torch.bool, device=cuda)
    mask[:, 40:57] = False
    mask[0, 128:256] = False
    bias = torch.zeros(1, Lk, device=cuda)
    bias[:, 5] = -math.inf
    want = ops.cross_attention(q, k, v, lengths=lengths, mask=mask, bias=bias)
    R.check(want, *R.cross_attention(q, k, v, lengths, mask, bias))
    gone = ~R.keep_mask(B, 1, 1, Lk, lengths, mask, bias, cuda)[:, 0, 0]
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2.transpose(1, 2)[gone] = bad
        v2.transpose(1, 2)[gone] = bad
        assert torch.equal(ops.cross_attention(q, k2, v2, lengths=lengths, mask=mask, bias=bias), want)


@pytest.mark.parametrize("Lq", [2, 150])
def test_cross_attention_bias_of_lowest(cuda, Lq):
    """A bias of the lowest finite value is no exclusion: a row with nothing else averages its values."""
    Lk, D = 200, 64
    q, k, v = states(cuda, 1, 2, Lq, D, FP, 1), states(cuda, 1, 2, Lk, D, FP, 2), states(cuda, 1, 2, Lk, D, FP, 3)
    low = torch.finfo(torch.float32).min
    bias = torch.full((1, Lk), low, device=cuda)
    got = ops.cross_attention(q, k, v, bias=bias)
    mean = v.double().mean(2).reshape(1, 1, 2 * D).expand(1, Lq, -1)
    u = R.UNIT[FP]
    # every probability is 1/200 exactly as stored (p = 1), so only the output is rounded
    assert float((got.double() - mean).abs().max()) <= u * float(mean.abs().max()) + 2.0 ** -20
    bias[0, :10] = 0.0
    R.check(ops.cross_attention(q, k, v, bias=bias), *R.cross_attention(q, k[:, :, :10], v[:, :, :10]))


@pytest.mark.parametrize("Lq", [1, 140])
def test_cross_attention_growing_scores(cuda, Lq):
    """Scores whose maximum keeps growing along the keys, by more than fp16's range of exponentials."""
    D, Lk = 128, 700
    q, k, v = states(cuda, 1, 4, Lq, D, BF, 1), states(cuda, 1, 4, Lk, D, BF, 2), states(cuda, 1, 4, Lk, D, BF, 3)
    k = (k.float() * torch.linspace(0.1, 6.0, Lk, device=cuda).view(1, 1, Lk, 1)).to(BF)
    for scale in (None, 1.0, -0.5, 0.0):
        R.check(ops.cross_attention(q, k, v, scale=scale), *R.cross_attention(q, k, v, scale=scale), str(scale))


def test_cross_attention_shared_and_strided(cuda):
    """K and V with a batch of one, head-major and sliced memory, a transposed mask, lengths outside 0..Lk."""
    B, H, Hk, D = 3, 8, 2, 128
    for Lq, Lk in ((4, 90), (300, 260)):
        gen = gen_of(cuda, Lq)
        q = torch.randn(B, H, Lq, D + 64, generator=gen, device=cuda).to(FP)[..., 64:]  # head-major, padded heads
        kv = torch.randn(1, Lk, 2, Hk, D, generator=gen, device=cuda).to(FP)
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        lengths = torch.tensor([-5, Lk + 100, Lk // 2], dtype=torch.int32, device=cuda)
        mask = (torch.rand(1, 1, Lk, Lq, generator=gen, device=cuda) < 0.5).transpose(2, 3)
        got = ops.cross_attention(q, k, v, lengths=lengths, mask=mask)
        R.check(got, *R.cross_attention(q, k, v, lengths, mask))
        whole = ops.cross_attention(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), lengths=lengths, mask=mask)
        R.check(whole, *R.cross_attention(q, k, v, lengths, mask))
        one = ops.cross_attention(q[:1], k, v)
        R.check(one, *R.cross_attention(q[:1], k, v))


def test_cross_attention_nothing(cuda):
    """No keys give zeros, no queries an empty result; a query of NaN stays in its row."""
    q, k = states(cuda, 2, 4, 5, 64, BF, 1), states(cuda, 2, 4, 9, 64, BF, 2)
    assert not ops.cross_attention(q, k[:, :, :0], k[:, :, :0]).any()
    assert tuple(ops.cross_attention(q[:, :, :0], k, k).shape) == (2, 0, 256)
    for Lq in (5, 300):
        q = states(cuda, 1, 4, Lq, 64, BF, 1)
        base = ops.cross_attention(q, k[:1], k[:1])
        q[0, 2, 3] = math.nan
        got = ops.cross_attention(q, k[:1], k[:1]).view(1, Lq, 4, 64)
        assert torch.isnan(got[0, 3, 2]).all()
        got[0, 3, 2] = base.view(1, Lq, 4, 64)[0, 3, 2]
        assert torch.equal(got.view(1, Lq, 256), base)


def test_in_a_graph(cuda):
    """The three operators captured and replayed on new inputs."""
    gen = gen_of(cuda, 21)
    packed, scales = R.random_w4(512, 256, gen, cuda)
    x = torch.randn(6, 256, generator=gen, device=cuda).to(BF)
    k = states(cuda, 1, 4, 50, 128, BF, 2)
    w = torch.zeros(128, device=cuda)

    def step():
        y = ops.w4_linear(x, packed, scales).view(1, 6, 4, 128).transpose(1, 2)
        y, kk = ops.qk_norm_rope(y, k, w, w)
        return ops.cross_attention(y, kk, k)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x.copy_(torch.randn(6, 256, generator=gen, device=cuda).to(BF))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, step())
