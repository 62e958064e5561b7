"""The conditioning operators at the ends of their ranges."""
import pytest
import torch

import _conditioning as R
from k2b import ops
from k2b._native import lib

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
# few-row kernel; many-query kernel with an even and an odd group, D 128 and 64
SHAPES = [(1, 8, 2, 3, 300, 128, FP), (1, 16, 4, 1000, 700, 128, FP), (1, 16, 4, 1000, 700, 128, BF),
          (1, 5, 5, 3000, 700, 64, FP), (2, 16, 4, 1500, 700, 64, BF)]


def gen_of(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def takes_tiles(B, H, Hk, Lq, Lk, D):
    return lib().k2b_cross_workspace_bytes(B, H, Hk, Lq, Lk, D, 0, 0, 1) > 0


def whole(cuda, B, H, L, D, dtype, seed):
    """Heads of whole numbers -2..2: their products are exact."""
    t = torch.randint(-2, 3, (B, L, H, D), generator=gen_of(cuda, seed), device=cuda)
    return t.to(dtype).transpose(1, 2)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [1e6, 1e8, 1e12])
def test_huge_scores(cuda, shape, scale):
    """Scores whose rounding alone is more than fp16's or fp32's range of exponents: each row is the mean of the values
    at its largest score."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    assert takes_tiles(*shape[:6]) == (Lq > 3)
    q, k = whole(cuda, B, H, Lq, D, dtype, 1), whole(cuda, B, Hk, Lk, D, dtype, 2)
    v = torch.randn(B, Hk, Lk, D, generator=gen_of(cuda, 3), device=cuda).to(dtype)
    for kk in (k, -k.abs()):  # the second: scores below zero for queries above
        qq = q if kk is k else q.abs() + 1
        s = qq.double() @ kk.double().repeat_interleave(H // Hk, 1).transpose(-1, -2)
        p = (s == s.amax(-1, keepdim=True)).double()
        p /= p.sum(-1, keepdim=True)
        vv = v.double().repeat_interleave(H // Hk, 1)
        want = (p @ vv).transpose(1, 2).reshape(B, Lq, H * D)
        # weights of 1 as stored; the sum and its reciprocal round in fp32, the output once
        bound = R.UNIT[dtype] * want.abs() + 2.0 ** -20 * float(v.abs().max())
        R.check(ops.cross_attention(qq, kk, v, scale=scale), want, bound)


@pytest.mark.parametrize("shape", SHAPES[1:])
def test_huge_scores_of_some_keys(cuda, shape):
    """The same where lengths, a mask per query and addends (to the keys past the first tile) take part."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    assert takes_tiles(*shape[:6])
    gen = gen_of(cuda, 9)
    q, k = whole(cuda, B, H, Lq, D, dtype, 1), whole(cuda, B, Hk, Lk, D, dtype, 2)
    v = torch.randn(B, Hk, Lk, D, generator=gen, device=cuda).to(dtype)
    lengths = torch.full((B,), Lk - 50, dtype=torch.int32, device=cuda)
    mask = torch.rand(1, 1, Lq, Lk, generator=gen, device=cuda) < 0.3
    mask[:, :, ::7] = False
    bias = torch.randint(0, 2, (1, Lk), generator=gen, device=cuda) * 5e7
    bias[:, :128] = 0.0
    gone = ~R.keep_mask(B, 1, 1, Lk, lengths, None, None, cuda)[0, 0, 0]
    v[:, :, gone] = float("nan")
    keep = R.keep_mask(B, H, Lq, Lk, lengths, mask, None, cuda)
    s = q.double() @ k.double().repeat_interleave(H // Hk, 1).transpose(-1, -2) * 1e8 + bias.double()
    s = torch.where(keep, s, -torch.inf)
    p = ((s == s.amax(-1, keepdim=True)) & keep).double()
    p /= p.sum(-1, keepdim=True).clamp(min=1)
    vv = torch.where(gone[:, None], 0.0, v.double()).repeat_interleave(H // Hk, 1)
    want = (p @ vv).transpose(1, 2).reshape(B, Lq, H * D)
    got = ops.cross_attention(q, k, v, scale=1e8, lengths=lengths, mask=mask, bias=bias)
    R.check(got, want, R.UNIT[dtype] * want.abs() + 2.0 ** -20 * float(vv.abs().max()))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("low,high", [(torch.finfo(torch.float32).min, -2.5e38), (2.5e38, torch.finfo(torch.float32).max),
                                      (torch.finfo(torch.float32).min, -2.9e38)])
@pytest.mark.parametrize("key", [3, 200])
def test_bias_of_extreme_size(cuda, shape, low, high, key):
    """Addends that log2 units cannot hold keep their order: the key with the larger one takes all of the weight."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    q, k = whole(cuda, B, H, Lq, D, dtype, 1), whole(cuda, B, Hk, Lk, D, dtype, 2)
    v = torch.randn(B, Hk, Lk, D, generator=gen_of(cuda, 3), device=cuda).to(dtype)
    bias = torch.full((1, Lk), low, device=cuda)
    bias[0, key] = high
    got = ops.cross_attention(q, k, v, bias=bias).view(B, Lq, H, D)
    assert torch.equal(got, v[:, :, key].repeat_interleave(H // Hk, 1)[:, None].expand(B, Lq, H, D))


@pytest.mark.parametrize("m,n,k", [(2, 64, 512), (8, 300, 1024), (20, 64, 640)])
@pytest.mark.parametrize("rotate", [False, True])
def test_w4_linear_large_activations(cuda, m, n, k, rotate):
    """Activations near the end of bf16's range, whose sums before the scales leave it: the products do not."""
    gen = gen_of(cuda, m)
    packed, scales = R.random_w4(n, k, gen, cuda)
    x = torch.randn(m, k, generator=gen, device=cuda) * 1e37
    x[-1] = 2e37  # every group's rotation adds up to 128 of these before it is scaled
    x = x.to(BF)
    want, bound = R.w4_linear(x, packed, scales, None, rotate, "none")
    assert float(want.abs().max()) < 3e38
    R.check(ops.w4_linear(x, packed, scales, rotate=rotate), want, bound)


def test_w4_linear_rows_past_a_grid_dimension(cuda):
    """More than 65535 blocks of 16 rows."""
    gen = gen_of(cuda, 5)
    m, n, k = 16 * 65535 + 21, 8, 128
    packed, scales = R.random_w4(n, k, gen, cuda)
    x = torch.randn(m, k, generator=gen, device=cuda).to(BF)
    got = ops.w4_linear(x, packed, scales)
    for rows in (slice(0, 40), slice(16 * 65535 - 20, m)):
        R.check(got[rows], *R.w4_linear(x[rows], packed, scales, None, True, "none"))


@pytest.mark.parametrize("per_head", [True, False])
def test_masks_past_a_grid_dimension(cuda, per_head):
    """A mask of its own for each of more than 65535 heads (or latents) on the many-query kernel."""
    H, Hk, Lq, Lk, D = 4, 2, 130, 40, 64
    B = 16400 if per_head else 65600
    assert takes_tiles(B, H, Hk, Lq, Lk, D)
    gen = gen_of(cuda, 6)
    q = torch.randn(B if per_head else 1, Lq, H, D, generator=gen, device=cuda).to(BF).transpose(1, 2)
    if not per_head:
        q = q.repeat(B, 1, 1, 1)
    k = torch.randn(1, Lk, Hk, D, generator=gen, device=cuda).to(BF).transpose(1, 2)
    mask = torch.rand((B, H, 1, Lk) if per_head else (B, 1, Lq, Lk), generator=gen, device=cuda) < 0.5
    got = ops.cross_attention(q, k, k, mask=mask)
    for i in (slice(0, 2), slice(B // 2, B // 2 + 2), slice(B - 2, B)):
        R.check(got[i], *R.cross_attention(q[i], k, k, None, mask[i]))


def test_cross_attention_no_keys_of_any_stride(cuda):
    """K and V without a key: nothing is read, so their strides do not matter."""
    q = torch.randn(2, 4, 5, 64, device=cuda).to(BF)
    k = torch.zeros(2, 9, 260, device=cuda, dtype=BF)[:, :, :256].unflatten(2, (4, 64)).transpose(1, 2)[:, :, :0]
    assert k.stride(2) % 8
    assert not ops.cross_attention(q, k, k).any()


@pytest.mark.parametrize("Lq", [1, 300])
def test_cross_attention_offsets_past_32_bits(cuda, Lq):
    """Keys whose elements lie beyond 2^31, on both kernels: a few at either end are left, the others excluded."""
    H, Hk, Lk, D = 16, 2, 8_500_001, 128
    assert takes_tiles(1, H, Hk, Lq, Lk, D) == (Lq > 1)
    gen = gen_of(cuda, 12)
    q = torch.randn(1, Lq, H, D, generator=gen, device=cuda).to(BF).transpose(1, 2)
    k, v = (torch.randn(1, Lk, Hk, D, generator=gen, device=cuda, dtype=BF).transpose(1, 2) for _ in range(2))
    assert k.stride(2) * (Lk - 1) > 2 ** 31
    left = torch.cat([torch.arange(7), torch.arange(Lk - 90, Lk - 1)]).to(cuda)
    bias = torch.full((1, Lk), -torch.inf, device=cuda)
    bias[0, left] = 0.5
    mask = torch.zeros(1, 1, 1, Lk, dtype=torch.bool, device=cuda)
    mask[..., left] = True
    lengths = torch.tensor([Lk - 1], dtype=torch.int32, device=cuda)
    want, bound = R.cross_attention(q, k[:, :, left], v[:, :, left])
    R.check(ops.cross_attention(q, k, v, bias=bias, lengths=lengths), want, bound + 2.0 ** -16 * float(v[:, :, left].abs().max()))
    R.check(ops.cross_attention(q, k, v, mask=mask), want, bound)


def test_qk_norm_rope_offsets_past_32_bits(cuda):
    gen = gen_of(cuda, 13)
    L, H, D = 8_500_001, 2, 128
    q = torch.randn(1, L, H, D, generator=gen, device=cuda, dtype=BF).transpose(1, 2)
    w = torch.rand(D, generator=gen, device=cuda) * 0.4 - 0.2
    a = torch.rand(L, D // 2, generator=gen, device=cuda) * 100.0
    f = torch.stack([a.cos(), -a.sin(), a.sin(), a.cos()], -1).unflatten(-1, (2, 2)).contiguous()
    got, _ = ops.qk_norm_rope(q, None, w, None, f)
    for rows in (slice(0, 50), slice(L - 50, L)):
        R.check(got[:, :, rows], *R.norm_rope(q[:, :, rows], w, f[rows], 1e-6))


def test_w4_linear_offsets_past_32_bits(cuda):
    gen = gen_of(cuda, 14)
    n, k = 300_001, 16384
    packed, scales = R.random_w4(n, k, gen, cuda)
    assert packed.numel() > 2 ** 31
    x = torch.randn(2, k, generator=gen, device=cuda).to(BF)
    got = ops.w4_linear(x, packed, scales)
    for cols in (slice(0, 40), slice(n - 40, n)):
        R.check(got[:, cols], *R.w4_linear(x, packed[cols], scales[cols], None, True, "none"))
