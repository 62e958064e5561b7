"""cross_attention's many-query (tcgen05) kernel at the sizes that the library's rule sends to it, each test asking the
rule first; and qk_norm_rope over several resident waves.  Against the definitions in 64 bits."""
import math

import pytest
import torch

import _conditioning as R
from k2b import ops
from k2b._native import lib

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def takes_tiles(B, H, Hk, Lq, Lk, D):
    """Whether these sizes go to the many-query kernel: only it packs a mask that depends on the query."""
    return lib().k2b_cross_workspace_bytes(B, H, Hk, Lq, Lk, D, 0, 0, 1) > 0


def items(H, Hk, Lq, B):
    """Its work items: two heads of an even group by 128 queries, one head of an odd group by 256."""
    g = H // Hk
    return (g * -(-Lq // 256) if g % 2 else g // 2 * -(-Lq // 128)) * Hk * B


def gen_of(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def states(cuda, B, H, L, D, dtype, seed):
    return torch.randn(B, L, H, D, generator=gen_of(cuda, seed), device=cuda).to(dtype).transpose(1, 2)


def inputs(cuda, B, H, Hk, Lq, Lk, D, dtype):
    return (states(cuda, B, H, Lq, D, dtype, 1), states(cuda, B, Hk, Lk, D, dtype, 2), states(cuda, B, Hk, Lk, D, dtype, 3))


# B, H, Hk, Lq, Lk, D, dtype: both group parities, head sizes and types; rings of two (D 128) and four (D 64) tiles that
# wrap
LONG = [
    (1, 4, 4, 2000, 700, 128, FP),
    (1, 16, 4, 1000, 700, 128, BF),
    (2, 16, 4, 1500, 700, 64, BF),
    (1, 5, 5, 3000, 700, 64, FP),
    (3, 7, 7, 900, 900, 64, BF),
]


@pytest.mark.parametrize("shape", LONG)
def test_growing_scores(cuda, shape):
    """Maxima that keep growing along the keys by more than 2^8 (O and its sum are rescaled, several times a row)."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    assert takes_tiles(*shape[:6])
    q, k, v = inputs(cuda, *shape)
    k = (k.float() * torch.linspace(0.1, 6.0, Lk, device=cuda).view(1, 1, Lk, 1)).to(dtype)
    for scale in (None, 1.0):
        R.check(ops.cross_attention(q, k, v, scale=scale), *R.cross_attention(q, k, v, scale=scale), str(scale))


@pytest.mark.parametrize("shape", [(1, 4, 4, 2000, 200, 128, BF), (1, 8, 4, 2000, 300, 64, FP)])
def test_bias_of_lowest(cuda, shape):
    """A bias of the lowest finite value is no exclusion: a row with nothing else averages its values, and one key
    with an ordinary bias takes all of the weight."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    assert takes_tiles(*shape[:6])
    q, k, v = inputs(cuda, *shape)
    bias = torch.full((1, Lk), torch.finfo(torch.float32).min, device=cuda)
    got = ops.cross_attention(q, k, v, bias=bias)
    mean = v.double().mean(2, keepdim=True).repeat_interleave(H // Hk, 1).expand(-1, -1, Lq, -1)
    mean = mean.transpose(1, 2).reshape(B, Lq, H * D)
    # every probability is 1/Lk exactly as stored (p = 1), so only the output is rounded
    assert float((got.double() - mean).abs().max()) <= R.UNIT[dtype] * float(mean.abs().max()) + 2.0 ** -20
    for first in (0, 150):  # the keys that count in the first tile, in a later one
        some = bias.clone()
        some[0, first:first + 10] = 0.0
        kept = slice(first, first + 10)
        R.check(ops.cross_attention(q, k, v, bias=some), *R.cross_attention(q, k[:, :, kept], v[:, :, kept]), str(first))


@pytest.mark.parametrize("shape", [(1, 8, 4, 2000, 300, 128, BF), (1, 8, 4, 2000, 300, 64, FP), (1, 5, 5, 3000, 300, 64, BF)])
@pytest.mark.parametrize("key", [5, 140, 299])
def test_infinite_scores_and_nan(cuda, shape, key):
    """A score of +inf makes its row NaN, one of -inf is a weight of zero, a query of NaN stays in its row."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    assert takes_tiles(*shape[:6])
    q, k, v = inputs(cuda, *shape)
    k[:, :, key, 7] = math.inf
    q[0, 1, 77] = math.nan
    got = ops.cross_attention(q, k, v).view(Lq, H, D).transpose(0, 1)
    up, down = q[0, :, :, 7] > 0, q[0, :, :, 7] < 0
    assert torch.isnan(got[up]).all() and torch.isnan(got[1, 77]).all()
    rest = torch.arange(Lk, device=cuda) != key
    clean = torch.where(torch.isnan(q), 0.0, q)
    want, bound = (t.view(Lq, H, D).transpose(0, 1)[down] for t in R.cross_attention(clean, k[:, :, rest], v[:, :, rest]))
    R.check(got[down], want, bound)


def test_few_row_kernel_infinite_scores(cuda):
    """The same on the few-row kernel."""
    shape = (1, 8, 2, 3, 300, 128)
    assert not takes_tiles(*shape)
    q, k, v = inputs(cuda, *shape, BF)
    for key in (5, 140):
        kk = k.clone()
        kk[:, :, key, 7] = math.inf
        got = ops.cross_attention(q, kk, v).view(3, 8, 128).transpose(0, 1)
        up, down = q[0, :, :, 7] > 0, q[0, :, :, 7] < 0
        assert torch.isnan(got[up]).all()
        rest = torch.arange(300, device=cuda) != key
        want, bound = (t.view(3, 8, 128).transpose(0, 1)[down] for t in R.cross_attention(q, kk[:, :, rest], v[:, :, rest]))
        R.check(got[down], want, bound)


# more items with keys than a B200 has SMs, so that CTAs go from item to item, over runs of one KV head and on to the
# next; prompts of at most the ring's tiles (K and V stay) and of more
MANY = [
    (4, 24, 6, 700, 250, 128, BF),    # stays, even group
    (4, 24, 6, 700, 500, 128, FP),    # does not stay
    (3, 48, 12, 700, 260, 64, BF),    # stays
    (3, 48, 12, 700, 700, 64, FP),    # does not
    (4, 20, 20, 1500, 130, 64, BF),   # group 1
    (4, 15, 5, 1300, 300, 128, BF),   # group 3
]


@pytest.mark.parametrize("shape", MANY)
@pytest.mark.parametrize("kind", ["plain", "lengths", "keys", "regions", "heads", "bias", "all"])
def test_many_items(cuda, shape, kind):
    B, H, Hk, Lq, Lk, D, dtype = shape
    n = items(H, Hk, Lq, B)
    assert takes_tiles(*shape[:6]) and n > 148
    gen = gen_of(cuda, Lq * 3 + Lk)
    q, k, v = inputs(cuda, *shape)
    lengths = mask = bias = None
    if kind in ("lengths", "all"):  # one latent without keys, one within a tile, one to the end
        lengths = torch.tensor([Lk - 1, 0, 20, Lk][:B], dtype=torch.int32, device=cuda)
    if kind == "keys":
        mask = torch.rand(B, Lk, generator=gen, device=cuda) < 0.6
        mask[0, :Lk // 2] = False
        mask[-1] = False
    if kind in ("regions", "all"):  # a region of queries sees its share of the keys: most tiles are skipped
        region = torch.arange(Lq, device=cuda)[:, None] * 3 // Lq == torch.arange(Lk, device=cuda) * 3 // Lk
        mask = (region & (torch.rand(Lq, 1, generator=gen, device=cuda) < 0.9)).view(1, 1, Lq, Lk).clone()
        mask[:, :, 256:512] = False  # whole items that see nothing
    if kind == "heads":
        mask = torch.rand(B, H, 1, Lk, generator=gen, device=cuda) < 0.3
        mask[:, ::4] = False
    if kind in ("bias", "all"):
        bias = torch.randn(B, Lk, generator=gen, device=cuda) * 2
        bias[:, ::5] = -math.inf
        bias[0] = 0.0  # a latent whose tiles have nothing to add
    got = ops.cross_attention(q, k, v, lengths=lengths, mask=mask, bias=bias)
    R.check(got, *R.cross_attention(q, k, v, lengths, mask, bias))
    gone = ~R.keep_mask(B, H, Lq, Lk, lengths, mask, bias, cuda).any(-1)
    assert not got.view(B, Lq, H, D).transpose(1, 2)[gone].any()
    assert torch.equal(got, ops.cross_attention(q, k, v, lengths=lengths, mask=mask, bias=bias))


def test_many_latents(cuda):
    """More than 64 latents with lengths (items are then shared out by number, not by cost), K and V shared."""
    B, H, Hk, Lq, Lk, D = 70, 4, 2, 130, 150, 64
    assert takes_tiles(B, H, Hk, Lq, Lk, D) and items(H, Hk, Lq, B) > 148
    q = states(cuda, B, H, Lq, D, FP, 1)
    k, v = states(cuda, 1, Hk, Lk, D, FP, 2), states(cuda, 1, Hk, Lk, D, FP, 3)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen_of(cuda, 4), device=cuda, dtype=torch.int32)
    R.check(ops.cross_attention(q, k, v, lengths=lengths), *R.cross_attention(q, k, v, lengths))


@pytest.mark.parametrize("B,H,Hk,Lq,Lk,D,dtype", [
    (1, 48, 12, 1300, 1300, 128, BF),
    (2, 20, 5, 1500, 700, 64, FP),    # 20 heads: items of twelve and of eight
    (2, 13, 1, 1300, 3000, 128, FP),
    (4, 5, 5, 3000, 1, 64, BF),
])
def test_qk_norm_rope_waves(cuda, B, H, Hk, Lq, Lk, D, dtype):
    """Many more items than resident warps (2368), on each side."""
    gen = gen_of(cuda, H)
    q = torch.randn(B, Lq, H + 1, D, generator=gen, device=cuda).to(dtype)[:, :, 1:].transpose(1, 2)
    k = torch.randn(B, Lk, Hk, D, generator=gen, device=cuda).to(dtype).transpose(1, 2)
    wq, wk = (torch.rand(D, generator=gen, device=cuda) * 0.4 - 0.2 for _ in range(2))

    def table(length):
        a = torch.rand(length, D // 2, generator=gen, device=cuda) * 100.0
        return torch.stack([a.cos(), -a.sin(), a.sin(), a.cos()], -1).unflatten(-1, (2, 2)).contiguous()

    fq, fk = table(Lq), table(Lk)
    qo, ko = ops.qk_norm_rope(q, k, wq, wk, fq, fk)
    R.check(qo, *R.norm_rope(q, wq, fq, 1e-6), "q")
    R.check(ko, *R.norm_rope(k, wk, fk, 1e-6), "k")


@pytest.mark.parametrize("shape", [(8, 48, 12, 2000, 40, 64, BF), (8, 40, 5, 2500, 150, 128, FP), (8, 18, 18, 5000, 40, 64, FP),
                                   (6, 36, 12, 2600, 300, 128, BF)])
@pytest.mark.parametrize("kind", ["lengths", "queries", "heads"])
def test_many_items_without_keys(cuda, shape, kind):
    """Long rows of items that see nothing, between items that do: latents without keys, blocks of queries or heads whose
    mask leaves none."""
    B, H, Hk, Lq, Lk, D, dtype = shape
    # each of a B200's CTAs gets at least sixteen in a row
    assert takes_tiles(*shape[:6]) and items(H, Hk, Lq, B) >= 16 * 148
    q, k, v = inputs(cuda, *shape)
    lengths = mask = None
    if kind == "lengths":
        lengths = torch.tensor([Lk, 0, 0, Lk - 1, 0, 0, 0, 5][:B], dtype=torch.int32, device=cuda)
    elif kind == "queries":
        mask = torch.ones(1, 1, Lq, Lk, dtype=torch.bool, device=cuda)
        mask[:, :, 300:] = False
    else:
        mask = torch.zeros(B, H, 1, Lk, dtype=torch.bool, device=cuda)
        mask[::3, ::9, :, ::2] = True
    got = ops.cross_attention(q, k, v, lengths=lengths, mask=mask)
    assert ops.device_error() == 0
    R.check(got, *R.cross_attention(q, k, v, lengths, mask))
    gone = ~R.keep_mask(B, H, Lq, Lk, lengths, mask, None, cuda).any(-1)
    assert not got.view(B, Lq, H, D).transpose(1, 2)[gone].any()
