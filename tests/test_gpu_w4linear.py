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
