"""The conditioning operators' two-launch forms (prepared rows and products, packed masks and attention) in CUDA graphs and
on several streams at once."""
import pytest
import torch

import _conditioning as R
from k2b import ops
from k2b._native import lib

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


class Work:
    """w4_linear with a prepare launch, head norms and many-query attention under a packed mask, in a row."""

    def __init__(self, cuda, seed, dtype=BF):
        self.gen = torch.Generator(device=cuda).manual_seed(seed)
        self.cuda, self.dtype = cuda, dtype
        self.packed, self.scales = R.random_w4(1024, 640, self.gen, cuda)
        self.w = torch.rand(128, generator=self.gen, device=cuda) * 0.2
        self.x = torch.empty(700, 640, dtype=dtype, device=cuda)
        self.mask = torch.empty(1, 1, 700, 300, dtype=torch.bool, device=cuda)
        self.k = torch.empty(1, 300, 2, 128, dtype=dtype, device=cuda).transpose(1, 2)
        assert lib().k2b_w4_workspace_bytes(700, 640) > 0
        assert lib().k2b_cross_workspace_bytes(1, 8, 2, 700, 300, 128, 0, 0, 300) > 0
        self.new_inputs()

    def new_inputs(self):
        self.x.copy_(torch.randn(self.x.shape, generator=self.gen, device=self.cuda))
        self.mask.copy_(torch.rand(self.mask.shape, generator=self.gen, device=self.cuda) < 0.4)
        self.k.copy_(torch.randn(self.k.shape, generator=self.gen, device=self.cuda))

    def __call__(self):
        y = ops.w4_linear(self.x, self.packed, self.scales).view(1, 700, 8, 128).transpose(1, 2)
        q, k = ops.qk_norm_rope(y, self.k, self.w, self.w)
        return y, q, ops.cross_attention(q, k, self.k, mask=self.mask)


def test_two_launches_in_a_graph(cuda):
    work = Work(cuda, 1)
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for _ in range(5):
        work.new_inputs()
        for _ in range(3):  # back to back: a replay's first launch behind the last one's
            graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = work()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    R.check(got[0].transpose(1, 2).reshape(700, 1024), *R.w4_linear(work.x, work.packed, work.scales, None, True, "none"))
    _, k = ops.qk_norm_rope(got[0], work.k, work.w, work.w)
    R.check(got[2], *R.cross_attention(got[1], k, work.k, None, work.mask))


def test_streams_at_once(cuda):
    """Three streams with their own inputs, nothing between them: workspaces and packed masks do not mix."""
    works = [Work(cuda, s, d) for s, d in ((2, BF), (3, FP), (4, BF))]
    want = [[t.clone() for t in w()] for w in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    got = [[] for _ in works]
    for _ in range(20):
        for i, (w, s) in enumerate(zip(works, streams)):
            with torch.cuda.stream(s):
                got[i].append(w())
    torch.cuda.synchronize()
    for mine, all_runs in zip(want, got):
        for run in all_runs:
            assert all(torch.equal(a, b) for a, b in zip(run, mine))
