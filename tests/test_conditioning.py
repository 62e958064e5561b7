"""The conditioning operators refuse what they do not take, before any launch.  No GPU."""
import ctypes
import os

import pytest
import torch

from k2b import ops

BF = torch.bfloat16


def w4_args(**change):
    a = dict(x=torch.zeros(2, 256, dtype=BF), packed=torch.zeros(8, 128, dtype=torch.uint8),
             scales=torch.zeros(8, 2, dtype=torch.float16), bias=torch.zeros(8, dtype=BF))
    a.update(change)
    return a.pop("x"), a.pop("packed"), a.pop("scales"), a


@pytest.mark.parametrize("change,what", [
    (dict(x=torch.zeros(2, 256)), "bf16 or fp16"),
    (dict(x=torch.zeros(2, 128, dtype=BF)), "do not fit"),
    (dict(packed=torch.zeros(8, 128, dtype=torch.int8)), "uint8"),
    (dict(packed=torch.zeros(8, 96, dtype=torch.uint8)), "do not fit"),
    (dict(packed=torch.zeros(128, 8, dtype=torch.uint8).t()), "contiguous"),
    (dict(scales=torch.zeros(8, 2)), "fp16 scales expected"),
    (dict(scales=torch.zeros(8, 3, dtype=torch.float16)), "do not fit"),
    (dict(bias=torch.zeros(7, dtype=BF)), "bias"),
    (dict(bias=torch.zeros(8)), "bias"),
    (dict(act="relu"), "act"),
    (dict(), "CUDA device"),  # all fits, but nothing here runs on the CPU
])
def test_w4_linear_refuses(change, what):
    x, packed, scales, rest = w4_args(**change)
    with pytest.raises(ValueError, match=what):
        ops.w4_linear(x, packed, scales, **rest)


def heads(B, H, L, D, dtype=BF):
    return torch.zeros(B, H, L, D, dtype=dtype)


@pytest.mark.parametrize("call,what", [
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 96), None, torch.zeros(96), None), "D 64 or 128"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64, torch.float32), None, torch.zeros(64), None), "bf16 or fp16"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64), None, torch.zeros(64, dtype=BF), None), "wq"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64), None, torch.zeros(64), torch.zeros(64)), "go with k"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64), heads(2, 2, 3, 64), torch.zeros(64), torch.zeros(64)), "does not go"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64), heads(1, 2, 3, 64), torch.zeros(64), None), "wk"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64), None, torch.zeros(64), None, torch.zeros(4, 32, 2, 2)), "freqs_q"),
    (lambda: ops.qk_norm_rope(torch.zeros(1, 2, 64, 3, dtype=BF).transpose(2, 3), None, torch.zeros(64), None),
     "contiguous heads"),
    (lambda: ops.qk_norm_rope(torch.zeros(1, 2, 3, 65, dtype=BF)[..., 1:], None, torch.zeros(64), None),
     "contiguous heads"),
    (lambda: ops.qk_norm_rope(heads(1, 2, 3, 64), None, torch.zeros(64), None), "CUDA device"),
])
def test_qk_norm_rope_refuses(call, what):
    with pytest.raises(ValueError, match=what):
        call()


Q, K = heads(2, 4, 3, 64), heads(2, 2, 5, 64)


@pytest.mark.parametrize("call,what", [
    (lambda: ops.cross_attention(Q, K, heads(2, 2, 6, 64)), "do not go together"),
    (lambda: ops.cross_attention(Q, heads(2, 3, 5, 64), heads(2, 3, 5, 64)), "do not go together"),
    (lambda: ops.cross_attention(heads(3, 4, 3, 64), K, K), "do not go together"),
    (lambda: ops.cross_attention(Q, K.half(), K.half()), "do not go together"),
    (lambda: ops.cross_attention(Q.float(), K, K), "bf16 or fp16"),
    (lambda: ops.cross_attention(Q[0], K[0], K[0]), "expected"),
    (lambda: ops.cross_attention(Q, K, K, lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (lambda: ops.cross_attention(Q, K, K, lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (lambda: ops.cross_attention(Q, K, K, mask=torch.zeros(2, 5)), "mask"),
    (lambda: ops.cross_attention(Q, K, K, mask=torch.zeros(2, 4, dtype=torch.bool)), "mask"),
    (lambda: ops.cross_attention(Q, K, K, mask=torch.zeros(2, 3, 3, 5, dtype=torch.bool)), "mask"),
    (lambda: ops.cross_attention(Q, K, K, bias=torch.zeros(2, 5, dtype=BF)), "bias"),
    (lambda: ops.cross_attention(Q, K, K, bias=torch.zeros(5)), "bias"),
    (lambda: ops.cross_attention(Q, K, K, bias=torch.zeros(5, 2).t()), "bias"),
    (lambda: ops.cross_attention(Q, K, K), "CUDA device"),
])
def test_cross_attention_refuses(call, what):
    with pytest.raises(ValueError, match=what):
        call()


@pytest.fixture(scope="module")
def lib():
    from k2b._native import LIB_PATH, lib as load

    if not os.path.exists(LIB_PATH):
        pytest.skip("libk2b not built (run __graft_entry__.build())")
    return load()


P = ctypes.c_void_p(1 << 20)  # never read: every call below fails on the host


def test_c_entries_refuse(lib):
    """cudaErrorInvalidValue for sizes, types, strides and pointers that the kernels do not take."""
    assert lib.k2b_w4_workspace_bytes(0, 128) == -1 and lib.k2b_w4_workspace_bytes(1, 100) == -1
    assert lib.k2b_w4_workspace_bytes(9, 256) >= 2 * 2 * (8 * 128 * 2)
    assert lib.k2b_w4_workspace_bytes(1, 256) == 0  # prepared inside the product kernel
    # a mask that depends on the query or the head is packed for the many-query kernel: 16 bytes per row and 128 keys,
    # and per 128 rows
    need = lib.k2b_cross_workspace_bytes
    assert need(1, 48, 12, 4096, 1000, 128, 0, 0, 1000) == 16 * 8 * (4096 + 32)
    assert need(2, 48, 12, 4096, 1000, 128, 1, 1, 1) == 2 * 48 * 16 * 8 * (4096 + 32)
    assert need(1, 48, 12, 4096, 1000, 128, 1000, 0, 0) == 0 and need(1, 48, 12, 1, 1000, 128, 0, 0, 1000) == 0
    assert need(1, 48, 12, 4096, 0, 128, 0, 0, 1) == 0 and need(1, 47, 12, 4096, 10, 128, 0, 0, 1) == -1
    w4 = lambda m=1, n=8, k=128, dtype=2, act=0, x=P, stride=128, work=P: lib.k2b_w4_linear(  # noqa: E731
        x, stride, P, P, None, P, work, m, n, k, dtype, 1, act, None)
    odd = ctypes.c_void_p((1 << 20) + 2)
    assert {w4(m=0), w4(n=0), w4(k=100), w4(dtype=0), w4(act=3), w4(x=None), w4(x=odd), w4(stride=126),
            w4(m=2, stride=64), w4(m=9, work=None), w4(k=4096, stride=4096, work=odd)} == {1}
    qk = lambda q=P, lq=1, heads=2, dim=64, st=64, fb=1, dtype=2: lib.k2b_qk_norm_rope(  # noqa: E731
        q, None, P, None, P, None, P, None, 2, lq, 0, heads, 1, dim, 64, 64, st, 0, 0, 0, fb, 1, 1e-6, 1e-6, dtype, None)
    assert {qk(q=None), qk(lq=0), qk(heads=0), qk(dim=32), qk(st=4), qk(fb=3), qk(dtype=0), qk(q=odd)} == {1}
    ca = lambda q=P, k=P, heads=2, hk=1, lq=1, lk=4, dim=64, st=64, dtype=2: lib.k2b_cross_attention(  # noqa: E731
        q, k, P, None, None, None, P, None, 1, heads, hk, lq, lk, dim, *([64] * 8), st, 0, 0, 0, 0, 0, 1.0, dtype, None)
    assert {ca(q=None), ca(k=None), ca(heads=3, hk=2), ca(lq=0), ca(lk=-1), ca(dim=96), ca(st=12), ca(st=-8),
            ca(dtype=0), ca(q=odd)} == {1}
