"""The block-scaled FP8 products at sizes that run every one of their kernels: which size
runs which is a host rule, checked without a GPU; the results need one.  Whole numbers,
so that every order of the sums gives the exact result."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib

BF16, FP16, FP32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn

# (m, k, n): whole blocks of K and a part of one, rows on and off 16 bytes
DENSE = [(3000, 128, 4096), (3000, 144, 4096), (3000, 2064, 4100), (8000, 272, 1024),
         (4096, 1024, 2048), (1000, 128, 2050), (600, 144, 4096), (257, 272, 4096),
         (200, 1040, 4100), (1000, 1024, 1028), (257, 272, 1024), (1000, 512, 260),
         (1, 128, 4096), (64, 144, 2050), (1000, 128, 33), (257, 2048, 2048), (100, 4096, 4100),
         (333, 2064, 1024), (33, 8192, 4100), (5, 4096, 4100), (64, 1040, 2050), (1, 144, 16),
         (64, 400, 260), (1, 2064, 33), (600, 1040, 33)]
# (tokens, top_k, experts, k, n)
GROUPED = [(30000, 1, 60, 144, 130), (15000, 2, 128, 512, 512), (16384, 1, 4, 144, 130),
           (15000, 2, 2, 512, 256), (40, 1, 60, 1040, 1028), (4000, 2, 2, 1040, 256),
           (8, 2, 16, 144, 2048), (509, 1, 1, 128, 1028), (255, 2, 16, 272, 256),
           (1, 1, 2, 144, 33), (20, 2, 128, 128, 1028), (128, 2, 60, 272, 2048),
           (3, 1, 16, 1040, 1028), (509, 1, 60, 512, 33), (50, 2, 2, 1040, 33),
           (1, 1, 1, 1040, 33)]


def kernel_of(routes, k, n, experts, out_bytes):
    f = _lib.load().mxfp4_test_fp8_kernel
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 2 + [ctypes.c_int64]
    return f(routes, k, n, experts, int(n * out_bytes % 16 == 0), 256)


def test_sizes_run_every_kernel():
    dense = {kernel_of(m, k, n, 0, b) for m, k, n in DENSE for b in (2, 4)}
    assert dense == set(range(kernel_of(0, 16, 1, 0, 2)))
    grouped = {kernel_of(m * t, k, n, e, b) for m, t, e, k, n in GROUPED for b in (2, 4)}
    assert grouped == set(range(kernel_of(0, 16, 1, 1, 2)))


def test_sizes_that_no_grid_holds_have_no_kernel():
    assert kernel_of(2 ** 31 - 1, 16, 2 ** 31 - 1, 0, 2) == -1
    assert kernel_of(2 ** 30 - 1, 16, 2 ** 20, 8, 2) == -1
    assert kernel_of(2 ** 26, 16, 1, 0, 2) >= 0


def blocks(k):
    return -(-k // 128)


def operands(g, rows, w_shape):
    """FP8 whole numbers -2 .. 2 and scales of 1/2 and 1."""
    k, n = w_shape[-1], w_shape[-2]

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=g, device="cuda", dtype=torch.int8)

    def powers(*shape):
        return 0.5 * torch.randint(1, 3, shape, generator=g, device="cuda").float()

    return (whole(rows, k).float().to(F8), powers(blocks(k), rows).t(),
            whole(*w_shape).float().to(F8), powers(*w_shape[:-2], blocks(n), blocks(k)))


def product(a, sa, w, sw):
    """a [m, k] by w [n, k], a block's sum before its scales: in FP32, which holds these
    sums exactly."""
    m, k, n = a.shape[0], a.shape[1], w.shape[0]
    out = torch.zeros((m, n), device="cuda")
    for b in range(blocks(k)):
        z = a[:, b * 128:(b + 1) * 128].float() @ w[:, b * 128:(b + 1) * 128].float().T
        out += z * sa[:, b:b + 1] * sw[:, b].repeat_interleave(128)[:n]
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,k,n", DENSE)
def test_dense(m, k, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    a, sa, w, sw = operands(g, m, (n, k))
    bias = torch.randint(-64, 65, (n,), generator=g, device="cuda").to(dtype)
    want = product(a, sa, w, sw)
    assert torch.equal(mx.linear_fp8_block(a, sa, w, sw, out_dtype=dtype), want.to(dtype))
    assert torch.equal(mx.linear_fp8_block(a, sa, w, sw, bias, dtype),
                       (want + bias.float()).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("gather", [True, False], ids=["gather", "sorted"])
@pytest.mark.parametrize("m,top_k,experts,k,n", GROUPED)
def test_grouped(m, top_k, experts, k, n, gather, dtype):
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    ids = torch.randint(-1, experts, (m, top_k), generator=g, device="cuda")
    order = mx.sort_routes(ids, experts)
    a, sa, w, sw = operands(g, m if gather else m * top_k, (experts, n, k))
    y = mx.grouped_linear_fp8_block(a, sa, w, sw, order, gather=gather, out_dtype=dtype)
    off = order.offsets.tolist()
    for e in range(experts):
        rows = slice(off[e], off[e + 1])
        at = order.routes[rows].long() // top_k if gather else rows
        assert torch.equal(y[rows], product(a[at], sa[at], w[e], sw[e]).to(dtype)), e
    assert not y[off[-1]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(257, 2176, 2048), (333, 2176, 1024), (333, 2192, 1024),
                                   (5, 1200, 40), (40, 400, 260), (3000, 400, 4096)])
def test_infinite_scales(m, k, n):
    # an infinite block scale gives infinities of its sums' signs, whichever waves add it
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    for block in (0, blocks(k) - 2, blocks(k) - 1):
        a, sa, w, sw = operands(g, m, (n, k))
        sa[m // 2, block] = math.inf
        want = product(a, sa, w, sw)
        y = mx.linear_fp8_block(a, sa, w, sw, out_dtype=FP32)
        assert torch.equal(y.nan_to_num(7e9), want.nan_to_num(7e9))
        assert want[m // 2].isinf().any() and torch.equal(y.isnan(), want.isnan())
