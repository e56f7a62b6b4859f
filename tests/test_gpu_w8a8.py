"""GPU: the W8A8 linear against FP64.  The int32 sum is exact; FP32 from there:
one rounding of the sum, two products, the bias' addition, 2^-24 each, then half
a step of the output type."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib

from _helpers import cuda

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24 * 1.01
HALF = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 0.0}
TINY = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -148}


def operands(m, k, n, seed=0, bias=None):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * k + 7 * n)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sa = torch.rand(m, generator=g, device="cuda") * 1e-2 + 1e-4
    sw = torch.rand(n, generator=g, device="cuda") * 1e-2 + 1e-4
    b = None
    if bias is not None:
        b = (torch.randn(n, generator=g, device="cuda") * 0.1 * math.sqrt(k)).to(bias)
    return a, sa, w, sw, b


def w8a8_tile(m, k, n, dtype, cus=256):
    """(rows, columns) of the tile that a size runs with."""
    f = _lib.load().mxfp4_test_w8a8_tile
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_int64]
    v = f(m, k, n, n * dtype.itemsize % 16 == 0, cus)
    return v >> 16, v & 65535


def agree(y, a, sa, w, sw, b=None, rows=slice(None)):
    dot = a[rows].double() @ w.double().T  # exact: below 2^53
    prod = dot * sa[rows].double()[:, None] * sw.double()
    want = prod if b is None else prod + b.double()
    tol = 3 * E * prod.abs() + (E + HALF[y.dtype]) * want.abs() + TINY[y.dtype]
    err = (y[rows].double() - want).abs()
    if y.dtype == FP16:  # half a step below the largest value rounds to infinity
        over = want.abs() >= 65519.99
        err = torch.where(over & (y[rows].double().abs() >= 65504), 0.0, err)
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128, 130, 255, 257, 520])
@pytest.mark.parametrize("k,n", [(32, 1), (64, 16), (96, 100), (160, 63), (256, 65), (1024, 256),
                                 (4096, 300), (2080, 1028)])
def test_sizes(m, k, n):
    dtype = (BF16, FP16, FP32)[(m + k + n) % 3]
    a, sa, w, sw, b = operands(m, k, n, bias=dtype if (m + n) % 2 else None)
    y = mx.linear_int8_w8a8(a, sa, w, sw, b, dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    agree(y, a, sa, w, sw, b)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,k,n", [(1, 2048, 5120), (48, 4096, 2048), (130, 2048, 5120),
                                   (1021, 4096, 2048), (2048, 1024, 4096), (4096, 2048, 5120),
                                   (2500, 544, 2570), (700, 8192, 1000), (4000, 288, 4001)])
def test_larger(m, k, n, dtype):
    a, sa, w, sw, b = operands(m, k, n, bias=dtype)
    agree(mx.linear_int8_w8a8(a, sa, w, sw, b, dtype), a, sa, w, sw, b)
    y = mx.linear_int8_w8a8(a, sa[:, None], w, sw[:, None], None, dtype)
    agree(y, a, sa, w, sw)


# a size of each tile, its last tile partly outside; K that ends inside a stage
TILES = {(256, 256): (3900, 8224, 4090), (256, 128): (2040, 8224, 4090),
         (128, 128): (2040, 1056, 2040), (128, 64): (1021, 4128, 2046), (64, 64): (130, 2080, 5118),
         (32, 32): (110, 2080, 1424), (16, 32): (45, 4128, 2046), (16, 16): (13, 12960, 70)}


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tile", TILES, ids=lambda t: f"{t[0]}x{t[1]}")
def test_every_tile(tile, dtype):
    m, k, n = TILES[tile]
    n = n // 16 * 16
    for cols in (n, n - 1, n - 2):  # rows on 16, 2 and 4 bytes (bf16)
        assert w8a8_tile(m, k, cols, dtype) == tile
        a, sa, w, sw, b = operands(m, k, cols, bias=dtype)
        for bias in (b, None):
            agree(mx.linear_int8_w8a8(a, sa, w, sw, bias, dtype), a, sa, w, sw, bias)


@pytest.mark.parametrize("m", [1, 40, 300, 4096])
def test_the_sum_is_exact_at_its_largest(m):
    k, n = (131040, 48) if m < 4096 else (8192, 4096)
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    a[m // 2] = 127
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    y = mx.linear_int8_w8a8(a, one[0], w, one[1], out_dtype=FP32)
    # int32 -> FP32 is the one rounding
    want = (a[:4].double() @ w.double().T).float()
    assert torch.equal(y[:4], want)
    assert torch.equal(y[m // 2], (a[m // 2].double() @ w.double().T).float())


@pytest.mark.parametrize("m", [3, 70, 600])
def test_layouts_and_leading_dimensions(m):
    k, n = 256, 130
    a, sa, w, sw, b = operands(m, k, n, bias=BF16)
    want = mx.linear_int8_w8a8(a, sa, w, sw, b)
    buf = torch.full((m + 1, k + 40), 9, dtype=torch.int8, device="cuda")
    for off in (0, 1, 16):
        buf[:m, off:off + k] = a
        assert torch.equal(mx.linear_int8_w8a8(buf[:m, off:off + k], sa, w, sw, b), want)
    wide = torch.full((n, k + 3), 9, dtype=torch.int8, device="cuda")
    wide[:, 3:] = w
    assert torch.equal(mx.linear_int8_w8a8(a, sa, wide[:, 3:], sw, b), want)
    flat = torch.zeros(n * k + 5, dtype=torch.int8, device="cuda")
    flat[5:] = w.reshape(-1)
    assert torch.equal(mx.linear_int8_w8a8(a, sa, flat[5:].view(n, k), sw, b), want)
    assert torch.equal(mx.linear_int8_w8a8(a, sa, w.T.contiguous().T, sw, b), want)
    # scales and bias that begin off 16 bytes
    s1, w1, b1 = (torch.cat([t[:1], t])[1:] for t in (sa, sw, b))
    assert torch.equal(mx.linear_int8_w8a8(a, s1, w, w1, b1), want)
    s2 = torch.stack([sa, sa + 1], 1)[:, 0]
    assert torch.equal(mx.linear_int8_w8a8(a, s2, w, torch.stack([sw, sw], 1)[:, 1], b), want)
    y = mx.linear_int8_w8a8(a[None, :, None], sa[None, :, None], w, sw, b)
    assert y.shape == (1, m, 1, n) and torch.equal(y[0, :, 0], want)
    y = mx.linear_int8_w8a8(a[0], sa[0], w, sw, b)
    assert y.shape == (n,) and torch.equal(y, mx.linear_int8_w8a8(a[:1], sa[:1], w, sw, b)[0])
    assert mx.linear_int8_w8a8(a[:0], sa[:0], w, sw, b).shape == (0, n)
    assert mx.linear_int8_w8a8(a, sa, w[:0], sw[:0]).shape == (m, 0)


@pytest.mark.parametrize("m,k,n", [(2, 2048, 64), (50, 96, 131), (333, 1024, 517), (4096, 256, 4096)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_scales_that_are_not_finite_stay_in_their_row_and_column(m, k, n, dtype):
    a, sa, w, sw, _ = operands(m, k, n)
    clean = mx.linear_int8_w8a8(a, sa, w, sw, out_dtype=dtype)
    sa2, sw2 = sa.clone(), sw.clone()
    sa2[m // 2], sw2[n // 3] = math.nan, math.nan
    y = mx.linear_int8_w8a8(a, sa2, w, sw2, out_dtype=dtype)
    assert y[m // 2].isnan().all() and y[:, n // 3].isnan().all()
    rows = torch.arange(m, device="cuda") != m // 2
    cols = torch.arange(n, device="cuda") != n // 3
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])


@pytest.mark.parametrize("m,k,n", [(1, 2048, 33), (17, 96, 20), (40, 4096, 2048), (100, 512, 70),
                                   (300, 96, 250), (2000, 160, 2100), (4096, 256, 4096)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_writes_its_output_only(m, k, n, dtype):
    # the C entry, its output inside a larger buffer; off a 16-byte boundary too
    a, sa, w, sw, b = operands(m, k, n, bias=dtype)
    want = mx.linear_int8_w8a8(a, sa, w, sw, b, dtype)
    for before in (64, 61):
        buf = torch.full((before + m * n + 64,), 3.0, dtype=dtype, device="cuda")
        _lib.check(_lib.load().mxfp4_linear_w8a8(
            _lib.ptr(a), _lib.ptr(sa), m, k, _lib.ptr(w), _lib.ptr(sw), n, _lib.ptr(b),
            ctypes.c_void_p(buf.data_ptr() + before * buf.element_size()),
            _lib.dtype_code(dtype), _lib.stream_of(a.device)))
        assert (buf[:before] == 3).all() and (buf[before + m * n:] == 3).all()
        assert torch.equal(buf[before:before + m * n].view(m, n), want)


def test_every_size_gives_the_same_bits_per_row():
    # a row's result does not depend on how many rows are beside it
    a, sa, w, sw, b = operands(4096, 1024, 4096, bias=BF16)
    full = mx.linear_int8_w8a8(a, sa, w, sw, b)
    for m in (1, 5, 40, 64, 100, 200, 500, 1000, 2000):
        assert torch.equal(mx.linear_int8_w8a8(a[:m], sa[:m], w, sw, b), full[:m]), m


def test_offsets_beyond_31_bits():
    m, k = 600000, 4096  # 2.46 GB of activations
    g = torch.Generator(device="cuda").manual_seed(1)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    _, _, w, sw, _ = operands(1, k, 80)
    sa = torch.rand(m, generator=g, device="cuda")
    y = mx.linear_int8_w8a8(a, sa, w, sw, out_dtype=FP32)
    agree(y, a, sa, w, sw, rows=slice(m - 300, m))
    # as many weights, and as many outputs
    y = mx.linear_int8_w8a8(w[:3], sw[:3], a, sa, out_dtype=FP32)
    agree(y.T.contiguous(), a, sa, w[:3], sw[:3], rows=slice(m - 300, m))
    del a, y
    a, sa, w, sw, _ = operands(50000, 32, 50000)
    y = mx.linear_int8_w8a8(a, sa, w, sw)
    agree(y, a, sa, w, sw, rows=slice(49900, 50000))
