"""What the FP8 quantizers, the FP8 products and the token sort refuse, on the CPU: the
Python surface's exception types and the C ABI's status codes, both before anything
is enqueued."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def order_of(m=2, top_k=2, experts=3):
    return mx.ExpertOrder(torch.zeros(experts + 1, dtype=torch.int32),
                          torch.zeros(m * top_k, dtype=torch.int32),
                          torch.zeros((m, top_k), dtype=torch.int32))


def test_native_calls_do_not_take_cpu_tensors():
    host = _lib.host()
    x = torch.zeros((4, 256), dtype=BF16)
    a, s = torch.zeros((4, 256)).to(F8), torch.ones((4, 2))
    w, ws = torch.zeros((3, 256, 256)).to(F8), torch.ones((3, 2, 2))
    o = order_of()
    assert host.fp8_quant(x, False) is None and host.fp8_quant(x, True) is None
    assert host.fp8_linear(a, s, w[0], ws[0], None, 0) is None
    assert host.fp8_grouped(a, s, w, ws, o, False, 0) is None
    assert host.fp8_grouped(a, s, w, ws, None, False, 0) is None
    assert host.sort_routes(torch.zeros((2, 2), dtype=torch.int64), 3) is None
    assert host.sort_tokens(x, o) is None and host.sort_tokens(x, None) is None
    assert host.combine_tokens(x, o, None) is None and host.combine_tokens(x, 1, None) is None
    for name in ("fp8_quant", "fp8_linear", "fp8_grouped", "sort_routes", "sort_tokens",
                 "combine_tokens"):
        with pytest.raises(TypeError, match="expected"):
            getattr(host, name)()


def test_quantizers():
    x = torch.zeros((4, 256), dtype=BF16)
    for f in (mx.dynamic_fp8_block_quant, mx.silu_mul_fp8_block_quant):
        with pytest.raises(TypeError, match="x must be"):
            f(x.double())
        with pytest.raises(ValueError, match="K >= 1"):
            f(x[:, :0])
        with pytest.raises(ValueError, match="K >= 1"):
            f(torch.tensor(1.0))
        with pytest.raises(RuntimeError, match="ROCm devices only"):
            f(x)
        with pytest.raises(ValueError, match="at most"):
            f(torch.zeros(2 * 1048576 + 2, dtype=BF16))
    with pytest.raises(ValueError, match="2 K"):
        mx.silu_mul_fp8_block_quant(x[:, :255])
    quant = mx.dynamic_fp8_block_quant
    with pytest.raises(ValueError, match="block_rows"):
        quant(x, block_rows=64)
    with pytest.raises(TypeError, match="x must be"):
        quant(x.double(), block_rows=128)
    for bad in (x[0], x[None, None], x[:, :0]):
        with pytest.raises(ValueError, match="weights"):
            quant(bad, block_rows=128)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        quant(x, block_rows=128)


def test_linear():
    a, sa = torch.zeros((2, 3, 256)).to(F8), torch.ones((2, 3, 2))
    w, sw = torch.zeros((200, 256)).to(F8), torch.ones((2, 2))
    f = mx.linear_fp8_block
    with pytest.raises(TypeError, match="a must be float8_e4m3fn"):
        f(a.to(torch.float8_e5m2), sa, w, sw)
    with pytest.raises(TypeError, match="w must be float8_e4m3fn"):
        f(a, sa, w.float(), sw)
    with pytest.raises(TypeError, match="output dtype"):
        f(a, sa, w, sw, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="does not match"):
        f(a[..., :128], sa, w, sw)
    with pytest.raises(ValueError, match="divisible by 16"):
        f(a[..., :40], sa, w[:, :40], sw)
    with pytest.raises(ValueError, match="divisible by 16"):
        f(a[..., :0], sa, w[:, :0], sw)
    with pytest.raises(ValueError, match="N, K"):
        f(a, sa, w[0], sw)
    for bad in (sa[:1], sa[..., :1], sa[..., None], torch.ones((6, 2))):
        with pytest.raises(ValueError, match="a_scales"):
            f(a, bad, w, sw)
    with pytest.raises(TypeError, match="a_scales"):
        f(a, sa.half(), w, sw)
    for bad in (sw[:1], sw[0], torch.ones((200, 2))):
        with pytest.raises(ValueError, match="w_scales"):
            f(a, sa, w, bad)
    with pytest.raises(TypeError, match="w_scales"):
        f(a, sa, w, sw.half())
    with pytest.raises(TypeError, match="bias"):
        f(a, sa, w, sw, torch.zeros(200))
    with pytest.raises(ValueError, match="bias"):
        f(a, sa, w, sw, torch.zeros(100, dtype=BF16))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        f(a, sa, w, sw, torch.zeros(200, dtype=BF16))


def test_grouped():
    a, sa = torch.zeros((4, 256)).to(F8), torch.ones((4, 2))
    w, sw = torch.zeros((3, 200, 256)).to(F8), torch.ones((3, 2, 2))
    f, o = mx.grouped_linear_fp8_block, order_of()
    with pytest.raises(ValueError, match="E, N, K"):
        f(a, sa, w[0], sw[0], o)
    with pytest.raises(ValueError, match="w_scales"):
        f(a, sa, w, sw[0], o)
    with pytest.raises(ValueError, match="experts"):
        f(a, sa, w, sw, order_of(experts=4))
    with pytest.raises(ValueError, match="a must be"):
        f(a[:2], sa[:2], w, sw, o)
    with pytest.raises(ValueError, match="a must be"):
        f(a, sa, w, sw, o, gather=True)
    with pytest.raises(ValueError, match="a must be"):
        f(a[None], sa[None], w, sw, o)
    with pytest.raises(ValueError, match="inconsistent order"):
        f(a, sa, w, sw, o._replace(routes=o.routes[:3]))
    with pytest.raises(TypeError, match="offsets must be int32"):
        f(a, sa, w, sw, o._replace(offsets=o.offsets.long()))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        f(a, sa, w, sw, o)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        f(a[:2], sa[:2], w, sw, o, gather=True)


def test_sort():
    ids = torch.zeros((4, 2), dtype=torch.int64)
    for bad in (ids.float(), ids.bool(), ids.to(torch.complex64)):
        with pytest.raises(TypeError, match="integers"):
            mx.sort_routes(bad, 4)
    for bad in (ids[0], ids[None], ids[:, :0], torch.zeros((1, 65), dtype=torch.int64)):
        with pytest.raises(ValueError, match="top_k"):
            mx.sort_routes(bad, 4)
    for e in (0, -1, 1025):
        with pytest.raises(ValueError, match="experts"):
            mx.sort_routes(ids, e)
    for e in (4.0, "4", None):
        with pytest.raises(TypeError):
            mx.sort_routes(ids, e)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        mx.sort_routes(ids, 4)
    o, x, y = order_of(), torch.zeros((2, 8)), torch.zeros((4, 8))
    with pytest.raises(TypeError, match="dtype"):
        mx.sort_tokens(x.double(), o)
    for bad in (y, x[0], x[None]):
        with pytest.raises(ValueError, match="x must be"):
            mx.sort_tokens(bad, o)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        mx.sort_tokens(x, o)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        mx.sort_tokens(x.clone().requires_grad_(), o)
    with pytest.raises(TypeError, match="y must be"):
        mx.combine_tokens(y.to(F8), o)
    for bad in (x, y[0], y[None]):
        with pytest.raises(ValueError, match="y must be"):
            mx.combine_tokens(bad, o)
    with pytest.raises(ValueError, match="topk_weights"):
        mx.combine_tokens(y, o, torch.ones(4))
    with pytest.raises(TypeError, match="topk_weights"):
        mx.combine_tokens(y, o, torch.ones((2, 2), dtype=torch.int64))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        mx.combine_tokens(y, o, torch.ones((2, 2)))
    for bad in (o._replace(offsets=o.offsets[:1]), o._replace(offsets=o.offsets[None]),
                o._replace(routes=o.routes[:3]), o._replace(position=o.position[0])):
        with pytest.raises(ValueError, match="inconsistent order"):
            mx.sort_tokens(x, bad)
        with pytest.raises(ValueError, match="inconsistent order"):
            mx.combine_tokens(y, bad)
    with pytest.raises(TypeError, match="position must be int32"):
        mx.sort_tokens(x, o._replace(position=o.position.long()))


def test_c_abi_status_codes():
    lib = _lib.load()
    nul = ctypes.c_void_p()
    T, V, OK = _lib.ERR_TYPE, _lib.ERR_VALUE, _lib.OK
    f32, bf, i8, i32 = _lib.DT_F32, _lib.DT_BF16, _lib.DT_I8, _lib.DT_I32

    def rows(dt=bf, rows=2, k=64, ld=64, silu=0, sr=1, sb=2):
        return lib.mxfp4_quant_fp8_rows(nul, dt, rows, k, ld, silu, nul, nul, sr, sb, nul)

    assert rows(dt=i8) == T and rows(rows=0) == OK
    for kw in (dict(k=0), dict(ld=63), dict(rows=-1), dict(silu=1), dict(sr=0), dict(sb=0),
               dict(k=1048577, ld=1048577)):
        assert rows(**kw) == V, kw
    blocks = lambda dt=bf, n=2, k=64, ld=64: lib.mxfp4_quant_fp8_blocks(  # noqa: E731
        nul, dt, n, k, ld, nul, nul, nul)
    assert blocks(dt=i8) == T and blocks(n=0) == OK
    for kw in (dict(k=0), dict(ld=63), dict(n=-1), dict(n=1 << 40)):
        assert blocks(**kw) == V, kw

    def linear(m=2, k=64, n=8, dt=bf, a=nul, sr=1, sb=2):
        return lib.mxfp4_linear_fp8(a, nul, sr, sb, m, k, nul, nul, n, nul, nul, dt, nul)

    assert linear(dt=i8) == T
    for kw in (dict(k=0), dict(k=40), dict(k=1048592), dict(m=-1), dict(n=-1), dict(m=1 << 31),
               dict(a=ctypes.c_void_p(8)), dict(m=(1 << 31) - 1, n=(1 << 31) - 1), dict(sr=0),
               dict(sb=0), dict(sb=1 << 29, k=256), dict(m=1 << 29, sr=2), dict(sr=1 << 40)):
        assert linear(**kw) == V, kw
    assert linear(m=0) == OK and linear(n=0) == OK

    def grouped(m=4, k=64, n=8, dt=bf, e=3, routes=nul, top=2, rows=4):
        return lib.mxfp4_grouped_linear_fp8(nul, nul, 1, max(m, 1), m, k, nul, nul, e, n, nul,
                                            routes, top, rows, nul, dt, nul)

    some = ctypes.c_void_p(16)
    assert grouped(dt=i8) == T
    for kw in (dict(e=0), dict(e=1025), dict(top=0), dict(rows=5), dict(k=8),
               dict(routes=some, m=1 << 25, rows=1 << 26), dict(routes=some, m=0)):
        assert grouped(**kw) == V, kw
    assert grouped(rows=0, m=0) == OK and grouped(n=0) == OK

    nbytes = ctypes.c_int64()
    size = lambda n, e: lib.mxfp4_sort_routes_workspace_size(  # noqa: E731
        n, e, ctypes.byref(nbytes))
    for bad in ((-1, 4), (1 << 30, 4), (8, 0), (8, 1025)):
        assert size(*bad) == V
    assert size(16384, 128) == OK and nbytes.value == 0
    assert size(16385, 128) == OK and nbytes.value > 0
    routes = lambda dt=i32, n=8, e=4, b=0: lib.mxfp4_sort_routes(  # noqa: E731
        nul, dt, n, e, nul, nul, nul, nul, b, nul)
    assert routes(dt=f32) == T
    for kw in (dict(n=-1), dict(e=0), dict(n=20000), dict(n=20000, b=64)):
        assert routes(**kw) == V, kw

    def tokens(dt=bf, m=2, h=8, ld=8, e=4, top=2):
        return lib.mxfp4_sort_tokens(nul, dt, m, h, ld, nul, nul, e, top, nul, nul)

    assert tokens(dt=9) == T and tokens(dt=-1) == T and tokens(m=0) == OK
    for kw in (dict(m=-1), dict(h=0), dict(ld=7), dict(e=0), dict(top=0), dict(top=65),
               dict(m=1 << 30)):
        assert tokens(**kw) == V, kw

    def combine(dt=bf, rows=4, m=2, h=8, ld=8, top=2):
        return lib.mxfp4_combine_tokens(nul, dt, rows, h, ld, nul, m, top, nul, nul, nul)

    assert combine(dt=i8) == T and combine(m=0) == OK
    for kw in (dict(m=-1), dict(h=0), dict(ld=7), dict(top=0), dict(top=65), dict(rows=-1)):
        assert combine(**kw) == V, kw

    def grad(dt=bf, m=2, h=8, ld=8, ldy=8, e=4, top=2, dy=nul, dw=nul):
        return lib.mxfp4_combine_tokens_grad(nul, dt, m, h, ld, nul, ldy, nul, nul, e, top, nul, dy,
                                             dw, nul)

    assert grad(dt=i8) == T and grad(m=0) == OK and grad() == OK
    for kw in (dict(m=-1), dict(h=0), dict(ld=7), dict(e=0), dict(top=0), dict(top=65),
               dict(dw=some, ldy=7)):
        assert grad(**kw) == V, kw
