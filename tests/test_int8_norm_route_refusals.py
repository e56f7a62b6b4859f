"""What the grouped router, the 8-bit norm, the int8 quantizer and the W8A8
linear refuse, on the CPU: the Python surface's exception types and the C ABI's
status codes, both before anything is enqueued."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib

INT8, BF16 = torch.int8, torch.bfloat16


def test_native_calls_do_not_take_cpu_tensors():
    host = _lib.host()
    x = torch.zeros((2, 64), dtype=BF16)
    a = torch.zeros((2, 64), dtype=INT8)
    s = torch.ones(2)
    assert host.route_topk_grouped(x, None, 2, 1, 1, 0, 0, True, 1.0, False) is None
    assert host.rms_norm_quant(x, x[0], None, 1e-6, _lib.DT_I8, False) is None
    assert host.int8_quant(x) is None
    assert host.w8a8(a, s, a, s, None, 0) is None
    for name in ("route_topk_grouped", "rms_norm_quant", "int8_quant", "w8a8"):
        with pytest.raises(TypeError, match="expected"):
            getattr(host, name)()


@pytest.mark.parametrize("kw,exc,what", [
    (dict(top_k=0), ValueError, "top_k"),
    (dict(top_k=17), ValueError, "top_k"),
    (dict(top_k=9, num_groups=4, topk_groups=2), ValueError, "top_k"),
    (dict(num_groups=3), ValueError, "groups"),
    (dict(num_groups=0), ValueError, "groups"),
    (dict(num_groups=4, topk_groups=5), ValueError, "groups"),
    (dict(num_groups=4, topk_groups=0), ValueError, "groups"),
    (dict(num_groups=16, topk_groups=4, group_score="top2"), ValueError, "two best"),
    (dict(scoring="tanh"), ValueError, "scoring"),
    (dict(group_score="mean"), ValueError, "group score"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(bias=torch.zeros(8)), ValueError, "bias"),
    (dict(bias=torch.zeros(16, dtype=torch.float64)), TypeError, "bias"),
    (dict(ids_dtype=torch.int16), TypeError, "ids"),
    (dict(), RuntimeError, "ROCm devices only"),
])
def test_router(kw, exc, what):
    with pytest.raises(exc, match=what):
        mx.route_topk_grouped(torch.zeros(4, 16), **{"top_k": 2, **kw})


def test_router_logits():
    with pytest.raises(TypeError):
        mx.route_topk_grouped(torch.zeros(4, 16, dtype=torch.float64), 2)
    with pytest.raises(ValueError):
        mx.route_topk_grouped(torch.tensor(1.0), 1)
    with pytest.raises(ValueError, match="experts"):
        mx.route_topk_grouped(torch.zeros(4, 1025), 2)
    with pytest.raises(ValueError, match="experts"):
        mx.route_topk_grouped(torch.zeros(4, 0), 1)


def test_norm():
    x, w = torch.zeros((2, 3, 64), dtype=BF16), torch.ones(64, dtype=BF16)
    with pytest.raises(ValueError, match="format"):
        mx.rms_norm_quant(x, w, fmt="fp4")
    for eps in (0.0, -1e-6, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            mx.rms_norm_quant(x, w, eps=eps)
    with pytest.raises(TypeError, match="x must be"):
        mx.rms_norm_quant(x.double(), w)
    with pytest.raises(TypeError, match="weight"):
        mx.rms_norm_quant(x, w.half())
    with pytest.raises(ValueError, match="weight"):
        mx.rms_norm_quant(x, w[:32])
    with pytest.raises(ValueError, match="divisible by 32"):
        mx.rms_norm_quant(x[..., :40], w[:40], fmt="mxfp8_e4m3")
    with pytest.raises(TypeError, match="residual"):
        mx.rms_norm_quant(x, w, x.float())
    with pytest.raises(ValueError, match="residual"):
        mx.rms_norm_quant(x, w, x[:1])
    with pytest.raises(ValueError, match="K >= 1"):
        mx.rms_norm_quant(x[..., :0], w[:0])
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        mx.rms_norm_quant(x, w.float(), x)


def test_int8_quant():
    with pytest.raises(TypeError):
        mx.dynamic_int8_quant(torch.zeros((2, 8), dtype=torch.float64))
    with pytest.raises(ValueError):
        mx.dynamic_int8_quant(torch.zeros((2, 0)))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        mx.dynamic_int8_quant(torch.zeros((2, 7)))


def test_w8a8():
    a, w = torch.zeros((2, 3, 64), dtype=INT8), torch.zeros((8, 64), dtype=INT8)
    sa, sw = torch.ones((2, 3)), torch.ones(8)
    f = mx.linear_int8_w8a8
    with pytest.raises(TypeError, match="a must be int8"):
        f(a.to(torch.uint8), sa, w, sw)
    with pytest.raises(TypeError, match="w must be int8"):
        f(a, sa, w.float(), sw)
    with pytest.raises(TypeError, match="output dtype"):
        f(a, sa, w, sw, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="does not match"):
        f(a[..., :32], sa, w, sw)
    with pytest.raises(ValueError, match="divisible by 32"):
        f(a[..., :40], sa, w[:, :40], sw)
    with pytest.raises(ValueError, match="divisible by 32"):
        f(a[..., :0], sa, w[:, :0], sw)
    big = torch.zeros((1, 131072), dtype=INT8)
    with pytest.raises(ValueError, match="131040"):
        f(big, sa[0, :1], big, sw[:1])
    for bad in (sa[:1], sa[..., None, None], torch.ones(6)):
        with pytest.raises(ValueError, match="a_scales"):
            f(a, bad, w, sw)
    with pytest.raises(ValueError, match="w_scales"):
        f(a, sa, w, sw[:4])
    with pytest.raises(TypeError, match="w_scales"):
        f(a, sa, w, sw.half())
    with pytest.raises(TypeError, match="bias"):
        f(a, sa, w, sw, torch.zeros(8))
    with pytest.raises(ValueError, match="bias"):
        f(a, sa, w, sw, torch.zeros(4, dtype=BF16))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        f(a, sa[..., None], w, sw[:, None], torch.zeros(8, dtype=BF16))


def test_c_abi_status_codes():
    lib = _lib.load()
    nul = ctypes.c_void_p()
    T, V, OK = _lib.ERR_TYPE, _lib.ERR_VALUE, _lib.OK
    f32, bf, i8, i64 = _lib.DT_F32, _lib.DT_BF16, _lib.DT_I8, _lib.DT_I64

    def route(dt=f32, m=4, e=16, ld=16, scoring=0, groups=1, keep=1, value=0, top=2, scale=1.0,
              ids=i64):
        return lib.mxfp4_moe_route_grouped(nul, dt, m, e, ld, nul, scoring, groups, keep, value,
                                           top, 1, scale, nul, nul, ids, nul)

    assert route(dt=_lib.DT_U8) == T and route(ids=f32) == T
    for kw in (dict(ld=8), dict(e=1025, ld=1025), dict(e=0), dict(m=-1), dict(scoring=2),
               dict(value=2), dict(groups=3), dict(groups=65, e=65, ld=65), dict(keep=2),
               dict(top=17), dict(top=0), dict(groups=16, keep=4, value=1),
               dict(scale=float("inf")), dict(m=1 << 40)):
        assert route(**kw) == V, kw
    assert route(m=0) == OK

    def norm(dt=bf, rows=2, k=64, ld=64, res=nul, ldr=0, wdt=bf, eps=1e-6, qdt=i8, out=nul):
        return lib.mxfp4_rms_norm_quant(nul, dt, rows, k, ld, res, ldr, nul, wdt, eps, qdt, nul,
                                        nul, out, nul, nul)

    assert norm(dt=i8) == T and norm(wdt=_lib.DT_F16) == T and norm(qdt=bf) == T
    some = ctypes.c_void_p(16)
    for kw in (dict(k=0, ld=0), dict(ld=32), dict(rows=-1), dict(k=40, qdt=_lib.DT_F8E4M3),
               dict(eps=0.0), dict(eps=float("nan")), dict(res=some, ldr=64), dict(out=some),
               dict(res=some, out=some, ldr=32), dict(k=(1 << 20) + 32, ld=(1 << 20) + 32)):
        assert norm(**kw) == V, kw
    assert norm(rows=0) == OK
    assert lib.mxfp4_quant_int8(nul, i8, 1, 8, 8, nul, nul, nul) == T
    assert lib.mxfp4_quant_int8(nul, bf, 1, 8, 4, nul, nul, nul) == V
    assert lib.mxfp4_quant_int8(nul, bf, 0, 8, 8, nul, nul, nul) == OK

    def w8a8(m=2, k=64, n=8, dt=bf, a=nul):
        return lib.mxfp4_linear_w8a8(a, nul, m, k, nul, nul, n, nul, nul, dt, nul)

    assert w8a8(dt=i8) == T
    for kw in (dict(k=0), dict(k=48), dict(k=131072), dict(m=-1), dict(n=-1), dict(m=1 << 31),
               dict(a=ctypes.c_void_p(8)), dict(m=(1 << 31) - 1, n=(1 << 31) - 1)):
        assert w8a8(**kw) == V, kw
    assert w8a8(m=0) == OK and w8a8(n=0) == OK


def test_rows_of():
    t = torch.arange(24.).reshape(4, 6)
    for v, ld, copied in ((t, 6, False), (t[:, :3], 6, False), (t[::2], 12, False),
                          (t.T, 4, True), (t[:1].expand(5, 6), 6, True), (t[:, :1], 6, False),
                          (t[2], 6, False), (t.reshape(2, 2, 6)[:, 1:], 12, False)):
        r, stride = _lib.rows_of(v)
        assert torch.equal(r, v.reshape(-1, v.shape[-1])) and stride == ld, (v, stride)
        assert (r.data_ptr() != v.data_ptr()) == copied
    r, stride = _lib.rows_of(torch.as_strided(t, (1, 6), (1, 1)))
    assert stride == 6 and torch.equal(r[0], t[0])


def test_norm_in_place_needs_rows_of_stride_k():
    # residual_out's rows are k apart: over an input whose rows are not, it would
    # write rows that other workgroups still read
    lib = _lib.load()
    nul, x, r, other = (ctypes.c_void_p(v) for v in (0, 1 << 20, 1 << 21, 1 << 22))

    def norm(ldx, ldr, out, rows=2, k=64):
        return lib.mxfp4_rms_norm_quant(x, _lib.DT_BF16, rows, k, ldx, r, ldr, other, _lib.DT_BF16,
                                        1e-6, _lib.DT_I8, other, other, out, nul, nul)

    assert norm(64, 80, r) == _lib.ERR_VALUE
    assert b"in place" in lib.mxfp4_last_error()
    assert norm(80, 64, x) == _lib.ERR_VALUE
    assert b"in place" in lib.mxfp4_last_error()
    # one row has no stride; no rows write nothing
    assert norm(80, 64, x, rows=0) == _lib.OK
