"""GPU: the 8-bit RMS norm and the int8 quantizer.

With h = x + residual in FP32, y = (h * w) * rs carries three FP32 roundings
(the product, rs from FP64, their product), 2^-24 each: U = 3.01 * 2^-24 of y.
A y rounded to a type is off by half its step more.  The 8-bit values follow
from y by exact rules, which are checked bit for bit on the FP32 y that
``normed`` returns for FP32 input; the other types are held to the FP64 oracle
within half a step of the 8-bit type."""

from __future__ import annotations

import math

import pytest
import torch

import mxfp4_amd as mx

from _helpers import cuda

pytestmark = pytest.mark.gpu
U = 3.01 * 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
MX = {"mxfp8_e4m3": (8, 448.0, torch.float8_e4m3fn, 2.0 ** -4, 2.0 ** -10),
      "mxfp8_e5m2": (15, 57344.0, torch.float8_e5m2, 2.0 ** -3, 2.0 ** -17)}
TINY = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}  # half the smallest step


def _rand(shape, seed, dtype=FP32, loud=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(4 * torch.rand((*shape[:-1], 1), generator=g))
    if loud and shape[-1] > 8:
        x[..., 5] *= 30
    return x.to(dtype)


def int8_of(y):
    """As FP32 gives it, on the CPU."""
    s = (y.abs().amax(-1) / 127).clamp(min=2.0 ** -126)
    return torch.round(y / s[..., None]).clamp(-127, 127).to(torch.int8), s


def mx_of(y, fmt):
    emax, most, f8 = MX[fmt][:3]
    b = y.double().reshape(*y.shape[:-1], -1, 32)
    amax = b.abs().amax(-1)
    e = (torch.frexp(amax)[1] - 1 - emax).clamp(-127, 127)
    e = torch.where(amax == 0, -127, e)
    q = torch.ldexp(b, -e[..., None]).clamp(-most, most).float()
    return q.to(f8).reshape(y.shape), (e + 127).to(torch.uint8)


def norm64(x, w, r=None, eps=1e-6):
    h = x.float() if r is None else x.float() + r.float()
    d = h.double()
    eps = float(torch.tensor(eps, dtype=FP32))
    y = d * w.double() / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return y, None if r is None else h.to(x.dtype)


def call(x, w, r=None, **kw):
    out = mx.rms_norm_quant(cuda(x), cuda(w), None if r is None else cuda(r), **kw)
    return [None if t is None else t.cpu() for t in out]


def near(got, want, dtype):
    """got of `dtype` against FP64 values: half a step of it and y's own roundings."""
    half = 0.0 if dtype == FP32 else torch.finfo(dtype).eps / 2
    got, want = got.double(), want.double()
    ok = (got - want).abs() <= (half + U) * want.abs() + TINY[dtype]
    assert ok.all(), float((got - want).abs().max())


def check(x, w, r=None, fmt="int8", eps=1e-6):
    y, sum_ = norm64(x, w, r, eps)
    q, s, res, normed = call(x, w, r, fmt=fmt, eps=eps, normed=True)
    assert (res is None) == (r is None) and q.shape == x.shape
    if r is not None:
        assert torch.equal(res, sum_)
    near(normed, y, x.dtype)
    if fmt == "int8":
        assert q.dtype == torch.int8 and s.dtype == FP32 and s.shape == x.shape[:-1]
        if x.dtype == FP32:
            wq, ws = int8_of(normed)
            assert torch.equal(s, ws) and torch.equal(q, wq)
        want = (y.abs().amax(-1) / 127).clamp(min=2.0 ** -126)
        assert ((s.double() - want).abs() <= (U + 2.0 ** -24) * want).all()
        # half an integer, and the roundings of y, s and the quotient
        err = (q.double() - y / want[..., None]).abs()
        assert float(err.max()) <= 0.5 + 127 * (2 * U + 2 * 2.0 ** -24)
    else:
        emax, most, f8, half, tiny = MX[fmt]
        assert q.dtype == f8 and s.dtype == torch.uint8
        assert s.shape == (*x.shape[:-1], x.shape[-1] // 32)
        if x.dtype == FP32:
            wq, ws = mx_of(normed, fmt)
            assert torch.equal(s, ws)
            assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8))
        amax = y.reshape(*s.shape, 32).abs().amax(-1)
        e = s.double() - 127
        lo, hi = torch.exp2(e + emax) * (1 - U), torch.exp2(e + emax + 1) * (1 + U)
        assert (((amax >= lo) | (s == 0)) & (amax < hi)).all()
        unit = torch.exp2(e).repeat_interleave(32, -1).reshape(y.shape)
        z = (y / unit).clamp(-most, most)
        err = (q.double() - z).abs()
        assert (err <= (half + U) * z.abs() + tiny).all()


@pytest.mark.parametrize("fmt", ["int8", *MX])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 2048), (3, 512), (5, 544), (2, 4096), (7, 4128),
                                    (2, 8192), (3, 14336), (2, 16384), (2, 16416), (1, 65536),
                                    (2, 1024), (2, 1056), (2, 3104), (513, 2048), (514, 4096)])
def test_norm_sizes(fmt, dtype, rows, k):
    w = _rand((k,), 1, FP32 if rows % 2 else dtype, loud=False)
    r = _rand((rows, k), 2, dtype) if rows != 5 else None
    check(_rand((rows, k), rows + k, dtype), w, r, fmt)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("k", [1, 2, 7, 8, 33, 127, 1000, 2049, 4097, 16385, 20000])
def test_norm_int8_odd_lengths(dtype, k):
    check(_rand((3, k), k, dtype), _rand((k,), 3, dtype), _rand((3, k), 4, dtype))


@pytest.mark.parametrize("fmt,k", [("int8", 100), ("mxfp8_e4m3", 96), ("mxfp8_e5m2", 20000)])
def test_norm_strides_and_alignment(fmt, k):
    x, r, w = _rand((4, k), 1, BF16), _rand((4, k), 2, BF16), _rand((k,), 3, BF16)
    want = call(x, w, r, fmt=fmt, normed=True)

    def same(a, b, c):
        got = mx.rms_norm_quant(a, c, b, fmt=fmt, normed=True)
        for g, o in zip(got, want):
            g = g.reshape(o.shape).cpu()
            assert torch.equal(g.view(torch.uint8) if g.dtype.itemsize == 1 else g,
                               o.view(torch.uint8) if o.dtype.itemsize == 1 else o)

    def wide(t, before, after):  # rows inside a wider tensor of NaN
        buf = torch.full((4, before + k + after), math.nan, dtype=BF16)
        buf[:, before:before + k] = t
        return cuda(buf)[:, before:before + k]

    same(wide(x, 8, 8), wide(r, 0, 16), cuda(w))
    same(wide(x, 1, 2), wide(r, 3, 0), cuda(w))
    same(cuda(x), cuda(r), wide(w.expand(4, k), 1, 0)[0])
    same(cuda(x.T.contiguous()).T, cuda(r), cuda(w))
    same(cuda(x).view(2, 2, k), cuda(r).view(2, 2, k), cuda(w))
    one = mx.rms_norm_quant(cuda(x)[1], cuda(w), cuda(r)[1], fmt=fmt)
    assert torch.equal(one.scales.cpu(), want[1][1]) and one.normed is None


def test_norm_broadcast_rows_and_empty():
    x, w = _rand((1, 64), 1, BF16), _rand((64,), 2, BF16)
    got = mx.rms_norm_quant(cuda(x).expand(5, 64), cuda(w), cuda(x).expand(5, 64))
    want = call(x, w, x)
    for g, o in zip(got[:3], want):
        assert torch.equal(g.cpu(), o.expand(5, *o.shape[1:]))
    e = mx.rms_norm_quant(cuda(x)[:0], cuda(w), cuda(x)[:0], fmt="mxfp8_e4m3", normed=True)
    assert [tuple(t.shape) for t in e] == [(0, 64), (0, 2), (0, 64), (0, 64)]


@pytest.mark.parametrize("fmt", ["int8", "mxfp8_e4m3"])
@pytest.mark.parametrize("k", [64, 20000])
def test_norm_rows_are_independent_and_special_values(fmt, k):
    x = _rand((12, k), 7, FP32)
    w = _rand((k,), 8, FP32, loud=False)
    clean = call(x, w, fmt=fmt)
    bad = x.clone()
    bad[2, 3] = math.nan
    bad[4, k - 1] = math.inf
    bad[5] = -math.inf
    got = call(bad, w, fmt=fmt)
    rest = [0, 1, 3, 6, 7, 8, 9, 10, 11]
    assert torch.equal(got[0][rest].view(torch.uint8), clean[0][rest].view(torch.uint8))
    assert torch.equal(got[1][rest], clean[1][rest])
    if fmt == "int8":
        assert got[1][[2, 4, 5]].isnan().all() and (got[0][[2, 4, 5]] == 0).all()
    else:
        assert (got[1][[2, 5]] == 255).all() and (got[0][[2, 4, 5]].float() == 0).all()
        # one infinity: its block is not a number, the others' y are 0
        assert int(got[1][4, -1]) == 255 and (got[1][4, :-1] == 0).all()
    # large and small rows: the mean of the squares stays in FP64's range
    for size in (3e38, 1e30, 1e-18, 1e-30, 0.0):
        v = torch.full((1, k), size)
        v[0, ::2] *= -1
        check(v, torch.full((k,), 0.5), fmt=fmt)
    check(x * 1e-20, w, fmt=fmt, eps=1e-45)
    check(torch.zeros(2, k), w, fmt=fmt)
    # a weight of 0, and one that leaves FP32 with one element
    check(x, torch.zeros(k), fmt=fmt)
    big = w.clone()
    big[1] = 3e38
    v = torch.full((1, k), 2.0)
    q, s, _, _ = call(v, big, fmt=fmt)
    assert s.isnan().all() if fmt == "int8" else int(s[0, 0]) == 255


@pytest.mark.parametrize("k", [2048, 20000])
def test_norm_writes_its_rows_only(k):
    # the C entry with outputs inside larger buffers, the residual in place
    from mxfp4_amd import _lib
    rows = 3
    x, r, w = (cuda(_rand(s, i, BF16)) for i, s in ((1, (rows, k)), (2, (rows, k)), (3, (k,))))
    want = mx.rms_norm_quant(x, w, r, normed=True)
    q = torch.full(((rows + 2) * k,), 77, dtype=torch.int8, device="cuda")
    s = torch.full((rows + 2,), 5.0, device="cuda")
    sums = torch.full((rows + 2, k), 9.0, dtype=BF16, device="cuda")
    sums[1:-1] = r
    y = torch.full((rows + 2, k), 9.0, dtype=BF16, device="cuda")
    p = lambda t: _lib.ctypes.c_void_p(t)  # noqa: E731
    _lib.check(_lib.load().mxfp4_rms_norm_quant(
        _lib.ptr(x), _lib.DT_BF16, rows, k, k, p(sums[1:].data_ptr()), k, _lib.ptr(w),
        _lib.DT_BF16, 1e-6, _lib.DT_I8, p(q.data_ptr() + k), p(s.data_ptr() + 4),
        p(sums[1:].data_ptr()), p(y[1:].data_ptr()), _lib.stream_of(x.device)))
    assert torch.equal(q[k:-k].view(rows, k), want.q) and torch.equal(s[1:-1], want.scales)
    assert torch.equal(sums[1:-1], want.residual) and torch.equal(y[1:-1], want.normed)
    assert (q[:k] == 77).all() and (q[-k:] == 77).all() and s[0] == s[-1] == 5
    for t in (sums, y):
        assert (t[0] == 9).all() and (t[-1] == 9).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4096), (5, 7), (3, 100), (9, 512), (130, 2048),
                                    (4, 5121), (2, 14336), (2, 30000), (70000, 40)])
def test_int8_quant_bit_for_bit(dtype, rows, k):
    x = _rand((rows, k), rows + k, dtype)
    x[0, k // 2] = 0
    q, s = mx.dynamic_int8_quant(cuda(x))
    wq, ws = int8_of(x.float())
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)


def test_int8_quant_ties_and_special_rows():
    # scales 1, 0.5 and 3: quotients on the half
    x = torch.zeros((9, 64))
    x[0, :8] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5])
    x[1, :4] = torch.tensor([63.5, 0.25, 0.75, -1.25])
    x[2, :4] = torch.tensor([-381.0, 1.5, 4.5, 7.5])
    x[3] = 1e-42
    x[4, 0] = torch.finfo(FP32).max
    x[5, 9] = math.nan
    x[6, 9] = math.inf
    x[7] = -0.0
    x[8] = torch.linspace(-1, 1, 64)
    q, s = (t.cpu() for t in mx.dynamic_int8_quant(cuda(x)))
    fine = [0, 1, 2, 3, 4, 7, 8]
    wq, ws = int8_of(x[fine])
    assert torch.equal(q[fine], wq) and torch.equal(s[fine], ws)
    assert s[[5, 6]].isnan().all() and (q[[5, 6]] == 0).all()
    # many quotients of many scales
    g = torch.Generator().manual_seed(1)
    amax = torch.exp2(60 * torch.rand(512, generator=g) - 30)
    x = amax[:, None] * (torch.randint(-127, 128, (512, 256), generator=g) + 0.5) / 127.5
    x[:, 0] = amax
    for t in (x, x.to(BF16), x.to(BF16).float() * 3):
        q, s = mx.dynamic_int8_quant(cuda(t))
        wq, ws = int8_of(t.float())
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)


def test_offsets_beyond_31_bits():
    rows, k = 300000, 8192  # 2.46e9 elements
    x = torch.empty((rows, k), dtype=BF16, device="cuda")
    x[:4], x[-4:] = 1.0, 1.0
    tail = _rand((4, k), 5, BF16)
    x[4:-4] = 0.25
    x[-4:] = cuda(tail)
    w = _rand((k,), 6, BF16)
    got = mx.rms_norm_quant(x, cuda(w))
    want = call(tail, w)
    assert torch.equal(got.q[-4:].cpu(), want[0]) and torch.equal(got.scales[-4:].cpu(), want[1])
    q, s = mx.dynamic_int8_quant(x)
    wq, ws = int8_of(tail.float())
    assert torch.equal(q[-4:].cpu(), wq) and torch.equal(s[-4:].cpu(), ws)
    assert (q[4:-4:4096] == 127).all()


@pytest.mark.parametrize("rows,k", [(3, 2048), (40, 1000), (2, 20000), (1, 96)])
def test_norm_sum_over_x_or_the_residual(rows, k):
    # the C entry with residual_out = x or the residual; one row of any stride
    from mxfp4_amd import _lib
    x, r, w = (cuda(_rand(s, i, BF16)) for i, s in ((1, (rows, k)), (2, (rows, k)), (3, (k,))))
    want = mx.rms_norm_quant(x, w, r)
    for over in (0, 1):
        ins = [x.clone(), r.clone()]
        q, s = torch.empty_like(want.q), torch.empty_like(want.scales)
        strides = [k + 8 if rows == 1 else k] * 2
        _lib.check(_lib.load().mxfp4_rms_norm_quant(
            _lib.ptr(ins[0]), _lib.DT_BF16, rows, k, strides[0], _lib.ptr(ins[1]), strides[1],
            _lib.ptr(w), _lib.DT_BF16, 1e-6, _lib.DT_I8, _lib.ptr(q), _lib.ptr(s),
            _lib.ptr(ins[over]), None, _lib.stream_of(x.device)))
        assert torch.equal(q, want.q) and torch.equal(s, want.scales)
        assert torch.equal(ins[over], want.residual)
        assert torch.equal(ins[1 - over], (r, x)[over])


@pytest.mark.parametrize("fmt", ["int8", *MX])
def test_norm_repeats_itself_bit_for_bit(fmt):
    for rows, k in ((700, 4096), (1, 2048), (9, 20000)):
        x, r, w = (cuda(_rand(s, i, BF16)) for i, s in ((1, (rows, k)), (2, (rows, k)), (3, (k,))))
        a, b = (mx.rms_norm_quant(x, w, r, fmt=fmt, normed=True) for _ in range(2))
        for p, q in zip(a, b):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
