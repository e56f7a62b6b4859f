"""GPU: the FP8 quantizers.  Scales bit for bit, values bit for bit with the exact
quotient's rounding; SiLU-mul within half a step of e4m3 and what FP32 may be off."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib

from _helpers import cuda

pytestmark = pytest.mark.gpu
BF16, FP16, FP32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def gen(*seed):
    return torch.Generator(device="cuda").manual_seed(hash(seed) % (1 << 31))


def blocked(v, rows):
    """[n, k] in blocks of rows x 128, filled up with zeros: [nb, rows, kb, 128]."""
    n, k = v.shape
    v = torch.nn.functional.pad(v, (0, -k % 128, 0, -n % rows))
    return v.view(-1, rows, v.shape[1] // 128, 128)


def expected(x, rows):
    """(values, scales [nb, kb]) from the definition, in FP64."""
    n, k = x.shape
    b = blocked(x.double(), rows)
    s = (b.abs().amax((1, 3)) / 448).float().clamp(min=2.0 ** -126)
    z = b / s.double()[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(z.abs())).clamp(min=-6) - 3)
    q = torch.where(z == 0, z, torch.round(z / step) * step)
    return q.reshape(-1, q.shape[2] * 128)[:n, :k], s


def inputs(g, m, k, dtype, kind):
    x = torch.randn((m, k), generator=g, device="cuda")
    if kind == "wide":
        x = x * torch.exp2(12 * torch.rand((m, k), generator=g, device="cuda") - 6)
    elif kind == "ties":  # few bits: quotients on and next to the middle of two steps
        x = torch.randint(-64, 65, (m, k), generator=g, device="cuda") / 8.0
        x[:, ::128] = 7.0 * 2.0 ** torch.randint(0, 4, (m, 1), generator=g, device="cuda")
    elif kind == "zeros":
        x[:, : k // 2] = 0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "zeros"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 7), (17, 136), (33, 515), (5, 2048), (130, 4096),
                                 (16, 1000)])
def test_rows_bit_for_bit(m, k, dtype, kind):
    x = inputs(gen(m, k), m, k, dtype, kind)
    q, s = mx.dynamic_fp8_block_quant(x)
    assert q.dtype == F8 and q.shape == x.shape and s.shape == (m, -(-k // 128))
    want, scales = expected(x, 1)
    assert torch.equal(s, scales)
    assert torch.equal(q.double(), want)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("kind", ["normal", "ties", "zeros"])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 136), (300, 515), (256, 2048)])
def test_blocks_bit_for_bit(n, k, dtype, kind):
    x = inputs(gen(n, k), n, k, dtype, kind)
    want, scales = expected(x, 128)
    q, s = mx.dynamic_fp8_block_quant(x, block_rows=128)
    assert torch.equal(s, scales) and torch.equal(q.double(), want)
    both = torch.stack([x, x * 2])  # experts: blocks begin anew
    q, s = mx.dynamic_fp8_block_quant(both, block_rows=128)
    least = scales == 2.0 ** -126  # of zeros
    assert torch.equal(s, torch.stack([scales, torch.where(least, scales, scales * 2)]))
    assert torch.equal(q.double(), torch.stack([want, want]))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,k", [(1, 1), (2, 128), (17, 136), (33, 515), (200, 768), (9, 2048)])
def test_silu_mul(m, k, dtype):
    g = gen(m, k)
    x = torch.randn((m, 2 * k), generator=g, device="cuda") * 4
    x[:, 0], x[0, k] = -90.0, 0.0
    x = x.to(dtype)
    q, s = mx.silu_mul_fp8_block_quant(x)
    gate, up = x.double().split(k, 1)
    h = gate * torch.sigmoid(gate) * up
    # exp2 of a product rounded once: |g| / ln 2 * 2^-24 * ln 2; exp2, 1 + e, the reciprocal
    # (an ulp each) and two products
    off = h.abs() * (gate.abs() + 8) * 2.0 ** -23 + 1e-37
    amax = blocked(h, 1).abs().amax((1, 3))
    worst = blocked(off, 1).amax((1, 3))
    lo, hi = (amax - worst) / 448 * (1 - 2.0 ** -23), (amax + worst) / 448 * (1 + 2.0 ** -23)
    assert ((s.double() >= lo) & (s.double() <= hi.clamp(min=2.0 ** -126))).all()
    unit = s.double().repeat_interleave(128, 1)[:, :k]
    step = torch.maximum(h.abs() * 2.0 ** -4, unit * 2.0 ** -10)  # half a step of e4m3
    # the last value may lie a rounding above 448 s
    assert ((q.double() * unit - h).abs() <= (step + off) * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("k", [512, 515])
def test_silu_mul_far_below_zero(k, dtype):
    # blocks of these only, so that their scale is no other value's: 1 / (1 + exp(-g)) lies
    # below the normal numbers from -87.3 on
    g = gen(k)
    gate = torch.empty((12, k), device="cuda").uniform_(-100, -80, generator=g).to(dtype)
    up = (torch.randn((12, k), generator=g, device="cuda") * 2.0 ** (12 if dtype is FP16 else 100))
    x = torch.cat([gate, up.to(dtype)], 1)
    q, s = mx.silu_mul_fp8_block_quant(x)
    gate, up = x.double().split(k, 1)
    h = gate * torch.sigmoid(gate) * up
    off = h.abs() * (gate.abs() + 8) * 2.0 ** -23 + 2.0 ** -148  # as above
    amax, worst = blocked(h, 1).abs().amax((1, 3)), blocked(off, 1).amax((1, 3))
    assert (amax / 448 > 2.0 ** -126).all()
    assert ((s.double() * 448 - amax).abs() <= worst + amax * 2.0 ** -23).all()
    unit = s.double().repeat_interleave(128, 1)[:, :k]
    step = torch.maximum(h.abs() * 2.0 ** -4, unit * 2.0 ** -10)  # half a step of e4m3
    assert ((q.double() * unit - h).abs() <= (step + off) * (1 + 2.0 ** -20)).all()


def test_values_that_are_not_finite_mark_their_block():
    x = torch.randn((20, 520), generator=gen(1), device="cuda")
    clean_q, clean_s = mx.dynamic_fp8_block_quant(x)
    x[3, 130], x[7, 519], x[8, 0], x[8, 1] = math.inf, math.nan, -math.inf, math.nan
    q, s = mx.dynamic_fp8_block_quant(x)
    bad = torch.zeros((20, 5), dtype=torch.bool, device="cuda")
    bad[3, 1] = bad[7, 4] = bad[8, 0] = True
    assert torch.equal(s.isnan(), bad) and torch.equal(s[~bad], clean_s[~bad])
    wide = bad.repeat_interleave(128, 1)[:, :520]
    assert (q.float()[wide] == 0).all()
    assert torch.equal(q.float()[~wide], clean_q.float()[~wide])
    q, s = mx.dynamic_fp8_block_quant(x, block_rows=128)
    assert s.isnan().tolist() == [[True, True, False, False, True]]
    assert (q.float()[:, :256] == 0).all() and (q.float()[:, 512:] == 0).all()
    y = torch.cat([x[:, :256], torch.ones((20, 256), device="cuda")], 1)
    assert mx.silu_mul_fp8_block_quant(y)[1].isnan().nonzero().tolist() == [[3, 1], [8, 0]]


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_the_ends_of_the_range(dtype):
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).tiny
    x = torch.zeros((4, 256), dtype=dtype, device="cuda")
    x[0, :3] = torch.tensor([big, -big, big / 2], dtype=dtype)
    x[1, 0], x[1, 200] = tiny, -tiny / 2
    x[2, 0] = 1.0
    q, s = mx.dynamic_fp8_block_quant(x)
    want, scales = expected(x, 1)
    assert torch.equal(s, scales) and torch.equal(q.double(), want)
    assert (s[3] == 2.0 ** -126).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("k", [512, 515])
def test_borders_among_the_smallest_numbers(k, dtype):
    # values on and next to the middles of two steps, of scales down to the smallest: the
    # quotient's remainder may lie below every FP32 number
    g = torch.Generator().manual_seed(k)
    rows = 37
    mid = 8.5 + torch.randint(0, 8, (rows * 64, k), generator=g).double()
    mid *= torch.exp2(4 - torch.randint(0, 15, mid.shape, generator=g).double())
    scale = torch.exp2(-126 + torch.arange(rows).repeat_interleave(64).double())
    scale *= 1 + torch.rand(rows * 64, generator=g).double()
    x = (mid * scale[:, None]).float()
    if dtype is FP32:
        x = (x.view(torch.int32) + torch.randint(-1, 2, x.shape, generator=g).int()).view(FP32)
    x[:, ::128] = (448 * scale[:, None]).float()
    x = x.to(dtype)
    want, scales = expected(x, 1)
    q, s = mx.dynamic_fp8_block_quant(cuda(x))
    assert torch.equal(s.cpu(), scales) and torch.equal(q.double().cpu(), want)
    want, scales = expected(x[:128], 128)
    q, s = mx.dynamic_fp8_block_quant(cuda(x[:128]), block_rows=128)
    assert torch.equal(s.cpu(), scales) and torch.equal(q.double().cpu(), want)


def test_layouts():
    g = gen(2)
    x = torch.randn((6, 8, 264), generator=g, device="cuda").to(BF16)
    q, s = mx.dynamic_fp8_block_quant(x)
    assert s.shape == (6, 8, 3) and s.view(48, 3).stride() == (1, 48)
    one = [mx.dynamic_fp8_block_quant(t) for t in x.view(48, 264)]
    assert torch.equal(torch.stack([t[0].float() for t in one]).view_as(x), q.float())
    assert torch.equal(torch.stack([t[1] for t in one]).view_as(s), s)
    wide = torch.full((48, 300), 9.0, dtype=BF16, device="cuda")
    for off in (0, 1, 8, 36):
        wide[:, off:off + 264] = x.view(48, 264)
        qw, sw = mx.dynamic_fp8_block_quant(wide[:, off:off + 264])
        assert torch.equal(qw.float(), q.view(48, 264).float()) and torch.equal(sw, s.view(48, 3))
    t = x.view(48, 264).t().contiguous().t()
    assert torch.equal(mx.dynamic_fp8_block_quant(t)[0].float(), q.view(48, 264).float())
    assert torch.equal(mx.silu_mul_fp8_block_quant(t[:, :256])[1],
                       mx.silu_mul_fp8_block_quant(x.view(48, 264)[:, :256].contiguous())[1])
    wq, ws = mx.dynamic_fp8_block_quant(x, block_rows=128)
    tq, ts = mx.dynamic_fp8_block_quant(x.transpose(1, 2).contiguous().transpose(1, 2),
                                        block_rows=128)
    assert torch.equal(wq.float(), tq.float()) and torch.equal(ws, ts)
    q, s = mx.dynamic_fp8_block_quant(x[:0])
    assert q.shape == (0, 8, 264) and s.shape == (0, 8, 3)
    assert mx.dynamic_fp8_block_quant(x[:, :0], block_rows=128)[1].shape == (6, 0, 3)
    assert mx.silu_mul_fp8_block_quant(x[:, :0])[0].shape == (6, 0, 132)


@pytest.mark.parametrize("k", [264, 261])
def test_writes_its_outputs_only(k):
    rows, kb = 37, 3
    x = torch.randn((rows, k), generator=gen(k), device="cuda").to(FP16)
    q, s = mx.dynamic_fp8_block_quant(x)
    for by_row in (True, False):
        for before in (64, 61):
            qb = torch.full((before + rows * k + 64,), 7, dtype=torch.uint8, device="cuda")
            sb = torch.full((rows * kb + 32,), -1.0, device="cuda")
            _lib.check(_lib.load().mxfp4_quant_fp8_rows(
                _lib.ptr(x), _lib.DT_F16, rows, k, k, 0,
                ctypes.c_void_p(qb.data_ptr() + before), ctypes.c_void_p(sb.data_ptr() + 64),
                kb if by_row else 1, 1 if by_row else rows, _lib.stream_of(x.device)))
            assert (qb[:before] == 7).all() and (qb[before + rows * k:] == 7).all()
            assert torch.equal(qb[before:before + rows * k].view(rows, k), q.view(torch.uint8))
            assert (sb[:16] == -1).all() and (sb[16 + rows * kb:] == -1).all()
            got = sb[16:16 + rows * kb]
            assert torch.equal(got.view(rows, kb) if by_row else got.view(kb, rows).t(), s)


def test_offsets_beyond_31_bits():
    m, k = 600000, 4096
    x = torch.zeros((m, k), dtype=BF16, device="cuda")
    x[-3:] = torch.randn((3, k), generator=gen(3), device="cuda").to(BF16)
    q, s = mx.dynamic_fp8_block_quant(x)
    want, scales = expected(x[-3:], 1)
    assert torch.equal(q[-3:].double(), want) and torch.equal(s[-3:], scales)
    assert (s[:-3] == 2.0 ** -126).all()
