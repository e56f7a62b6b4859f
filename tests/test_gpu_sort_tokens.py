"""GPU: tokens sorted by expert and back.  The order and the moves are exact; sums are
FP32: top_k products and additions of 2^-24 each, then half a step of the type."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import mxfp4_amd as mx
from mxfp4_amd import _lib

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -149}
FLOATS = [BF16, FP16, FP32]


def gen(*seed):
    return torch.Generator(device="cuda").manual_seed(hash(seed) % (1 << 31))


def make_ids(g, m, top_k, experts, kind="drop", dtype=torch.int64):
    ids = torch.randint(0, experts, (m, top_k), generator=g, device="cuda")
    if kind == "drop":
        out = torch.randint(0, 4, (m, top_k), generator=g, device="cuda")
        ids = torch.where(out == 0, -1, torch.where(out == 1, experts, ids))
    elif kind == "one":
        ids[:] = experts // 2
    elif kind == "none":
        ids[:] = -1
    elif kind == "skewed":
        ids = torch.where(torch.rand((m, top_k), generator=g, device="cuda") < 0.9, 0, ids)
    return ids.to(dtype)


def expected_order(ids, experts):
    """(offsets, routes, position) by a host sort."""
    flat = ids.reshape(-1).tolist()
    lists = [[] for _ in range(experts)]
    for r, e in enumerate(flat):
        if 0 <= e < experts:
            lists[e].append(r)
    offsets, routes = [0], []
    for v in lists:
        routes += v
        offsets.append(len(routes))
    position = [-1] * len(flat)
    for p, r in enumerate(routes):
        position[r] = p
    return offsets, routes + [-1] * (len(flat) - len(routes)), position


@pytest.mark.parametrize("kind", ["spread", "drop", "one", "none", "skewed"])
@pytest.mark.parametrize("m,top_k,experts", [
    (1, 1, 1), (1, 8, 128), (5, 3, 2), (64, 8, 128), (65, 8, 7), (171, 6, 1024), (500, 4, 60),
    (2048, 8, 256), (2049, 8, 128), (4096, 8, 128), (16384, 8, 64), (16400, 8, 1024),
    (50000, 3, 1000)])
def test_order(m, top_k, experts, kind):
    g = gen(m, top_k, experts)
    ids = make_ids(g, m, top_k, experts, kind, (torch.int64, torch.int32)[m % 2])
    order = mx.sort_routes(ids, experts)
    offsets, routes, position = expected_order(ids, experts)
    assert order.offsets.tolist() == offsets
    assert order.routes.tolist() == routes
    assert order.position.shape == (m, top_k) and order.position.reshape(-1).tolist() == position


@pytest.mark.parametrize("m,top_k", [(16384, 64), (16400, 64), (70000, 33)])
@pytest.mark.parametrize("experts", [1, 60, 1024])
def test_order_of_a_million_routes(m, top_k, experts):
    # 2^20 routes are the most whose workgroups sum all counts themselves
    ids = torch.randint(-1, experts + 1, (m, top_k), generator=gen(m, experts), device="cuda")
    order = mx.sort_routes(ids, experts)
    flat = ids.reshape(-1)
    bucket = torch.where((flat >= 0) & (flat < experts), flat, experts)
    counts = torch.bincount(bucket, minlength=experts + 1)
    live = int(counts[:experts].sum())
    assert order.offsets[0] == 0 and torch.equal(order.offsets[1:].long(),
                                                 counts[:experts].cumsum(0))
    routes = torch.sort(bucket, stable=True).indices
    assert torch.equal(order.routes[:live].long(), routes[:live])
    assert (order.routes[live:] == -1).all()
    position = torch.full_like(flat, -1)
    position[routes[:live]] = torch.arange(live, device="cuda")
    assert torch.equal(order.position.reshape(-1).long(), position)


def test_order_of_other_types_and_layouts():
    ids = make_ids(gen(1), 300, 4, 16)
    want = mx.sort_routes(ids, 16)
    for other in (ids.to(torch.int16), ids.t().contiguous().t(), torch.cat([ids, ids], 1)[:, 4:],
                  ids.to(torch.int8)):
        for a, b in zip(mx.sort_routes(other, 16), want):
            assert torch.equal(a, b)
    # ids far outside the experts
    far = torch.tensor([[1 << 40, 3], [-(1 << 40), 1 << 32]], device="cuda")
    order = mx.sort_routes(far, 4)
    assert order.offsets.tolist() == [0, 0, 0, 0, 1] and order.routes.tolist() == [1, -1, -1, -1]
    order = mx.sort_routes(ids[:0], 16)
    assert order.offsets.tolist() == [0] * 17 and order.position.shape == (0, 4)


def picked(y, order):
    """y's rows by slot, zeros for a dropped one, in FP64."""
    p = order.position.long()
    return torch.where((p >= 0)[..., None], y.double()[p.clamp(min=0)], 0.0)


def agree(got, terms, extra=0.0):
    """got = terms summed over dim 1, in FP32."""
    want = terms.sum(1)
    n = terms.shape[1]
    # a product and an addition a term; the rounding is of the computed value
    off = (2 * n + extra) * 2.0 ** -24 * terms.abs().sum(1)
    tol = off * 1.01 + HALF[got.dtype] * (want.abs() + off) + TINY[got.dtype]
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", ["spread", "drop", "one", "none"])
@pytest.mark.parametrize("m,top_k,h", [(1, 1, 1), (1, 8, 2048), (7, 3, 129), (60, 64, 40),
                                       (300, 9, 1407), (1000, 8, 512), (33, 2, 4104), (9, 4, 70001)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_there_and_back(m, top_k, h, dtype, kind):
    g = gen(m, top_k, h)
    experts = 12
    order = mx.sort_routes(make_ids(g, m, top_k, experts, kind), experts)
    live = int(order.offsets[-1])
    x = torch.randn((m, h), generator=g, device="cuda").to(dtype)
    rows = mx.sort_tokens(x, order)
    assert rows.shape == (m * top_k, h) and rows.dtype == dtype
    assert torch.equal(rows[:live], x[order.routes[:live].long() // top_k])
    assert (rows[live:] == 0).all()
    y = torch.randn((m * top_k, h), generator=g, device="cuda").to(dtype)
    w = torch.rand((m, top_k), generator=g, device="cuda")
    agree(mx.combine_tokens(y, order, w), picked(y, order) * w.double()[..., None])
    agree(mx.combine_tokens(y, order), picked(y, order))


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.int8, torch.uint8,
                                   torch.int32, torch.int64])
@pytest.mark.parametrize("h", [1, 3, 64, 130])
def test_rows_of_any_type_are_moved(h, dtype):
    g = gen(h)
    order = mx.sort_routes(make_ids(g, 50, 3, 8), 8)
    live = int(order.offsets[-1])
    x = torch.randint(0, 120, (50, h), generator=g, device="cuda", dtype=torch.uint8)
    x = x.view(dtype) if dtype.itemsize == 1 else x.to(dtype)
    rows = mx.sort_tokens(x, order)
    bits = torch.uint8 if dtype.itemsize == 1 else dtype
    assert rows.dtype == dtype
    assert torch.equal(rows[:live].view(bits), x.view(bits)[order.routes[:live].long() // 3])
    assert (rows[live:].view(bits) == 0).all()


def test_strides_and_alignment():
    g = gen(4)
    m, top_k, h = 90, 4, 128
    order = mx.sort_routes(make_ids(g, m, top_k, 10), 10)
    x = torch.randn((m, h), generator=g, device="cuda").to(BF16)
    y = torch.randn((m * top_k, h), generator=g, device="cuda").to(BF16)
    w = torch.rand((m, top_k), generator=g, device="cuda")
    rows, out = mx.sort_tokens(x, order), mx.combine_tokens(y, order, w)
    for off in (0, 1, 2, 8):
        xb = torch.zeros((m, h + 24), dtype=BF16, device="cuda")
        yb = torch.zeros((m * top_k, h + 24), dtype=BF16, device="cuda")
        xb[:, off:off + h], yb[:, off:off + h] = x, y
        assert torch.equal(mx.sort_tokens(xb[:, off:off + h], order), rows)
        assert torch.equal(mx.combine_tokens(yb[:, off:off + h], order, w), out)
    assert torch.equal(mx.sort_tokens(x.t().contiguous().t(), order), rows)
    assert torch.equal(mx.combine_tokens(y.t().contiguous().t(), order, w.t().contiguous().t()), out)
    assert torch.equal(mx.sort_tokens(x[:1].expand(m, h), order),
                       mx.sort_tokens(x[:1].repeat(m, 1), order))
    spread = mx.ExpertOrder(order.offsets, torch.stack([order.routes] * 2, 1)[:, 0],
                            order.position.t().contiguous().t())
    assert torch.equal(mx.combine_tokens(y, spread, w), out)
    assert torch.equal(mx.combine_tokens(y, order, w.double()), out)
    assert mx.sort_tokens(x[:, :0], order).shape == (m * top_k, 0)
    assert mx.combine_tokens(y[:, :0], order, w).shape == (m, 0)
    none = mx.sort_routes(torch.zeros((0, 4), dtype=torch.int64, device="cuda"), 10)
    assert mx.sort_tokens(x[:0], none).shape == (0, h)
    assert mx.combine_tokens(y[:0], none, w[:0]).shape == (0, h)


def test_dropped_rows_do_not_enter_the_sums():
    # what lies behind the last expert's rows is not read, whatever it holds
    g = gen(6)
    order = mx.sort_routes(make_ids(g, 40, 4, 8), 8)
    live = int(order.offsets[-1])
    y = torch.randn((160, 64), generator=g, device="cuda")
    w = torch.rand((40, 4), generator=g, device="cuda")
    want = mx.combine_tokens(y, order, w)
    bad_y, bad_w = y.clone(), w.clone()
    bad_y[live:] = float("nan")
    bad_w[order.position < 0] = float("inf")
    assert torch.equal(mx.combine_tokens(bad_y, order, bad_w), want)
    # and what is not finite stays in its token
    bad_y[order.position[7].max().long()] = float("inf")
    got = mx.combine_tokens(bad_y, order, w)
    assert not got[7].isfinite().any()
    rest = torch.arange(40, device="cuda") != 7
    assert torch.equal(got[rest], want[rest])


# -------------------------------------------------------------- gradients

@pytest.mark.parametrize("kind", ["spread", "drop", "none"])
@pytest.mark.parametrize("m,top_k,h", [(1, 1, 1), (1, 8, 2048), (7, 3, 129), (60, 20, 40),
                                       (300, 9, 1407), (500, 8, 4104)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_gradients(m, top_k, h, dtype, kind):
    g = gen(m, top_k, h)
    order = mx.sort_routes(make_ids(g, m, top_k, 12, kind), 12)
    live = int(order.offsets[-1])
    x = torch.randn((m, h), generator=g, device="cuda").to(dtype).requires_grad_()
    y = torch.randn((m * top_k, h), generator=g, device="cuda").to(dtype).requires_grad_()
    w = torch.rand((m, top_k), generator=g, device="cuda").requires_grad_()
    g_rows = torch.randn((m * top_k, h), generator=g, device="cuda").to(dtype)
    g_out = torch.randn((m, h), generator=g, device="cuda").to(dtype)
    rows, out = mx.sort_tokens(x, order), mx.combine_tokens(y, order, w)
    dx, dy, dw = torch.autograd.grad((rows, out), (x, y, w), (g_rows, g_out))
    assert dx.dtype == dy.dtype == dtype and dw.dtype == FP32
    with torch.no_grad():
        agree(dx, picked(g_rows, order))
        routes = order.routes[:live].long()
        want = torch.zeros((m * top_k, h), dtype=torch.float64, device="cuda")
        want[:live] = w.double().reshape(-1)[routes][:, None] * g_out.double()[routes // top_k]
        # one product, one rounding
        tol = (HALF[dtype] * (1 + 2.0 ** -24) + 2.0 ** -24) * want.abs() + TINY[dtype]
        assert ((dy.double() - want).abs() <= tol).all()
        terms = picked(y, order) * g_out.double()[:, None]
        # a thread adds ceil(h / 256) or more units in order, then 6 + 2 steps of a tree
        off = (h / 256 + 8 + 8) * 2.0 ** -24 * terms.abs().sum(-1)
        assert ((dw.double() - terms.sum(-1)).abs() <= off * 1.01 + 1e-38).all()
        assert (dw[order.position < 0] == 0).all() and (dy[live:] == 0).all()


def test_gradients_against_differences():
    # both moves are linear in every input: the difference quotient is exact but for FP32
    g = gen(8)
    m, top_k, h = 30, 4, 50
    order = mx.sort_routes(make_ids(g, m, top_k, 6), 6)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, w, c = rnd(m, h).requires_grad_(), rnd(m, top_k).requires_grad_(), rnd(m, h)
    scale = rnd(m * top_k, 1)

    def loss(x, w):
        rows = mx.sort_tokens(x, order) * scale  # in the experts' place
        return (mx.combine_tokens(rows, order, w).double() * c.double()).sum()

    dx, dw = torch.autograd.grad(loss(x, w), (x, w))
    with torch.no_grad():
        for v, d, at in ((rnd(m, h), dx, 0), (rnd(m, top_k), dw, 1)):
            plus = loss(x + v, w) if at == 0 else loss(x, w + v)
            minus = loss(x - v, w) if at == 0 else loss(x, w - v)
            size = (c.abs().double().sum() * 100) * 2.0 ** -24 * 100
            assert abs((plus - minus) / 2 - (d.double() * v.double()).sum()) <= size


def test_gradient_of_one_input_only_and_of_other_layouts():
    g = gen(9)
    order = mx.sort_routes(make_ids(g, 40, 4, 8), 8)
    y = torch.randn((160, 96), generator=g, device="cuda")
    w = torch.rand((40, 4), generator=g, device="cuda")
    up = torch.randn((40, 96), generator=g, device="cuda")

    def grads(y, w, up=up):
        leaves = [t for t in (y, w) if t is not None and t.requires_grad]
        return torch.autograd.grad(mx.combine_tokens(y, order, w), leaves, up)

    dy, dw = grads(y.clone().requires_grad_(), w.clone().requires_grad_())
    assert torch.equal(grads(y.clone().requires_grad_(), w)[0], dy)
    assert torch.equal(grads(y, w.clone().requires_grad_())[0], dw)
    ones = torch.ones_like(w)
    assert torch.equal(grads(y.clone().requires_grad_(), None)[0],
                       grads(y.clone().requires_grad_(), ones)[0])
    half = w.to(FP16).requires_grad_()
    assert grads(y, half)[0].dtype == FP16
    wide = torch.zeros((40, 100), device="cuda")
    wide[:, 2:98] = up
    for other in (wide[:, 2:98], up.t().contiguous().t()):
        got = grads(y.clone().requires_grad_(), w.clone().requires_grad_(), other)
        assert torch.equal(got[0], dy)
        # rows off 16 bytes are added in another order: both are within 17 roundings of it
        terms = (picked(y, order) * up.double()[:, None]).abs().sum(-1)
        assert ((got[1] - dw).abs() <= 2 * 17 * 2.0 ** -24 * terms).all()
    # an expanded gradient, as a sum's is
    x = torch.randn((40, 96), generator=g, device="cuda").requires_grad_()
    mx.sort_tokens(x, order).sum().backward()
    assert torch.equal(x.grad, (order.position >= 0).sum(1, keepdim=True).expand(40, 96).float())
    with torch.no_grad():
        assert not mx.sort_tokens(x, order).requires_grad
    with pytest.raises(RuntimeError):  # no second derivative
        v = w.clone().requires_grad_()
        d, = torch.autograd.grad(mx.combine_tokens(y, order, v).square().sum(), v,
                                 create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("w_dtype", [FP32, BF16])
def test_second_derivatives_of_a_linear_loss_are_refused(native, w_dtype, monkeypatch):
    # dw = <g, y> and dy = w * g, also where the loss' own gradient g is a constant
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: None)
    g = gen(12)
    order = mx.sort_routes(make_ids(g, 40, 4, 8), 8)
    x = torch.randn((40, 96), generator=g, device="cuda").requires_grad_()
    y = torch.randn((160, 96), generator=g, device="cuda").requires_grad_()
    w = torch.rand((40, 4), generator=g, device="cuda").to(w_dtype).requires_grad_()
    dy, dw = torch.autograd.grad(mx.combine_tokens(y, order, w).sum(), (y, w), create_graph=True)
    dx, = torch.autograd.grad(mx.sort_tokens(x, order).sum(), x, create_graph=True)
    for d, leaf in ((dw, y), (dy, w), (dx, x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            (d.square().sum() + leaf.square().sum()).backward(retain_graph=True)


@pytest.mark.parametrize("native", [True, False])
def test_hooks_on_saved_tensors(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: None)
    g = gen(14)
    order = mx.sort_routes(make_ids(g, 40, 4, 8), 8)
    x = torch.randn((40, 96), generator=g, device="cuda").requires_grad_()
    y = torch.randn((160, 96), generator=g, device="cuda").requires_grad_()
    w = torch.rand((40, 4), generator=g, device="cuda").requires_grad_()
    up = torch.randn((40, 96), generator=g, device="cuda")
    g_rows = torch.randn((160, 96), generator=g, device="cuda")

    def grads(unpack=None, pack=lambda t: t.clone()):
        hooks = torch.autograd.graph.saved_tensors_hooks
        with hooks(pack, unpack) if unpack else contextlib.nullcontext():
            out, rows = mx.combine_tokens(y, order, w), mx.sort_tokens(x, order)
        return torch.autograd.grad((out, rows), (x, y, w), (up, g_rows))

    want = grads()
    turned = lambda t: t.t().contiguous().t() if t.ndim == 2 else t  # noqa: E731
    spread = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    for unpack, pack in ((lambda t: t, lambda t: t.clone()), (turned, lambda t: t),
                         (spread, lambda t: t), (lambda t: t.cuda(), lambda t: t.cpu())):
        assert all(torch.equal(a, b) for a, b in zip(grads(unpack, pack), want))
    with torch.autograd.graph.save_on_cpu():
        out = mx.combine_tokens(y, order, w)
    got = torch.autograd.grad(out, (y, w), up)
    assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[2])
    # what cannot be read as the saved ones: each of y, weights, offsets, position, and all
    for bad in (lambda t: t.to(FP16), lambda t: t[:-1], lambda t: t.cpu(), lambda t: t[None],
                lambda t: t.to_sparse()):
        for which in (0, 1, 2, 3, None):
            count = iter(range(100))
            with torch.autograd.graph.saved_tensors_hooks(
                    lambda t: (t, next(count)),
                    lambda p: bad(p[0]) if which is None or p[1] == which else p[0]):
                out = mx.combine_tokens(y, order, w)
            with pytest.raises(RuntimeError, match="hooks gave back"):
                torch.autograd.grad(out, (y, w), up)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
            rows = mx.sort_tokens(x, order)
        with pytest.raises(RuntimeError, match="hooks gave back"):
            torch.autograd.grad(rows, x, g_rows)


@pytest.mark.parametrize("native", [True, False])
def test_forward_mode_is_refused(native, monkeypatch):
    # a dual tensor need not require grad; its tangent would be lost
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: None)
    g = gen(13)
    order = mx.sort_routes(make_ids(g, 40, 4, 8), 8)
    x = torch.randn((40, 96), generator=g, device="cuda")
    y = torch.randn((160, 96), generator=g, device="cuda")
    w = torch.rand((40, 4), generator=g, device="cuda")
    rows, out = mx.sort_tokens(x, order), mx.combine_tokens(y, order, w)
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: mx.sort_tokens(dual(x), order),
                     lambda: mx.sort_tokens(dual(x.clone().requires_grad_()), order),
                     lambda: mx.combine_tokens(dual(y), order, w),
                     lambda: mx.combine_tokens(y, order, dual(w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(mx.sort_tokens(x, order), rows)
        assert torch.equal(mx.combine_tokens(y, order, w), out)


def test_the_same_bits_on_every_call():
    g = gen(10)
    order = mx.sort_routes(make_ids(g, 2000, 8, 64, "skewed"), 64)
    y = torch.randn((16000, 512), generator=g, device="cuda").to(BF16).requires_grad_()
    w = torch.rand((2000, 8), generator=g, device="cuda").requires_grad_()
    up = torch.randn((2000, 512), generator=g, device="cuda").to(BF16)
    first = None
    for _ in range(4):
        out = mx.combine_tokens(y, order, w)
        got = (out.detach(), *torch.autograd.grad(out, (y, w), up))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("h", [96, 97])
def test_writes_its_outputs_only(h):
    g = gen(h)
    m, top_k, experts = 37, 3, 5
    order = mx.sort_routes(make_ids(g, m, top_k, experts), experts)
    x = torch.randn((m, h), generator=g, device="cuda").to(BF16)
    y = torch.randn((m * top_k, h), generator=g, device="cuda").to(BF16)
    w = torch.rand((m, top_k), generator=g, device="cuda")
    lib, st = _lib.load(), _lib.stream_of(x.device)
    pos, off = _lib.ptr(order.position), _lib.ptr(order.offsets)
    rows, out = mx.sort_tokens(x, order), mx.combine_tokens(y, order, w)
    for before in (64, 61):
        def guarded(n, call, want):
            buf = torch.full((before + n + 64,), 3.0, dtype=BF16, device="cuda")
            _lib.check(call(ctypes.c_void_p(buf.data_ptr() + 2 * before)))
            assert (buf[:before] == 3).all() and (buf[before + n:] == 3).all()
            if want is not None:
                assert torch.equal(buf[before:before + n].view_as(want), want)

        guarded(rows.numel(), lambda p: lib.mxfp4_sort_tokens(
            _lib.ptr(x), _lib.DT_BF16, m, h, h, pos, off, experts, top_k, p, st), rows)
        guarded(out.numel(), lambda p: lib.mxfp4_combine_tokens(
            _lib.ptr(y), _lib.DT_BF16, m * top_k, h, h, pos, m, top_k, _lib.ptr(w), p, st), out)
        guarded(rows.numel(), lambda p: lib.mxfp4_combine_tokens_grad(
            _lib.ptr(x), _lib.DT_BF16, m, h, h, None, 0, pos, off, experts, top_k, None, p, None,
            st), rows)


def test_positions_that_lie():
    # device data: a place outside the rows counts as none
    pos = torch.tensor([[0, 99], [-7, 1]], dtype=torch.int32, device="cuda")
    off = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    order = mx.ExpertOrder(off, torch.zeros(4, dtype=torch.int32, device="cuda"), pos)
    y = torch.arange(8.0, device="cuda").view(4, 2)
    assert mx.combine_tokens(y, order).tolist() == [[0, 1], [2, 3]]
    assert mx.sort_tokens(y[:2], order).tolist() == [[0, 1], [2, 3], [0, 0], [0, 0]]


def test_offsets_beyond_31_bits():
    m, top_k, h = 140000, 2, 8192  # 2.3 G values, 4.6 GB
    g = gen(11)
    ids = make_ids(g, m, top_k, 16, "spread")
    order = mx.sort_routes(ids, 16)
    x = torch.zeros((m, h), dtype=BF16, device="cuda")
    x[:, 0] = (torch.arange(m, device="cuda") % 256).to(BF16)
    x[:, -1] = (torch.arange(m, device="cuda") // 1024).to(BF16)
    rows = mx.sort_tokens(x, order)
    token = order.routes.long() // top_k
    assert torch.equal(rows[:, 0], x[token, 0]) and torch.equal(rows[:, -1], x[token, -1])
    back = mx.combine_tokens(rows, order)
    assert torch.equal(back[:, 0].float(), (2 * x[:, 0].float()).to(BF16).float())
    assert torch.equal(back[:, -1].float(), (2 * x[:, -1].float()).to(BF16).float())
