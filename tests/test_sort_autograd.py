"""The autograd side of the token moves' general path, on the CPU: the kernel calls are
replaced by plain torch, so that what is recorded, kept and refused around them shows."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import mxfp4_amd as mx
from mxfp4_amd import _lib, sort

M, TOP_K, E, H = 5, 2, 3, 4


@pytest.fixture
def order(monkeypatch):
    """Every second slot dropped in token 0; the kernel calls in plain torch."""
    def take(y, position):
        return torch.where((position >= 0)[..., None], y[position.clamp(min=0).long()], 0)

    def _sort(x, offsets, position):
        rows = x.new_zeros((position.numel(), x.shape[1]))
        at = position >= 0
        rows[position[at].long()] = x[:, None].expand(-1, position.shape[1], -1)[at]
        return rows

    def _combine(y, position, weights):
        picked = take(y, position)
        return (picked if weights is None else picked * weights[..., None]).sum(1).to(y.dtype)

    def _combine_grad(g, y, weights, offsets, position, want_dy, want_dw):
        w = torch.ones(position.shape) if weights is None else weights
        dy = dw = None
        if want_dy:
            dy = g.new_zeros((position.numel(), g.shape[1]))
            at = position >= 0
            dy[position[at].long()] = (w[..., None] * g[:, None])[at].to(g.dtype)
        if want_dw:
            dw = (take(y, position).float() * g[:, None].float()).sum(-1)
        return dy, dw

    monkeypatch.setattr(_lib, "host", lambda: None)
    for f in (_sort, _combine, _combine_grad):
        monkeypatch.setattr(sort, f.__name__, f)
    ids = torch.tensor([[0, -1], [1, 2], [2, 0], [0, 0], [1, 1]])
    routes = torch.argsort(torch.where(ids.reshape(-1) < 0, E, ids.reshape(-1)), stable=True)
    position = torch.empty(M * TOP_K, dtype=torch.int32)
    position[routes] = torch.arange(M * TOP_K, dtype=torch.int32)
    position[1], routes[-1] = -1, -1
    offsets = torch.tensor([0, 4, 7, 9], dtype=torch.int32)
    return mx.ExpertOrder(offsets, routes.int(), position.view(M, TOP_K))


def leaves(w_dtype=torch.float32):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((M, H), generator=g, requires_grad=True)
    y = torch.randn((M * TOP_K, H), generator=g, requires_grad=True)
    w = torch.rand((M, TOP_K), generator=g).to(w_dtype).requires_grad_()
    return x, y, w


def test_first_derivatives(order):
    x, y, w = leaves()
    dx, = torch.autograd.grad(mx.sort_tokens(x, order).sum(), x)
    assert torch.equal(dx, (order.position >= 0).sum(1, keepdim=True).expand(M, H).float())
    dy, dw = torch.autograd.grad(mx.combine_tokens(y, order, w).sum(), (y, w))
    assert torch.equal(dy[order.position[2].long()], w.detach()[2, :, None].expand(2, H))
    assert dw[0, 1] == 0 and not (dx.requires_grad or dy.requires_grad or dw.requires_grad)


@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16])
def test_second_derivatives_are_refused_whatever_the_loss(order, w_dtype):
    # the incoming gradient of a linear loss is a constant, dw = <g, y> is none
    x, y, w = leaves(w_dtype)
    out = mx.combine_tokens(y, order, w)
    dy, dw = torch.autograd.grad(out.sum(), (y, w), create_graph=True)
    for again in (dw.square().sum() + (y ** 2).sum(), dy.square().sum() + (w ** 2).sum()):
        with pytest.raises(RuntimeError, match="differentiable once"):
            again.backward(retain_graph=True)
    dx, = torch.autograd.grad(mx.sort_tokens(x, order).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (dx.square().sum() + (x ** 2).sum()).backward()


def test_forward_mode_is_refused(order):
    x, y, w = (t.detach() for t in leaves())
    w16 = w.bfloat16()
    with fwAD.dual_level():
        rows, out = mx.sort_tokens(x, order), mx.combine_tokens(y, order, w)  # no tangent: as ever
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for grad in (torch.enable_grad, torch.no_grad):
            for call in (lambda: mx.sort_tokens(dual(x), order),
                         lambda: mx.sort_tokens(dual(x.clone().requires_grad_()), order),
                         lambda: mx.combine_tokens(dual(y), order, w),
                         lambda: mx.combine_tokens(dual(y), order),
                         lambda: mx.combine_tokens(y, order, dual(w)),
                         lambda: mx.combine_tokens(y, order, dual(w16))):
                with grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        xd, yd, wd = dual(x), dual(y), dual(w)
        with torch.inference_mode():  # records no tangent of anything
            assert torch.equal(mx.sort_tokens(xd, order), rows)
            assert torch.equal(mx.combine_tokens(yd, order, wd), out)


def gradients(order):
    x, y, w = leaves()
    g = torch.Generator().manual_seed(4)
    up = torch.randn((M, H), generator=g), torch.randn((M * TOP_K, H), generator=g)
    return torch.autograd.grad((mx.combine_tokens(y, order, w), mx.sort_tokens(x, order)),
                               (x, y, w), up)


def turned(t):
    return t.t().contiguous().t() if t.ndim == 2 else t


def test_saved_tensors_may_come_back_in_another_layout(order, monkeypatch):
    want = gradients(order)
    seen = []
    for name in ("_combine", "_combine_grad"):  # which take y and the weights of any strides
        def call(*a, f=getattr(sort, name)):
            seen.extend(t for t in a if isinstance(t, torch.Tensor) and t.dtype == torch.int32)
            return f(*a)
        monkeypatch.setattr(sort, name, call)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), turned):
        got = gradients(order)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert len(seen) == 4 and all(t.is_contiguous() for t in seen)


@pytest.mark.parametrize("bad", [lambda t: t.to(torch.float16), lambda t: t[:1],
                                 lambda t: t.to("meta"), lambda t: t.to_sparse()],
                         ids=["type", "shape", "device", "layout"])
def test_saved_tensors_that_come_back_as_others_are_refused(order, bad):
    # each of offsets, position, y and the weights by itself, and all
    for which in (0, 1, 2, 3, None):
        x, y, w = leaves()
        count = iter(range(100))
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: (t, next(count)),
                lambda p: bad(p[0]) if which is None or p[1] == which else p[0]):
            out = mx.combine_tokens(y, order, w)
        with pytest.raises(RuntimeError, match="hooks gave back"):
            out.sum().backward()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
            rows = mx.sort_tokens(x, order)
        with pytest.raises(RuntimeError, match="hooks gave back"):
            rows.sum().backward()
