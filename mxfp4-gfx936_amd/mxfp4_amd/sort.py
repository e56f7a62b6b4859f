# SPDX-License-Identifier: MIT
"""Tokens sorted by expert and back, with their weights and gradients, on MI355X.

``sort_routes`` orders the routes of ``topk_ids`` by expert, ``sort_tokens`` moves the
tokens' rows there, and ``combine_tokens`` sums what the experts gave back into tokens.
``make_routing`` is the padded order that the MXFP4 products read; this one has no
padding, and its moves are differentiable.  No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import functools
import operator
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODES = {**_lib._DTYPE_CODES, torch.int8: _lib.DT_I8}


class ExpertOrder(NamedTuple):
    """The routes r = t * top_k + s of ``topk_ids`` [M, top_k] by expert (all int32).

    * offsets [E + 1]: expert e has places offsets[e] .. offsets[e + 1];
    * routes [M * top_k]: the route at a place, each expert's in ascending order; -1
      from offsets[E] on (as many as were dropped);
    * position [M, top_k]: a route's place, -1 for one whose id is outside [0, E).
    """

    offsets: torch.Tensor
    routes: torch.Tensor
    position: torch.Tensor


def sort_routes(topk_ids: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The order of ``topk_ids`` [M, top_k] (int32 or int64; others are converted) by
    expert, on the device and without a host round trip: a stable sort.  Ids outside
    [0, num_experts) (another rank's experts, unused slots) are dropped.  At most 1024
    experts, top_k 64 and 2^30 - 1 routes."""
    host = _lib.host()
    out = host and host.sort_routes(topk_ids, num_experts)
    if out is not None:
        return ExpertOrder(*out)
    if topk_ids.is_floating_point() or topk_ids.is_complex() or topk_ids.dtype == torch.bool:
        raise TypeError(f"topk_ids must be integers, got {topk_ids.dtype}")
    if topk_ids.ndim != 2 or not 1 <= topk_ids.shape[1] <= 64:
        raise ValueError(f"topk_ids must be [M, top_k] with top_k of 1 to 64, got "
                         f"{tuple(topk_ids.shape)}")
    num_experts = operator.index(num_experts)
    if not 1 <= num_experts <= 1024 or topk_ids.numel() >= 1 << 30:
        raise ValueError(f"unsupported sizes: {num_experts} experts, {topk_ids.numel()} routes")
    device = _lib.require_device(topk_ids)
    lib = _lib.load()
    ids = topk_ids if topk_ids.dtype in (torch.int32, torch.int64) else topk_ids.to(torch.int64)
    ids = ids.contiguous()
    n = ids.numel()
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    routes = torch.empty(n, dtype=torch.int32, device=device)
    position = torch.empty(ids.shape, dtype=torch.int32, device=device)
    nbytes = ctypes.c_int64()
    _lib.check(lib.mxfp4_sort_routes_workspace_size(n, num_experts, ctypes.byref(nbytes)))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device) if nbytes.value else None
    with _lib.on_device(device):
        _lib.check(lib.mxfp4_sort_routes(
            _lib.ptr(ids), _lib.dtype_code(ids.dtype), n, num_experts, _lib.ptr(offsets),
            _lib.ptr(routes), _lib.ptr(position), _lib.ptr(ws), nbytes.value,
            _lib.stream_of(device)))
    return ExpertOrder(offsets, routes, position)


def check_order(order: ExpertOrder):
    """The order's tensors, contiguous; TypeError / ValueError unless they fit together."""
    offsets, routes, position = order
    for t, name in ((offsets, "offsets"), (routes, "routes"), (position, "position")):
        if t.dtype != torch.int32:
            raise TypeError(f"the order's {name} must be int32, got {t.dtype}")
    if (position.ndim != 2 or not 1 <= position.shape[1] <= 64 or offsets.ndim != 1
            or not 2 <= offsets.numel() <= 1025 or routes.shape != (position.numel(),)
            or position.numel() >= 1 << 30):
        raise ValueError(f"inconsistent order: offsets {tuple(offsets.shape)}, routes "
                         f"{tuple(routes.shape)}, position {tuple(position.shape)}")
    return offsets.contiguous(), routes.contiguous(), position.contiguous()


def _sort(x, offsets, position):
    device = _lib.require_device(x, offsets, position, recorders=True)
    lib = _lib.load()
    m, top_k = position.shape
    h = x.shape[1]
    rows = torch.empty((m * top_k, h), dtype=x.dtype, device=device)
    if rows.numel():
        x2, ldx = _lib.rows_of(x)
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_sort_tokens(
                _lib.ptr(x2), _CODES[x.dtype], m, h, ldx, _lib.ptr(position), _lib.ptr(offsets),
                offsets.numel() - 1, top_k, _lib.ptr(rows), _lib.stream_of(device)))
    return rows


def _combine(y, position, weights):
    device = _lib.require_device(y, position, weights, recorders=True)
    lib = _lib.load()
    m, top_k = position.shape
    out = torch.empty((m, y.shape[1]), dtype=y.dtype, device=device)
    if out.numel():
        y2, ldy = _lib.rows_of(y)
        w = None if weights is None else weights.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_combine_tokens(
                _lib.ptr(y2), _CODES[y.dtype], y2.shape[0], y2.shape[1], ldy, _lib.ptr(position),
                m, top_k, _lib.ptr(w), _lib.ptr(out), _lib.stream_of(device)))
    return out


def _combine_grad(g, y, weights, offsets, position, want_dy, want_dw):
    """(dy or None, dweights or None)"""
    device = _lib.require_device(g, y, weights, offsets, position, recorders=True)
    lib = _lib.load()
    m, top_k = position.shape
    h = g.shape[1]
    dy = torch.empty((m * top_k, h), dtype=g.dtype, device=device) if want_dy else None
    dw = torch.empty((m, top_k), dtype=torch.float32, device=device) if want_dw else None
    if m and h:
        g2, ldg = _lib.rows_of(g)
        y2, ldy = _lib.rows_of(y) if want_dw else (None, 0)
        w = None if weights is None else weights.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_combine_tokens_grad(
                _lib.ptr(g2), _CODES[g.dtype], m, h, ldg, _lib.ptr(y2), ldy, _lib.ptr(position),
                _lib.ptr(offsets), offsets.numel() - 1, top_k, _lib.ptr(w), _lib.ptr(dy),
                _lib.ptr(dw), _lib.stream_of(device)))
    elif want_dw:
        dw.zero_()
    return dy, dw


def _check_tangents(*inputs):
    """NotImplementedError for an input with a tangent (forward-mode differentiation), which
    the output would not have."""
    if torch.is_inference_mode_enabled():
        return
    for t in inputs:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the moves of tokens by expert have no forward-mode "
                                      "derivative")


def _check_capture(*leaves):
    """RuntimeError for a leaf whose backward pass a capture could not take."""
    host = _lib.host()
    if host and leaves[0].is_cuda and torch.cuda.is_current_stream_capturing():
        for t in leaves:
            if t is not None:
                host.leaf_in_capture(t)


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g):
        return g.view_as(g)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("the moves of tokens by expert are differentiable once")


def _differentiable_once(backward):
    """A backward pass whose gradients, where they are recorded, raise when they are
    differentiated: whether the incoming gradient is recorded does not matter, dy and dw
    are functions of the saved weights and rows too."""
    @functools.wraps(backward)
    def run(ctx, g):
        with torch.no_grad():
            grads = backward(ctx, g)
        if not torch.is_grad_enabled():
            return grads
        return tuple(None if d is None else _Once.apply(d.detach().requires_grad_())
                     for d in grads)

    return run


def _saved(t, name, like, dtype, shape):
    """``t``, which hooks on saved tensors may have replaced: RuntimeError unless it can be
    read as the ``name`` that was saved."""
    if (t.dtype != dtype or t.shape != shape or t.device != like.device
            or t.layout != torch.strided):
        raise RuntimeError(f"the {name} that saved-tensor hooks gave back are not {dtype} "
                           f"{tuple(shape)} on {like.device}: {t.dtype} {tuple(t.shape)} on "
                           f"{t.device}, {t.layout}")
    return t


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, position):
        ctx.save_for_backward(position)
        ctx.order = position.shape
        return _sort(x, offsets, position)

    @staticmethod
    @_differentiable_once
    def backward(ctx, g):
        position = _saved(*ctx.saved_tensors, "positions", g, torch.int32, ctx.order)
        return _combine(g, position.contiguous(), None), None, None


class _CombineTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, offsets, position):
        # y itself only where the weights' gradient reads it
        keep = weights is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(y if keep else None, weights, offsets, position)
        ctx.order = offsets.shape, position.shape
        return _combine(y, position, weights)

    @staticmethod
    @_differentiable_once
    def backward(ctx, g):
        y, weights, offsets, position = ctx.saved_tensors
        bounds, slots = ctx.order
        if y is not None:
            _saved(y, "rows", g, g.dtype, (slots.numel(), g.shape[1]))
        if weights is not None:
            _saved(weights, "weights", g, torch.float32, slots)
        offsets = _saved(offsets, "offsets", g, torch.int32, bounds).contiguous()
        position = _saved(position, "positions", g, torch.int32, slots).contiguous()
        grads = _combine_grad(g, y, weights, offsets, position, *ctx.needs_input_grad[:2])
        return *grads, None, None


def sort_tokens(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """x [M, H] (floating types of 8 to 32 bits, int8, uint8, int32, int64) -> rows [M *
    top_k, H]: each token's row at the places of its routes, zeros behind the last
    expert's.  Differentiable for bf16, fp16 and fp32: dx is the sum of the token's rows
    of the gradient, in FP32, rounded once."""
    host = _lib.host()
    out = host and host.sort_tokens(x, order)
    if out is not None:
        return out
    offsets, routes, position = check_order(order)
    if x.dtype not in _CODES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    if x.ndim != 2 or x.shape[0] != position.shape[0]:
        raise ValueError(f"x must be [{position.shape[0]}, H], got {tuple(x.shape)}")
    _check_tangents(x)
    grad = x.requires_grad and torch.is_grad_enabled()
    _lib.refuse_recorder(grad)
    if grad:
        if x.dtype not in _FLOATS:
            raise TypeError(f"no gradient for {x.dtype}")
        _check_capture(x)
        return _SortTokens.apply(x, offsets, position)
    return _sort(x, offsets, position)


def combine_tokens(y: torch.Tensor, order: ExpertOrder,
                   topk_weights: torch.Tensor | None = None) -> torch.Tensor:
    """y [M * top_k, H] (bf16, fp16 or fp32) by expert -> [M, H]: out[t] = the sum over s of
    topk_weights[t, s] * y[position[t, s]], in FP32 in the slots' order, rounded once.
    Dropped routes add nothing; without weights ([M, top_k], converted to float32) all
    are 1.  Differentiable in y and in the weights; the same inputs give the same bits
    on every call, gradients too."""
    host = _lib.host()
    out = host and host.combine_tokens(y, order, topk_weights)
    if out is not None:
        return out
    offsets, routes, position = check_order(order)
    if y.dtype not in _FLOATS:
        raise TypeError(f"y must be bf16, fp16 or fp32, got {y.dtype}")
    if y.ndim != 2 or y.shape[0] != routes.numel():
        raise ValueError(f"y must be [{routes.numel()}, H], got {tuple(y.shape)}")
    _check_tangents(y, topk_weights)
    w = topk_weights
    if w is not None:
        if not w.is_floating_point():
            raise TypeError(f"topk_weights must be floating point, got {w.dtype}")
        if w.shape != position.shape:
            raise ValueError(f"topk_weights must be {tuple(position.shape)}, got {tuple(w.shape)}")
        w = w.to(torch.float32)
    grad = torch.is_grad_enabled() and (y.requires_grad or (w is not None and w.requires_grad))
    _lib.refuse_recorder(grad)
    if grad:
        _check_capture(y, topk_weights)
        return _CombineTokens.apply(y, w, offsets, position)
    return _combine(y, position, w)
