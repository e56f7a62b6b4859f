# SPDX-License-Identifier: MIT
"""FP8 (e4m3) products with a scale for each 128 values, and their quantizers, on MI355X.

The pair for layers that a checkpoint keeps in FP8 with block scales: activations
[..., K] carry a float32 scale for each 128 values of a row, weights [N, K] one for
each block of 128 x 128.  ``linear_fp8_block`` is the dense product,
``grouped_linear_fp8_block`` the one by expert, on rows in the order of
``sort_routes``.  No counterpart in the reference.  Inference only: no gradients.
"""

from __future__ import annotations

import torch

from . import _lib
from .sort import ExpertOrder, check_order, sort_tokens

BLOCK = 128
MAX_K = 1048576

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_OUT_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


def _row_outputs(x: torch.Tensor, k: int):
    """q [..., k] and scales [..., blocks], whose blocks are outermost in memory."""
    lead = x.shape[:-1]
    rows = lead.numel()
    q = torch.empty((*lead, k), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((_blocks(k), rows), dtype=torch.float32, device=x.device)
    return q, scales.t().view(*lead, _blocks(k)), rows


def _quant_rows(x: torch.Tensor, silu: bool):
    host = _lib.host()
    out = host and host.fp8_quant(x, silu)
    if out is not None:
        return out
    if x.dtype not in _FLOATS:
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1 or (silu and x.shape[-1] % 2):
        raise ValueError(f"x must be [..., {'2 K' if silu else 'K'}] with K >= 1, got "
                         f"{tuple(x.shape)}")
    k = x.shape[-1] // 2 if silu else x.shape[-1]
    if k > MAX_K:
        raise ValueError(f"K must be at most {MAX_K}, got {k}")
    device = _lib.require_device(x)
    lib = _lib.load()
    q, scales, rows = _row_outputs(x, k)
    if rows:
        x2, ldx = _lib.rows_of(x)
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_quant_fp8_rows(
                _lib.ptr(x2), _lib.dtype_code(x.dtype), rows, k, ldx, int(silu), _lib.ptr(q),
                _lib.ptr(scales), 1, rows, _lib.stream_of(device)))
    return q, scales


def dynamic_fp8_block_quant(x: torch.Tensor, *, block_rows: int = 1):
    """Quantize ``x`` (bf16, fp16 or fp32) to FP8 e4m3; returns (q, scales).

    * ``block_rows=1``: activations [..., K], a float32 scale for each 128 values of a
      row: scales [..., ceil(K/128)], laid out with the blocks outermost (as the
      products read them fastest; any layout is taken);
    * ``block_rows=128``: weights [N, K] or [E, N, K], one for each block of 128 x
      128: scales [..., ceil(N/128), ceil(K/128)].

    scale = max|x| / 448 (2^-126 at least), q = x / scale to the nearest (even) e4m3
    value.  A block with a value that is not finite has scale NaN and q = 0; the
    last block of a row (or column) may be a part."""
    if block_rows == 1:
        return _quant_rows(x, False)
    if block_rows != BLOCK:
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.ndim not in (2, 3) or not 1 <= x.shape[-1] <= MAX_K:
        raise ValueError(f"weights must be [N, K] or [E, N, K] with K of 1 to {MAX_K}, got "
                         f"{tuple(x.shape)}")
    device = _lib.require_device(x)
    lib = _lib.load()
    n, k = x.shape[-2:]
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty((*x.shape[:-2], _blocks(n), _blocks(k)), dtype=torch.float32,
                         device=device)
    if x.numel():
        with _lib.on_device(device):
            for xe, qe, se in (zip(x, q, scales) if x.ndim == 3 else ((x, q, scales),)):
                x2, ldx = _lib.rows_of(xe)
                _lib.check(lib.mxfp4_quant_fp8_blocks(
                    _lib.ptr(x2), _lib.dtype_code(x.dtype), n, k, ldx, _lib.ptr(qe),
                    _lib.ptr(se), _lib.stream_of(device)))
    return q, scales


def silu_mul_fp8_block_quant(x: torch.Tensor):
    """x [..., 2 K], gate before up -> (q e4m3 [..., K], scales [..., ceil(K/128)]) of
    g / (1 + exp(-g)) * u, taken in FP32, as ``dynamic_fp8_block_quant`` quantizes it:
    the step between an expert's (or a dense layer's) gate_up and down products."""
    return _quant_rows(x, True)


def _scale_rows(scales: torch.Tensor, lead, kb: int, name: str):
    """Activation scales [..., kb] as rows, and their strides (row's, block's)."""
    if scales.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {scales.dtype}")
    if tuple(scales.shape) != (*lead, kb):
        raise ValueError(f"{name} must be {(*lead, kb)}: one scale for each {BLOCK} values, got "
                         f"{tuple(scales.shape)}")
    s = scales.reshape(-1, kb)
    row, block = s.stride() if s.shape[0] > 1 else (1, s.stride(1))
    block = block if kb > 1 else 1
    if row < 1 or block < 1:  # an expanded dimension
        s = s.contiguous()
        row, block = kb, 1
    return s, row, block


def _check_product(a, a_scales, w, w_scales, out_dtype, w_ndim):
    """Types and shapes both products check; (scale rows, strides, n, k)."""
    for t, name in ((a, "a"), (w, "w")):
        if t.dtype != torch.float8_e4m3fn:
            raise TypeError(f"{name} must be float8_e4m3fn, got {t.dtype}")
    if out_dtype not in _OUT_CODES:
        raise TypeError(f"unsupported output dtype {out_dtype}")
    if a.ndim < 1 or w.ndim != w_ndim:
        raise ValueError(f"a must be [..., K] and w [{'E, ' if w_ndim == 3 else ''}N, K]")
    n, k = w.shape[-2:]
    if a.shape[-1] != k:
        raise ValueError(f"activation K {a.shape[-1]} does not match weight K {k}")
    if k == 0 or k % 16 or k > MAX_K:
        raise ValueError(f"K must be divisible by 16 and at most {MAX_K}, got {k}")
    if w_scales.dtype != torch.float32:
        raise TypeError(f"w_scales must be float32, got {w_scales.dtype}")
    want = (*w.shape[:-2], _blocks(n), _blocks(k))
    if tuple(w_scales.shape) != want:
        raise ValueError(f"w_scales must be {want}: one scale for each {BLOCK} x {BLOCK}, got "
                         f"{tuple(w_scales.shape)}")
    return _scale_rows(a_scales, a.shape[:-1], _blocks(k), "a_scales"), n, k


def linear_fp8_block(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor,
                     w_scales: torch.Tensor, bias: torch.Tensor | None = None,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out [..., N] = sum over blocks b of K of a_scales[..., b] * w_scales[n / 128, b] *
    (a . w^T over the block) (+ bias): a e4m3 [..., K] with scales [..., ceil(K/128)]
    in any layout, w e4m3 [N, K] with scales [ceil(N/128), ceil(K/128)], bias [N] of
    ``out_dtype`` (bf16, fp16 or fp32).

    A block's sum is the FP8 MFMA's, which drops the lowest bits of small products
    beside large ones: about 1e-5 of the result, whatever ``out_dtype``.  Scales and the
    sum over the blocks are FP32, rounded once.  K is a multiple of 16."""
    host = _lib.host()
    out = host and host.fp8_linear(a, a_scales, w, w_scales, bias, _OUT_CODES.get(out_dtype, -1))
    if out is not None:
        return out
    (sa, row, block), n, k = _check_product(a, a_scales, w, w_scales, out_dtype, 2)
    if bias is not None:
        if bias.dtype != out_dtype:
            raise TypeError(f"bias must be {out_dtype}, got {bias.dtype}")
        if bias.shape != (n,):
            raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    device = _lib.require_device(a, sa, w, w_scales, bias)
    lib = _lib.load()
    m = a.numel() // k
    out = torch.empty((*a.shape[:-1], n), dtype=out_dtype, device=device)
    if m and n:
        a2, w2 = _lib.aligned(a), _lib.aligned(w)
        ws = w_scales.contiguous()
        b = None if bias is None else bias.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_linear_fp8(
                _lib.ptr(a2), _lib.ptr(sa), row, block, m, k, _lib.ptr(w2), _lib.ptr(ws), n,
                _lib.ptr(b), _lib.ptr(out), _lib.dtype_code(out_dtype), _lib.stream_of(device)))
    return out


def grouped_linear_fp8_block(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor,
                             w_scales: torch.Tensor, order: ExpertOrder, *, gather: bool = False,
                             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``linear_fp8_block`` by expert: w e4m3 [E, N, K], scales [E, ceil(N/128),
    ceil(K/128)], out [R, N] for the R = M * top_k rows of ``order`` (``sort_routes`` of
    the same E): row p by the weights of the expert whose rows p lies in, zeros behind
    the last expert's.

    ``a`` is sorted already, [R, K], or with ``gather`` the tokens' own rows [M, K], each
    read for all its routes (quantized once a token, and never copied)."""
    host = _lib.host()
    out = host and host.fp8_grouped(a, a_scales, w, w_scales, order, bool(gather),
                                    _OUT_CODES.get(out_dtype, -1))
    if out is not None:
        return out
    (sa, row, block), n, k = _check_product(a, a_scales, w, w_scales, out_dtype, 3)
    offsets, routes, position = check_order(order)
    experts = w.shape[0]
    if offsets.numel() != experts + 1:
        raise ValueError(f"the order is of {offsets.numel() - 1} experts, w of {experts}")
    m, top_k = position.shape
    rows = m * top_k
    if a.ndim != 2 or a.shape[0] != (m if gather else rows):
        raise ValueError(f"a must be [{m if gather else rows}, K], got {tuple(a.shape)}")
    device = _lib.require_device(a, sa, w, w_scales, offsets, routes, position)
    lib = _lib.load()
    if gather and m * k >= 1 << 31:  # past the gathering kernels' offsets: copied once
        moved = ExpertOrder(offsets, routes, position)
        a, gather = sort_tokens(a, moved), False
        sa, row, block = sort_tokens(sa.contiguous(), moved), _blocks(k), 1
    out = torch.empty((rows, n), dtype=out_dtype, device=device)
    if rows and n:
        a2, w2 = _lib.aligned(a), _lib.aligned(w)
        ws = w_scales.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_grouped_linear_fp8(
                _lib.ptr(a2), _lib.ptr(sa), row, block, a2.shape[0], k, _lib.ptr(w2),
                _lib.ptr(ws), experts, n, _lib.ptr(offsets),
                _lib.ptr(routes if gather else None), top_k, rows, _lib.ptr(out),
                _lib.dtype_code(out_dtype), _lib.stream_of(device)))
    return out
