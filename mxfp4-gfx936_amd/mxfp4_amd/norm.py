# SPDX-License-Identifier: MIT
"""RMS norm with the residual's addition and an 8-bit output, on MI355X.

``rms_norm_quant`` is the step between two projections of a decoder layer in
one pass over the data: it adds the residual, normalises, and writes what the
next product reads -- int8 with a scale per token for ``linear_int8_w8a8``, or
OCP MX FP8 blocks for ``fused_moe_mxfp4`` -- beside the new residual.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

# fmt -> (output dtype, its code in the C ABI)
_FORMATS = {
    "int8": (torch.int8, _lib.DT_I8),
    "mxfp8_e4m3": (torch.float8_e4m3fn, _lib.DT_F8E4M3),
    "mxfp8_e5m2": (torch.float8_e5m2, _lib.DT_F8E5M2),
}


class QuantizedNorm(NamedTuple):
    """What ``rms_norm_quant`` returns; None where it was not asked for."""

    q: torch.Tensor
    scales: torch.Tensor
    residual: torch.Tensor | None
    normed: torch.Tensor | None


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                   eps: float = 1e-6, fmt: str = "int8", normed: bool = False) -> QuantizedNorm:
    """Normalise the last dimension of ``x`` (bf16, fp16 or fp32, [..., K]):

        h = x + residual                                      (FP32)
        y = h * weight / sqrt(mean(h^2) + eps)

    ``weight`` [K] is of x's dtype or fp32, ``residual`` of x's shape and dtype.
    Returns (q, scales, residual, normed):

    * ``fmt="int8"``: q int8 [..., K], scales float32 [...]: one per token,
      max|y| / 127 (2^-126 at least), q = y / scale to the nearest (even)
      integer; a token with a value that is not finite has scale NaN, q = 0;
    * ``fmt="mxfp8_e4m3"`` / ``"mxfp8_e5m2"``: q [..., K] of that float8
      dtype, scales uint8 [..., K/32] (E8M0, E = floor(log2 max|y|) - 8 / 15),
      saturating; a block with a value that is not finite has byte 255, q = 0;
    * residual: h rounded to x's dtype, None without a ``residual``.  The norm
      takes h before that rounding;
    * ``normed=True``: y rounded to x's dtype as well (what a router's gate
      reads); else None.

    h * weight is FP32; where it leaves that range y is not finite.  y is that
    product times 1 / sqrt(..): three FP32 roundings, in another order than
    (h / sqrt(..)) * weight.  An 8-bit value whose quotient lies that close to
    the middle between two steps can come out one step apart from such a form's;
    neither is the nearer one to the exact result.  The same inputs give the same
    bits on every call.
    """
    if fmt not in _FORMATS:
        raise ValueError(f"unknown output format {fmt!r}")
    eps = float(eps)
    if not 0 < eps < math.inf:
        raise ValueError(f"eps must be positive and finite, got {eps}")
    host = _lib.host()
    q_dtype, q_code = _FORMATS[fmt]
    out = host and host.rms_norm_quant(x, weight, residual, eps, q_code, bool(normed))
    if out is not None:
        return QuantizedNorm(*out)
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"weight must be {x.dtype} or fp32, got {weight.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., K] with K >= 1, got {tuple(x.shape)}")
    k = x.shape[-1]
    if weight.shape != (k,):
        raise ValueError(f"weight must be [{k}], got {tuple(weight.shape)}")
    if fmt != "int8" and k % 32:
        raise ValueError(f"MX blocks need K divisible by 32, got {k}")
    if residual is not None:
        if residual.dtype != x.dtype:
            raise TypeError(f"residual must be {x.dtype}, got {residual.dtype}")
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} is not of x's shape "
                             f"{tuple(x.shape)}")
    device = _lib.require_device(x, weight, residual)
    lib = _lib.load()
    q = torch.empty(x.shape, dtype=q_dtype, device=device)
    if fmt == "int8":
        scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    else:
        scales = torch.empty((*x.shape[:-1], k // 32), dtype=torch.uint8, device=device)
    res_out = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=device)
    y = torch.empty(x.shape, dtype=x.dtype, device=device) if normed else None
    rows = x.numel() // k
    if rows:
        x2, ldx = _lib.rows_of(x)
        r2, ldr = (None, 0) if residual is None else _lib.rows_of(residual)
        w = weight.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_rms_norm_quant(
                _lib.ptr(x2), _lib.dtype_code(x.dtype), rows, k, ldx, _lib.ptr(r2), ldr,
                _lib.ptr(w), _lib.dtype_code(w.dtype), eps, q_code, _lib.ptr(q),
                _lib.ptr(scales), _lib.ptr(res_out), _lib.ptr(y), _lib.stream_of(device)))
    return QuantizedNorm(q, scales, res_out, y)
