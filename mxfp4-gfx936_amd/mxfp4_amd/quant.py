# SPDX-License-Identifier: MIT
"""Activation quantizers and the dense linears that read them, on MI355X.

``dynamic_mxfp4_quant(x, mode)`` turns [..., K] bf16/fp16/fp32 activations
into packed E2M1 [..., K/2] + E8M0 [..., K/32] on the device:

* ``mode="ties_away"`` reproduces the reference test quantizer
  ``torch_dynamic_mxfp4_quant`` (tests/test_moe_mxfp4_soft.py:28-60 of
  lutianshu824/mxfp4-gfx936) bit for bit;
* ``mode="rne"`` is the OCP MX rule used for the W4A4 benchmark
  configuration: E = floor(log2(amax)) - 2, E2M1 round-to-nearest-even,
  saturation at +-6.

``linear_mxfp4_w4a4`` multiplies packed activations by packed weights on
gfx950's block-scaled FP4 MFMA (the packed-A semantics of
integration/aiter/moe_op_mxfp4.py:206-214, 329-338 with a single expert).

``dynamic_int8_quant`` and ``linear_int8_w8a8`` are the pair for the layers that
a checkpoint keeps in 8 bits (attention projections beside MXFP4 experts): int8
rows with one float32 scale each -- a token's activations, an output channel's
weights -- and their product, exact in int32.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from . import _lib

_MODES = {"ties_away": _lib.QUANT_TIES_AWAY, "rne": _lib.QUANT_RNE}

_OUT_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def dynamic_mxfp4_quant(x: torch.Tensor, mode: str = "ties_away"):
    """Quantize the last dimension of ``x`` in blocks of 32; returns
    (packed uint8 [..., K/2], scales uint8 [..., K/32])."""
    if mode not in _MODES:
        raise ValueError(f"unknown quantizer mode {mode!r}")
    host = _lib.host()
    out = host and host.quant(x, _MODES[mode])
    if out is not None:
        return out
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    k = x.shape[-1]
    if k % 32:
        raise ValueError("test quantizer requires K divisible by 32")
    device = _lib.require_device(x)
    lib = _lib.load()
    rows = x.numel() // k if k else 0
    packed = torch.empty((*x.shape[:-1], k // 2), dtype=torch.uint8, device=device)
    scales = torch.empty((*x.shape[:-1], k // 32), dtype=torch.uint8, device=device)
    if rows and k:
        x2 = x.reshape(rows, k)
        if x2.stride(-1) != 1:
            x2 = x2.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_quant(
                _lib.ptr(x2), _lib.dtype_code(x.dtype), rows, k, x2.stride(0), _MODES[mode],
                _lib.ptr(packed), _lib.ptr(scales), _lib.stream_of(device)))
    return packed, scales


def linear_mxfp4_w4a4(a_packed: torch.Tensor, a_scales: torch.Tensor, w_packed: torch.Tensor,
                      w_scales: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out [M, N] = dequant(a) . dequant(w)^T with FP32 accumulation, rounded
    once to ``out_dtype`` (bf16, fp16 or fp32)."""
    host = _lib.host()
    out = host and host.w4a4(a_packed, a_scales, w_packed, w_scales, _OUT_CODES.get(out_dtype, -1))
    if out is not None:
        return out
    for t, name in ((a_packed, "a_packed"), (a_scales, "a_scales"), (w_packed, "w_packed"),
                    (w_scales, "w_scales")):
        if t.dtype != torch.uint8:
            raise TypeError(f"{name} must be uint8, got {t.dtype}")
    if out_dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"unsupported output dtype {out_dtype}")
    if a_packed.ndim != 2 or w_packed.ndim != 2:
        raise ValueError("packed operands must be 2D")
    m, n, k = a_packed.shape[0], w_packed.shape[0], a_packed.shape[1] * 2
    if w_packed.shape[1] * 2 != k:
        raise ValueError(f"activation K {k} does not match weight K {w_packed.shape[1] * 2}")
    if k % 32:
        raise ValueError(f"logical K must be divisible by 32, got {k}")
    if a_scales.shape != (m, k // 32) or w_scales.shape != (n, k // 32):
        raise ValueError("one E8M0 scale is required for every 32 MXFP4 values")
    device = _lib.require_device(a_packed, a_scales, w_packed, w_scales)
    lib = _lib.load()
    out = torch.empty((m, n), dtype=out_dtype, device=device)
    if m and n:
        a = _lib.aligned(a_packed)
        w = _lib.aligned(w_packed)
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_linear_w4a4(
                _lib.ptr(a), _lib.ptr(a_scales.contiguous()), m, k, _lib.ptr(w),
                _lib.ptr(w_scales.contiguous()), n, _lib.ptr(out), _lib.dtype_code(out_dtype),
                _lib.stream_of(device)))
    return out


def dynamic_int8_quant(x: torch.Tensor):
    """Quantize the rows of ``x`` [..., K] (bf16, fp16 or fp32) to int8; returns
    (q int8 [..., K], scales float32 [...]): scale = max|x| / 127 (2^-126 at
    least), q = round(x / scale), ties to even, both as FP32 gives them.  A row
    with a value that is not finite has scale NaN and q = 0.  Activations
    [..., K] get a scale per token, weights [N, K] one per output channel."""
    host = _lib.host()
    out = host and host.int8_quant(x)
    if out is not None:
        return out
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., K] with K >= 1, got {tuple(x.shape)}")
    device = _lib.require_device(x)
    lib = _lib.load()
    k = x.shape[-1]
    rows = x.numel() // k
    q = torch.empty(x.shape, dtype=torch.int8, device=device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    if rows:
        x2, ldx = _lib.rows_of(x)
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_quant_int8(
                _lib.ptr(x2), _lib.dtype_code(x.dtype), rows, k, ldx, _lib.ptr(q),
                _lib.ptr(scales), _lib.stream_of(device)))
    return q, scales


def _row_scales(scales: torch.Tensor, lead, name: str) -> torch.Tensor:
    """One float32 scale per row: [...] or [..., 1] -> contiguous."""
    if scales.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {scales.dtype}")
    if tuple(scales.shape) not in (tuple(lead), (*lead, 1)):
        raise ValueError(f"{name} must be {tuple(lead)}: one scale per row, got "
                         f"{tuple(scales.shape)}")
    return scales.contiguous()


def linear_int8_w8a8(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor,
                     w_scales: torch.Tensor, bias: torch.Tensor | None = None,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out [..., N] = (a . w^T) * a_scales * w_scales (+ bias): a int8 [..., K]
    with a float32 scale per row, w int8 [N, K] with one per output channel
    (both [...] or [..., 1]), bias [N] of ``out_dtype`` (bf16, fp16 or fp32).
    The sum is exact in int32, FP32 from there, rounded once.  K is a multiple
    of 32, at most 131040."""
    host = _lib.host()
    out = host and host.w8a8(a, a_scales, w, w_scales, bias, _OUT_CODES.get(out_dtype, -1))
    if out is not None:
        return out
    for t, name in ((a, "a"), (w, "w")):
        if t.dtype != torch.int8:
            raise TypeError(f"{name} must be int8, got {t.dtype}")
    if out_dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"unsupported output dtype {out_dtype}")
    if a.ndim < 1 or w.ndim != 2:
        raise ValueError("a must be [..., K] and w [N, K]")
    n, k = w.shape
    if a.shape[-1] != k:
        raise ValueError(f"activation K {a.shape[-1]} does not match weight K {k}")
    if k == 0 or k % 32 or k > 131040:
        raise ValueError(f"K must be divisible by 32 and at most 131040, got {k}")
    sa = _row_scales(a_scales, a.shape[:-1], "a_scales")
    sw = _row_scales(w_scales, (n,), "w_scales")
    if bias is not None:
        if bias.dtype != out_dtype:
            raise TypeError(f"bias must be {out_dtype}, got {bias.dtype}")
        if bias.shape != (n,):
            raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    device = _lib.require_device(a, sa, w, sw, bias)
    lib = _lib.load()
    m = a.numel() // k
    out = torch.empty((*a.shape[:-1], n), dtype=out_dtype, device=device)
    if m and n:
        a2, w2 = _lib.aligned(a), _lib.aligned(w)
        b = None if bias is None else bias.contiguous()
        with _lib.on_device(device):
            _lib.check(lib.mxfp4_linear_w8a8(
                _lib.ptr(a2), _lib.ptr(sa), m, k, _lib.ptr(w2), _lib.ptr(sw), n, _lib.ptr(b),
                _lib.ptr(out), _lib.dtype_code(out_dtype), _lib.stream_of(device)))
    return out
