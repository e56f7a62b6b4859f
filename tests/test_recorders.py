"""torch's recorders of tensor calls (torch.jit.trace, make_fx on real tensors) do not see the
library's: a recording would replay an operator's torch.empty and no kernel.  The operators
refuse to be recorded."""

from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import mxfp4_amd as mx
from mxfp4_amd import _lib

from _helpers import cuda, rand_act

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning",
                                        "ignore::DeprecationWarning")
BF16, F8, U8 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8
RECORDERS = {
    "jit.trace": lambda f, x: torch.jit.trace(f, x, check_trace=False),
    "make_fx": lambda f, x: make_fx(f, tracing_mode="real")(x),
}


def order_of(device="cpu"):
    return mx.ExpertOrder(*(t.to(device) for t in (
        torch.tensor([0, 2, 3, 4], dtype=torch.int32), torch.tensor([0, 3, 1, 2], dtype=torch.int32),
        torch.tensor([[0, 2], [3, 1]], dtype=torch.int32))))


def calls(device="cpu"):
    """name -> (operator of one tensor, that tensor)"""
    zeros = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    ones = lambda *s, dtype=torch.float32: torch.ones(s, dtype=dtype, device=device)  # noqa: E731
    o = order_of(device)
    x = zeros(2, 256, dtype=BF16)
    w4, s4 = zeros(32, 128, dtype=U8), ones(32, 8, dtype=U8)
    ids = zeros(2, 2, dtype=torch.int64)
    layer = (zeros(4, 256, 128, dtype=U8), ones(4, 256, 8, dtype=U8),
             zeros(4, 256, 64, dtype=U8), ones(4, 256, 4, dtype=U8), ones(2, 2), ids)
    a8, w8 = zeros(2, 256).to(F8), zeros(3, 128, 256).to(F8)
    i8 = zeros(2, 256, dtype=torch.int8)
    return {
        "dequant": (lambda t: mx.dequant_mxfp4(t, s4), w4),
        "linear": (lambda t: mx.linear_mxfp4_soft(t, w4, s4), x),
        "layer": (lambda t: mx.moe_layer(t, *layer), x),
        "quant": (lambda t: mx.dynamic_mxfp4_quant(t), x),
        "w4a4": (lambda t: mx.linear_mxfp4_w4a4(t, s4, w4, s4), w4),
        "route": (lambda t: mx.route_topk(t, 2), zeros(2, 8)),
        "route_grouped": (lambda t: mx.route_topk_grouped(t, 2), zeros(2, 8)),
        "norm": (lambda t: mx.rms_norm_quant(t, ones(256, dtype=BF16)), x),
        "int8": (lambda t: mx.dynamic_int8_quant(t), x),
        "w8a8": (lambda t: mx.linear_int8_w8a8(t, ones(2, 1), i8, ones(2)), i8),
        "routing": (lambda t: mx.make_routing_device(t, 4, 16), ids),
        "fp8_quant": (lambda t: mx.dynamic_fp8_block_quant(t), x),
        "fp8_blocks": (lambda t: mx.dynamic_fp8_block_quant(t, block_rows=128), x),
        "fp8_silu": (lambda t: mx.silu_mul_fp8_block_quant(t), x),
        "fp8_linear": (lambda t: mx.linear_fp8_block(t, ones(2, 2), w8[0], ones(1, 2)), a8),
        "fp8_grouped": (lambda t: mx.grouped_linear_fp8_block(t, ones(2, 2), w8, ones(3, 1, 2), o,
                                                              gather=True), a8),
        "sort_routes": (lambda t: mx.sort_routes(t, 3), ids),
        "sort_tokens": (lambda t: mx.sort_tokens(t, o), x),
        "combine": (lambda t: mx.combine_tokens(t, o, ones(2, 2)), zeros(4, 256)),
    }


@pytest.mark.parametrize("recorder", sorted(RECORDERS))
@pytest.mark.parametrize("name", sorted(calls()))
def test_recording_is_refused(name, recorder):
    f, x = calls()[name]
    with pytest.raises(RuntimeError, match="ROCm devices only"):  # not what a recorder says
        f(x)
    with pytest.raises(RuntimeError, match=recorder):
        RECORDERS[recorder](f, x)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("recorder", sorted(RECORDERS))
def test_recording_on_the_gpu(recorder, native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: None)
    for name, (f, x) in calls("cuda").items():
        with pytest.raises(RuntimeError, match=recorder):
            RECORDERS[recorder](f, x)
        f(x)  # and afterwards runs as ever


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_recording_of_the_moves_with_gradients(native, monkeypatch):
    # torch.jit.trace keeps an autograd function as a call; make_fx looks into it
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: None)
    o = order_of("cuda")
    w = torch.tensor([[0.5, 2.0], [1.0, -1.0]], device="cuda")

    def there_and_back(t):
        return mx.combine_tokens(mx.sort_tokens(t, o) * 3, o, w)

    x, other = (cuda(rand_act(i, (2, 64))).float().requires_grad_() for i in (1, 2))
    with pytest.raises(RuntimeError, match="make_fx"):
        RECORDERS["make_fx"](there_and_back, x)
    traced = RECORDERS["jit.trace"](there_and_back, x)
    for t in (x, other):
        want, got = there_and_back(t), traced(t)
        assert torch.equal(got, want)
        assert torch.equal(*(torch.autograd.grad(v.sum(), t)[0] for v in (got, want)))
