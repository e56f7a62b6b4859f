# SPDX-License-Identifier: MIT
"""mxfp4_amd -- MI355X (gfx950) MXFP4 backend behind the ``moe_op_mxfp4_soft``
operator surface of lutianshu824/mxfp4-gfx936.

Operators (all compute in libmxfp4_gfx950.so, on the tensors' device and
current stream; no host synchronisation, no fallback path):

* ``dequant_mxfp4``, ``linear_mxfp4_soft``, ``fused_moe_mxfp4_soft`` --
  drop-in for src/aiter/ops/triton/moe_op_mxfp4_soft.py;
* ``fused_moe_mxfp4`` -- AITER's entry (integration/aiter/moe_op_mxfp4.py);
* ``moe_layer`` / ``make_routing`` -- the vLLM MoE layer and routing
  metadata (integration/vllm/vllm_mxfp4_gfx936.py:119-146, 233-265);
  ``route_topk`` -- router logits -> the layer's top-k weights and ids;
  ``route_topk_grouped`` -- the same with sigmoid scores, a balance bias and
  groups of experts;
* ``dynamic_mxfp4_quant`` / ``linear_mxfp4_w4a4`` -- activation quantizer
  and dense W4A4 on the block-scaled FP4 MFMA;
* ``rms_norm_quant`` -- RMS norm with the residual's addition, to int8 with a
  scale per token or MX FP8; ``dynamic_int8_quant`` / ``linear_int8_w8a8`` --
  int8 quantizer by rows and dense W8A8 on the integer MFMA;
* ``dynamic_fp8_block_quant`` / ``silu_mul_fp8_block_quant`` -- quantizers to FP8
  with a scale for each 128 values; ``linear_fp8_block`` and
  ``grouped_linear_fp8_block`` -- the products of such operands, dense and by
  expert;
* ``sort_routes`` / ``sort_tokens`` / ``combine_tokens`` -- tokens sorted by expert
  and back with their weights, differentiable;
* ``prepack_w4a16`` -- the fragment-ordered weight copy the prefill GEMMs
  read when given one (``prepacked=`` / ``prepacked13=``, ``prepacked2=``);
  ``register_prepacked`` records one for expert weights, which
  ``fused_moe_mxfp4_soft`` / ``fused_moe_mxfp4`` then find by address.

``mxfp4_amd.vllm_adapter.install()`` points vLLM's compressed-tensors MXFP4
schemes at these operators (integration/vllm/vllm_mxfp4_gfx936.py).
"""

from .moe_op_mxfp4_soft import (  # noqa: F401
    _MXFP4_E2M1_VALUES,
    dequant_mxfp4,
    fused_moe_mxfp4_soft,
    linear_mxfp4_soft,
    make_routing_device,
)
from .moe_op_mxfp4 import fused_moe_mxfp4  # noqa: F401
from .moe_layer import make_routing, moe_layer, route_topk, route_topk_grouped  # noqa: F401
from .fp8 import (  # noqa: F401
    dynamic_fp8_block_quant,
    grouped_linear_fp8_block,
    linear_fp8_block,
    silu_mul_fp8_block_quant,
)
from .norm import QuantizedNorm, rms_norm_quant  # noqa: F401
from .quant import (  # noqa: F401
    dynamic_int8_quant,
    dynamic_mxfp4_quant,
    linear_int8_w8a8,
    linear_mxfp4_w4a4,
)
from .prepack import (  # noqa: F401
    PrepackedWeights,
    lookup_prepacked,
    prepack_w4a16,
    register_prepacked,
    unregister_prepacked,
)
from .sort import ExpertOrder, combine_tokens, sort_routes, sort_tokens  # noqa: F401
from . import _lib  # noqa: F401

__all__ = [
    "dequant_mxfp4",
    "linear_mxfp4_soft",
    "fused_moe_mxfp4_soft",
    "fused_moe_mxfp4",
    "moe_layer",
    "make_routing",
    "route_topk",
    "route_topk_grouped",
    "make_routing_device",
    "dynamic_mxfp4_quant",
    "linear_mxfp4_w4a4",
    "rms_norm_quant",
    "QuantizedNorm",
    "dynamic_int8_quant",
    "linear_int8_w8a8",
    "dynamic_fp8_block_quant",
    "silu_mul_fp8_block_quant",
    "linear_fp8_block",
    "grouped_linear_fp8_block",
    "ExpertOrder",
    "sort_routes",
    "sort_tokens",
    "combine_tokens",
    "prepack_w4a16",
    "PrepackedWeights",
    "register_prepacked",
    "unregister_prepacked",
    "lookup_prepacked",
]
