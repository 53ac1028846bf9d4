"""MI355X-native quantized-weight matmul behind the ``max.graph.ops.qmatmul`` call shape.

``qmatmul(encoding, config, lhs, *rhs)``, ``dequantize`` and the
``QuantizationEncoding`` / ``QuantizationConfig`` types mirror the MAX graph API;
the arithmetic runs in hand-written HIP kernels for gfx950 reached through the
C ABI of ``libqmm.so`` (``include/qmm.h``).  There is no CPU fallback: a missing
library or a non-GPU tensor is an error.
"""
from .quantization import BlockParameters, QuantizationConfig, QuantizationEncoding
from .ops import (
    block_dots_q4_0,
    dequantize,
    qmatmul,
    qmatmul_grouped,
    qmatmul_repacked,
    qmatmul_rmsnorm,
    qmatmul_swiglu,
    quantize,
    quantize_gptq,
    repack_weights,
    RepackedWeights,
)
from .experts import (
    ExpertRouting,
    group_experts,
    qmatmul_experts,
    qmatmul_experts_sum,
    qmatmul_experts_swiglu,
    route_experts,
)
from .scores import LogProbs, logprobs, qmatmul_logprobs
from .weights import GGUFWeights, load_gptq_config, load_gptq_linear

__all__ = [
    "BlockParameters",
    "QuantizationConfig",
    "QuantizationEncoding",
    "qmatmul",
    "qmatmul_grouped",
    "qmatmul_repacked",
    "repack_weights",
    "RepackedWeights",
    "qmatmul_rmsnorm",
    "qmatmul_swiglu",
    "route_experts",
    "group_experts",
    "ExpertRouting",
    "qmatmul_experts",
    "qmatmul_experts_swiglu",
    "qmatmul_experts_sum",
    "logprobs",
    "qmatmul_logprobs",
    "LogProbs",
    "dequantize",
    "quantize",
    "quantize_gptq",
    "block_dots_q4_0",
    "GGUFWeights",
    "load_gptq_config",
    "load_gptq_linear",
]
