"""MI355X (gfx950) implementation of the dropless MoE expert-MLP hot path behind the plugin surface of
foundation-model-stack/moe-distributed-training: `scattermoe_utils` (parallel_linear_lora, ParallelLinearLora,
kernels.ops) plus the scattermoe pieces those scripts import (parallel_linear, ParallelExperts,
flatten_and_sort, padded_block_indices) and `megablocks_utils` (router, the fused expert-MLP caller).

All device work runs in libmoe_hip.so (hand-written HIP, C ABI in include/moe_hip.h); importing the ops on a
machine without that library raises immediately -- there is no host fallback.
"""
from . import _lib  # noqa: F401
from .scattermoe_utils.kernels.ops import (  # noqa: F401
    flatten_and_sort, padded_block_indices, scatter2scatter, scatter2scatter_lora, group, group_bwd_AB, group_bwd_W,
    quantize_rows,
)
from .scattermoe_utils.parallel_linear_lora import ParallelLinearLora, parallel_linear_lora  # noqa: F401
from .scattermoe_utils.parallel_experts import ParallelLinear, parallel_linear, ParallelExperts  # noqa: F401
from .scattermoe_utils.parallel_linear_int8 import parallel_linear_int8, quantize_expert_weights  # noqa: F401
from .megablocks_utils.router import forward_router, route_and_sort  # noqa: F401
from .megablocks_utils.moe_mlp import (  # noqa: F401
    scattermoe_permute_and_compute, fused_expert_mlp, moe_layer_forward, ScatterMoEBlock,
    Int8ExpertWeights, fused_expert_mlp_int8, moe_layer_forward_int8,
)

__all__ = [
    "flatten_and_sort", "padded_block_indices", "scatter2scatter", "scatter2scatter_lora", "group", "group_bwd_AB",
    "group_bwd_W", "ParallelLinearLora", "parallel_linear_lora", "ParallelLinear", "parallel_linear",
    "ParallelExperts", "forward_router", "route_and_sort", "scattermoe_permute_and_compute", "fused_expert_mlp",
    "moe_layer_forward", "ScatterMoEBlock", "quantize_rows", "quantize_expert_weights", "parallel_linear_int8",
    "Int8ExpertWeights", "fused_expert_mlp_int8", "moe_layer_forward_int8",
]
