"""B200-native SonicMoE layer: the reference's Python surface over libsonicmoe_b200.so.

Exports match the reference package (sonicmoe/__init__.py:5-8).
"""

from .count_cumsum import count_cumsum
from .enums import ActivationType, KernelBackendMoE
from .functional import enable_quack_gemm, moe_general_routing_inputs, moe_TC_softmax_topk_layer
from .functional.adapters import adapter_linear, adapter_permutation
from .functional.norm import NormedRows, rms_norm, rms_norm_quantize
from .functional.permutation import TokenPermutation, permute_tokens, token_permutation, unpermute_tokens
from .moe import MoE
from ._lib import SonicMoEError, check_status

__all__ = [
    "ActivationType",
    "KernelBackendMoE",
    "MoE",
    "count_cumsum",
    "enable_quack_gemm",
    "moe_TC_softmax_topk_layer",
    "moe_general_routing_inputs",
    # beyond the reference's exports: the status check of the bounded-wait GEMM kernels
    "SonicMoEError",
    "check_status",
    # and tokens sorted by expert and back, for experts of the caller's own
    "TokenPermutation",
    "token_permutation",
    "permute_tokens",
    "unpermute_tokens",
    # the norm in front of the layer, in the activations' type or as 8-bit rows
    "NormedRows",
    "rms_norm",
    "rms_norm_quantize",
    # low-rank adapters of many requests beside a shared projection
    "adapter_linear",
    "adapter_permutation",
]
