"""B200-native (sm_100a) routed-attention hot path of Double Attention.

Drop-in for the reference package's module/config API
(src/double_attention/__init__.py): the same constructors, parameters and
state_dict keys, with the dictionary normalisation, fused Q/K projection,
dictionary route and outer routed attention running in hand-written
tcgen05 kernels (``libda_b200.so``, C ABI in ``include/da_b200.h``).
"""

from .config import DoubleAttentionConfig, experiment_config, experiment_names
from .eight_bit import (
    Checkpoint8,
    Int8Rows,
    add_layernorm_int8,
    add_rmsnorm_int8,
    checkpoint8,
    feedforward_checkpoint8,
    gelu_checkpoint8,
    gelu_checkpoint8_backward,
    int8_linear,
    layernorm_int8,
    linear_checkpoint8,
    quantize_int8,
    rmsnorm_int8,
    weight_grad_checkpoint8,
)
from .graphs import GraphedModuleStep
from .int8_model import Int8DoubleAttentionLM, Int8Linear
from .modules import (
    DoubleAttentionAux,
    DoubleAttentionBlock,
    DoubleAttentionLM,
    DoubleAttentionStack,
    SharedDictionaryAttention,
    SharedDictionaryBank,
)
from .ops import assemble_score_maps, dictionary_route, routed_attention

__all__ = [
    "Checkpoint8",
    "DoubleAttentionAux",
    "DoubleAttentionBlock",
    "DoubleAttentionConfig",
    "DoubleAttentionLM",
    "DoubleAttentionStack",
    "GraphedModuleStep",
    "Int8DoubleAttentionLM",
    "Int8Linear",
    "Int8Rows",
    "SharedDictionaryAttention",
    "SharedDictionaryBank",
    "add_layernorm_int8",
    "add_rmsnorm_int8",
    "assemble_score_maps",
    "checkpoint8",
    "dictionary_route",
    "experiment_config",
    "experiment_names",
    "feedforward_checkpoint8",
    "gelu_checkpoint8",
    "gelu_checkpoint8_backward",
    "int8_linear",
    "layernorm_int8",
    "linear_checkpoint8",
    "quantize_int8",
    "rmsnorm_int8",
    "routed_attention",
    "weight_grad_checkpoint8",
]
