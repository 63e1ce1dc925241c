"""fastmoe_amd: fastmoe's grouped pointer-indirection MoE combine on MI355X (gfx950).

The operator API mirrors ``fastmoe.kernels.ops``; the work runs in hand-written HIP kernels of
``libfastmoe_amd.so`` through its C ABI (``include/fastmoe_amd.h``).
"""
from .consts import MoEImplementation
from .dispatch import PermutedTokens, permute_tokens
from .moe import (
    Int8MoEFeedForward,
    MoEFeedForward,
    NormedMoEFeedForward,
    compute_experts,
    gate_and_sort,
    unpermute,
)
from .ops import (
    GroupedMetadata,
    GroupedWeightedScatterAdd,
    build_plan,
    grouped_weighted_scatter_add,
    invert_scatter_index,
    prepare_grouped_metadata,
    prepare_metadata_and_plan,
    weighted_scatter_add,
)
from .quantize import (
    CompressedRows,
    Int8NormedRows,
    Int8Weights,
    QuantizedRows,
    add_rms_norm,
    add_rms_norm_int8,
    compress_rows,
    gelu_compress,
    gelu_compressed_backward,
    int8_linear,
    quantize_rows,
    quantize_weights,
    restore_rows,
)

__all__ = [
    "CompressedRows",
    "GroupedMetadata",
    "GroupedWeightedScatterAdd",
    "Int8MoEFeedForward",
    "Int8NormedRows",
    "Int8Weights",
    "MoEFeedForward",
    "MoEImplementation",
    "NormedMoEFeedForward",
    "PermutedTokens",
    "QuantizedRows",
    "add_rms_norm",
    "add_rms_norm_int8",
    "compress_rows",
    "compute_experts",
    "gate_and_sort",
    "gelu_compress",
    "gelu_compressed_backward",
    "int8_linear",
    "permute_tokens",
    "quantize_rows",
    "quantize_weights",
    "restore_rows",
    "unpermute",
    "build_plan",
    "grouped_weighted_scatter_add",
    "invert_scatter_index",
    "prepare_grouped_metadata",
    "prepare_metadata_and_plan",
    "weighted_scatter_add",
]
