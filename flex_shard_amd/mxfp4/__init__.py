from .mxfp4_linear import (
    FlexShardMxFp4Linear,
    convert_to_flex_shard_mxfp4_linear,
    mxfp4_expert_linear,
    mxfp4_linear,
)
from .mxfp4_matrix import (
    MxFp4Matrix,
    MxFp4Weight,
    mxfp4_quantize,
    mxfp4_quantize_both,
    mxfp4_quantize_transposed,
    quantize_mxfp4_weight,
)

__all__ = [
    "FlexShardMxFp4Linear", "MxFp4Matrix", "MxFp4Weight", "convert_to_flex_shard_mxfp4_linear", "mxfp4_expert_linear",
    "mxfp4_linear", "mxfp4_quantize", "mxfp4_quantize_both", "mxfp4_quantize_transposed", "quantize_mxfp4_weight",
]
