"""nnue_pytorch_b200: sm_100a kernels for the sparse feature-transformer hot
path of nnue-pytorch, behind the reference's own operator interface."""

from .composed_feature_transformer import ComposedFeatureTransformer
from .double_ft_functions import double_feature_transform
from .fp8_functions import Fp8Blocks, linear_fp8, quantize_fp8_rows, quantize_fp8_tiles
from .fused_ft_functions import FusedDoubleFtFunction
from .grouped_linear_functions import GroupedLinearFunction, GroupPlan, grouped_linear
from .sparse_linear_functions import SparseLinearFunction

__all__ = [
    "ComposedFeatureTransformer",
    "Fp8Blocks",
    "FusedDoubleFtFunction",
    "GroupPlan",
    "GroupedLinearFunction",
    "SparseLinearFunction",
    "double_feature_transform",
    "grouped_linear",
    "linear_fp8",
    "quantize_fp8_rows",
    "quantize_fp8_tiles",
]
