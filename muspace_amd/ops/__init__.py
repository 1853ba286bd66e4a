"""Canonical operator exports (the MSDA path of /root/reference/mu_space/ops/__init__.py:24-28)."""

from .multi_scale_deformable_attn import (
    explain_dispatch,
    level_start_index_from_shapes,
    multi_scale_deformable_attn,
    multi_scale_deformable_attn_pytorch,
    multi_scale_deformable_attn_pytorch_compat,
)
from .scatter_div import multi_scale_deformable_attn_scatter_div
from .msda_softmax import attention_softmax, multi_scale_deformable_attn_softmax
from .deformable_aggregation import (
    deformable_aggregation,
    deformable_aggregation_function,
    deformable_aggregation_reference,
    feature_maps_format,
)
from .dropout import dropout, dropout_pytorch
from .gated_linear import gated_linear, gated_linear_pytorch
from .layer_norm import layer_norm, layer_norm_pytorch
from .linear import checkpoint_int8, checkpoint_restore, linear, linear_pytorch
from .linear_int8 import (
    linear_int8,
    linear_int8_pytorch,
    quantize_int8,
    quantize_int8_pytorch,
)
from .residual_norm import residual_norm, residual_norm_pytorch

__all__ = [
    "attention_softmax",
    "checkpoint_int8",
    "checkpoint_restore",
    "deformable_aggregation",
    "deformable_aggregation_function",
    "deformable_aggregation_reference",
    "dropout",
    "dropout_pytorch",
    "feature_maps_format",
    "explain_dispatch",
    "gated_linear",
    "gated_linear_pytorch",
    "layer_norm",
    "layer_norm_pytorch",
    "level_start_index_from_shapes",
    "linear",
    "linear_int8",
    "linear_int8_pytorch",
    "linear_pytorch",
    "multi_scale_deformable_attn",
    "multi_scale_deformable_attn_pytorch",
    "multi_scale_deformable_attn_pytorch_compat",
    "multi_scale_deformable_attn_scatter_div",
    "multi_scale_deformable_attn_softmax",
    "quantize_int8",
    "quantize_int8_pytorch",
    "residual_norm",
    "residual_norm_pytorch",
]
