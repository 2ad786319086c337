"""Canonical operator exports of the B200 build: the MSDA operator, the fused
spatial-cross-attention scatter built on it, FlashSCA, SparseDrive's deformable
aggregation, and the layer around them: the linear product with its epilogue, the gated
feed-forward product, layer norm, norms with their residual, dropout and 8-bit
activation checkpoints."""

from .checkpoint8 import Checkpoint8, checkpoint_pack, checkpoint_unpack
from .deformable_aggregation import (
    deformable_aggregation,
    deformable_aggregation_function,
    feature_maps_format,
)
from .dropout import dropout
from .multi_scale_deformable_attn import (
    explain_dispatch,
    multi_scale_deformable_attn,
    multi_scale_deformable_attn_pytorch_compat,
)
from .flash_sca import flash_bevpool_sca
from .gated_linear import gated_linear
from .layer_norm import layer_norm
from .linear_act import linear_act
from .residual_norm import add_norm, norm_add
from .sca_scatter import ms_deform_attn_scatter_div, sca_rebatch_scatter

__all__ = [
    "Checkpoint8",
    "add_norm",
    "checkpoint_pack",
    "checkpoint_unpack",
    "deformable_aggregation",
    "deformable_aggregation_function",
    "dropout",
    "explain_dispatch",
    "feature_maps_format",
    "flash_bevpool_sca",
    "gated_linear",
    "layer_norm",
    "linear_act",
    "ms_deform_attn_scatter_div",
    "multi_scale_deformable_attn",
    "multi_scale_deformable_attn_pytorch_compat",
    "norm_add",
    "sca_rebatch_scatter",
]
