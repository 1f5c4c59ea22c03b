from . import conv
from .attention import AttentionSegments, sparse_attention
from .conv import build_out_coords, compute_neighbor_indices, sparse_conv3d, sparse_conv3d_fused
from .norm import sparse_batch_norm, sparse_batch_norm_act, sparse_layer_norm
from .rotary import RotaryAxes, sparse_rotary
from .spatial import sparse_pooling, sparse_upsample

__all__ = ["conv", "sparse_conv3d", "sparse_conv3d_fused", "compute_neighbor_indices", "build_out_coords", "sparse_batch_norm",
           "sparse_batch_norm_act", "sparse_layer_norm", "RotaryAxes", "sparse_rotary", "AttentionSegments", "sparse_attention", "sparse_pooling", "sparse_upsample"]
