"""pack3d_b200: a Blackwell (sm_100a) backend for the PACK3D attention operator.

Drop-in for the reference ``pack3d`` package's operator path: the same layer
(``PACK3DAttention``), geometry (``build_layout``, ``prepare_geometry``,
``TokenLayout``) and operator (``pack3d_streamed``, ``rotate_projections``)
APIs, with every stage of the hot path in hand-written CUDA behind the C-ABI
library ``lib/libpack3d_b200.so``.  There is no CPU path: compute entry points
raise if the native library or a CUDA sm_100 device is missing.
"""
from .attention import PACK3DAttention
from .cache import PagedCache, paged_attention
from .feedforward import FeedForward
from .fp8 import Fp8Matrix, fp8_linear, fp8_matmul, quantize, quantize_weight
from .geometry import Pack3DGeometry, TokenLayout, build_layout, grid_coordinates, prepare_geometry
from .ops import pack3d_streamed
from .residual import NormSpec, dropout, norm, residual_norm
from .rope import balanced_pairs, rotate_projections
from .sequence import norm_rotate, sequence_attention
from .sequence_layer import SequenceAttention

__version__ = "0.1.0"
__all__ = ["FeedForward", "Fp8Matrix", "NormSpec", "PACK3DAttention", "Pack3DGeometry", "PagedCache",
           "SequenceAttention", "TokenLayout", "balanced_pairs", "build_layout", "dropout", "fp8_linear", "fp8_matmul",
           "grid_coordinates", "norm", "norm_rotate", "pack3d_streamed", "paged_attention", "prepare_geometry",
           "quantize", "quantize_weight", "residual_norm", "rotate_projections", "sequence_attention"]
