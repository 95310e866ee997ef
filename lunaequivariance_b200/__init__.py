"""B200-native UVU TensorProductConv hot path (sm_100a CUDA behind a C-ABI) with the reference's Python surface.

Public names follow HPC-AI-Team/LunaEquivariance (``src/__init__.py:3-45``) for the path this library covers:
``TensorProductConv``, ``TensorProduct`` / ``tensor_product`` (uvu), ``TensorProductConfig``, ``make_graph`` / ``LunaTPGraph``, ``prepare_tensor_product``,
``tensor_product_conv``, ``SphericalHarmonics`` / ``spherical_harmonics``, ``Irrep`` / ``Irreps`` and the ``o3``
namespace.  Beside them stand the operators of attention over a node's neighbours: ``LayerNorm`` / ``layer_norm`` over irreps,
``RelativeBias`` / ``relative_bias`` / ``distance_buckets`` (a learned bias by distance) and ``graph_softmax``.  ``HostStreamedConv`` (per-edge tensors streamed from host memory) and the ``sharded`` module (graphs
partitioned over GPUs) have no counterpart there.
"""

from . import o3
from .conv import LunaTPUVUConv, create_uvu_conv_operator
from .functional import prepare_tensor_product, tensor_product, tensor_product_conv
from .graph import LunaTPGraph, make_graph
from .graph_softmax import graph_softmax
from .irreps import Irrep, Irreps
from .layer_norm import LayerNormConfig, layer_norm
from .modules import LayerNorm, LunaEqSphericalHarmonics, RelativeBias, SphericalHarmonics, TensorProduct, TensorProductConv
from .relative_bias import distance_buckets, relative_bias
from .streaming import HostStreamedConv
from .tensor_product import LunaTPUVU
from .paths import Instruction, TensorProductConfig, TensorProductPaths, build_uvu_conv_metadata
from .spherical_harmonics import spherical_harmonics

__all__ = [
    "TensorProductConv", "TensorProduct", "tensor_product", "LunaTPUVU", "TensorProductConfig", "TensorProductPaths", "Instruction", "build_uvu_conv_metadata",
    "LunaTPGraph", "make_graph", "prepare_tensor_product", "tensor_product_conv", "LunaTPUVUConv",
    "create_uvu_conv_operator", "SphericalHarmonics", "LunaEqSphericalHarmonics", "spherical_harmonics",
    "Irrep", "Irreps", "o3", "HostStreamedConv",
    "LayerNorm", "LayerNormConfig", "layer_norm", "RelativeBias", "relative_bias", "distance_buckets", "graph_softmax",
]
