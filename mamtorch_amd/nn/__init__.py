"""``FullyConnected`` is the MAM layer (mamtorch/nn/__init__.py:6 exports the v4 module); ``encoder``
has the rest of an encoder layer; ``convert``
holds the model-surgery helpers of the reference's ViT example; ``v1`` / ``v4`` are the reference's
sub-package names (mamtorch/nn/__init__.py:1-4)."""
from .fullyconnected import FullyConnected
from .convert import MAMMlp, add_mam_to_model, get_layers
from .legacy import FullyConnectedV1, MAMDense
from .conv import MAMConv1d, MAMConv2d
from .encoder import LayerNorm, Dropout, DiffAttention, DiffAttentionCache, MAMEncoderLayer
from . import compat, v1, v4

__all__ = ["FullyConnected", "MAMMlp", "add_mam_to_model", "get_layers", "FullyConnectedV1", "MAMDense", "MAMConv1d", "MAMConv2d", "LayerNorm", "Dropout", "DiffAttention",
           "DiffAttentionCache", "MAMEncoderLayer", "compat", "v1", "v4"]
