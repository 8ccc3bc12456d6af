"""Operators of an encoder layer around the MAM layers: layer norm, dropout whose mask is never stored, their join between a layer's
halves, and differential attention.  No upstream names (the reference's ViT example takes these parts from its model library,
examples/vitb16_imagenet1k/utils.py)."""
from .norm import layer_norm, add_dropout_layer_norm
from .dropout import dropout
from .attention import diff_attention

__all__ = ["layer_norm", "add_dropout_layer_norm", "dropout", "diff_attention"]
