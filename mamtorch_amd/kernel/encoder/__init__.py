"""Operators of an encoder layer around the MAM layers: layer norm, dropout whose mask is never stored, their join between a layer's
halves, differential attention, norms of its queries and keys with the position rotation, and its cache in pages: their bookkeeping, trees of drafted
tokens, attention over them.  No upstream names (the reference's ViT example takes these parts from its model library,
examples/vitb16_imagenet1k/utils.py)."""
from .norm import layer_norm, add_dropout_layer_norm
from .dropout import dropout
from .attention import diff_attention
from .rotary import rotary_frequencies, norm_rotate
from .pages import (pages_extend, pages_fork, pages_trim, pages_copy, pages_compact, draft_tree, norm_rotate_append,
                    diff_attention_pages)

__all__ = ["layer_norm", "add_dropout_layer_norm", "dropout", "diff_attention", "rotary_frequencies", "norm_rotate", "pages_extend", "pages_fork",
           "pages_trim", "pages_copy", "pages_compact", "draft_tree", "norm_rotate_append", "diff_attention_pages"]
