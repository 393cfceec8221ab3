"""B200-native (sm_100a) complex-valued Conv2d for PyTorch.

Drop-in for the ``complex_conv2d`` package of cutlass-complex-conv
(``complex_conv2d/__init__.py:3-5``): the public object is ``ComplexConv2d``.
Beyond it: operators on the rows of features its planes hold (``token_ops``).
"""

from .modules import ComplexConv2d
from .token_ops import (Dropout, GatedFeedForward, LayerNorm, dropout, gated_feed_forward,
                        gated_feed_forward_backward, gated_feed_forward_with_saved, layer_norm,
                        layer_norm_backward, layer_norm_with_stats)

__all__ = [
    "ComplexConv2d",
    "layer_norm", "layer_norm_with_stats", "layer_norm_backward",
    "gated_feed_forward", "gated_feed_forward_with_saved", "gated_feed_forward_backward",
    "dropout", "LayerNorm", "GatedFeedForward", "Dropout",
]
