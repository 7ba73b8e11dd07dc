"""Layer norm on this library's kernels (``dcn_layer_norm_forward`` / ``dcn_layer_norm_backward``):
``layer_norm`` with the arguments of ``torch.nn.functional.layer_norm`` and ``LayerNorm`` with those of
``torch.nn.LayerNorm`` (the 'LN' layer of mmcv/cnn/bricks/norm.py).  There is no CPU path.
"""
import numbers

import torch
import torch.nn as nn

from .. import _layers


def layer_norm(input, normalized_shape, weight=None, bias=None, eps=1e-5):
    """Layer norm of ``input`` over its last ``len(normalized_shape)`` dimensions, statistics in fp32.
    input float32, bfloat16 or float16 on a CUDA device; weight and bias of shape normalized_shape,
    both of input's type or both float32, or None.  The result has input's type; under autocast it
    is float32, as ``torch.nn.functional.layer_norm`` has it there.  Second derivatives,
    forward-mode differentiation and tracing are refused."""
    if isinstance(normalized_shape, numbers.Integral):
        normalized_shape = (int(normalized_shape),)
    if torch.is_autocast_enabled('cuda'):
        input, weight, bias = (_layers.autocast(t, torch.float32) for t in (input, weight, bias))
    return _layers.native.layer_norm(input, normalized_shape, weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` (same arguments, parameters and state) whose forward is ``layer_norm``."""

    def forward(self, input):
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
