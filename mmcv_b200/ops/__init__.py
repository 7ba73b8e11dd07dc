"""The deformable-convolution names of ``mmcv.ops`` and their sibling sampler (reference:
mmcv/ops/__init__.py), and the operators of the transformer layer around that sampler."""
from .deform_conv import DeformConv2d, DeformConv2dFunction, DeformConv2dPack, deform_conv2d
from .deformable_encoder_layer import DeformableEncoderLayer
from .fused_linear import FFN, FusedLinear, feed_forward, fused_linear
from .layer_norm import LayerNorm, layer_norm
from .modulated_deform_conv import (ModulatedDeformConv2d, ModulatedDeformConv2dFunction,
                                    ModulatedDeformConv2dPack, modulated_deform_conv2d)
from .multi_scale_deform_attn import (MultiScaleDeformableAttention,
                                      MultiScaleDeformableAttnFunction)
from .saconv import SAConv2d

__all__ = ['DeformConv2d', 'DeformConv2dFunction', 'DeformConv2dPack', 'deform_conv2d',
           'ModulatedDeformConv2d', 'ModulatedDeformConv2dFunction',
           'ModulatedDeformConv2dPack', 'modulated_deform_conv2d', 'SAConv2d',
           'MultiScaleDeformableAttention', 'MultiScaleDeformableAttnFunction',
           'DeformableEncoderLayer', 'FFN', 'FusedLinear', 'LayerNorm', 'feed_forward', 'fused_linear',
           'layer_norm']
