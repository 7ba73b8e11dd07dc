"""One post-norm encoder layer of Deformable DETR on this library's operators: multi-scale deformable
self-attention with its identity, layer norm, feed-forward block with its identity, layer norm (the
operation order 'self_attn', 'norm', 'ffn', 'norm' of mmcv/cnn/bricks/transformer.py,
BaseTransformerLayer).
"""
import torch.nn as nn

from .fused_linear import FFN
from .layer_norm import LayerNorm
from .multi_scale_deform_attn import MultiScaleDeformableAttention


class DeformableEncoderLayer(nn.Module):
    """``attentions.0``, ``ffns.0`` and ``norms.0`` / ``norms.1`` are the names under which the
    reference's layer of this operation order keeps its parameters."""

    def __init__(self, embed_dims=256, num_heads=8, num_levels=4, num_points=4, feedforward_channels=1024,
                 attn_drop=0., ffn_drop=0., act_cfg=None, batch_first=True, im2col_step=64):
        super().__init__()
        self.embed_dims = embed_dims
        self.batch_first = batch_first
        self.attentions = nn.ModuleList([MultiScaleDeformableAttention(
            embed_dims=embed_dims, num_heads=num_heads, num_levels=num_levels, num_points=num_points,
            im2col_step=im2col_step, dropout=attn_drop, batch_first=batch_first, fused_proj=True)])
        self.ffns = nn.ModuleList([FFN(embed_dims, feedforward_channels, act_cfg=act_cfg, ffn_drop=ffn_drop)])
        self.norms = nn.ModuleList([LayerNorm(embed_dims), LayerNorm(embed_dims)])

    def forward(self, query, query_pos=None, key_padding_mask=None, reference_points=None, spatial_shapes=None,
                level_start_index=None, **kwargs):
        x = self.attentions[0](query, query_pos=query_pos, key_padding_mask=key_padding_mask,
                               reference_points=reference_points, spatial_shapes=spatial_shapes,
                               level_start_index=level_start_index, **kwargs)
        x = self.norms[0](x)
        x = self.ffns[0](x)
        return self.norms[1](x)
