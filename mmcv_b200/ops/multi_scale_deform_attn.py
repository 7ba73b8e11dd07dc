"""``MultiScaleDeformableAttnFunction`` and ``MultiScaleDeformableAttention`` under the reference's
names and argument conventions (mmcv/ops/multi_scale_deform_attn.py:23-110, :172-384), on this
library's sampler kernels (``dcn_msda_forward`` / ``dcn_msda_backward``).

There is no CPU path here: the reference's pure-PyTorch function
``multi_scale_deformable_attn_pytorch`` (same file, :113-170) is restated under ``oracle/`` as a
checker only, and CPU tensors raise ``RuntimeError`` as they do for the deformable convolutions.
"""
import math
import warnings
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from .. import _ext as ext_module
from .. import _layers
from .fused_linear import fused_linear
from .modulated_deform_conv import register_layer


class MultiScaleDeformableAttnFunction(Function):

    @staticmethod
    def forward(ctx, value, value_spatial_shapes, value_level_start_index, sampling_locations,
                attention_weights, im2col_step):
        """value (bs, num_keys, num_heads, embed_dims // num_heads); value_spatial_shapes
        (num_levels, 2) as (h, w); sampling_locations (bs, num_queries, num_heads, num_levels,
        num_points, 2) as (x, y) in [0, 1]; attention_weights the same without the last axis.
        Returns (bs, num_queries, embed_dims)."""
        ctx.im2col_step = im2col_step
        # the flag for fp16 / autocast is value's dtype: the other two follow it
        # (mmcv/ops/multi_scale_deform_attn.py:53-63)
        sampling_locations = sampling_locations.type_as(value)
        attention_weights = attention_weights.type_as(value)
        output = ext_module.ms_deform_attn_forward(
            value, value_spatial_shapes, value_level_start_index, sampling_locations,
            attention_weights, im2col_step=ctx.im2col_step)
        ctx.save_for_backward(value, value_spatial_shapes, value_level_start_index,
                              sampling_locations, attention_weights)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        value, value_spatial_shapes, value_level_start_index, sampling_locations, \
            attention_weights = ctx.saved_tensors
        grad_value = torch.zeros_like(value)
        grad_sampling_loc = torch.zeros_like(sampling_locations)
        grad_attn_weight = torch.zeros_like(attention_weights)
        ext_module.ms_deform_attn_backward(
            value, value_spatial_shapes, value_level_start_index, sampling_locations,
            attention_weights, grad_output.contiguous(), grad_value, grad_sampling_loc,
            grad_attn_weight, im2col_step=ctx.im2col_step)
        return grad_value, None, None, grad_sampling_loc, grad_attn_weight, None


def _is_power_of_2(n):
    if (not isinstance(n, int)) or (n < 0):
        raise ValueError(f'invalid input for _is_power_of_2: {n} (type: {type(n)})')
    return (n & (n - 1) == 0) and n != 0


class MultiScaleDeformableAttention(nn.Module):
    """The attention module of Deformable DETR: same constructor arguments, parameters
    (``sampling_offsets``, ``attention_weights``, ``value_proj``, ``output_proj``), initialisation
    and forward arithmetic as the reference layer (mmcv/ops/multi_scale_deform_attn.py:172-384).

    fused_proj (not in the reference): the four projections run on this library's matrix product
    (``fused_linear``), the last one with the identity in its epilogue while no dropout is active.
    The sums are the same, rounded once where the default rounds twice.  A projection that carries hooks,
    or was replaced or parametrized, is called as it is."""

    def __init__(self, embed_dims: int = 256, num_heads: int = 8, num_levels: int = 4,
                 num_points: int = 4, im2col_step: int = 64, dropout: float = 0.1,
                 batch_first: bool = False, norm_cfg: Optional[dict] = None, init_cfg=None,
                 value_proj_ratio: float = 1.0, fused_proj: bool = False):
        super().__init__()
        if embed_dims % num_heads != 0:
            raise ValueError(f'embed_dims must be divisible by num_heads, '
                             f'but got {embed_dims} and {num_heads}')
        dim_per_head = embed_dims // num_heads
        self.norm_cfg = norm_cfg
        self.init_cfg = init_cfg
        self.dropout = nn.Dropout(dropout)
        self.batch_first = batch_first
        self.fused_proj = fused_proj
        if not _is_power_of_2(dim_per_head):
            warnings.warn("You'd better set embed_dims in MultiScaleDeformAttention to make the "
                          'dimension of each attention head a power of 2 which is more efficient '
                          'in the CUDA implementation.')
        self.im2col_step = im2col_step
        self.embed_dims = embed_dims
        self.num_levels = num_levels
        self.num_heads = num_heads
        self.num_points = num_points
        self.sampling_offsets = nn.Linear(embed_dims, num_heads * num_levels * num_points * 2)
        self.attention_weights = nn.Linear(embed_dims, num_heads * num_levels * num_points)
        value_proj_size = int(embed_dims * value_proj_ratio)
        self.value_proj = nn.Linear(embed_dims, value_proj_size)
        self.output_proj = nn.Linear(value_proj_size, embed_dims)
        self.init_weights()

    def init_weights(self) -> None:
        nn.init.constant_(self.sampling_offsets.weight, 0.)
        device = next(self.parameters()).device
        thetas = torch.arange(self.num_heads, dtype=torch.float32, device=device) * \
            (2.0 * math.pi / self.num_heads)
        grid_init = torch.stack([thetas.cos(), thetas.sin()], -1)
        grid_init = (grid_init / grid_init.abs().max(-1, keepdim=True)[0]).view(
            self.num_heads, 1, 1, 2).repeat(1, self.num_levels, self.num_points, 1)
        for i in range(self.num_points):
            grid_init[:, :, i, :] *= i + 1
        self.sampling_offsets.bias.data = grid_init.view(-1)
        nn.init.constant_(self.attention_weights.weight, 0.)
        nn.init.constant_(self.attention_weights.bias, 0.)
        nn.init.xavier_uniform_(self.value_proj.weight)
        nn.init.constant_(self.value_proj.bias, 0.)
        nn.init.xavier_uniform_(self.output_proj.weight)
        nn.init.constant_(self.output_proj.bias, 0.)
        self._is_init = True

    def _project(self, linear, x):
        if self.fused_proj and _layers.untouched((linear, nn.Linear)):
            return fused_linear(x, linear.weight, linear.bias)
        return linear(x)

    def forward(self, query, key=None, value=None, identity=None, query_pos=None,
                key_padding_mask=None, reference_points=None, spatial_shapes=None,
                level_start_index=None, **kwargs):
        if 'residual' in kwargs:        # the reference's deprecated name of `identity`
            identity = kwargs.pop('residual')
        if value is None:
            value = query
        if identity is None:
            identity = query
        if query_pos is not None:
            query = query + query_pos
        if not self.batch_first:
            query = query.permute(1, 0, 2)
            value = value.permute(1, 0, 2)
        bs, num_query, _ = query.shape
        bs, num_value, _ = value.shape
        assert (spatial_shapes[:, 0] * spatial_shapes[:, 1]).sum() == num_value

        value = self._project(self.value_proj, value)
        if key_padding_mask is not None:
            value = value.masked_fill(key_padding_mask[..., None], 0.0)
        value = value.view(bs, num_value, self.num_heads, -1)
        sampling_offsets = self._project(self.sampling_offsets, query).view(
            bs, num_query, self.num_heads, self.num_levels, self.num_points, 2)
        attention_weights = self._project(self.attention_weights, query).view(
            bs, num_query, self.num_heads, self.num_levels * self.num_points)
        attention_weights = attention_weights.softmax(-1)
        attention_weights = attention_weights.view(bs, num_query, self.num_heads,
                                                   self.num_levels, self.num_points)
        if reference_points.shape[-1] == 2:
            offset_normalizer = torch.stack([spatial_shapes[..., 1], spatial_shapes[..., 0]], -1)
            sampling_locations = reference_points[:, :, None, :, None, :] \
                + sampling_offsets / offset_normalizer[None, None, None, :, None, :]
        elif reference_points.shape[-1] == 4:
            sampling_locations = reference_points[:, :, None, :, None, :2] \
                + sampling_offsets / self.num_points * reference_points[:, :, None, :, None, 2:] * 0.5
        else:
            raise ValueError(f'Last dim of reference_points must be 2 or 4, but get '
                             f'{reference_points.shape[-1]} instead.')
        if not value.is_cuda:
            raise RuntimeError('mmcv_b200: multi-scale deformable attention has no CPU path '
                               '(value must be a CUDA tensor)')
        output = MultiScaleDeformableAttnFunction.apply(
            value.contiguous(), spatial_shapes, level_start_index, sampling_locations.contiguous(),
            attention_weights.contiguous(), self.im2col_step)
        if self.fused_proj and _layers.untouched((self.output_proj, nn.Linear)) and _layers.passes_on(self.dropout):
            if not self.batch_first:
                identity = identity.permute(1, 0, 2)
            output = fused_linear(output, self.output_proj.weight, self.output_proj.bias, identity)
            return output if self.batch_first else output.permute(1, 0, 2)
        output = self._project(self.output_proj, output)
        if not self.batch_first:
            output = output.permute(1, 0, 2)
        return self.dropout(output) + identity


register_layer('MultiScaleDeformableAttention', MultiScaleDeformableAttention)
