"""Layer norm on this library's kernels (``dcn_layer_norm_forward`` / ``dcn_layer_norm_backward``):
``layer_norm`` with the arguments of ``torch.nn.functional.layer_norm`` and ``LayerNorm`` with those of
``torch.nn.LayerNorm`` (the 'LN' layer of mmcv/cnn/bricks/norm.py).  There is no CPU path.
"""
import numbers

import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from .. import _layers


class LayerNormFunction(Function):

    @staticmethod
    def forward(ctx, input, weight, bias, cols, eps):
        """Arguments checked by layer_norm; weight and bias are contiguous or None."""
        y, stats = _layers.norm_forward(input, weight, bias, cols, eps, True)
        p = weight if weight is not None else bias
        ctx.cols = cols
        ctx.param_dtype = input.dtype if p is None else p.dtype
        ctx.param_shape = None if p is None else p.shape
        ctx.save_for_backward(input, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, weight, stats = ctx.saved_tensors
        gx, gw, gb = _layers.norm_backward(grad_output, input, weight, stats, ctx.cols, ctx.needs_input_grad[:3],
                                           ctx.param_dtype)
        return (gx, None if gw is None else gw.view(ctx.param_shape),
                None if gb is None else gb.view(ctx.param_shape), None, None)


def layer_norm(input, normalized_shape, weight=None, bias=None, eps=1e-5):
    """Layer norm of ``input`` over its last ``len(normalized_shape)`` dimensions, statistics in fp32.
    input float32, bfloat16 or float16 on a CUDA device; weight and bias of shape normalized_shape,
    both of input's type or both float32, or None.  The result has input's type; under autocast it
    is float32, as ``torch.nn.functional.layer_norm`` has it there."""
    if isinstance(normalized_shape, numbers.Integral):
        normalized_shape = (int(normalized_shape),)
    shape = tuple(normalized_shape)
    if torch.is_autocast_enabled('cuda'):
        input = input.float()
        weight = None if weight is None else weight.float()
        bias = None if bias is None else bias.float()
    op = 'layer_norm'
    _layers.dtype_code(op, input.dtype)
    if not input.is_cuda:
        raise RuntimeError(f'dcn_b200: {op}: input must be a CUDA tensor (this build has no CPU '
                           'implementation)')
    if not shape or tuple(input.shape[input.dim() - len(shape):]) != shape or input.dim() < len(shape):
        raise RuntimeError(f'dcn_b200: {op}: input of shape {tuple(input.shape)} does not end in '
                           f'normalized_shape {shape}')
    cols = 1
    for n in shape:
        cols *= n
    if cols == 0:
        raise RuntimeError(f'dcn_b200: {op}: normalized_shape {shape} has no elements')
    for name, p in (('weight', weight), ('bias', bias)):
        if p is None:
            continue
        if tuple(p.shape) != shape:
            raise RuntimeError(f'dcn_b200: {op}: {name} has shape {tuple(p.shape)}, expected {shape}')
        if p.dtype != input.dtype and p.dtype != torch.float32:
            raise RuntimeError(f'dcn_b200: {op}: {name} has dtype {p.dtype}, expected {input.dtype} or float32')
        if not p.is_cuda or p.device != input.device:
            raise RuntimeError(f'dcn_b200: {op}: {name} is on {p.device}, expected {input.device}')
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f'dcn_b200: {op}: weight has dtype {weight.dtype}, bias {bias.dtype}')
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (input.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return LayerNormFunction.apply(input, weight, bias, cols, float(eps))
    return _layers.norm_forward(input, weight, bias, cols, float(eps), False)[0]


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` (same arguments, parameters and state) whose forward is ``layer_norm``."""

    def forward(self, input):
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
