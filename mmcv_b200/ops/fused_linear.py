"""Matrix product with bias, activation and residual in its epilogue (``fused_linear``,
``FusedLinear``) and the pair of two such products that makes a transformer layer's feed-forward
block (``feed_forward``, ``FFN``), on this library's kernels (``dcn_linear_forward`` /
``dcn_linear_backward``).

``FFN`` follows the layer of that name in mmcv/cnn/bricks/transformer.py: the same constructor
arguments (of the two-layer form with ReLU or GELU), parameter names and arithmetic.  There is no CPU
path: CPU tensors raise ``RuntimeError``.
"""
import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from .. import _layers, _lib
from .modulated_deform_conv import register_layer


class FusedLinearFunction(Function):

    @staticmethod
    def forward(ctx, input, weight, bias, residual, activation):
        """activation is a DCN_ACT_* code; shapes and types have been checked by fused_linear."""
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        y, saved = _layers.linear_forward(input, weight, bias, residual, activation,
                                          need_x or need_w or need_b)
        ctx.activation = activation
        ctx.x_shape = input.shape
        ctx.save_for_backward(input if need_w else None, weight if need_x or not need_w else None, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, weight, saved = ctx.saved_tensors
        want = ctx.needs_input_grad
        gx = gw = gb = None
        if want[0] or want[1] or want[2]:
            gx, gw, gb = _layers.linear_backward(grad_output, input, weight, saved, ctx.activation,
                                                 want[:3], x_shape=ctx.x_shape)
        return gx, gw, gb, (grad_output if want[3] else None), None


def _check_linear(op, input, weight, bias, names=('weight', 'bias')):
    _layers.dtype_code(op, input.dtype)
    if not input.is_cuda:
        raise RuntimeError(f'dcn_b200: {op}: input must be a CUDA tensor (this build has no CPU '
                           'implementation)')
    _layers.require(op, input.dtype, input.device, **{names[0]: weight, names[1]: bias})
    if weight.dim() != 2 or input.dim() < 1 or input.shape[-1] != weight.shape[1]:
        raise RuntimeError(f'dcn_b200: {op}: {names[0]} has shape {tuple(weight.shape)}, which does not '
                           f'fit input {tuple(input.shape)} (expected [out, {input.shape[-1] if input.dim() else 1}])')
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise RuntimeError(f'dcn_b200: {op}: {names[0]} must not be empty')
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise RuntimeError(f'dcn_b200: {op}: {names[1]} has shape {tuple(bias.shape)}, expected '
                           f'({weight.shape[0]},)')


def _check_residual(op, input, cout, residual):
    shape = input.shape[:-1] + (cout,)
    _layers.require(op, input.dtype, input.device, residual=residual)
    if residual.shape != shape:
        residual = residual.expand(shape)   # its gradient is summed where it was broadcast
    return residual


def fused_linear(input, weight, bias=None, residual=None, activation=None):
    """``act(input @ weight.T + bias) + residual`` as one kernel; the gradients of input, weight and
    bias are this library's products too.

    input (..., in), weight (out, in), bias (out,) or None, residual broadcastable to (..., out) or
    None, all of one type (float32, bfloat16 or float16) on one CUDA device; activation None,
    'relu' or 'gelu' (the exact form).  Everything is accumulated in fp32 and rounded once.  Under
    autocast, input, weight and bias are cast as ``torch.nn.functional.linear`` casts them, and a
    residual of another type is added outside the kernel."""
    act = _layers.activation_code(activation)
    dt = _layers.autocast_dtype()
    if dt is not None:
        input, weight, bias = input.to(dt), _layers.cast_weight(weight, dt), _layers.cast_weight(bias, dt)
        if residual is not None and residual.dtype != dt:
            return fused_linear(input, weight, bias, None, activation) + residual
    _check_linear('fused_linear', input, weight, bias)
    if residual is not None:
        residual = _check_residual('fused_linear', input, weight.shape[0], residual)
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return FusedLinearFunction.apply(input, weight, bias, residual, act)
    return _layers.linear_forward(input, weight, bias, residual, act, False)[0]


class FeedForwardFunction(Function):
    """Two products back to back.  The gradient between them passes the activation's derivative in
    the epilogue of the product that computes it, so that no separate pass reads or writes it."""

    @staticmethod
    def forward(ctx, input, weight1, bias1, weight2, bias2, residual, activation, identity):
        """identity: the residual is the input itself (residual is None then)."""
        need = ctx.needs_input_grad
        inner = need[0] or need[1] or need[2]
        h, saved = _layers.linear_forward(input, weight1, bias1, None, activation, inner)
        y, _ = _layers.linear_forward(h, weight2, bias2, input if identity else residual, _lib.ACT_NONE, False)
        ctx.activation, ctx.identity, ctx.inner = activation, identity, inner
        ctx.save_for_backward(input, weight1, weight2, h if need[3] else None, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, weight1, weight2, h, saved = ctx.saved_tensors
        want = ctx.needs_input_grad
        gz, gw2, gb2 = _layers.linear_backward(
            grad_output, h, weight2, None, _lib.ACT_NONE, (ctx.inner, want[3], want[4]), in_saved=saved,
            in_act=ctx.activation, x_shape=input.shape[:-1] + (weight1.shape[0],))
        gx = gw1 = gb1 = None
        if ctx.inner:
            gx, gw1, gb1 = _layers.linear_backward(
                gz, input, weight1, None, _lib.ACT_NONE, want[:3],
                gx_add=grad_output if ctx.identity and want[0] else None, x_shape=input.shape)
        return gx, gw1, gb1, gw2, gb2, (grad_output if want[5] else None), None, None


def feed_forward(input, weight1, bias1, weight2, bias2, residual=None, activation='relu'):
    """``act(input @ weight1.T + bias1) @ weight2.T + bias2 + residual``: the feed-forward block of a
    transformer layer.  weight1 (hidden, in), weight2 (out, hidden); the biases may be None; types,
    devices, activations and autocast as for ``fused_linear``.  The hidden activations are kept in
    the tensors' type.  Pass the input itself as residual (the usual identity) and its two gradients
    come out of one kernel, already added."""
    act = _layers.activation_code(activation)
    dt = _layers.autocast_dtype()
    if dt is not None:
        same = residual is input
        input = input.to(dt)
        weight1, bias1, weight2, bias2 = (_layers.cast_weight(t, dt) for t in (weight1, bias1, weight2, bias2))
        if residual is not None and residual.dtype != dt:
            return feed_forward(input, weight1, bias1, weight2, bias2, None, activation) + residual
        if same:
            residual = input
    op = 'feed_forward'
    _check_linear(op, input, weight1, bias1, ('weight1', 'bias1'))
    _layers.require(op, input.dtype, input.device, weight2=weight2, bias2=bias2)
    if weight2.dim() != 2 or weight2.shape[1] != weight1.shape[0] or weight2.shape[0] == 0:
        raise RuntimeError(f'dcn_b200: {op}: weight2 has shape {tuple(weight2.shape)}, expected '
                           f'[out, {weight1.shape[0]}]')
    if bias2 is not None and tuple(bias2.shape) != (weight2.shape[0],):
        raise RuntimeError(f'dcn_b200: {op}: bias2 has shape {tuple(bias2.shape)}, expected '
                           f'({weight2.shape[0]},)')
    identity = residual is input and weight2.shape[0] == input.shape[-1]
    if residual is not None and not identity:
        residual = _check_residual(op, input, weight2.shape[0], residual)
    tensors = (input, weight1, bias1, weight2, bias2, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return FeedForwardFunction.apply(input, weight1, bias1, weight2, bias2, None if identity else residual, act,
                                         identity)
    h = _layers.linear_forward(input, weight1, bias1, None, act, False)[0]
    return _layers.linear_forward(h, weight2, bias2, residual, _lib.ACT_NONE, False)[0]


class FusedLinear(nn.Linear):
    """``nn.Linear`` whose forward is ``fused_linear``; ``activation`` is part of the layer, the
    residual an argument of the call."""

    def __init__(self, in_features, out_features, bias=True, activation=None, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        _layers.activation_code(activation)
        self.activation = activation

    def forward(self, input, residual=None):
        return fused_linear(input, self.weight, self.bias, residual, self.activation)

    def extra_repr(self):
        return f'{super().extra_repr()}, activation={self.activation!r}'


class FFN(nn.Module):
    """Feed-forward block with identity: Linear, activation, Dropout, Linear, Dropout, and the
    dropout of the residual branch (mmcv/cnn/bricks/transformer.py, class FFN; parameter names
    ``layers.0.0.*`` and ``layers.1.*``).  While no dropout is active the whole block is
    ``feed_forward``; with an active dropout the two products are ``fused_linear`` around it."""

    def __init__(self, embed_dims=256, feedforward_channels=1024, num_fcs=2, act_cfg=None, ffn_drop=0.,
                 dropout_layer=None, add_identity=True, init_cfg=None):
        super().__init__()
        if num_fcs != 2:
            raise ValueError(f'FFN is built for num_fcs=2, but got {num_fcs}')
        kind = (act_cfg or dict(type='ReLU')).get('type')
        if kind not in ('ReLU', 'GELU'):
            raise ValueError(f"FFN takes act_cfg of type 'ReLU' or 'GELU', but got {kind!r}")
        if dropout_layer is not None and dropout_layer.get('type') != 'Dropout':
            raise ValueError(f"FFN takes a dropout_layer of type 'Dropout', but got {dropout_layer!r}")
        self.embed_dims = embed_dims
        self.feedforward_channels = feedforward_channels
        self.num_fcs = num_fcs
        self.init_cfg = init_cfg
        self.add_identity = add_identity
        self.activation = kind.lower()
        act = nn.ReLU() if kind == 'ReLU' else nn.GELU()
        self.layers = nn.Sequential(
            nn.Sequential(nn.Linear(embed_dims, feedforward_channels), act, nn.Dropout(ffn_drop)),
            nn.Linear(feedforward_channels, embed_dims), nn.Dropout(ffn_drop))
        self.dropout_layer = (nn.Dropout(dropout_layer.get('drop_prob', 0.5)) if dropout_layer
                              else nn.Identity())

    def forward(self, x, identity=None):
        fc1, _, drop1 = self.layers[0]
        fc2, drop2 = self.layers[1], self.layers[2]
        if self.add_identity and identity is None:
            identity = x
        if not self.add_identity:
            identity = None
        p_out = getattr(self.dropout_layer, 'p', 0.)
        if not self.training or (drop1.p == 0 and drop2.p == 0 and p_out == 0):
            return feed_forward(x, fc1.weight, fc1.bias, fc2.weight, fc2.bias, identity, self.activation)
        h = drop1(fused_linear(x, fc1.weight, fc1.bias, None, self.activation))
        out = self.dropout_layer(drop2(fused_linear(h, fc2.weight, fc2.bias)))
        return out if identity is None else identity + out


register_layer('FFN', FFN)
