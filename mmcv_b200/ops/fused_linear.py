"""Matrix product with bias, activation and residual in its epilogue (``fused_linear``,
``FusedLinear``) and the pair of two such products that makes a transformer layer's feed-forward
block (``feed_forward``, ``FFN``), on this library's kernels (``dcn_linear_forward`` /
``dcn_linear_backward``).

``FFN`` follows the layer of that name in mmcv/cnn/bricks/transformer.py: the same constructor
arguments (of the two-layer form with ReLU or GELU), parameter names and arithmetic.  There is no CPU
path: CPU tensors raise ``RuntimeError``.
"""
import torch.nn as nn

from .. import _layers


def fused_linear(input, weight, bias=None, residual=None, activation=None):
    """``act(input @ weight.T + bias) + residual`` as one kernel; the gradients of input, weight and
    bias are this library's products too.

    input (..., in), weight (out, in), bias (out,) or None, residual broadcastable to (..., out) or
    None, all of one type (float32, bfloat16 or float16) on one CUDA device; activation None,
    'relu' or 'gelu' (the exact form).  Everything is accumulated in fp32 and rounded once.  Under
    autocast, input, weight and bias are cast as ``torch.nn.functional.linear`` casts them, and a
    residual of another type is added outside the kernel.  Second derivatives, forward-mode
    differentiation and tracing (torch.jit.trace, make_fx, torch.export) are refused; torch.compile runs
    the call as it is, between two graphs."""
    act = _layers.activation_code(activation)
    dt = _layers.autocast_dtype()
    if dt is not None:
        input = _layers.autocast(input, dt)
        weight, bias = _layers.autocast_weight(weight, dt), _layers.autocast_weight(bias, dt)
        if residual is not None and residual.dtype != dt:
            return fused_linear(input, weight, bias, None, activation) + residual
    return _layers.native.fused_linear(input, weight, bias, residual, act)


def feed_forward(input, weight1, bias1, weight2, bias2, residual=None, activation='relu'):
    """``act(input @ weight1.T + bias1) @ weight2.T + bias2 + residual``: the feed-forward block of a
    transformer layer.  weight1 (hidden, in), weight2 (out, hidden); the biases may be None; types,
    devices, activations, autocast and refusals as for ``fused_linear``.  The hidden activations are kept in
    the tensors' type.  The gradient between the two products passes the activation's derivative in
    the epilogue of the product that computes it, and is rounded to that type as well (bias1's
    gradient is summed before that rounding up to 2^22 hidden values, after it beyond).  Pass the input
    itself as residual (the usual identity) and its two gradients come out of one kernel, already added."""
    act = _layers.activation_code(activation)
    dt = _layers.autocast_dtype()
    if dt is not None:
        same = residual is input
        input = _layers.autocast(input, dt)
        weight1, bias1, weight2, bias2 = (_layers.autocast_weight(t, dt) for t in (weight1, bias1, weight2, bias2))
        if residual is not None and residual.dtype != dt:
            return feed_forward(input, weight1, bias1, weight2, bias2, None, activation) + residual
        if same:
            residual = input
    return _layers.native.feed_forward(input, weight1, bias1, weight2, bias2, residual, act)


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
    ``layers.0.0.*`` and ``layers.1.*``).  It takes a part of what that layer takes, so it does not stand
    under its registry name: configurations build the layer they always built.  init_cfg is kept and not
    acted upon.  While no dropout is active the whole block is
    ``feed_forward``; with an active dropout the two products are ``fused_linear`` around it.  Children
    that carry hooks, or were replaced or parametrized, are called as they are."""

    def __init__(self, embed_dims=256, feedforward_channels=1024, num_fcs=2, act_cfg=None, ffn_drop=0.,
                 dropout_layer=None, add_identity=True, init_cfg=None):
        super().__init__()
        if num_fcs != 2:
            raise ValueError(f'FFN is built for num_fcs=2, but got {num_fcs}')
        act_cfg = act_cfg or dict(type='ReLU')
        kind = act_cfg.get('type')
        if kind not in ('ReLU', 'GELU'):
            raise ValueError(f"FFN takes act_cfg of type 'ReLU' or 'GELU', but got {kind!r}")
        # in place or not is the kernels' own affair; whatever else would change the arithmetic
        if set(act_cfg) - {'type', 'inplace' if kind == 'ReLU' else 'approximate'} or \
                act_cfg.get('approximate', 'none') != 'none':
            raise ValueError(f'FFN has ReLU and the exact GELU without further options, but got {act_cfg!r}')
        if dropout_layer is not None and (dropout_layer.get('type') != 'Dropout' or
                                          set(dropout_layer) - {'type', 'drop_prob', 'inplace'}):
            raise ValueError("FFN takes a dropout_layer of type 'Dropout' with drop_prob, "
                             f'but got {dropout_layer!r}')
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

    def _as_built(self):
        """(fc1, dropout, fc2, dropout) while the children are those of the constructor, else None."""
        kind = nn.ReLU if self.activation == 'relu' else nn.GELU
        if type(self.layers) is not nn.Sequential or len(self.layers._modules) != 3:
            return None
        inner, fc2, drop2 = self.layers._modules.values()
        if type(inner) is not nn.Sequential or len(inner._modules) != 3:
            return None
        fc1, act, drop1 = inner._modules.values()
        if not _layers.untouched((self.layers, nn.Sequential), (inner, nn.Sequential), (fc1, nn.Linear), (act, kind),
                                 (fc2, nn.Linear)) or kind is nn.GELU and act.approximate != 'none':
            return None
        return fc1, drop1, fc2, drop2

    def forward(self, x, identity=None):
        if self.add_identity and identity is None:
            identity = x
        if not self.add_identity:
            identity = None
        parts = self._as_built()
        if parts is None:
            out = self.dropout_layer(self.layers(x))
            return out if identity is None else identity + out
        fc1, drop1, fc2, drop2 = parts
        if _layers.passes_on(drop1, drop2, self.dropout_layer):
            return feed_forward(x, fc1.weight, fc1.bias, fc2.weight, fc2.bias, identity, self.activation)
        h = drop1(fused_linear(x, fc1.weight, fc1.bias, None, self.activation))
        out = self.dropout_layer(drop2(fused_linear(h, fc2.weight, fc2.bias)))
        return out if identity is None else identity + out
