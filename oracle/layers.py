"""Plain 64-bit forms of the transformer-layer operators, with bounds on how far an implementation
that keeps sums in fp32 and rounds tensors to `dtype` may be from them, element by element.

u is half a step of the tensors' type (relative), acc(n) bounds the relative error, against the sum of
magnitudes, of a sum of n products in fp32: a chain of at most n / 16 + 24 additions of 2^-23 each
(sixteen products are added at a time; 2^-23, not 2^-24, because a tensor core truncates).
"""
import math

import torch

STEP32 = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half of the smallest subnormal: what a value near zero may lose to rounding."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def acc(n):
    return STEP32 * (n / 16 + 24)


def activation(z, act):
    """(value, first derivative, bound of the value's slope, bound of the derivative's slope)"""
    if act == 'relu':
        return z.clamp(min=0), (z > 0).double(), 1.0, 0.0
    if act == 'gelu':
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, 1.13, 0.8
    return z, torch.ones_like(z), 1.0, 0.0


class Value:
    """A tensor in 64 bits and how far an implementation may be from it."""

    def __init__(self, v, e=None):
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def rounded(self, dtype):
        return Value(self.v, self.e + half_step(dtype) * (self.v.abs() + self.e) + floor_of(dtype))

    def t(self):
        return Value(self.v.t(), self.e.t())


def product(a, b):
    """a b^T over the last dimension of both."""
    size = a.v.abs() @ b.v.abs().t()
    e = a.e @ b.v.abs().t() + a.v.abs() @ b.e.t() + a.e @ b.e.t()
    return Value(a.v @ b.v.t(), e + acc(a.v.shape[1]) * size)


def column_sum(a):
    return Value(a.v.sum(0), a.e.sum(0) + acc(a.v.shape[0]) * a.v.abs().sum(0))


def add(a, v):
    return Value(a.v + v, a.e + STEP32 * (a.v.abs() + v.abs()))


def apply(z, act):
    y, _, slope, _ = activation(z.v, act)
    extra = 2.0 ** -20 * z.v.abs() if act == 'gelu' else 0.0
    return Value(y, slope * z.e + extra)


def through(g, z, act, kept=None):
    """g * act'(z); `kept`: what the forward pass keeps for the derivative is bounded by z's rounding to that
    type."""
    _, d, _, curve = activation(z.v, act)
    ez = z.e if kept is None else z.rounded(kept).e
    if act == 'relu':
        return Value(g.v * d, g.e + (g.v.abs() + g.e) * (z.v.abs() <= z.e))
    if act == 'gelu':
        return Value(g.v * d, 1.13 * g.e + (g.v.abs() + g.e) * (curve * ez + 2.0 ** -19))
    return g


def linear(x, w, b, res, act, gy=None):
    """{'y', 'gx', 'gw', 'gb'} of act(x w^T + b) + res; tensors of one type, [rows, in] and [out, in]."""
    t = x.dtype
    X, W = Value(x), Value(w)
    z = product(X, W)
    if b is not None:
        z = add(z, b.double())
    y = apply(z, act)
    if res is not None:
        y = add(y, res.double())
    out = {'y': y.rounded(t)}
    if gy is not None:
        gz = Value(gy)
        if act is not None:
            gz = through(gz, z, act, kept=t).rounded(t)
        out['gx'] = product(gz, W.t()).rounded(t)
        out['gw'] = product(gz.t(), X.t()).rounded(t)
        out['gb'] = column_sum(gz).rounded(t)
    return out


def feed_forward(x, w1, b1, w2, b2, res, act, gy=None):
    t = x.dtype
    X, W1, W2 = Value(x), Value(w1), Value(w2)
    z = add(product(X, W1), b1.double())
    h = apply(z, act).rounded(t)
    y = add(product(h, W2), b2.double())
    if res is not None:
        y = add(y, res.double())
    out = {'y': y.rounded(t)}
    if gy is not None:
        G = Value(gy)
        out['gw2'] = product(G.t(), h.t()).rounded(t)
        out['gb2'] = column_sum(G).rounded(t)
        gz = through(product(G, W2.t()), z, act, kept=t).rounded(t)
        out['gx'] = product(gz, W1.t()).rounded(t)
        out['gw1'] = product(gz.t(), X.t()).rounded(t)
        out['gb1'] = column_sum(gz).rounded(t)
    return out


def layer_norm(x, w, b, eps, gy=None):
    """x [rows, cols].  A thread adds at most 32 (or cols / 1024) elements before the sums of the
    threads are joined in a tree: k additions, each within half a step of fp32."""
    t = x.dtype
    rows, cols = x.shape
    k = (48 + cols / 1024) * STEP32
    X = x.double()
    d = X - X.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    n = d * rstd
    en = k * (n.abs() + 1)
    W = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.double()
    B = torch.zeros(cols, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = Value(n * W + B, en * W.abs() + STEP32 * (n * W).abs() + STEP32 * B.abs())
    out = {'y': y.rounded(t)}
    if gy is not None:
        G = gy.double()
        g = G * W
        mg, mgn = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
        ag, agn = g.abs().mean(1, keepdim=True), (g.abs() * (n.abs() + en)).mean(1, keepdim=True)
        gx = rstd * (g - mg - n * mgn)
        e = rstd * (4 * k * (g.abs() + ag + (n.abs() + 1) * agn) + n.abs() * (g.abs() * en).mean(1, keepdim=True))
        out['gx'] = Value(gx, e).rounded(t)
        p = x.dtype if w is None else w.dtype
        long = STEP32 * (rows / 592 + 64)
        out['gw'] = Value((G * n).sum(0), (G.abs() * en).sum(0) + long * (G * n).abs().sum(0)).rounded(p)
        out['gb'] = Value(G.sum(0), long * G.abs().sum(0)).rounded(p)
    return out


def excess(got, want):
    """The largest error of `got` in units of its bound (at most 1 passes); finite values only."""
    d = (got.double() - want.v).abs()
    if not torch.isfinite(d).all():
        return math.inf
    return (d / want.e.clamp_min(1e-300)).max().item() if d.numel() else 0.0
