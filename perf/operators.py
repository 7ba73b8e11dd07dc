"""Workloads of the transformer-layer operators that surround multi-scale deformable attention:
the matrix product with bias, activation and residual in its epilogue, the feed-forward pair of
two such products, and layer norm, each as a forward pass and as a training step.

Every case runs either the plain form (elementary torch operations in 32 bits) or, with ``own``
set, this package's operators.
"""
import math

import torch

own = False

_TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}

# Tokens of two images on the four feature levels that the repository's attention workload uses
# (100x134, 50x67, 25x34, 13x17), every key a query.
_ENCODER = 2 * (100 * 134 + 50 * 67 + 25 * 34 + 13 * 17)
_LARGEST = 8192 * 4096 * 4096


def listed():
    return [
        # one token through the first feed-forward product: pure latency
        dict(name='linear one token', op='linear', train=False, rows=1, cin=256, cout=1024, dtype='bf16',
             act='relu', residual=False, bias=True),
        # second product of a decoder layer on 300 queries of two images
        dict(name='linear decoder queries', op='linear', train=False, rows=600, cin=1024, cout=256, dtype='fp16',
             act='none', residual=True, bias=True),
        # ragged everything in full precision: no dimension is a multiple of a vector or a tile
        dict(name='linear odd sizes fp32', op='linear', train=False, rows=1237, cin=250, cout=387, dtype='fp32',
             act='gelu', residual=True, bias=True),
        # generic wide layer, bound by the tensor cores
        dict(name='linear wide', op='linear', train=False, rows=8192, cin=4096, cout=4096, dtype='bf16',
             act='gelu', residual=False, bias=True),
        # training step of the attention's output projection, identity added in the epilogue
        dict(name='linear train projection', op='linear', train=True, rows=_ENCODER, cin=256, cout=256,
             dtype='fp32', act='none', residual=True, bias=True),
        # training step of a generic layer with the gradient of a smooth activation
        dict(name='linear train gelu', op='linear', train=True, rows=4096, cin=1024, cout=2048, dtype='fp16',
             act='gelu', residual=False, bias=True),
        # feed-forward block of a decoder layer in serving: 300 queries of one image
        dict(name='ffn decoder queries', op='ffn', train=False, rows=300, cin=256, hidden=1024, dtype='bf16',
             act='relu', residual=True),
        # feed-forward block of an encoder layer, training step
        dict(name='ffn train encoder', op='ffn', train=True, rows=_ENCODER, cin=256, hidden=1024, dtype='bf16',
             act='relu', residual=True),
        # norm of the decoder queries in serving
        dict(name='norm decoder queries', op='norm', train=False, rows=300, cols=256, dtype='fp32'),
        # norm of all encoder tokens
        dict(name='norm encoder', op='norm', train=False, rows=_ENCODER, cols=256, dtype='bf16'),
        # the same as a training step
        dict(name='norm train encoder', op='norm', train=True, rows=_ENCODER, cols=256, dtype='bf16'),
        # odd, wider rows in full precision: no vector loads
        dict(name='norm train odd fp32', op='norm', train=True, rows=5003, cols=1537, dtype='fp32'),
    ]


def _size(rng, lo, hi):
    """Log-uniform over [lo, hi]; two in three are multiples of 8 (as most layers are), the rest as they fall."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    if rng.random() < 2 / 3 and n >= 8:
        n = n // 8 * 8
    return n


def draw(rng):
    op = rng.choice(['linear', 'linear', 'ffn', 'norm', 'norm'])
    train = rng.random() < 0.5
    dtype = rng.choice(['bf16', 'fp16', 'fp32'])
    rows = max(1, int(round(math.exp(rng.uniform(0.0, math.log(_ENCODER))))))
    if op == 'norm':
        return dict(op='norm', train=train, rows=rows, cols=_size(rng, 16, 4096), dtype=dtype)
    # a gradient through the kink of relu is a coin toss where the pre-activation is within the rounding
    # error of zero; in full precision one such element is more than the type's bound
    acts = ['gelu', 'none'] if train and dtype == 'fp32' else ['relu', 'gelu', 'none']
    act = rng.choice(acts)
    passes = 3 if train else 1
    if op == 'linear':
        cin, cout = _size(rng, 16, 4096), _size(rng, 16, 4096)
        rows = max(1, min(rows, _LARGEST // (cin * cout * passes)))
        return dict(op='linear', train=train, rows=rows, cin=cin, cout=cout, dtype=dtype, act=act,
                    residual=rng.random() < 0.5, bias=rng.random() < 0.8)
    cin, hidden = _size(rng, 16, 1024), _size(rng, 32, 4096)
    rows = max(1, min(rows, _LARGEST // (2 * cin * hidden * passes)))
    return dict(op='ffn', train=train, rows=rows, cin=cin, hidden=hidden, dtype=dtype,
                act='gelu' if act == 'none' else act, residual=rng.random() < 0.7)


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = _TYPES[case['dtype']]
    rows, train = case['rows'], case['train']

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dtype)

    def uniform(*shape, bound):
        return ((torch.rand(*shape, generator=gen, device=dev) * 2 - 1) * bound).to(dtype)

    s = dict(case=case)
    leaves = []
    if case['op'] == 'norm':
        cols = case['cols']
        # post-norm activations: every row has a mean and a scale of its own
        mean = torch.randn(rows, 1, generator=gen, device=dev) * 0.5
        spread = torch.rand(rows, 1, generator=gen, device=dev) + 0.5
        s['x'] = (torch.randn(rows, cols, generator=gen, device=dev) * spread + mean).to(dtype)
        s['w'] = normal(cols, scale=0.1, shift=1.0)
        s['b'] = normal(cols, scale=0.1)
        s['gy'] = normal(rows, cols) if train else None
        leaves = ['x', 'w', 'b']
    elif case['op'] == 'linear':
        cin, cout = case['cin'], case['cout']
        s['x'] = normal(rows, cin)
        s['w'] = uniform(cout, cin, bound=math.sqrt(6.0 / (cin + cout)))   # xavier
        s['b'] = uniform(cout, bound=1.0 / math.sqrt(cin)) if case['bias'] else None
        s['res'] = normal(rows, cout) if case['residual'] else None
        s['gy'] = normal(rows, cout) if train else None
        leaves = ['x', 'w', 'b', 'res']
    else:
        cin, hidden = case['cin'], case['hidden']
        s['x'] = normal(rows, cin)
        s['w1'] = uniform(hidden, cin, bound=math.sqrt(6.0 / (cin + hidden)))
        s['b1'] = uniform(hidden, bound=1.0 / math.sqrt(cin))
        s['w2'] = uniform(cin, hidden, bound=math.sqrt(6.0 / (cin + hidden)))
        s['b2'] = uniform(cin, bound=1.0 / math.sqrt(hidden))
        s['res'] = normal(rows, cin) if case['residual'] else None
        s['gy'] = normal(rows, cin) if train else None
        leaves = ['x', 'w1', 'b1', 'w2', 'b2', 'res']
    if train:
        for k in leaves:
            if s[k] is not None:
                s[k].requires_grad_(True)
        s['leaves'] = [k for k in leaves if s[k] is not None]
    return s


# ---- plain forms -----------------------------------------------------------------------------

def _act(z, act):
    if act == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, act, g):
    if act == 'relu':
        return torch.where(z > 0, g, torch.zeros_like(g))
    if act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return g * (cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    return g


def _plain_linear(s):
    case, t = s['case'], s['x'].dtype
    x, w = s['x'].float(), s['w'].float()
    z = x @ w.t()
    if s['b'] is not None:
        z = z + s['b'].float()
    y = _act(z, case['act'])
    if s['res'] is not None:
        y = y + s['res'].float()
    y = y.to(t)
    if not case['train']:
        return {'y': y}
    gz = _act_grad(z, case['act'], s['gy'].float())
    out = {'y': y, 'gx': (gz @ w).to(t), 'gw': (gz.t() @ x).to(t)}
    if s['b'] is not None:
        out['gb'] = gz.sum(0).to(t)
    if s['res'] is not None:
        out['gres'] = s['gy']
    return out


def _plain_ffn(s):
    case, t = s['case'], s['x'].dtype
    x, w1, w2 = s['x'].float(), s['w1'].float(), s['w2'].float()
    z = x @ w1.t() + s['b1'].float()
    h = _act(z, case['act'])
    y = h @ w2.t() + s['b2'].float()
    if s['res'] is not None:
        y = y + s['res'].float()
    y = y.to(t)
    if not case['train']:
        return {'y': y}
    gy = s['gy'].float()
    gz = _act_grad(z, case['act'], gy @ w2)
    out = {'y': y, 'gx': (gz @ w1).to(t), 'gw1': (gz.t() @ x).to(t), 'gb1': gz.sum(0).to(t),
           'gw2': (gy.t() @ h).to(t), 'gb2': gy.sum(0).to(t)}
    if s['res'] is not None:
        out['gres'] = s['gy']
    return out


_EPS = 1e-5


def _plain_norm(s):
    case, t = s['case'], s['x'].dtype
    x, w = s['x'].float(), s['w'].float()
    d = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + _EPS)
    n = d * rstd
    y = (n * w + s['b'].float()).to(t)
    if not case['train']:
        return {'y': y}
    gy = s['gy'].float()
    g = gy * w
    gx = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    return {'y': y, 'gx': gx.to(t), 'gw': (gy * n).sum(0).to(t), 'gb': gy.sum(0).to(t)}


# ---- this package's operators ----------------------------------------------------------------

def _own_forward(s):
    from mmcv_b200 import ops
    case = s['case']
    if case['op'] == 'norm':
        return ops.layer_norm(s['x'], (case['cols'],), s['w'], s['b'], _EPS)
    act = None if case['act'] == 'none' else case['act']
    if case['op'] == 'linear':
        return ops.fused_linear(s['x'], s['w'], s['b'], residual=s['res'], activation=act)
    return ops.feed_forward(s['x'], s['w1'], s['b1'], s['w2'], s['b2'], residual=s['res'], activation=act)


def _own(s):
    y = _own_forward(s)
    if not s['case']['train']:
        return {'y': y}
    names = s['leaves']
    grads = torch.autograd.grad(y, [s[k] for k in names], s['gy'])
    out = {'g' + k: g for k, g in zip(names, grads)}
    out['y'] = y.detach()
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {'linear': _plain_linear, 'ffn': _plain_ffn, 'norm': _plain_norm}[state['case']['op']](state)


def work(case):
    e = 4 if case['dtype'] == 'fp32' else 2
    rows, train = case['rows'], case['train']
    if case['op'] == 'norm':
        cols = case['cols']
        n = rows * cols
        # forward: x in, y out; training reads the incoming gradient and writes gx, gw and gb too
        return {'bytes': e * ((4 * n + 4 * cols) if train else (2 * n + 2 * cols)),
                'flops': (20 if train else 8) * n}
    if case['op'] == 'linear':
        cin, cout = case['cin'], case['cout']
        inputs = rows * cin + cin * cout + (cout if case['bias'] else 0) + (rows * cout if case['residual'] else 0)
        grads = rows * cin + cin * cout + (cout if case['bias'] else 0)
        flops = 2 * rows * cin * cout
        outputs = rows * cout
        # training: the gradient of y in as well, the gradients of x, weight and bias out
        return {'bytes': e * (inputs + outputs + ((rows * cout + grads) if train else 0)),
                'flops': flops * (3 if train else 1)}
    cin, hidden = case['cin'], case['hidden']
    weights = 2 * cin * hidden + cin + hidden
    # the hidden activations need not leave the chip in a forward pass, nor between two passes of a training step
    inputs = rows * cin * (2 if case['residual'] else 1) + weights
    return {'bytes': e * (inputs + rows * cin + ((2 * rows * cin + weights) if train else 0)),
            'flops': 4 * rows * cin * hidden * (3 if train else 1)}


# ---- the same from the definitions, in 64 bits -----------------------------------------------

def _phi(z):
    """Standard normal distribution function and density."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)), torch.exp(-z.square() / 2) / math.sqrt(2.0 * math.pi)


def _exact_act(z, act):
    """Value and derivative."""
    if act == 'relu':
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == 'gelu':
        cdf, pdf = _phi(z)
        return z * cdf, cdf + z * pdf
    return z, torch.ones_like(z)


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
        train = case['train']
        if case['op'] == 'norm':
            var, mean = torch.var_mean(d['x'], dim=1, unbiased=False, keepdim=True)
            inv = (var + _EPS).rsqrt()
            n = (d['x'] - mean) * inv
            out = {'y': torch.addcmul(d['b'], n, d['w'])}
            if train:
                g = d['gy'] * d['w']
                cols = case['cols']
                # the Jacobian (I - 1 1^T / c - n n^T / c) / sigma applied to g
                out['gx'] = (g - g.sum(1, keepdim=True) / cols - n * ((g * n).sum(1, keepdim=True) / cols)) * inv
                out['gw'] = torch.einsum('rc,rc->c', d['gy'], n)
                out['gb'] = torch.einsum('rc->c', d['gy'])
            return out
        if case['op'] == 'linear':
            z = torch.einsum('rk,nk->rn', d['x'], d['w'])
            if 'b' in d:
                z += d['b']
            a, slope = _exact_act(z, case['act'])
            out = {'y': a + d['res'] if 'res' in d else a}
            if train:
                gz = d['gy'] * slope
                out['gx'] = torch.einsum('rn,nk->rk', gz, d['w'])
                out['gw'] = torch.einsum('rn,rk->nk', gz, d['x'])
                if 'b' in d:
                    out['gb'] = torch.einsum('rn->n', gz)
                if 'res' in d:
                    out['gres'] = d['gy']
            return out
        z = torch.addmm(d['b1'], d['x'], d['w1'].t())
        h, slope = _exact_act(z, case['act'])
        y = torch.addmm(d['b2'], h, d['w2'].t())
        out = {'y': y + d['res'] if 'res' in d else y}
        if train:
            gz = torch.einsum('rc,ch->rh', d['gy'], d['w2']) * slope
            out['gx'] = torch.einsum('rh,hc->rc', gz, d['w1'])
            out['gw1'] = torch.einsum('rh,rc->hc', gz, d['x'])
            out['gb1'] = torch.einsum('rh->h', gz)
            out['gw2'] = torch.einsum('rc,rh->ch', d['gy'], h)
            out['gb2'] = torch.einsum('rc->c', d['gy'])
            if 'res' in d:
                out['gres'] = d['gy']
        return out
