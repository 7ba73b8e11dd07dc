"""The transformer-layer operators on the GPU against 64-bit forms, element by element within bounds
that oracle/layers.py derives from the roundings: fused_linear, feed_forward, layer_norm, the layers
that call them, and a whole encoder layer."""
import pytest
import torch

from mmcv_b200 import ops
from oracle import layers as plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def tensors(seed, dtype, *shapes, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [None if s is None else (torch.randn(s, generator=gen) * scale).to(dtype).cuda() for s in shapes]


def hold(got, want):
    for key, value in want.items():
        over = plain.excess(got[key], value)
        assert over <= 1.0, f'{key}: {over:.3g} of its bound'


def linear_case(rows, cin, cout, dtype, act, bias=True, res=True, seed=0):
    x, r, gy = tensors(seed, dtype, (rows, cin), (rows, cout) if res else None, (rows, cout))
    w, b = tensors(seed + 1, dtype, (cout, cin), (cout,) if bias else None, scale=cin ** -0.5)
    return x, w, b, r, gy


def run_linear(x, w, b, r, gy, act):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = ops.fused_linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
    given = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(('gx', 'gw', 'gb', 'gr'), leaves) if t is not None],
                     torch.autograd.grad(y, given, gy)))
    return {'y': y.detach(), **grads}


SIZES = [(1, 256, 1024), (1, 1, 1), (3, 8, 8), (5, 7, 3), (8, 100, 130), (9, 64, 64), (64, 40, 200),
         (129, 72, 136), (300, 256, 1024), (257, 250, 387), (130, 520, 264), (1000, 1032, 72), (2500, 96, 40)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,cout', SIZES)
def test_linear_forward_and_gradients(rows, cin, cout, dtype):
    for k, (act, bias, res) in enumerate([(None, True, False), ('relu', True, True), ('gelu', False, True),
                                          (None, False, False)]):
        x, w, b, r, gy = linear_case(rows, cin, cout, dtype, act, bias, res, seed=k)
        want = plain.linear(x, w, b, r, act, gy)
        if b is None:
            want.pop('gb')
        got = run_linear(x, w, b, r, gy, act)
        hold(got, want)
        if r is not None:
            assert torch.equal(got['gr'], gy)
        with torch.no_grad():   # the serving call gives the same bits
            assert torch.equal(ops.fused_linear(x, w, b, r, act), got['y'])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,cout', [(9, 2048, 64), (300, 1024, 256), (130, 576, 40), (257, 1600, 100), (33, 4104, 72),
                                           (20, 1030, 130), (140, 513, 90)])
def test_linear_long_sums_of_few_tiles(rows, cin, cout, dtype):
    """Sums over k that several blocks of a cluster share, forward and (with the sides swapped) backward,
    ranges of uneven length among them."""
    for act, res in ((None, True), ('relu', False), ('gelu', True)):
        x, w, b, r, gy = linear_case(rows, cin, cout, dtype, act, True, res)
        got = run_linear(x, w, b, r, gy, act)
        hold(got, plain.linear(x, w, b, r, act, gy))
        with torch.no_grad():
            assert torch.equal(ops.fused_linear(x, w, b, r, act), got['y'])
        x, w, b, r, gy = linear_case(rows, cout, cin, dtype, act, False, res)
        got = run_linear(x, w, b, r, gy, act)
        want = plain.linear(x, w, b, r, act, gy)
        want.pop('gb')
        hold(got, want)
        again = run_linear(x, w, b, r, gy, act)
        assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize('dtype', DTYPES)
def test_linear_few_rows_and_small_problems(dtype):
    """One to eight rows, with everything an epilogue has; weights and inputs off 16 bytes; rows that leave
    the kernels for few of them and for small problems."""
    big, = tensors(7, dtype, (700, 300))
    for rows in (1, 2, 3, 4, 5, 8, 9, 33, 640):
        for cin, cout in ((1, 33), (96, 200), (257, 31), (2100, 40), (72, 1300), (264, 4801 if rows == 3 else 64)):
            x, w, b, r, gy = linear_case(rows, cin, cout, dtype, None, True, True, seed=rows)
            for act in (None, 'relu', 'gelu'):
                got = run_linear(x, w, b, r, gy, act)
                hold(got, plain.linear(x, w, b, r, act, gy))
                with torch.no_grad():
                    assert torch.equal(ops.fused_linear(x, w, b, r, act), got['y'])
            if cin == 257:
                x = big[:rows, 3:3 + cin]
                hold(run_linear(x, w, b, r, gy, 'gelu'), plain.linear(x, w, b, r, 'gelu', gy))
                x = big[:rows, 8:8 + cin]      # rows on 16 bytes whose length is odd
                hold(run_linear(x, w, None, r, gy, 'relu'),
                     {k: v for k, v in plain.linear(x, w, None, r, 'relu', gy).items() if k != 'gb'})


def test_first_call_of_a_thread():
    """A new thread has no CUDA context bound to it; a call that allocates nothing binds none before the
    tensor maps are encoded."""
    import threading
    x, w, b, _, _ = linear_case(64, 64, 64, torch.bfloat16, None)
    want, got = ops.fused_linear(x, w, b), []
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream()

    def call():
        got.append(ops.fused_linear(x, w, b))

    for _ in range(2):
        t = threading.Thread(target=call)
        t.start()
        t.join()
    stream.synchronize()
    assert len(got) == 2 and all(torch.equal(g, want) for g in got)


def test_backward_as_the_first_work_of_the_process():
    """The engine's thread starts with this backward pass: nothing has bound a context to it."""
    import os
    import subprocess
    import sys
    code = ("import torch\nfrom mmcv_b200 import ops\n"
            "x, w, b, g = (torch.randn(s, device='cuda').bfloat16() for s in ((300, 256), (1024, 256), (1024,), (300, 1024)))\n"
            "x.requires_grad_(True); w.requires_grad_(True); b.requires_grad_(True)\n"
            "gx, gw, gb = torch.autograd.grad(ops.fused_linear(x, w, b), [x, w, b], g)\n"
            "err = ((gw.double() - g.double().t() @ x.double()).norm() / gw.double().norm()).item()\n"
            "assert err < 2 ** -8, err\n"
            "print('done')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'done' in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize('dtype', DTYPES)
def test_linear_many_rows_and_splits(dtype):
    """Enough rows that the weight gradient's sum is divided among blocks."""
    for rows, cin, cout, act in [(20011, 64, 72, 'gelu'), (6000, 256, 264, 'relu'), (3000, 130, 33, None),
                                 (19000, 136, 264, 'gelu'), (9600, 264, 520, 'relu'), (9500, 257, 300, None)]:
        x, w, b, r, gy = linear_case(rows, cin, cout, dtype, act)
        got = run_linear(x, w, b, r, gy, act)
        hold(got, plain.linear(x, w, b, r, act, gy))
        again = run_linear(x, w, b, r, gy, act)
        assert all(torch.equal(got[k], again[k]) for k in got)   # no order left to chance


@pytest.mark.parametrize('dtype', DTYPES)
def test_linear_strides_and_alignment(dtype):
    """Row strides, views that start off a 16-byte boundary, a transposed weight, expanded gradients
    and residuals, leading dimensions."""
    rows, cin, cout = 77, 48, 56
    wide, = tensors(3, dtype, (rows, 128))
    w_big, b, gy = tensors(4, dtype, (64, 80), (cout,), (rows, cout))
    for x in (wide[:, :cin], wide[:, 8:8 + cin], wide[:, 3:3 + cin], wide[::2][:, 1:1 + cin],
              wide.t()[:cin].t(), wide[:1, :cin].expand(rows, cin)):
        for w in (w_big[:cout, :cin], w_big[1:1 + cout, 5:5 + cin], w_big.t()[:cin, :cout].t(),
                  w_big[:cin, :cout].t()):
            g = gy[:x.shape[0]]
            hold(run_linear(x, w, b, None, g, 'gelu'), plain.linear(x, w, b, None, 'gelu', g))
    x, w = wide[:, :cin].reshape(7, 11, cin), w_big[:cout, :cin]
    res, = tensors(5, dtype, (11, 1))
    leaf, rleaf = x.detach().requires_grad_(True), res.detach().requires_grad_(True)
    y = ops.fused_linear(leaf, w, b[::1], rleaf, 'relu')
    assert y.shape == (7, 11, cout)
    y.sum().backward()      # an expanded gradient
    want = plain.linear(x.reshape(-1, cin), w, b, res.expand(7, 11, cout).reshape(-1, cout), 'relu',
                        torch.ones(rows, cout, dtype=dtype, device='cuda'))
    hold({'y': y.detach().reshape(rows, cout), 'gx': leaf.grad.reshape(rows, cin)}, {k: want[k] for k in ('y', 'gx')})
    assert torch.equal(rleaf.grad, torch.full_like(res, 7 * cout))


def test_linear_partial_gradients_and_empty_batch():
    x, w, b, r, gy = linear_case(40, 24, 32, torch.bfloat16, 'gelu')
    full = run_linear(x, w, b, r, gy, 'gelu')
    for mask in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b, r))]
        y = ops.fused_linear(*leaves, activation='gelu')
        y.backward(gy)
        for name, t in zip(('gx', 'gw', 'gb', 'gr'), leaves):
            if t.requires_grad:
                if name == 'gb' and not leaves[1].requires_grad:
                    hold({'gb': t.grad}, {'gb': plain.linear(x, w, b, r, 'gelu', gy)['gb']})
                else:
                    assert torch.equal(t.grad, full[name]), (mask, name)
            else:
                assert t.grad is None
    leaves = [t.detach().requires_grad_(True) for t in (x[:0], w, b)]
    y = ops.fused_linear(*leaves, activation='relu')
    assert y.shape == (0, 32)
    y.sum().backward()
    assert leaves[0].grad.shape == (0, 24) and not leaves[1].grad.any() and not leaves[2].grad.any()


def test_linear_non_finite_rows_stay_alone():
    """A NaN row of x reaches its own row of y only; NaN passes relu and gelu."""
    for dtype in DTYPES:
        x, w, b, _, _ = linear_case(200, 64, 136, dtype, 'relu')
        x = x.clone()
        x[37] = float('nan')
        for act in (None, 'relu', 'gelu'):
            y = ops.fused_linear(x, w, b, activation=act)
            bad = torch.isnan(y).all(1)
            assert bad[37] and int(torch.isnan(y).any(1).sum()) == 1


@pytest.mark.parametrize('dtype', DTYPES)
def test_linear_infinities(dtype):
    """An infinite element of x makes its row of z infinite with the sign of the weight (NaN where that is
    zero), whatever the finite ones are; the same in the gradients."""
    inf = float('inf')
    x, w, b, _, gy = linear_case(140, 600, 72, dtype, None)
    w[5] = 1.0                     # nothing below the leading bits
    x[3, 17], x[9, 400], x[130, 599] = inf, -inf, inf
    y = ops.fused_linear(x, w, b)
    want = x.double() @ w.double().t() + b.double()
    assert not torch.isfinite(want[[3, 9, 130]]).any()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(torch.sign(y[[3, 9, 130]]), torch.sign(want[[3, 9, 130]]).to(dtype))
    x = linear_case(140, 600, 72, dtype, None)[0]
    gy[70, 5] = inf
    got = run_linear(x, w, b, None, gy, None)
    for key, ref in (('gx', gy.double() @ w.double()), ('gw', gy.double().t() @ x.double()), ('gb', gy.double().sum(0))):
        assert torch.equal(torch.isnan(got[key]), torch.isnan(ref)), key
        assert torch.equal(got[key][torch.isinf(ref)].double(), ref[torch.isinf(ref)]), key
    y = ops.fused_linear(torch.full((4, 600), -inf, dtype=dtype, device='cuda'), w.abs() + 0.5, b, activation='gelu')
    assert torch.equal(y, torch.zeros_like(y))      # gelu(-inf)


def test_gelu_gradient_keeps_fine_and_huge_pre_activations():
    """One element per row with a weight of one: gz alone is tested, through gx.  Its pre-activation is
    kept in fp16 for bf16 tensors: half a step of 2^-11 of |z| (slope's slope at most 0.8), then the two
    roundings of gz and gx to bf16; beyond fp16's range the derivative is 0 or 1 exactly."""
    z = torch.cat([torch.linspace(-6, 6, 400), torch.tensor([1e5, -1e5, 3e38, -3e38, 70.0, -70.0])])
    x = torch.zeros(z.numel(), 8)
    x[:, 0] = z
    x = x.bfloat16().cuda().requires_grad_(True)
    w = torch.zeros(8, 8)
    w[0, 0] = 1
    w = w.bfloat16().cuda()
    y = ops.fused_linear(x, w, activation='gelu')
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    v = x.detach()[:, 0].double()
    slope = plain.activation(v, 'gelu')[1]
    bound = 0.8 * v.abs().clamp(max=40) * 2.0 ** -11 + slope.abs() * (2 * 2.0 ** -8 + 2.0 ** -16) + 2.0 ** -19
    assert ((gx[:, 0].double() - slope).abs() <= bound).all()
    assert gx[-6:, 0].tolist() == [1, 0, 1, 0, 1, 0]


def test_linear_gradient_against_differences():
    """The directional derivative of sum(y * gy) along random directions, by central differences of
    the 64-bit form; the gradients are fp32: relative error of a sum of n products, and the
    differences' own h^2."""
    x, w, b, r, gy = linear_case(50, 40, 30, torch.float32, 'gelu')
    got = run_linear(x, w, b, r, gy, 'gelu')
    d = tensors(9, torch.float64, x.shape, w.shape, b.shape)
    h = 1e-4

    def f(s):
        z = (x.double() + s * d[0]) @ (w.double() + s * d[1]).t() + b.double() + s * d[2]
        return (plain.activation(z, 'gelu')[0] * gy.double()).sum()

    slope = ((f(h) - f(-h)) / (2 * h)).item()
    mine = sum((got[k].double() * v).sum().item() for k, v in zip(('gx', 'gw', 'gb'), d))
    size = sum((got[k].double() * v).abs().sum().item() for k, v in zip(('gx', 'gw', 'gb'), d))
    assert abs(mine - slope) <= 1e-5 * size


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,hidden', [(1, 16, 32), (300, 256, 1024), (45, 33, 70), (2049, 64, 96)])
def test_feed_forward(rows, cin, hidden, dtype):
    for act in ('relu', 'gelu'):
        x, r, gy = tensors(1, dtype, (rows, cin), (rows, cin), (rows, cin))
        w1, w2 = tensors(2, dtype, (hidden, cin), (cin, hidden), scale=(cin + hidden) ** -0.5)
        b1, b2 = tensors(3, dtype, (hidden,), (cin,), scale=0.1)
        want = plain.feed_forward(x, w1, b1, w2, b2, r, act, gy)
        leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2, r)]
        y = ops.feed_forward(*leaves, activation=act)
        grads = torch.autograd.grad(y, leaves, gy)
        hold({'y': y.detach(), **dict(zip(('gx', 'gw1', 'gb1', 'gw2', 'gb2'), grads))}, want)
        assert torch.equal(grads[5], gy)
        with torch.no_grad():
            assert torch.equal(ops.feed_forward(x, w1, b1, w2, b2, r, act), y.detach())
        # the input as its own residual: one gradient, both parts in it
        leaf = x.detach().requires_grad_(True)
        y = ops.feed_forward(leaf, w1, b1, w2, b2, leaf, act)
        g, = torch.autograd.grad(y, leaf, gy)
        both = plain.feed_forward(x, w1, b1, w2, b2, x, act, gy)
        gx = plain.add(plain.Value(both['gx'].v, both['gx'].e), gy.double())
        hold({'y': y.detach(), 'gx': g}, {'y': both['y'], 'gx': gx.rounded(dtype)})


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,hidden', [(1, 16, 32), (31, 24, 70), (333, 40, 48), (2500, 64, 520)])
def test_feed_forward_bias_gradient_is_summed_before_rounding(rows, cin, hidden, dtype):
    """bias1's gradient within one rounding of the sum of the unrounded gradients, which the hidden
    gradient's own rounding would exceed."""
    for act in ('relu', 'gelu'):
        x, gy = tensors(1, dtype, (rows, cin), (rows, cin))
        w1, w2 = tensors(2, dtype, (hidden, cin), (cin, hidden), scale=(cin + hidden) ** -0.5)
        b1, b2 = tensors(3, dtype, (hidden,), (cin,), scale=0.1)
        z = plain.add(plain.product(plain.Value(x), plain.Value(w1)), b1.double())
        gz = plain.through(plain.product(plain.Value(gy), plain.Value(w2).t()), z, act,
                           kept=torch.float32 if dtype == torch.float32 else torch.float16)
        want = plain.column_sum(gz).rounded(dtype)
        leaf = b1.detach().requires_grad_(True)
        g, = torch.autograd.grad(ops.feed_forward(x, w1, leaf, w2, b2, None, act), leaf, gy)
        hold({'gb1': g}, {'gb1': want})
        # the same bits beside the other gradients
        leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
        grads = torch.autograd.grad(ops.feed_forward(*leaves, None, act), leaves, gy)
        assert torch.equal(grads[2], g)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,hidden', [(300, 48, 768), (70, 40, 1000)])
def test_feed_forward_many_hidden_columns(rows, cin, hidden, dtype):
    """bias1's gradient from the rounded hidden gradient, and each gradient wanted alone."""
    x, gy = tensors(1, dtype, (rows, cin), (rows, cin))
    w1, w2 = tensors(2, dtype, (hidden, cin), (cin, hidden), scale=(cin + hidden) ** -0.5)
    b1, b2 = tensors(3, dtype, (hidden,), (cin,), scale=0.1)
    for act in ('relu', 'gelu'):
        want = plain.feed_forward(x, w1, b1, w2, b2, x, act, gy)
        leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
        y = ops.feed_forward(*leaves, leaves[0], act)
        grads = dict(zip(('gx', 'gw1', 'gb1', 'gw2', 'gb2'), torch.autograd.grad(y, leaves, gy)))
        want['gx'] = plain.add(want['gx'], gy.double()).rounded(dtype)
        hold({'y': y.detach(), **grads}, want)
        for only in range(5):
            parts = [t.detach().requires_grad_(i == only) for i, t in enumerate((x, w1, b1, w2, b2))]
            g, = torch.autograd.grad(ops.feed_forward(*parts, parts[0], act), parts[only], gy)
            hold({'g': g}, {'g': want[('gx', 'gw1', 'gb1', 'gw2', 'gb2')[only]]})


def test_graphs_are_used_once_unless_retained():
    x, w, b, r, gy = linear_case(20, 24, 32, torch.bfloat16, 'gelu')
    w2, = tensors(5, torch.bfloat16, (24, 32))
    for f in (lambda t: ops.fused_linear(t, w, b, activation='gelu'), lambda t: ops.layer_norm(t, (24,), t[0], None),
              lambda t: ops.feed_forward(t, w, b, w2, None, t)):
        leaf = x.detach().requires_grad_(True)
        y = f(leaf)
        one, = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
        two, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert torch.equal(one, two)
        with pytest.raises(RuntimeError, match='second time'):
            torch.autograd.grad(y, leaf, torch.ones_like(y))
    leaf, wl = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    y = ops.fused_linear(leaf, wl)
    with torch.no_grad():
        leaf.add_(1)           # what the backward pass needs has changed
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    x, w, b, _, _ = linear_case(20, 24, 32, torch.bfloat16, None)
    w2, = tensors(5, torch.bfloat16, (24, 32))
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda t: ops.fused_linear(t, w, b), lambda t: ops.layer_norm(t, (24,)),
                  lambda t: ops.feed_forward(t, w, b, w2, None)):
            with pytest.raises(RuntimeError, match='forward-mode'):
                f(dual)
        with pytest.raises(RuntimeError, match='forward-mode'):
            ops.fused_linear(x, w, fwd.make_dual(b, torch.ones_like(b)))


NORM_SIZES = [(1, 1), (1, 256), (3, 8), (300, 256), (77, 100), (9, 1024), (5, 1537), (40, 2048), (3, 8192), (2, 8200),
              (3, 9001), (5000, 64), (1203, 384), (700, 4096)]


def norm_case(rows, cols, dtype, wdtype=None, shift=0.0, seed=0):
    x, gy = tensors(seed, dtype, (rows, cols), (rows, cols))
    w, b = tensors(seed + 1, wdtype or dtype, (cols,), (cols,))
    return x + shift, w, b, gy


def run_norm(x, w, b, gy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(leaves[0], x.shape[1:], leaves[1], leaves[2], eps)
    given = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(('gx', 'gw', 'gb'), leaves) if t is not None],
                     torch.autograd.grad(y, given, gy)))
    return {'y': y.detach(), **grads}


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cols', NORM_SIZES)
def test_norm_forward_and_gradients(rows, cols, dtype):
    x, w, b, gy = norm_case(rows, cols, dtype)
    got = run_norm(x, w, b, gy)
    hold(got, plain.layer_norm(x, w, b, 1e-5, gy))
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, (cols,), w, b), got['y'])
    again = run_norm(x, w, b, gy)
    assert all(torch.equal(got[k], again[k]) for k in got)
    plain_only = run_norm(x, None, None, gy)
    hold(plain_only, {k: v for k, v in plain.layer_norm(x, None, None, 1e-5, gy).items() if k in ('y', 'gx')})


def test_norm_mixed_parameter_type_and_partial_gradients():
    for dtype in (torch.bfloat16, torch.float16):
        x, w, b, gy = norm_case(70, 264, dtype, torch.float32)
        got = run_norm(x, w, b, gy)
        assert got['gw'].dtype == torch.float32 and got['y'].dtype == dtype
        hold(got, plain.layer_norm(x, w, b, 1e-5, gy))
    for mask in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        ops.layer_norm(leaves[0], (264,), leaves[1], leaves[2]).backward(gy)
        for name, t in zip(('gx', 'gw', 'gb'), leaves):
            assert (t.grad is None) == (not t.requires_grad)
            if t.requires_grad:
                assert torch.equal(t.grad, got[name]), (mask, name)
    hold(run_norm(x, w, None, gy), {k: v for k, v in plain.layer_norm(x, w, None, 1e-5, gy).items() if k != 'gb'})


def test_norm_large_means_constant_rows_and_non_finite_rows():
    # a mean 10000 times the spread: the input itself is exact in fp32, so the statistics must be too
    x, w, b, gy = norm_case(60, 256, torch.float32)
    x = (x * 64).round() / 64 + 10000.0
    hold(run_norm(x, w, b, gy), plain.layer_norm(x, w, b, 1e-5, gy))
    # constant rows: variance 0, the result is the bias (to what (x - mean) leaves: nothing)
    flat = torch.full((5, 256), 3.25, device='cuda')
    y = ops.layer_norm(flat, (256,), w, b)
    assert torch.equal(y, b.expand(5, 256))
    x[7, 3] = float('inf')
    x[9, 0] = float('nan')
    y = ops.layer_norm(x, (256,), w, b)
    bad = torch.isnan(y).any(1)
    assert bad[7] and bad[9] and int(bad.sum()) == 2


@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_strides_shapes_and_empty(dtype):
    big, = tensors(0, dtype, (50, 300))
    w, b, gy = tensors(1, dtype, (256,), (256,), (50, 256))
    for x in (big[:, :256], big[:, 40:296], big[:, 3:259], big[::2, 1:257], big[:1, :256].expand(50, 256)):
        g = gy[:x.shape[0]]
        hold(run_norm(x, w, b, g), plain.layer_norm(x, w, b, 1e-5, g))
        wm = torch.cat([w, w])[5:261]     # parameters off a 16-byte boundary
        hold(run_norm(x, wm, b, g), plain.layer_norm(x, wm, b, 1e-5, g))
    x4 = big[:, :256].reshape(5, 10, 16, 16)
    y = ops.layer_norm(x4, (16, 16), w.view(16, 16), b.view(16, 16))
    assert torch.equal(y.view(50, 256), ops.layer_norm(big[:, :256], 256, w, b))
    leaves = [t.detach().requires_grad_(True) for t in (big[:0, :256], w, b)]
    y = ops.layer_norm(leaves[0], (256,), leaves[1], leaves[2])
    y.sum().backward()
    assert y.shape == (0, 256) and not leaves[1].grad.any() and not leaves[2].grad.any()
    leaf = big[:, :256].detach().requires_grad_(True)
    ops.layer_norm(leaf, (256,), w, b).sum().backward()    # an expanded gradient
    one = torch.ones(50, 256, dtype=dtype, device='cuda')
    hold({'gx': leaf.grad}, {'gx': plain.layer_norm(big[:, :256], w, b, 1e-5, one)['gx']})


@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_over_all_dimensions_of_a_strided_matrix(dtype):
    """One row made of a whole matrix whose own rows do not follow one another."""
    big, w, b, gy = tensors(0, dtype, (16, 300), (16, 16), (16, 16), (16, 16))
    for x in (big[:, :16], big[:, 3:19], big[:, :16].t(), big[::2, :32].reshape(16, 16)):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.layer_norm(leaves[0], (16, 16), leaves[1], leaves[2])
        grads = torch.autograd.grad(y, leaves, gy.t())
        flat = lambda t: t.reshape(1, 256)   # noqa: E731
        want = plain.layer_norm(flat(x), w.flatten(), b.flatten(), 1e-5, flat(gy.t()))
        hold({'y': flat(y.detach()), 'gx': flat(grads[0]), 'gw': grads[1].flatten(), 'gb': grads[2].flatten()}, want)


def test_norm_gradient_against_differences():
    x, w, b, gy = norm_case(30, 40, torch.float32)
    got = run_norm(x, w, b, gy)
    d = tensors(9, torch.float64, x.shape, w.shape, b.shape)
    h = 1e-4

    def f(s):
        t = x.double() + s * d[0]
        c = t - t.mean(1, keepdim=True)
        y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * (w.double() + s * d[1]) + b.double() + s * d[2]
        return (y * gy.double()).sum()

    slope = ((f(h) - f(-h)) / (2 * h)).item()
    mine = sum((got[k].double() * v).sum().item() for k, v in zip(('gx', 'gw', 'gb'), d))
    size = sum((got[k].double() * v).abs().sum().item() for k, v in zip(('gx', 'gw', 'gb'), d))
    assert abs(mine - slope) <= 1e-5 * size


def block_inputs(dtype, rows=70, cin=64, hidden=96, seed=0):
    x, gy = tensors(seed, dtype, (rows, cin), (rows, cin))
    w1, w2 = tensors(seed + 1, dtype, (hidden, cin), (cin, hidden), scale=0.1)
    b1, b2, g, b = tensors(seed + 2, dtype, (hidden,), (cin,), (cin,), (cin,))
    return x, gy, w1, b1, w2, b2, g, b


def block(x, w1, b1, w2, b2, g, b):
    return ops.layer_norm(ops.feed_forward(x, w1, b1, w2, b2, x, 'gelu'), (x.shape[-1],), g, b)


def test_another_stream_and_two_at_once():
    """Two streams at once, each with its own tensors; results equal to those of one stream."""
    sets = [block_inputs(torch.bfloat16, rows=3000, seed=10 * k) for k in range(2)]
    want = [block(s[0], *s[2:]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(block(sets[k][0], *sets[k][2:]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in got[k])


def test_threads_with_a_stream_each():
    """Training steps of four threads at once, sizes that run on every kernel."""
    import threading
    sets = [block_inputs(dt, rows=rows, seed=10 * k)
            for k, (dt, rows) in enumerate([(torch.bfloat16, 3000), (torch.float32, 70), (torch.float16, 3),
                                            (torch.float32, 2500)])]

    def step(x, gy, *params):
        leaves = [t.detach().requires_grad_(True) for t in (x, *params)]
        y = block(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[k] = step(*sets[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    for k in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows of the result and of the gradients against a call on those rows."""
    rows, cin, cout = 2_150_000, 16, 1024
    x, w, b, _, _ = linear_case(rows, cin, cout, torch.bfloat16, None)
    tail = slice(rows - 300, rows)
    for act in ('relu', 'gelu'):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.fused_linear(*leaves, activation=act)
        assert y.numel() > 2 ** 31
        gy = torch.zeros_like(y)
        gy[tail] = tensors(5, torch.bfloat16, (300, cout))[0]
        got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(y, leaves, gy)))
        want = plain.linear(x[tail], w, b, None, act, gy[tail])
        hold({'y': y.detach()[tail], 'gx': got['gx'][tail], 'gw': got['gw'], 'gb': got['gb']}, want)
        assert not got['gx'][:rows - 300].any()
        del y, gy, got, leaves
    del x
    rows, cols = 530_000, 4104
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(0))
    w, b = tensors(1, torch.bfloat16, (cols,), (cols,))
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = ops.layer_norm(leaves[0], (cols,), leaves[1], leaves[2])
    gy = torch.zeros_like(y)
    gy[-200:] = tensors(5, torch.bfloat16, (200, cols))[0]
    got = dict(zip(('gx', 'gw', 'gb'), torch.autograd.grad(y, leaves, gy)))
    hold({'y': y.detach()[-200:], 'gx': got['gx'][-200:], 'gw': got['gw'], 'gb': got['gb']},
         plain.layer_norm(x[-200:], w, b, 1e-5, gy[-200:]))
    assert not got['gx'][:-200].any()


@pytest.mark.parametrize('dtype', DTYPES)
def test_captured_training_step(dtype):
    """Forward and backward in a CUDA graph while an eager graph of the same leaves lives (made on a side
    stream: torch cannot capture a backward pass over leaves whose accumulation node belongs to the
    default stream, whatever the operators); replayed on new values it gives the eager results."""
    x, gy, *params = block_inputs(dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, *params)]

    def step():
        y = block(*leaves)
        return (y, *torch.autograd.grad(y, leaves, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = block(*leaves)          # an eager graph that outlives the capture
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    del alive
    for seed in (20, 30):
        nx, ngy, *nparams = block_inputs(dtype, seed=seed)
        with torch.no_grad():
            for t, v in zip((*leaves, gy), (nx, *nparams, ngy)):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_status_reading_and_capture():
    """With the status word read after every call, a capture still works (it reads nothing), eager calls are
    checked, and the results are those without."""
    from mmcv_b200 import _ext
    x, gy, *params = block_inputs(torch.bfloat16)
    want = block(x, *params)
    before = _ext._check_status
    _ext.set_check_status(True)
    try:
        assert torch.equal(block(x, *params), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = block(x, *params)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        leaf = x.detach().requires_grad_(True)
        torch.autograd.grad(block(leaf, *params), leaf, gy)
    finally:
        _ext.set_check_status(before)


def test_autocast_follows_torch():
    x, gy, w1, b1, w2, b2, g, b = block_inputs(torch.float32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1)]
    with torch.autocast('cuda', dtype=torch.bfloat16):
        y = ops.fused_linear(*leaves, activation='relu')
        n = ops.layer_norm(y, (96,))
        z = ops.feed_forward(x, w1, b1, w2, b2, x)
    assert y.dtype == torch.bfloat16 and n.dtype == torch.float32 and z.dtype == torch.float32
    y.sum().backward()
    assert all(t.grad.dtype == torch.float32 for t in leaves)
    ref = ops.fused_linear(x.bfloat16(), w1.bfloat16(), b1.bfloat16(), activation='relu')
    assert torch.equal(y, ref)


def test_a_second_derivative_is_refused():
    x, gy, w1, b1, w2, b2, g, b = block_inputs(torch.float32)
    for f in (lambda t: ops.fused_linear(t, w1, b1, activation='gelu'), lambda t: ops.layer_norm(t, (64,), g, b),
              lambda t: ops.feed_forward(t, w1, b1, w2, b2, t)):
        leaf = x.detach().requires_grad_(True)
        first, = torch.autograd.grad(f(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match='cannot be differentiated again'):
            first.sum().backward()


def test_layers_match_their_torch_forms():
    torch.manual_seed(0)
    for act in ('ReLU', 'GELU'):
        ffn = ops.FFN(64, 160, act_cfg=dict(type=act)).cuda()
        assert set(ffn.state_dict()) == {'layers.0.0.weight', 'layers.0.0.bias', 'layers.1.weight', 'layers.1.bias'}
        x = torch.randn(3, 50, 64, device='cuda')
        other = torch.randn_like(x)
        ref = ffn.double().layers(x.double())
        ffn.float()
        for ident, want in ((None, x + ref), (other, other + ref)):
            assert torch.allclose(ffn(x, ident).double(), want, rtol=0, atol=2e-5)
    drop = ops.FFN(64, 160, ffn_drop=0.5, dropout_layer=dict(type='Dropout', drop_prob=0.25)).cuda()
    y = drop(x)
    y.sum().backward()
    assert drop.layers[1].weight.grad is not None and not torch.equal(y, drop(x))
    drop.eval()
    assert torch.equal(drop(x), drop(x))
    norm = ops.LayerNorm(64).cuda()
    assert torch.allclose(norm(x), torch.nn.functional.layer_norm(x, (64,)), atol=1e-5)
    lin = ops.FusedLinear(64, 24, activation='relu').cuda()
    res = torch.randn(3, 50, 24, device='cuda')
    assert torch.allclose(lin(x, res), torch.relu(x @ lin.weight.t() + lin.bias) + res, atol=2e-5)


@pytest.mark.parametrize('batch_first', [True, False])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_encoder_layer_runs_the_operators_together(batch_first, dtype):
    """The encoder layer against the same layer built from the default attention layer and 64-bit
    torch, forward and gradients.  fp32: the operators' own errors are below 1e-6 of a row's size and
    four follow one another, the sampler's tolerance is 1e-4.  bf16: relative L2 within six roundings
    of 2^-8 along the path."""
    from oracle.msda import msda_forward
    torch.manual_seed(0)
    layer = ops.DeformableEncoderLayer(64, num_heads=4, num_levels=2, num_points=3, feedforward_channels=160,
                                       batch_first=batch_first)
    att = layer.attentions[0]
    for p in (att.sampling_offsets.weight, att.attention_weights.weight):
        p.data.normal_(0, 0.05)
    layer = layer.to(dtype).cuda()
    shapes = torch.tensor([[6, 5], [3, 2]])
    S = 36
    x, gy = tensors(0, dtype, (2, S, 64), (2, S, 64))
    pos, = tensors(1, dtype, (2, S, 64), scale=0.1)
    refp = torch.rand(2, S, 2, 2, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    mask = torch.zeros(2, S, dtype=torch.bool, device='cuda')
    mask[1, 30:] = True                                     # a padded batch
    flip = (lambda t: t) if batch_first else (lambda t: t.transpose(0, 1))
    leaf = flip(x).contiguous().detach().requires_grad_(True)
    y = layer(leaf, query_pos=flip(pos), key_padding_mask=mask, reference_points=refp,
              spatial_shapes=shapes.cuda(), level_start_index=torch.tensor([0, 30]).cuda())
    params = dict(layer.named_parameters())
    grads = torch.autograd.grad(y, [leaf, *params.values()], flip(gy).contiguous())
    # 64 bits, on the CPU
    P = {k: v.detach().double().cpu().requires_grad_(True) for k, v in params.items()}
    X = x.double().cpu().requires_grad_(True)

    def lin(t, name):
        return t @ P[name + '.weight'].t() + P[name + '.bias']

    def norm(t, name):
        return torch.nn.functional.layer_norm(t, (64,), P[name + '.weight'], P[name + '.bias'])

    q = X + pos.double().cpu()
    v = lin(X, 'attentions.0.value_proj').masked_fill(mask.cpu()[..., None], 0.0).view(2, S, 4, 16)
    off = lin(q, 'attentions.0.sampling_offsets').view(2, S, 4, 2, 3, 2)
    aw = lin(q, 'attentions.0.attention_weights').view(2, S, 4, 6).softmax(-1).view(2, S, 4, 2, 3)
    scale = torch.stack([shapes[:, 1], shapes[:, 0]], -1).double()
    loc = refp.double().cpu()[:, :, None, :, None, :] + off / scale[None, None, None, :, None, :]
    a = norm(lin(msda_forward(v, shapes, loc, aw), 'attentions.0.output_proj') + X, 'norms.0')
    h = torch.relu(lin(a, 'ffns.0.layers.0.0'))
    want = norm(a + lin(h, 'ffns.0.layers.1'), 'norms.1')
    wgrads = torch.autograd.grad(want, [X, *P.values()], gy.double().cpu())
    tol = 1e-4 if dtype == torch.float32 else 6 * 2.0 ** -8
    rel = lambda g, w: ((g.double().cpu() - w).norm() / w.norm()).item()   # noqa: E731
    assert rel(flip(y.detach()), want.detach()) <= tol
    # the sampler's location gradients jump at cell borders, which rounded locations cross: the
    # gradients that do not pass through them are compared.  In bf16 a location is off by up to 2^-9
    # of a map, 0.01 pixels, and the gradients of the attention weights are differences of samples.
    names = [None, *params]
    for name, g, w in zip(names, grads, wgrads):
        if name is None:
            g = flip(g)
        if name is None or 'sampling_offsets' in name or (dtype != torch.float32 and 'attention_weights' in name):
            assert torch.isfinite(g).all()
            continue
        assert rel(g, w) <= (tol if dtype == torch.float32 else 2 * tol), name


def test_fused_projections_of_the_attention_layer():
    """fused_proj changes roundings only; the default layer is untouched."""
    torch.manual_seed(1)
    a = ops.MultiScaleDeformableAttention(64, 4, 2, 3, dropout=0.1, batch_first=True).cuda()
    b = ops.MultiScaleDeformableAttention(64, 4, 2, 3, dropout=0.1, batch_first=True, fused_proj=True).cuda()
    b.load_state_dict(a.state_dict())
    assert a.fused_proj is False
    q, = tensors(0, torch.float32, (2, 36, 64))
    kw = dict(reference_points=torch.rand(2, 36, 2, 2, device='cuda'), spatial_shapes=torch.tensor([[6, 5], [3, 2]]).cuda(),
              level_start_index=torch.tensor([0, 30]).cuda())
    a.eval(), b.eval()
    assert torch.allclose(a(q, **kw), b(q, **kw), atol=2e-5)
    b.train()
    assert torch.isfinite(b(q, **kw)).all()     # dropout active: the identity is added outside


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,cout', [(1237, 250, 388), (2500, 264, 384), (4000, 512, 520), (300, 1024, 256)])
def test_residual_off_16_bytes_gives_the_bits_of_an_aligned_one(rows, cin, cout, dtype):
    """The residual's element-by-element form (several staging chunks to an epilogue warp) against the tensor
    load's, and both against the bounds."""
    x, w, b, r, _ = linear_case(rows, cin, cout, dtype, None)
    wide = torch.zeros(rows, cout + 9, dtype=dtype, device='cuda')
    wide[:, 1:1 + cout] = r
    for act in (None, 'relu', 'gelu'):
        leaf = w.detach().requires_grad_(True)   # what the backward pass needs is kept: another epilogue
        y = ops.fused_linear(x, w, b, r, act)
        hold({'y': y}, plain.linear(x, w, b, r, act))
        for _ in range(3):
            assert torch.equal(ops.fused_linear(x, w, b, wide[:, 1:1 + cout], act), y)
            assert torch.equal(ops.fused_linear(x, leaf, b, wide[:, 1:1 + cout], act).detach(), y)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cin,hidden', [(1, 16, 32), (45, 33, 70), (300, 48, 768), (2049, 64, 1000)])
def test_feed_forward_without_activation(rows, cin, hidden, dtype):
    """activation=None: all gradients together, and each alone."""
    x, r, gy = tensors(1, dtype, (rows, cin), (rows, cin), (rows, cin))
    w1, w2 = tensors(2, dtype, (hidden, cin), (cin, hidden), scale=(cin + hidden) ** -0.5)
    b1, b2 = tensors(3, dtype, (hidden,), (cin,), scale=0.1)
    want = plain.feed_forward(x, w1, b1, w2, b2, r, None, gy)
    # oracle.layers passes the hidden gradient on unrounded where there is no activation; it is stored in the
    # tensors' type: rounded here, before the products that read it
    gz = plain.product(plain.Value(gy), plain.Value(w2).t()).rounded(dtype)
    want['gx'] = plain.product(gz, plain.Value(w1).t()).rounded(dtype)
    want['gw1'] = plain.product(gz.t(), plain.Value(x).t()).rounded(dtype)
    want['gb1'] = plain.column_sum(gz).rounded(dtype)
    names = ('gx', 'gw1', 'gb1', 'gw2', 'gb2')
    leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = ops.feed_forward(*leaves, r, None)
    hold({'y': y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, gy)))}, want)
    for only in range(5):
        parts = [t.detach().requires_grad_(i == only) for i, t in enumerate((x, w1, b1, w2, b2))]
        g, = torch.autograd.grad(ops.feed_forward(*parts, r, None), parts[only], gy)
        hold({'g': g}, {'g': want[names[only]]})


def test_kept_casts_and_captures():
    """frozen_weights(): what a capture would make is not kept (an eager call after it would find it unmade),
    what eager calls have kept serves a capture, and other streams find it complete."""
    import mmcv_b200
    from mmcv_b200 import _ext
    x, w, b, _, _ = linear_case(300, 2048, 4096, torch.float32, None)
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        want = ops.fused_linear(x, w, b)
        with mmcv_b200.frozen_weights():
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = ops.fused_linear(x, w, b)
            assert not _ext._frozen.casts
            assert torch.equal(ops.fused_linear(x, w, b), want)
            assert len(_ext._frozen.casts) == 2
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want)
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                ops.fused_linear(x, w, b)
            assert len(_ext._frozen.casts) == 2
        for _ in range(3):
            with mmcv_b200.frozen_weights():
                one, two = torch.cuda.Stream(), torch.cuda.Stream()
                torch.cuda.synchronize()
                with torch.cuda.stream(one):
                    torch.cuda._sleep(20_000_000)
                    ops.fused_linear(x, w, b)
                with torch.cuda.stream(two):
                    y = ops.fused_linear(x, w, b)
                torch.cuda.synchronize()
                assert torch.equal(y, want)


def test_kept_weight_images_and_captures(monkeypatch):
    """The same for the convolution's re-laid-out weights."""
    import mmcv_b200
    from mmcv_b200 import _ext
    monkeypatch.setattr(_ext, '_check_status', False)   # its reading waits, which a capture does not allow
    torch.manual_seed(5)
    layer = ops.ModulatedDeformConv2dPack(64, 64, 3, padding=1, deform_groups=2).cuda().bfloat16()
    x = torch.randn(2, 64, 24, 40, device='cuda', dtype=torch.bfloat16)
    with torch.no_grad():
        want = layer(x)
        with mmcv_b200.frozen_weights():
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = layer(x)
            assert all(image is None for _, image in _ext._frozen.images.values())
            assert torch.equal(layer(x), want)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want)


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_compile_runs_the_operators_between_its_graphs(backend):
    """torch.compile breaks its graph at the operators: new inputs give new results, and gradients."""
    x, w, b, _, _ = linear_case(40, 24, 24, torch.float32, None)

    def f(t):
        return ops.layer_norm(torch.relu(ops.fused_linear(t * 2, w, b)) * 3, (24,)) + t

    g = torch.compile(f, backend=backend)
    for seed in (1, 2):
        a, gy = tensors(seed, torch.float32, (40, 24), (40, 24))
        leaf, other = a.detach().requires_grad_(True), a.detach().requires_grad_(True)
        y, want = g(leaf), f(other)
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y, leaf, gy)[0], torch.autograd.grad(want, other, gy)[0])


def test_tracing_is_refused_on_the_device():
    x, w, b, _, _ = linear_case(40, 24, 24, torch.float32, None)
    with torch.no_grad(), pytest.raises(RuntimeError, match='tracing is not supported'):
        torch.jit.trace(lambda t: torch.relu(ops.fused_linear(t, w, b)) * 2, x)


class Adapter(torch.nn.Module):
    """A low-rank addition around a linear layer whose weight and bias it exposes."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.down = torch.nn.Linear(base.in_features, 2, bias=False)
        self.up = torch.nn.Linear(2, base.out_features, bias=False)

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return self.base(x) + self.up(self.down(x))


def altered_children(parent, name):
    """(what was done, how to undo it) of each way in which users change a child's call."""
    child = getattr(parent, name)
    seen = []
    handle = child.register_forward_hook(lambda m, a, out: out * 2)
    yield 'hook', handle.remove
    handle = child.register_forward_pre_hook(lambda m, a: (a[0] + 1,))
    yield 'pre-hook', handle.remove
    child.forward = lambda x: torch.nn.functional.linear(x, child.weight) * 3
    yield 'forward of its own', lambda: delattr(child, 'forward')
    torch.nn.utils.parametrizations.weight_norm(child)
    yield 'parametrization', lambda: torch.nn.utils.parametrize.remove_parametrizations(child, 'weight')
    setattr(parent, name, Adapter(child).cuda())
    yield 'adapter', lambda: setattr(parent, name, child)
    handle = torch.nn.modules.module.register_module_forward_hook(
        lambda m, a, out: out + 1 if m is child else None)
    yield 'hook on all modules', handle.remove
    handle = child.register_full_backward_hook(lambda m, gi, go: seen.append(1))
    yield 'backward hook', handle.remove
    assert seen


def test_children_of_the_block_are_called_where_they_were_changed():
    torch.manual_seed(0)
    x, gy = tensors(0, torch.float32, (2, 50, 64), (2, 50, 64))
    ffn = ops.FFN(64, 96, act_cfg=dict(type='GELU')).cuda()
    untouched = ffn(x)
    assert torch.equal(untouched, ops.feed_forward(x, ffn.layers[0][0].weight, ffn.layers[0][0].bias,
                                                   ffn.layers[1].weight, ffn.layers[1].bias, x, 'gelu'))
    for parent, name in ((ffn.layers[0], '0'), (ffn.layers, '1')):
        for what, undo in altered_children(parent, name):
            leaf = x.detach().requires_grad_(True)
            y = ffn(leaf)
            want = leaf + ffn.layers(leaf)
            assert torch.equal(y, want), (name, what)
            assert torch.isfinite(torch.autograd.grad(y, leaf, gy)[0]).all()
            undo()
        # the weight went through a norm and back: as good as untouched
        assert torch.allclose(ffn(x), untouched, atol=2e-5)
    for module in (ffn.layers, ffn.layers[0], ffn.layers[0][1], ffn.layers[2], ffn.dropout_layer):
        handle = module.register_forward_hook(lambda m, a, out: out * 2)
        assert torch.allclose(ffn(x), x + ffn.dropout_layer(ffn.layers(x)), atol=1e-4)
        assert not torch.allclose(ffn(x), untouched, atol=1e-2)
        handle.remove()
    ffn.layers[0][1] = torch.nn.SiLU()
    assert torch.equal(ffn(x), x + ffn.layers(x))
    ffn.layers[0] = torch.nn.Linear(64, 96).cuda()
    assert torch.equal(ffn(x), x + ffn.layers(x))
    ffn.layers = torch.nn.Identity()
    assert torch.equal(ffn(x), x + x)


@pytest.mark.parametrize('dtype', DTYPES)
def test_feed_forward_of_no_rows(dtype):
    _, _, w1, b1, w2, b2, _, _ = block_inputs(dtype)
    x = w1.new_empty(3, 0, 64)
    for act in (None, 'relu', 'gelu'):
        for same in (False, True):
            leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
            y = ops.feed_forward(*leaves, leaves[0] if same else None, act)
            grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
            assert y.shape == grads[0].shape == (3, 0, 64) and not any(g.any() for g in grads[1:])


def test_projections_of_the_attention_layer_are_called_where_they_were_changed():
    torch.manual_seed(1)
    layer = ops.MultiScaleDeformableAttention(64, 4, 2, 3, dropout=0., batch_first=True, fused_proj=True).cuda()
    q, = tensors(0, torch.float32, (2, 36, 64))
    kw = dict(reference_points=torch.rand(2, 36, 2, 2, device='cuda'), spatial_shapes=torch.tensor([[6, 5], [3, 2]]).cuda(),
              level_start_index=torch.tensor([0, 30]).cuda())
    for name in ('value_proj', 'sampling_offsets', 'attention_weights', 'output_proj'):
        for what, undo in altered_children(layer, name):
            leaf = q.detach().requires_grad_(True)
            y = layer(leaf, **kw)
            y.sum().backward()
            layer.fused_proj = False
            want = layer(q, **kw)
            layer.fused_proj = True
            assert torch.allclose(y, want, atol=1e-4), (name, what)
            undo()
    handle = layer.dropout.register_forward_hook(lambda m, a, out: out * 0)
    assert torch.equal(layer(q, **kw), q)
    handle.remove()


def test_dropouts_go_by_their_own_mode():
    """Dropouts switched on in a model that evaluates (sampling its uncertainty), or off in one that trains."""
    torch.manual_seed(0)
    x, = tensors(0, torch.float32, (2, 36, 64))
    kw = dict(reference_points=torch.rand(2, 36, 2, 2, device='cuda'), spatial_shapes=torch.tensor([[6, 5], [3, 2]]).cuda(),
              level_start_index=torch.tensor([0, 30]).cuda())
    ffn = ops.FFN(64, 96, ffn_drop=0.5, dropout_layer=dict(type='Dropout', drop_prob=0.5)).cuda()
    att = ops.MultiScaleDeformableAttention(64, 4, 2, 3, dropout=0.5, batch_first=True, fused_proj=True).cuda()
    for layer, call in ((ffn, lambda: ffn(x)), (att, lambda: att(x, **kw))):
        drops = [m for m in layer.modules() if isinstance(m, torch.nn.Dropout)]
        layer.eval()
        quiet = call()
        assert torch.equal(call(), quiet)
        for drop in drops:
            drop.train()
            assert not torch.equal(call(), call())
            drop.eval()
        layer.train()
        assert not torch.equal(call(), call())
        for drop in drops:
            drop.eval()
        assert torch.equal(call(), quiet)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows,cin,hidden', [(1, 16, 1024), (70, 40, 1000), (300, 48, 2048), (2048, 32, 2048), (2049, 32, 2048),
                                             (9001, 24, 520)])
def test_feed_forward_bias_gradient_by_the_number_of_hidden_values(rows, cin, hidden, dtype):
    """Summed before the hidden gradient's rounding up to 2^22 hidden values, whatever the width; after it
    beyond."""
    x, gy = tensors(1, dtype, (rows, cin), (rows, cin))
    w1, w2 = tensors(2, dtype, (hidden, cin), (cin, hidden), scale=(cin + hidden) ** -0.5)
    b1, b2 = tensors(3, dtype, (hidden,), (cin,), scale=0.1)
    z = plain.add(plain.product(plain.Value(x), plain.Value(w1)), b1.double())
    for act in ('relu', 'gelu'):
        gz = plain.through(plain.product(plain.Value(gy), plain.Value(w2).t()), z, act, kept=torch.float16)
        if rows * hidden > 2 ** 22:
            gz = gz.rounded(dtype)
        leaf = b1.detach().requires_grad_(True)
        g, = torch.autograd.grad(ops.feed_forward(x, w1, leaf, w2, b2, None, act), leaf, gy)
        hold({'gb1': g}, {'gb1': plain.column_sum(gz).rounded(dtype)})


def kept_slope_bound(z, dtype):
    """How far gelu's derivative at z (16-bit tensors, |z| <= 6) may be off as the backward pass has it.  Computed:
    |z| Phi(-|z|) within 0.0073 of half a step of fp16 (2^-11 of it, at least 2^-25), the density from an
    exponent of up to 26 with two roundings of 2^-24, and one addition.  Kept: 2^-16 if positive, else 2^-11 of it
    and 2^-30."""
    a = z.abs().clamp(min=1e-2)
    tail = 0.5 * torch.special.erfc(a / 2 ** 0.5)
    weighted = a * torch.exp(-a * a / 2) / (2 * torch.pi) ** 0.5
    slope = plain.activation(z, 'gelu')[1]
    computed = 0.0073 * torch.maximum(2.0 ** -11 * tail, 2.0 ** -25 / a) + 4e-6 * weighted + 2.0 ** -23 * (slope.abs() + tail + weighted)
    kept = torch.where(slope >= -computed, 2.0 ** -16, 2.0 ** -11 * slope.abs() + 2.0 ** -30)
    return slope, computed + kept


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows,cols', [(8, 8), (8, 9), (600, 8), (600, 9), (600, 264), (5000, 72)])
def test_kept_derivative_of_gelu_keeps_its_digits(rows, cols, dtype):
    """One element per row with a weight of one: gx is the derivative, rounded once.  Relative precision on the
    negative side as well, where the derivative falls to 4e-8 (gy lifts it out of fp16's subnormals), through
    every kernel that keeps or reads it."""
    z = torch.linspace(-6, 6, rows) if rows > 8 else torch.tensor([-6, -5.5, -5, -4.5, -4, -2, 0.5, 3])
    x = torch.zeros(rows, cols)
    x[:, 0] = z
    x = x.to(dtype).cuda()
    eye = torch.eye(cols, dtype=dtype, device='cuda')
    gy = torch.full((rows, cols), 16384.0, dtype=dtype, device='cuda')
    res = torch.zeros(rows, cols, dtype=dtype, device='cuda')
    zd = x[:, 0].double()
    slope, off = kept_slope_bound(zd, dtype)
    bound = off + plain.half_step(dtype) * (slope.abs() + off) + plain.floor_of(dtype) / 16384
    for f in (lambda t: ops.fused_linear(t, eye, activation='gelu'), lambda t: ops.fused_linear(t, eye, None, res, 'gelu'),
              lambda t: ops.feed_forward(t, eye, None, eye, None, None, 'gelu')):
        leaf = x.detach().requires_grad_(True)
        gx, = torch.autograd.grad(f(leaf), leaf, gy)
        over = ((gx[:, 0].double() / 16384 - slope).abs() / bound).max().item()
        assert over <= 1.0, over
        assert (gx[:, 0][zd < -1] < 0).all()


def test_kept_derivative_of_gelu_beyond_its_range():
    """Far on the negative side the derivative is 0, far on the positive one 1, and a NaN stays one."""
    inf = float('inf')
    z = torch.tensor([-7.0, -20.0, -1e4, -inf, 7.0, 20.0, 1e4, inf, float('nan')])
    for dtype in (torch.bfloat16, torch.float16):
        for rows in (9, 300):
            x = torch.zeros(rows, 8)
            x[:9, 0] = z
            x = x.to(dtype).cuda().requires_grad_(True)
            w = torch.zeros(8, 8, dtype=dtype, device='cuda')
            w[:, 0] = 1
            y = ops.fused_linear(x, w, activation='gelu')
            gx, = torch.autograd.grad(y, x, torch.ones_like(y))
            assert gx[:8, 0].tolist() == [0, 0, 0, 0, 8, 8, 8, 8] and torch.isnan(gx[8, 0])


def test_fp32_products_keep_fp32_accuracy_element_by_element():
    """Sums of one product each, on the tensor cores.  Three planes of 8 bits rounded to nearest leave out at
    most 2^-24 + 2^-34 of the product; adding the small products to the leading one (exact: 16 bits) rounds by
    2^-24, the small ones' own sum by five truncations of 2^-23 at 2^-7 of it: 2.5 * 2^-24 in all, and the error has no
    sign."""
    rows, cin, cout = 2048, 64, 1024
    gen = torch.Generator().manual_seed(0)

    def values(n):
        v = (1 + torch.rand(n, generator=gen)) * torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0)
        v[:4] = torch.tensor([0x3f80ffff, 0x3f807fff, 0x3f808001, 0x3fffffff], dtype=torch.int32).view(torch.float32)
        return v.cuda()

    def check(got, p, q):
        want = p.double()[:, None] * q.double()[None, :]
        rel = got.double() / want - 1
        assert rel.abs().max().item() <= 2.5 * 2.0 ** -24, rel.abs().max().item() * 2 ** 24
        assert abs(rel.mean().item()) <= 0.1 * 2.0 ** -24, rel.mean().item() * 2 ** 24

    x, w, gy = (torch.zeros(s, device='cuda') for s in ((rows, cin), (cout, cin), (rows, cout)))
    p, q = values(rows), values(cout)
    x[:, 3], w[:, 3] = p, q
    check(ops.fused_linear(x, w), p, q)
    x = torch.randn(rows, cin, device='cuda').requires_grad_(True)
    w = torch.zeros(cout, cin, device='cuda')
    k = values(cin)
    w[5], gy[:, 5] = k, p
    check(torch.autograd.grad(ops.fused_linear(x, w), x, gy)[0], p, k)
    x, gy, w = torch.zeros(rows, cin, device='cuda'), torch.zeros(rows, cout, device='cuda'), w.requires_grad_(True)
    x[7], gy[7] = k, q
    check(torch.autograd.grad(ops.fused_linear(x, w), w, gy)[0], q, k)


def test_fp32_largest_values():
    """The largest and the lowest finite value, and a little below, stay what they are."""
    big = torch.finfo(torch.float32).max
    x = torch.zeros(2048, 64, device='cuda')
    x[:, 0] = torch.tensor([big, -big, big / 2 * 1.999, 3.396e38, 3.397e38, 3.39e38, -3.4e38, 1e38]).repeat(256).cuda()
    w = torch.zeros(1024, 64, device='cuda')
    w[:, 0] = 1
    y = ops.fused_linear(x, w)
    assert torch.isfinite(y).all()
    assert (y.double() / x[:, :1].double() - 1).abs().max().item() <= 2.5 * 2.0 ** -24


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_lazily_negated_views_have_their_sign(dtype):
    """Inputs, parameters, residuals and gradients whose memory holds the opposite sign."""
    lazy = torch._neg_view
    x, gy, w1, b1, w2, b2, g, b = block_inputs(dtype)
    half = lazy(x)
    assert half.is_neg() and torch.equal(half, -x)
    cases = [(lambda n, t, w, c, r: ops.fused_linear(n(t), n(w), n(c), n(r), 'gelu'), (x, w1, b1, gy.new_ones(70, 96))),
             (lambda n, t, w, c, r: ops.feed_forward(n(t), n(w), n(c), n(r), None, None, 'gelu'), (x, w1, b1, w2)),
             (lambda n, t, w, c, r: ops.feed_forward(t, n(w), n(c), n(r), None, t), (lazy(x), w1, b1, w2)),
             (lambda n, t, w, c, r: ops.layer_norm(n(t), (64,), n(w), n(c)) + r, (x, g, b, x)),
             (lambda n, t, w, c, r: ops.fused_linear(n(t), n(w), n(c)) + r, (x[:, :1], w1[:, :1], b1, gy.new_ones(70, 96)))]
    for f, given in cases:
        out = []
        for n, flip in ((lambda t: -t, lambda t: -t), (lazy, lazy)):
            leaves = [t.detach().clone().requires_grad_(True) if not t.is_neg() else t.detach().requires_grad_(True)
                      for t in given]
            y = f(n, *leaves)
            dy = tensors(8, dtype, y.shape)[0]
            out.append([y.detach(), *torch.autograd.grad(y, leaves, flip(dy))])
        assert all(torch.equal(p, q) for p, q in zip(*out))
    w = torch.randn(1, 64, device='cuda')       # a gradient of one column that autograd itself negates lazily
    leaf = torch.randn(70, 64, device='cuda', requires_grad=True)
    y = ops.fused_linear(leaf, w)
    torch.complex(y * 0, y).conj().imag.sum().backward()
    assert torch.equal(leaf.grad, -w.expand(70, 64))


def test_autocast_leaves_other_types_to_their_refusal():
    """autocast does not touch fp64 or whole numbers; the operators refuse them there as elsewhere."""
    x, w, b, r, _ = linear_case(20, 24, 24, torch.float32, None)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        for t in (x.double(), x.int(), x.bool()):
            for f in (lambda: ops.fused_linear(t, w), lambda: ops.fused_linear(x, t), lambda: ops.fused_linear(x, w, t[0]),
                      lambda: ops.feed_forward(t, w, b, w, b), lambda: ops.feed_forward(x, w, b, t, b),
                      lambda: ops.layer_norm(t, (24,)), lambda: ops.layer_norm(x, (24,), t[0])):
                with pytest.raises(RuntimeError, match='dtype'):
                    f()
        assert ops.fused_linear(x.half(), w, b).dtype == torch.bfloat16
        # a residual of another type is added outside, whatever it is
        y = ops.fused_linear(x, w, b, r.double())
        assert y.dtype == torch.float64
        assert torch.equal(y, ops.fused_linear(x, w, b) + r.double())
