"""The transformer-layer operators without a GPU: refusals, argument checks of the C entries, layer
construction, and the 64-bit forms against torch."""
import ctypes

import pytest
import torch

from mmcv_b200 import _lib, ops
from oracle import layers as plain


def test_cpu_tensors_fail_loudly():
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        ops.fused_linear(x, w)
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        ops.feed_forward(x, w, None, torch.randn(4, 5), None)
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        ops.layer_norm(x, (4,))
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        ops.FFN(4, 8)(x)


def test_types_and_names_are_checked():
    with pytest.raises(RuntimeError, match='unsupported dtype'):
        ops.fused_linear(torch.randn(3, 4).double(), torch.randn(5, 4).double())
    with pytest.raises(RuntimeError, match='unsupported dtype'):
        ops.layer_norm(torch.randn(3, 4).double(), (4,))
    for bad in ('silu', 1, []):
        with pytest.raises(ValueError, match='unknown activation'):
            ops.fused_linear(torch.randn(3, 4), torch.randn(5, 4), activation=bad)
    with pytest.raises(ValueError, match='unknown activation'):
        ops.FusedLinear(4, 4, activation='tanh')
    for kw in (dict(num_fcs=3), dict(act_cfg=dict(type='SiLU')), dict(dropout_layer=dict(type='DropPath'))):
        with pytest.raises(ValueError):
            ops.FFN(4, 8, **kw)


def test_c_entries_reject_bad_arguments_without_a_device():
    lib = _lib.load()
    n = ctypes.c_size_t(0)

    def last():
        return lib.dcn_last_error().decode()

    assert lib.dcn_linear_workspace_bytes(7, 1, 8, 8, 0, ctypes.byref(n)) == -2
    assert lib.dcn_linear_workspace_bytes(1, 1, 0, 8, 0, ctypes.byref(n)) == -1 and 'positive' in last()
    assert lib.dcn_linear_workspace_bytes(1, -1, 8, 8, 0, ctypes.byref(n)) == -1
    assert lib.dcn_linear_workspace_bytes(1, 1, 8, 1 << 21, 0, ctypes.byref(n)) == -2
    assert lib.dcn_linear_workspace_bytes(1, 1, 8, 8, 0, None) == -1
    assert lib.dcn_linear_backward_workspace_bytes(1, 9, 1, 8, 8, 0, 1, 1, 1, ctypes.byref(n)) == -1
    p = 4096   # never dereferenced: the checks come first
    fwd = lib.dcn_linear_forward
    assert fwd(None, 8, p, 8, None, None, 0, p, None, 1, 0, 4, 8, 8, 0, None, 0, None) == -1 and 'non-NULL' in last()
    assert fwd(p, 7, p, 8, None, None, 0, p, None, 1, 0, 4, 8, 8, 0, None, 0, None) == -1 and 'stride' in last()
    assert fwd(p, 8, p, 8, None, p, 7, p, None, 1, 0, 4, 8, 8, 0, None, 0, None) == -1 and 'stride' in last()
    assert fwd(p, 8, p, 8, None, None, 0, p, None, 1, 1, 4, 8, 8, 0, None, 0, None) == -1 and 'activation' in last()
    assert fwd(None, 8, None, 8, None, None, 0, None, None, 1, 0, 0, 8, 8, 0, None, 0, None) == 0   # no rows
    norm = lib.dcn_layer_norm_forward
    assert norm(None, 8, None, None, p, None, 0, 0, 4, 8, 1e-5, 0, None) == -1
    assert norm(p, 7, None, None, p, None, 0, 0, 4, 8, 1e-5, 0, None) == -1 and 'stride' in last()
    assert norm(p, 8, None, None, p, None, 0, 1, 4, 8, 1e-5, 0, None) == -1 and 'type' in last()
    assert norm(p, 8, None, None, p, None, 5, 5, 4, 8, 1e-5, 0, None) == -2
    assert norm(p, 0, None, None, p, None, 0, 0, 4, 0, 1e-5, 0, None) == -1
    assert lib.dcn_layer_norm_workspace_bytes(10, 16, ctypes.byref(n)) == 0 and n.value >= 10 * 2 * 16 * 4


def test_plain_forms_against_torch():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).float()   # noqa: E731
    x, w, b, res, gy = r(7, 5), r(6, 5), r(6), r(7, 6), r(7, 6)
    for act, f in ((None, lambda t: t), ('relu', torch.relu), ('gelu', torch.nn.functional.gelu)):
        leaves = [t.double().requires_grad_(True) for t in (x, w, b)]
        y = f(torch.nn.functional.linear(*leaves)) + res.double()
        grads = torch.autograd.grad(y, leaves, gy.double())
        out = plain.linear(x, w, b, res, act, gy)
        for key, ref in zip(('y', 'gx', 'gw', 'gb'), (y, *grads)):
            assert torch.allclose(out[key].v, ref.detach(), rtol=1e-12, atol=1e-12)
    w2, b2, gx = r(5, 6), r(5), r(7, 5)
    leaves = [t.double().requires_grad_(True) for t in (x, w, b, w2, b2)]
    y = torch.nn.functional.linear(torch.relu(torch.nn.functional.linear(*leaves[:3])), *leaves[3:]) + x.double()
    grads = torch.autograd.grad(y, leaves, gx.double())
    out = plain.feed_forward(x, w, b, w2, b2, x, 'relu', gx)
    for key, ref in zip(('y', 'gx', 'gw1', 'gb1', 'gw2', 'gb2'), (y, *grads)):
        assert torch.allclose(out[key].v, ref.detach(), rtol=1e-12, atol=1e-12)
    g, c = r(5), r(5)
    leaves = [t.double().requires_grad_(True) for t in (x, g, c)]
    y = torch.nn.functional.layer_norm(leaves[0], (5,), leaves[1], leaves[2], 1e-5)
    grads = torch.autograd.grad(y, leaves, gx.double())
    out = plain.layer_norm(x, g, c, 1e-5, gx)
    for key, ref in zip(('y', 'gx', 'gw', 'gb'), (y, *grads)):
        assert torch.allclose(out[key].v, ref.detach(), rtol=1e-12, atol=1e-12)


def test_layer_parameters_carry_the_reference_names():
    layer = ops.DeformableEncoderLayer(32, num_heads=4, num_levels=2, num_points=2, feedforward_channels=48)
    names = set(layer.state_dict())
    assert {'attentions.0.value_proj.weight', 'ffns.0.layers.0.0.weight', 'ffns.0.layers.1.bias', 'norms.0.weight',
            'norms.1.bias'} <= names
    assert layer.attentions[0].fused_proj and layer.ffns[0].feedforward_channels == 48
    with pytest.raises(ValueError, match='divisible'):
        ops.DeformableEncoderLayer(30, num_heads=4)


def test_kept_casts_tell_layouts_apart():
    """frozen_weights(): a square weight and its transpose, and two views from one start, are different weights."""
    import mmcv_b200
    from mmcv_b200 import _ext
    w = torch.randn(8, 8)
    with torch.no_grad(), mmcv_b200.frozen_weights():
        for t in (w, w.t(), w[:4], w[::2], w.t()[:4], torch._neg_view(w)):
            for _ in range(2):
                assert torch.equal(_ext.cast_weight(t, torch.bfloat16), t.to(torch.bfloat16))
        assert _ext.cast_weight(w.t(), torch.bfloat16) is _ext.cast_weight(w.t(), torch.bfloat16)


def traced_calls():
    return [lambda t: ops.fused_linear(t, t), lambda t: ops.feed_forward(t, t, None, t, None, t),
            lambda t: ops.layer_norm(t, (4,))]


def test_tracing_is_refused():
    """A traced program would keep the example's results; the check stands before those on devices."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 4)
    for f in traced_calls():
        with torch.no_grad(), pytest.raises(RuntimeError, match='tracing is not supported'):
            torch.jit.trace(lambda t: torch.relu(f(t)) * 2, x)   # noqa: B023
        for mode in ('real', 'fake'):
            with pytest.raises(RuntimeError, match='tracing is not supported'):
                make_fx(lambda t: f(t) * 2 + t, tracing_mode=mode)(x)   # noqa: B023


def test_export_is_refused():
    class Model(torch.nn.Module):
        def __init__(self, f):
            super().__init__()
            self.f = f

        def forward(self, t):
            return torch.relu(self.f(t)) * 2

    for f in traced_calls():
        with pytest.raises(RuntimeError, match='tracing is not supported'):
            torch.export.export(Model(f), (torch.randn(4, 4),), strict=False)


def test_import_leaves_a_registered_ffn_alone():
    """Configurations that name 'FFN' build what they built before: a stand-in for the registry package."""
    import os
    import subprocess
    import sys
    code = ("import sys, types\n"
            "class Registry(dict):\n"
            "    def register_module(self, name=None, force=False, module=None):\n"
            "        assert force or name not in self\n"
            "        self[name] = module\n"
            "package, registry = types.ModuleType('mmengine'), types.ModuleType('mmengine.registry')\n"
            "registry.MODELS = package.MODELS = Registry(FFN='theirs')\n"
            "package.registry = registry\n"
            "sys.modules.update({'mmengine': package, 'mmengine.registry': registry})\n"
            "import mmcv_b200.ops\n"
            "assert registry.MODELS['FFN'] == 'theirs', registry.MODELS\n"
            "assert {'DCN', 'DCNv2', 'MultiScaleDeformableAttention'} <= set(registry.MODELS)\n"
            "print('done')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'done' in r.stdout, r.stdout + r.stderr


def test_ffn_options_that_it_does_not_have_are_refused():
    for kw in (dict(act_cfg=dict(type='GELU', approximate='tanh')), dict(act_cfg=dict(type='ReLU', negative_slope=0.1)),
               dict(act_cfg=dict(type='GELU', inplace=True)), dict(dropout_layer=dict(type='Dropout', p=0.1))):
        with pytest.raises(ValueError):
            ops.FFN(4, 8, **kw)
    for kw in (dict(act_cfg=dict(type='ReLU', inplace=True)), dict(act_cfg=dict(type='GELU', approximate='none')),
               dict(act_cfg=dict(type='GELU')), dict(dropout_layer=dict(type='Dropout', drop_prob=0.1, inplace=True)),
               dict(dropout_layer=dict(type='Dropout')), dict(act_cfg={})):
        ops.FFN(4, 8, **kw)


def run_python(code):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'done' in r.stdout, r.stdout + r.stderr


def test_only_the_layer_operators_need_the_tensor_front():
    """Without it the package imports, other layers are built, and these operators say what is missing."""
    run_python("import os, torch\n"
               "real = os.path.exists\n"
               "os.path.exists = lambda p: '_layers_native' not in str(p) and real(p)\n"
               "from mmcv_b200 import ops\n"
               "ops.ModulatedDeformConv2dPack(8, 8, 3), ops.MultiScaleDeformableAttention(32, 4), ops.DeformableEncoderLayer(32, 4)\n"
               "for f in (lambda: ops.fused_linear(torch.ones(2, 2), torch.ones(2, 2)), lambda: ops.layer_norm(torch.ones(2, 2), 2)):\n"
               "    try:\n"
               "        f()\n"
               "        raise SystemExit('no error')\n"
               "    except ImportError as e:\n"
               "        assert 'build_ext' in str(e)\n"
               "print('done')\n")


def test_status_flag_reaches_a_tensor_front_loaded_later():
    run_python("from mmcv_b200 import _ext, _layers\n"
               "_ext.set_check_status(True)\n"
               "assert 'native' not in vars(_layers) and not _ext._status_listeners\n"
               "_layers.native\n"
               "assert 'native' in vars(_layers) and len(_ext._status_listeners) == 1\n"
               "_ext.set_check_status(False)\n"
               "print('done')\n")


def test_the_tensor_front_is_this_torch_s():
    """Another torch (or Python) has a file of its own: it is neither loaded nor counted as built."""
    import sys
    from mmcv_b200 import _layers, build_ext
    assert _layers.NATIVE_PATH == build_ext.binding_path()
    assert torch.__version__.replace('+', '_') in _layers.NATIVE_PATH and sys.implementation.cache_tag in _layers.NATIVE_PATH
    run_python("import torch\n"
               "torch.__version__ = '0.0.1+other'\n"
               "from mmcv_b200 import _layers\n"
               "try:\n"
               "    _layers.native\n"
               "except ImportError as e:\n"
               "    assert '0.0.1_other' in str(e) and 'build_ext' in str(e)\n"
               "    print('done')\n")
