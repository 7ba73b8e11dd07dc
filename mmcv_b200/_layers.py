"""Loads ``lib/_layers_native.*.so``, the C++ tensor front of the transformer-layer entries of the library
(``dcn_linear_*``, ``dcn_layer_norm_*``; mmcv_b200/csrc/layers_binding.cpp): argument checks, row
strides, workspaces, streams and autograd nodes.  ``mmcv_b200.ops`` documents the operators.

There is no fallback: if the module is missing, the first call of such an operator raises.
"""
import importlib.machinery
import importlib.util
import os
import threading

import torch
import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from . import _ext, _lib, build_ext

ACTIVATIONS = {None: _lib.ACT_NONE, 'relu': _lib.ACT_RELU, 'gelu': _lib.ACT_GELU}
NATIVE_PATH = build_ext.binding_path()   # of this Python and torch


def _load():
    _lib.load()   # the library that the module calls; raises if it is missing or of another version
    if not os.path.exists(NATIVE_PATH):
        raise ImportError(f'{NATIVE_PATH} is missing: build it with `python -m mmcv_b200.build_ext` '
                          '(there is no fallback implementation)')
    loader = importlib.machinery.ExtensionFileLoader('_layers_native', NATIVE_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader('_layers_native', loader))
    loader.exec_module(module)
    return module


_loading = threading.Lock()


def __getattr__(name):
    # `native` at its first use: the convolutions and the sampler need the C library only
    if name != 'native':
        raise AttributeError(f'module {__name__!r} has no attribute {name!r}')
    with _loading:
        if name not in globals():
            module = _load()
            module.set_check_status(_ext._check_status)
            _ext._status_listeners.append(module.set_check_status)
            globals()[name] = module
    return globals()[name]


def activation_code(name):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {name!r} (None, 'relu' and 'gelu' are available)") from None


def autocast_dtype():
    """The type that an active autocast wants for a matrix product, or None."""
    return torch.get_autocast_dtype('cuda') if torch.is_autocast_enabled('cuda') else None


_CAST = (torch.float32, torch.bfloat16, torch.float16)


def autocast(t, dtype):
    """t as an active autocast hands it on: fp64 and whole numbers stay, and are refused, as without it."""
    return t.to(dtype) if t is not None and t.dtype in _CAST else t


def autocast_weight(t, dtype):
    return _ext.cast_weight(t, dtype) if t is not None and t.dtype in _CAST else t


def untouched(*pairs):
    """Whether, for each (module, kind), a call of the module is `kind`'s forward on its parameters and nothing
    besides: the very type (no adapter, no parametrization), no hooks, no forward of its own.  Only then may a
    layer take its child's parameters instead of calling it."""
    if _has_any_global_hook():
        return False
    for module, kind in pairs:
        if type(module) is not kind or 'forward' in module.__dict__ or module._forward_hooks or \
                module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks:
            return False
    return True


def passes_on(*dropouts):
    """Whether dropouts hand their input on: by their own mode, which need not be their parent's."""
    for drop in dropouts:
        if type(drop) is nn.Dropout and drop.p and drop.training:
            return False
    return untouched(*((drop, nn.Identity if type(drop) is nn.Identity else nn.Dropout) for drop in dropouts))
