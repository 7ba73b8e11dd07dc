"""Binding of the transformer-layer entries of the library (``dcn_linear_*``, ``dcn_layer_norm_*``):
argument checks, row strides, workspaces and streams.  The differentiable functions and layers on
top of it are in ``mmcv_b200.ops``.
"""
import ctypes
import functools

import torch

from . import _ext, _lib

ACTIVATIONS = {None: _lib.ACT_NONE, 'relu': _lib.ACT_RELU, 'gelu': _lib.ACT_GELU}
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_raw_stream = torch._C._cuda_getCurrentRawStream


def activation_code(name):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {name!r} (None, 'relu' and 'gelu' are available)") from None


def require(op, dtype, device, **tensors):
    """Every given tensor is a CUDA tensor of this type on this device."""
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f'dcn_b200: {op}: {name} must be a CUDA tensor (this build has no CPU '
                               'implementation)')
        if t.device != device:
            raise RuntimeError(f'dcn_b200: {op}: {name} is on {t.device}, expected {device}')
        if t.dtype != dtype:
            raise RuntimeError(f'dcn_b200: {op}: {name} has dtype {t.dtype}, expected {dtype}')


def dtype_code(op, dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        raise RuntimeError(f'dcn_b200: {op}: unsupported dtype {dtype} (float32, bfloat16 and float16 only)')
    return code


def as_rows(t, cols):
    """(t as [rows, cols] with neighbouring columns next to each other in memory, its row stride).
    Anything that a row stride can describe is taken as it lies; the rest is copied."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    sr, sc = t.stride()
    if (sc != 1 and cols > 1) or (sr < cols and t.size(0) > 1):
        t = t.contiguous()
        sr = cols
    return t, (sr if t.size(0) > 1 else cols)


def _ptr(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _linear_bytes(code, rows, cin, cout, alignment):
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().dcn_linear_workspace_bytes(code, rows, cin, cout, alignment, ctypes.byref(n)))
    return n.value


@functools.lru_cache(maxsize=4096)
def _linear_backward_bytes(code, act, rows, cin, cout, alignment, want_gx, want_gw):
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().dcn_linear_backward_workspace_bytes(code, act, rows, cin, cout, alignment, want_gx,
                                                               want_gw, ctypes.byref(n)))
    return n.value


@functools.lru_cache(maxsize=4096)
def _norm_bytes(rows, cols):
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().dcn_layer_norm_workspace_bytes(rows, cols, ctypes.byref(n)))
    return n.value


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _check_waits(device):
    status = ctypes.c_int32(0)
    _lib.check(_lib.load().dcn_linear_read_status(device.index, _raw_stream(device.index), ctypes.byref(status)))
    if status.value:
        raise RuntimeError(f'dcn_b200: device-side wait {status.value} timed out; the output is not valid')


def linear_forward(x, weight, bias, residual, act, save):
    """act(x weight^T + bias) + residual of checked tensors; with `save`, what the activation's
    derivative needs as well.  Returns (y, saved)."""
    lib = _lib.load()
    code, dev, esize = _DTYPES[x.dtype], x.device, x.element_size()
    cout, cin = weight.shape
    x2, ldx = as_rows(x, cin)
    w2, ldw = as_rows(weight, cin)
    rows = x2.size(0)
    y = x.new_empty(x.shape[:-1] + (cout,))
    r2, ldr = (None, 0) if residual is None else as_rows(residual, cout)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    saved = None
    if save and act == _lib.ACT_RELU:
        saved = torch.empty((rows, (cout + 31) // 32), dtype=torch.int32, device=dev)
    elif save and act == _lib.ACT_GELU:
        saved = x.new_empty((rows, (cout + 7) // 8 * 8))
    xp, wp = x2.data_ptr(), w2.data_ptr()
    nbytes = _linear_bytes(code, rows, cin, cout, (xp | wp | (ldx | ldw) * esize) & 15)
    ws = _workspace(nbytes, dev)
    _lib.check(lib.dcn_linear_forward(xp, ldx, wp, ldw, _ptr(bias), _ptr(r2), ldr, y.data_ptr(), _ptr(saved),
                                      code, act, rows, cin, cout, dev.index, _ptr(ws), nbytes,
                                      _raw_stream(dev.index)))
    if _ext._check_status:
        _check_waits(dev)
    return y, saved


def linear_backward(gy, x, weight, saved, act, want, in_saved=None, in_act=_lib.ACT_NONE, gx_add=None,
                    x_shape=None):
    """The gradients of linear_forward that `want` = (x, weight, bias) asks for.  in_saved / in_act:
    the gradient of x is taken on through the activation that made x; gx_add is added to it."""
    lib = _lib.load()
    code, dev, esize = _DTYPES[gy.dtype], gy.device, gy.element_size()
    cout = gy.shape[-1]
    g2, ldg = as_rows(gy, cout)
    rows = g2.size(0)
    cin = weight.shape[1] if weight is not None else x.shape[-1]
    x2, ldx = as_rows(x, cin) if want[1] else (None, cin)
    w2, ldw = as_rows(weight, cin) if want[0] else (None, cin)
    gx = gy.new_empty(x_shape) if want[0] else None
    gw = gy.new_empty((cout, cin)) if want[1] else None
    gb = gy.new_empty((cout,)) if want[2] else None
    if gx_add is not None:
        gx_add = gx_add.contiguous()
    gp, xp, wp = g2.data_ptr(), _ptr(x2), _ptr(w2)
    nbytes = _linear_backward_bytes(code, act, rows, cin, cout,
                                    (gp | (xp or 0) | (wp or 0) | (ldg | ldx | ldw) * esize) & 15, int(want[0]),
                                    int(want[1]))
    ws = _workspace(nbytes, dev)
    _lib.check(lib.dcn_linear_backward(gp, ldg, xp, ldx, wp, ldw, _ptr(saved), _ptr(in_saved), _ptr(gx_add),
                                       _ptr(gx), _ptr(gw), _ptr(gb), code, act, in_act, rows, cin, cout,
                                       dev.index, _ptr(ws), nbytes, _raw_stream(dev.index)))
    if _ext._check_status:
        _check_waits(dev)
    return gx, gw, gb


def norm_forward(x, weight, bias, cols, eps, save):
    """Layer norm over the last `cols` elements.  Returns (y, stats or None)."""
    lib = _lib.load()
    code, dev = _DTYPES[x.dtype], x.device
    x2, ldx = as_rows(x, cols)
    rows = x2.size(0)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats = torch.empty((3, rows), dtype=torch.float32, device=dev) if save else None
    p = weight if weight is not None else bias
    wcode = code if p is None else _DTYPES[p.dtype]
    _lib.check(lib.dcn_layer_norm_forward(x2.data_ptr(), ldx, _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(stats),
                                          code, wcode, rows, cols, eps, dev.index, _raw_stream(dev.index)))
    return y, stats


def norm_backward(gy, x, weight, stats, cols, want, wdtype):
    """The gradients of norm_forward that `want` = (x, weight, bias) asks for (flat, [cols], for the
    last two)."""
    lib = _lib.load()
    code, dev = _DTYPES[x.dtype], x.device
    g2, ldg = as_rows(gy, cols)
    x2, ldx = as_rows(x, cols)
    rows = x2.size(0)
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want[0] else None
    gw = torch.empty(cols, dtype=wdtype, device=dev) if want[1] else None
    gb = torch.empty(cols, dtype=wdtype, device=dev) if want[2] else None
    nbytes = _norm_bytes(rows, cols) if want[1] or want[2] else 0
    ws = _workspace(nbytes, dev)
    _lib.check(lib.dcn_layer_norm_backward(g2.data_ptr(), ldg, x2.data_ptr(), ldx, _ptr(weight), stats.data_ptr(),
                                           _ptr(gx), _ptr(gw), _ptr(gb), code, _DTYPES[wdtype], rows, cols,
                                           dev.index, _ptr(ws), nbytes, _raw_stream(dev.index)))
    return gx, gw, gb


def autocast_dtype(*tensors):
    """The type that an active autocast wants for a matrix product of these tensors, or None."""
    if not torch.is_autocast_enabled('cuda'):
        return None
    return torch.get_autocast_dtype('cuda')


cast_weight = _ext.cast_weight
