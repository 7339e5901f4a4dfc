"""Root-mean-square norm with the residual's addition: autograd wrapper over
the HIP library (kernels/rms_norm.hip).

``rms_norm`` is the norm in front of a transformer's layers, forward and
backward; ``rms_norm_quantized`` the same for inference, with its output in
8 bits as a block-scaled product reads it.  There is no CPU path: without a GPU
the library refuses to load.
"""

import functools
import os

import torch

from framework import capi, e4m3
from framework.loader import load_kernel
from framework.once import differentiated, once

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "rms_norm_hip"
SOURCES = ["rms_norm.hip"]


def bind_library(lib):
    V, I64, I, F, S = capi.c_void_p, capi.c_int64, capi.c_int, capi.c_float, capi.c_size_t
    rows = [V, I, I64, V, I, I64, V, I]
    capi.bind(lib, "rms_norm_forward", rows + [V, V, V, I64, I64, F, V])
    capi.bind(lib, "rms_norm_quant", rows + [V, I64, V, I, V, I64, I64, F, V])
    capi.bind(lib, "rms_norm_backward_workspace_bytes", [I64, I64], S)
    capi.bind(lib, "rms_norm_backward",
              [V, I, I64, V, I, I64, V, I64, V, I, V, V, V, V, I64, I64, V, S, V])
    capi.bind_last_error(lib, "rms_norm_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows, D):
    return _lib().rms_norm_backward_workspace_bytes(rows, D)


def _check(x, weight, residual):
    device, shape = x.get_device(), x.shape
    # the common case in one expression; what is wrong with another is said below
    if (device >= 0 and weight.get_device() == device and shape and shape[-1] >= 1 and
            weight.shape == shape[-1:] and x.dtype in e4m3.DTYPES and weight.dtype in e4m3.DTYPES and
            (residual is None or residual.get_device() == device and residual.shape == shape and
             (residual.dtype == x.dtype or residual.dtype == torch.float32))):
        return device
    capi.require(device >= 0 and weight.is_cuda and (residual is None or residual.is_cuda),
                 "x, weight and residual must be GPU tensors")
    capi.require(weight.get_device() == device and
                 (residual is None or residual.get_device() == device),
                 "weight and residual must be on the GPU of x")
    capi.require(x.dtype in e4m3.DTYPES and weight.dtype in e4m3.DTYPES,
                 "x and weight must be float32, bfloat16 or float16")
    capi.require(len(shape) >= 1 and shape[-1] >= 1 and weight.shape == shape[-1:],
                 "x must be [..., D] with D >= 1 and weight [D]")
    raise RuntimeError("residual must have x's shape, and its type or float32")


def _inputs(x, weight, residual):
    """What the C entries take of x, the residual and the weight, the tensors that they read, and
    the rows."""
    x, rows, D, stride = e4m3.rows_of(x)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if residual is None:
        r, r_ptr, r_type, r_stride = None, 0, 0, 0
    else:
        r, _, _, r_stride = e4m3.rows_of(residual)
        r_ptr, r_type = r.data_ptr(), e4m3.DTYPES[r.dtype]
    return ((x.data_ptr(), e4m3.DTYPES[x.dtype], stride, r_ptr, r_type, r_stride,
             weight.data_ptr(), e4m3.DTYPES[weight.dtype]), (x, weight, r), rows, D)


def _dense(t):
    """A dense tensor of t's shape and type beside it."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _forward(x, weight, residual, eps, keep):
    """(y, h or None, rstd or None, weight as read)."""
    device = _check(x, weight, residual)
    lib = _lib()
    args, held, rows, D = _inputs(x, weight, residual)
    y = _dense(x)
    h = None if residual is None else _dense(residual)
    rstd = x.new_empty(rows, dtype=torch.float32) if keep else None
    st = capi.launch(lib.rms_norm_forward, device, *args, y.data_ptr(),
                     0 if h is None else h.data_ptr(), rstd.data_ptr() if keep else 0, rows, D,
                     eps)
    if st:
        capi.check(st, lib.rms_norm_last_error, "rms_norm")
    return y, h, rstd, held[1]


def _backward(dy, dh, h, weight, rstd, dtype, want_weight):
    """(dx, dresidual, dweight): dx of ``dtype``, dresidual of h's type."""
    lib = _lib()
    shape, device = h.shape, h.get_device()
    h, rows, D, h_stride = e4m3.rows_of(h)
    # what autograd gives back of what was saved: every read lies within it
    capi.require(0 <= device == weight.get_device() == rstd.get_device() and
                 weight.numel() == D and rstd.numel() == rows and rstd.dtype == torch.float32 and
                 dy.dtype == dtype and (dh is None or dh.dtype == h.dtype),
                 "autograd gave back other tensors than were saved")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if not rstd.is_contiguous():
        rstd = rstd.contiguous()
    dy, _, _, dy_stride = e4m3.rows_of(dy)
    dh_ptr = dh_stride = 0
    if dh is not None:
        dh, _, _, dh_stride = e4m3.rows_of(dh)
        dh_ptr = dh.data_ptr()
    dx = _dense(dy)
    dres = dx if h.dtype == dtype else h.new_empty(shape)
    dw_ptr = ws_ptr = ws_bytes = 0
    dw = None
    if want_weight:
        dw = torch.empty_like(weight)
        ws_bytes = _workspace_bytes(rows, D)
        ws = rstd.new_empty(max(ws_bytes, 16) // 4)
        dw_ptr, ws_ptr = dw.data_ptr(), ws.data_ptr()
    types = e4m3.DTYPES
    st = capi.launch(lib.rms_norm_backward, device, dy.data_ptr(), types[dtype], dy_stride,
                     h.data_ptr(), types[h.dtype], h_stride, dh_ptr, dh_stride, weight.data_ptr(),
                     types[weight.dtype], rstd.data_ptr(), dx.data_ptr(),
                     0 if dres is dx else dres.data_ptr(), dw_ptr, rows, D, ws_ptr, ws_bytes)
    if st:
        capi.check(st, lib.rms_norm_last_error, "rms_norm backward")
    return dx, dres, dw


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, h, rstd, weight = _forward(x, weight, residual, eps, True)
        ctx.dtype, ctx.summed = x.dtype, residual is not None
        ctx.save_for_backward(h if ctx.summed else x, weight, rstd)
        return (y, h) if ctx.summed else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        if dy is None and dh is None:
            return None, None, None, None
        h, weight, rstd = ctx.saved_tensors
        if dy is None:      # the norm itself has no part in the answer
            dy = torch.zeros(h.shape, dtype=ctx.dtype, device=h.device)
        capi.require(dy.shape == h.shape and (dh is None or dh.shape == h.shape),
                     "autograd gave back other tensors than were saved")
        dx, dres, dw = _backward(dy, dh, h, weight, rstd, ctx.dtype, ctx.needs_input_grad[1])
        return *once("rms_norm", dx, dw, dres if ctx.summed else None), None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, of x's type;
    with a residual (y, h), h = x + residual rounded to the residual's type, else
    h = x.  Differentiable in x, weight and residual, once and in reverse.

    x [..., D] of float32, bfloat16 or float16, the residual of its type or
    float32, weight [D] of any of the three.
    """
    if differentiated(x, weight, residual):
        return RMSNormFunction.apply(x, weight, residual, eps)
    y, h = _forward(x, weight, residual, eps, False)[:2]
    return y if residual is None else (y, h)


def rms_norm_quantized(x, weight, residual=None, eps=1e-6, scale_dtype=torch.float8_e8m0fnu):
    """``rms_norm`` with y in 8 bits, never stored in more: (codes, scales) as
    ``quantize_rows`` gives them, and h where there is a residual.  For inference:
    inputs that need a gradient are refused."""
    capi.require(not differentiated(x, weight, residual),
                 "rms_norm_quantized has no gradient: use rms_norm, or torch.no_grad()")
    device = _check(x, weight, residual)
    e4m3.require_scales(scale_dtype)
    lib = _lib()
    args, held, rows, D = _inputs(x, weight, residual)
    shape = x.shape
    lead = shape[:-1]
    codes, pitch = e4m3.new_codes(x, lead, D)
    scales = e4m3.new_scales(x, lead, D, scale_dtype)
    h = None if residual is None else _dense(residual)
    st = capi.launch(lib.rms_norm_quant, device, *args, codes.data_ptr(), pitch,
                     scales.data_ptr(), e4m3.SCALES[scale_dtype], 0 if h is None else h.data_ptr(),
                     rows, D, eps)
    if st:
        capi.check(st, lib.rms_norm_last_error, "rms_norm_quantized")
    return (codes, scales) if h is None else (codes, scales, h)


def candidate(inputs, params):
    """Framework candidate contract: inputs={"X","R","W"} -> y."""
    return rms_norm(inputs["X"], inputs["W"], inputs["R"], params.get("eps", 1e-6))[0]


def forward_only(inputs, params):
    """Forward without autograd."""
    with torch.no_grad():
        return candidate(inputs, params)
