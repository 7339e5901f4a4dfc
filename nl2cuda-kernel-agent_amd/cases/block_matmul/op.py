"""Matrix product in 8-bit floating point with a scale for each block of 128
numbers, and the trainable layer made of it: wrapper over the HIP library
(kernels/block_matmul.hip).

``block_matmul`` multiplies what ``quantize_rows``, ``quantize_tiles`` and
``rms_norm_quantized`` give; ``block_linear`` is x weight^T with all three of
its products in 8 bits, forward and backward.  There is no CPU path: without a
GPU the library refuses to load.
"""

import collections
import functools
import math
import os

import torch

from cases.block_quant.op import quantize_tiles
from framework import capi, e4m3
from framework.loader import load_kernel
from framework.once import differentiated, once

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "block_matmul_hip"
SOURCES = ["block_matmul.hip"]
LONGEST = 1 << 22     # of the kernels' offsets within a tile
FARTHEST = 1 << 36    # scales of one row may lie apart

QuantizedWeight = collections.namedtuple("QuantizedWeight", "codes scales codes_t scales_t")


def bind_library(lib):
    V, I64, I, S = capi.c_void_p, capi.c_int64, capi.c_int, capi.c_size_t
    capi.bind(lib, "block_matmul_workspace_bytes", [I64, I64, I64, I], S)
    capi.bind(lib, "block_matmul", [V, I64, V, I64, I64, I] * 2 + [I, V, I, I64, I64, I64, V, S, V])
    capi.bind(lib, "block_linear_kept_bytes", [I64, I64, I64, I, I, I, I], S)
    capi.bind(lib, "block_linear_workspace_bytes", [I64, I64, I64, I, I, I, I], S)
    weight = [V, I64, V, I64, I64]
    capi.bind(lib, "block_linear_forward",
              [V, I, I64, V, I, I64] + weight + [I, I, I, V, V, I64, I64, I64, V, S, V])
    capi.bind(lib, "block_linear_backward",
              [V, I, I64] + weight + [I, V, V, V, I, I64, I64, I64, V, S, V])
    capi.bind_last_error(lib, "block_matmul_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(M, N, K, out_dtype):
    return _lib().block_matmul_workspace_bytes(M, N, K, out_dtype)


@functools.lru_cache(maxsize=1024)
def _layer_bytes(M, N, K, scale_type, x_type, w_type, want_x, want_w, have_codes):
    """(workspace of the forward, of the backward, what is kept between them)."""
    lib = _lib()
    sizes = (M, N, K, scale_type)
    return (lib.block_linear_workspace_bytes(*sizes, x_type, w_type, 0),
            lib.block_linear_workspace_bytes(*sizes, x_type, w_type, 1),
            lib.block_linear_kept_bytes(*sizes, want_x, want_w, have_codes))


def _codes(c, rows, K):
    """(codes, bytes between rows) as the kernels read them: rows a multiple of 16 bytes apart, the
    last one's memory up to the next 16; copied only if they lie otherwise."""
    whole = (K + 15) // 16 * 16
    pitch, step = c.stride()
    if rows == 1:
        pitch = whole
    if ((step == 1 or K == 1) and pitch >= K and pitch % 16 == 0 and
            pitch <= 2 * LONGEST and c.data_ptr() % 16 == 0 and
            (whole == K or c.storage_offset() + (rows - 1) * pitch + whole <=
             c.untyped_storage().nbytes())):
        return c, pitch
    copy, pitch = e4m3.new_codes(c, (rows,), K)
    copy.view(torch.uint8).copy_(c.view(torch.uint8))
    return copy, pitch


def _scales(name, s, rows, K):
    """(scales, row stride, block stride, whether they are of tiles)."""
    n, tiles, shape = (K + 127) // 128, (rows + 127) // 128, s.shape
    of_tiles = shape == (tiles, n)
    if not of_tiles and shape != (rows, n):
        raise RuntimeError(name)
    row, block = s.stride()
    if row > LONGEST or block > FARTHEST:
        # strides of a dimension of one are never taken, and may be anything
        row, block = row if shape[0] > 1 else 0, block if n > 1 else 0
        if row > LONGEST or block > FARTHEST:
            s = s.contiguous()
            row, block = n, 1
    return s, row, block, of_tiles


def _product(a, a_scales, b, b_scales, out, M, N, K):
    """out = a b^T for matrices of codes and their scales on one GPU."""
    lib = _lib()
    a, a_pitch = _codes(a, M, K)
    b, b_pitch = _codes(b, N, K)
    a_scales, a_row, a_block, a_tiles = _scales(
        "a_scales must be [rows, blocks] of a or [tiles, blocks]", a_scales, M, K)
    b_scales, b_row, b_block, b_tiles = _scales(
        "b_scales must be [rows, blocks] of b or [tiles, blocks]", b_scales, N, K)
    dtype = e4m3.DTYPES[out.dtype]
    ws_bytes, ws_ptr = _workspace_bytes(M, N, K, dtype), 0
    if ws_bytes:
        ws = a.new_empty(ws_bytes // 4, dtype=torch.float32)
        ws_ptr = ws.data_ptr()
    st = capi.launch(lib.block_matmul, a.get_device(), a.data_ptr(), a_pitch, a_scales.data_ptr(),
                     a_row, a_block, a_tiles, b.data_ptr(), b_pitch, b_scales.data_ptr(), b_row,
                     b_block, b_tiles, e4m3.SCALES[a_scales.dtype], out.data_ptr(), dtype, M, N, K,
                     ws_ptr, ws_bytes)
    if st:
        capi.check(st, lib.block_matmul_last_error, "block_matmul")
    return out


def block_matmul(a, a_scales, b, b_scales, out_dtype=torch.bfloat16):
    """a b^T for a [..., K] and b [N, K], codes with a scale for each block of 128:
    [..., N] of out_dtype (float32, bfloat16 or float16); without a gradient.

    Scales are of rows, [..., ceil(K / 128)], or of tiles of 128 x 128,
    [ceil(M / 128), ceil(K / 128)] for M rows in all; float32 or float8_e8m0fnu, the same for
    both.  Codes in another layout than the quantisers' are copied.  Sums are
    held in float32.  The 8-bit matrix instruction, which adds up 16-bit results, drops
    what lies 13 bits below the largest of each eight products: a result is off by at
    most 7 * 2^-13 of the sum of those, of random numbers by 1.5e-5 of the results'
    root mean square, before it is rounded.  A float32 one takes the 16-bit
    instruction, 2.5 times as long, and has its 24 bits.
    """
    device, shape, scale_dtype = a.get_device(), a.shape, a_scales.dtype
    # the common case in one expression; what is wrong with another is said below
    if not (device >= 0 and
            device == a_scales.get_device() == b.get_device() == b_scales.get_device() and
            a.dtype == b.dtype == e4m3.CODES and scale_dtype == b_scales.dtype and
            scale_dtype in e4m3.SCALES and out_dtype in e4m3.DTYPES and len(shape) >= 1 and
            b.dim() == 2 and shape[-1] == b.shape[1] >= 1):
        capi.require(device >= 0 and a_scales.is_cuda and b.is_cuda and b_scales.is_cuda,
                     "codes and scales must be GPU tensors")
        capi.require(device == a_scales.get_device() == b.get_device() == b_scales.get_device(),
                     "codes and scales must be on one GPU")
        capi.require(a.dtype == b.dtype == e4m3.CODES, "a and b must be float8_e4m3fn")
        capi.require(scale_dtype == b_scales.dtype and scale_dtype in e4m3.SCALES,
                     "scales must both be float32 or both float8_e8m0fnu")
        capi.require(out_dtype in e4m3.DTYPES, "out_dtype must be float32, bfloat16 or float16")
        raise RuntimeError("a must be [..., K] and b [N, K] with K >= 1")
    capi.require(not differentiated(a, a_scales, b, b_scales),
                 "block_matmul has no gradient: use block_linear, or torch.no_grad()")
    N, K = b.shape
    if len(shape) == 2:
        M = shape[0]
        out = a.new_empty(M, N, dtype=out_dtype)
    else:
        out = a.new_empty((*shape[:-1], N), dtype=out_dtype)
        M, blocks = math.prod(shape[:-1]), e4m3.blocks(K)
        rows, tiles = (*shape[:-1], blocks), (e4m3.blocks(M), blocks)
        capi.require(a_scales.shape == rows or a_scales.shape == tiles,
                     f"a_scales must be {rows} or {tiles}, got {tuple(a_scales.shape)}")
        if M:
            a = a.reshape(M, K)
            if a_scales.shape == rows:
                a_scales = a_scales.reshape(M, -1)
    if M == 0 or N == 0:
        return out
    return _product(a, a_scales, b, b_scales, out, M, N, K)


def quantize_weight(weight, scale_dtype=torch.float8_e8m0fnu):
    """What ``block_linear`` makes of a weight [N, K] in every call, for programs that
    use it more than once between two updates."""
    return QuantizedWeight(*quantize_tiles(weight, scale_dtype, transposed=True))


def _tiles(codes, scales, rows, n):
    """A quantised weight, or its transpose, as the C entries take it."""
    codes, pitch = _codes(codes, rows, n)
    scales, row, block, _ = _scales("quantized must be quantize_weight's", scales, rows, n)
    return (codes.data_ptr(), pitch, scales.data_ptr(), row, block), (codes, scales)


def _layer_forward(x, weight, quantized, scale_dtype, want_x, want_w):
    """(y, what the backward needs or None)."""
    lib = _lib()
    N, K = weight.shape
    rows, M, _, x_stride = e4m3.rows_of(x)
    types = e4m3.DTYPES
    x_type, w_type, s_type = types[x.dtype], types[weight.dtype], e4m3.SCALES[scale_dtype]
    y = x.new_empty((*x.shape[:-1], N))
    if M == 0:
        return y, None
    if quantized is None:
        weight, _, _, w_stride = e4m3.rows_of(weight)
        w, held = (weight.data_ptr(), w_type, w_stride, 0, 0, 0, 0, 0), weight
    else:
        codes, held = _tiles(quantized[0], quantized[1], N, K)
        w = (0, w_type, 0) + codes
    ws_bytes, _, kept_bytes = _layer_bytes(M, N, K, s_type, x_type, w_type, want_x, want_w,
                                           quantized is not None)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    kept = x.new_empty(kept_bytes, dtype=torch.uint8) if kept_bytes else None
    st = capi.launch(lib.block_linear_forward, x.get_device(), rows.data_ptr(), x_type, x_stride,
                     *w, s_type, want_x, want_w, y.data_ptr(),
                     kept.data_ptr() if kept_bytes else 0, M, N, K, ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, lib.block_matmul_last_error, "block_linear")
    return y, kept


class BlockLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, quantized, scale_dtype):
        ctx.want = ctx.needs_input_grad[:2]
        y, kept = _layer_forward(x, weight, quantized, scale_dtype, *ctx.want)
        ctx.scale_dtype, ctx.dtypes = scale_dtype, (x.dtype, weight.dtype)
        ctx.x_shape, ctx.w_shape = x.shape, weight.shape
        ctx.quantized = quantized is not None
        ctx.save_for_backward(kept, *(quantized[2:] if ctx.quantized and ctx.want[0] else ()))
        return y

    @staticmethod
    def backward(ctx, dy):
        kept, *codes_t = ctx.saved_tensors
        want_x, want_w = ctx.want
        N, K = ctx.w_shape
        dy, M, _, dy_stride = e4m3.rows_of(dy)
        dx = dy.new_empty(ctx.x_shape, dtype=ctx.dtypes[0]) if want_x else None
        if M == 0:
            dw = dy.new_zeros((N, K), dtype=ctx.dtypes[1]) if want_w else None
            return *once("block_linear", dx, dw), None, None
        lib, device = _lib(), dy.get_device()
        types = e4m3.DTYPES
        x_type, w_type = types[ctx.dtypes[0]], types[ctx.dtypes[1]]
        s_type = e4m3.SCALES[ctx.scale_dtype]
        _, ws_bytes, kept_bytes = _layer_bytes(M, N, K, s_type, x_type, w_type, want_x, want_w,
                                               ctx.quantized)
        # what autograd gives back of what was saved: every read lies within it
        message = "autograd gave back other tensors than were saved"
        if kept_bytes:
            capi.require(kept.get_device() == device and kept.dtype == torch.uint8 and
                         kept.numel() == kept_bytes, message)
            kept = kept.contiguous()
        w = (0, 0, 0, 0, 0)
        if codes_t:
            codes_t, scales_t = codes_t
            capi.require(codes_t.shape == (K, N) and codes_t.dtype == e4m3.CODES and
                         scales_t.shape == (e4m3.blocks(K), e4m3.blocks(N)) and
                         scales_t.dtype == ctx.scale_dtype and
                         codes_t.get_device() == device == scales_t.get_device(), message)
            w, held = _tiles(codes_t, scales_t, K, N)
        dw = dy.new_empty((N, K), dtype=ctx.dtypes[1]) if want_w else None
        ws = dy.new_empty(ws_bytes, dtype=torch.uint8)
        st = capi.launch(lib.block_linear_backward, device, dy.data_ptr(), x_type, dy_stride, *w,
                         s_type, kept.data_ptr() if kept_bytes else 0,
                         dx.data_ptr() if want_x else 0, dw.data_ptr() if want_w else 0, w_type, M,
                         N, K, ws.data_ptr(), ws_bytes)
        if st:
            capi.check(st, lib.block_matmul_last_error, "block_linear backward")
        return *once("block_linear", dx, dw), None, None


def block_linear(x, weight, quantized=None, scale_dtype=torch.float8_e8m0fnu):
    """x weight^T, x [..., K] and weight [N, K] of float32, bfloat16 or float16, in 8
    bits: [..., N] of x's type.

        y  = Q(x) Q(weight)^T          blocks along K, tiles of the weight
        dx = Q(dy) Q(weight)           blocks along N, the same tiles
        dweight = Q(dy^T) Q(x^T)^T     blocks along the tokens

    Gradients pass through the roundings Q as if they were not there; dx and
    dweight come in x's and the weight's type.  Differentiable once and in
    reverse.  quantized: what ``quantize_weight`` gave for this weight.
    """
    device = x.get_device()
    capi.require(device >= 0 and device == weight.get_device(),
                 "x and weight must be GPU tensors on one GPU")
    capi.require(x.dtype in e4m3.DTYPES and weight.dtype in e4m3.DTYPES,
                 "x and weight must be float32, bfloat16 or float16")
    capi.require(x.dim() >= 1 and weight.dim() == 2 and x.shape[-1] == weight.shape[1] >= 1 and
                 weight.shape[0] >= 1, "x must be [..., K] and weight [N, K] with N, K >= 1")
    e4m3.require_scales(scale_dtype)
    if quantized is not None:
        N, K = weight.shape
        for codes, scales, shape in ((*quantized[:2], (N, K)), (*quantized[2:], (K, N))):
            capi.require(codes.shape == shape and codes.dtype == e4m3.CODES and
                         scales.shape == (e4m3.blocks(shape[0]), e4m3.blocks(shape[1])) and
                         scales.dtype == scale_dtype and
                         codes.get_device() == device == scales.get_device(),
                         "quantized must be quantize_weight's, of this weight and scale_dtype")
    if differentiated(x, weight):
        return BlockLinearFunction.apply(x, weight, quantized, scale_dtype)
    return _layer_forward(x.detach(), weight.detach(), quantized, scale_dtype, False, False)[0]


def candidate(inputs, params):
    """Framework candidate contract: inputs={"X","W"} -> X W^T in 8 bits."""
    return block_linear(inputs["X"], inputs["W"],
                        scale_dtype=params.get("scale_dtype", torch.float8_e8m0fnu))


def forward_only(inputs, params):
    """Forward without autograd."""
    with torch.no_grad():
        return candidate(inputs, params)
