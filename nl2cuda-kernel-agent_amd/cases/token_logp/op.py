"""Log-probabilities of given tokens: autograd wrapper over the HIP library
(kernels/token_logp.hip).

``token_logp(logits, labels)`` is what scoring an answer, a reference model's
share of a loss, or a sampler's record of what it chose needs.  The forward
reads the logits once and, where a gradient is wanted, keeps each row's maximum
and sum for a backward of one streaming pass.  There is no CPU path: without a
GPU the library refuses to load.
"""

import functools
import os

import torch

from framework import capi, token_rows
from framework.loader import load_kernel

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "token_logp_hip"
SOURCES = ["token_logp.hip"]


def bind_library(lib):
    V, I64, I, F = capi.c_void_p, capi.c_int64, capi.c_int, capi.c_float
    rows = [I64, I64, I64, I64, I64, I64, F]
    capi.bind(lib, "token_logp_forward", [V, I, V, V, V] + rows + [V])
    capi.bind(lib, "token_logp_backward", [V, I, V, V, V, V, V] + rows + [V])
    capi.bind_last_error(lib, "token_logp_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


def logp_forward(logits, labels, temperature=1.0, ignore_index=-100, keep_stats=False):
    """(logp, stats): stats [..., 2] hold each row's maximum and sum of
    exponentials for ``logp_backward`` (None unless ``keep_stats``)."""
    token_rows.check(logits, labels)
    x, B, S, V, bs, rs = token_rows.layout(logits)
    return _forward(x, labels.contiguous(), (B, S, V, bs, rs, ignore_index, temperature),
                    keep_stats)


def _forward(x, labels, rows, keep_stats):
    lib = _lib()
    logp = torch.empty(labels.shape, dtype=torch.float32, device=x.device)
    stats = logp.new_empty(labels.shape + (2,)) if keep_stats else None
    st = capi.launch(lib.token_logp_forward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), logp.data_ptr(),
                     stats.data_ptr() if keep_stats else 0, *rows)
    if st:
        capi.check(st, lib.token_logp_last_error, "token_logp")
    return logp, stats


def logp_backward(logits, labels, stats, dlogp, temperature=1.0, ignore_index=-100):
    """dlogits = dlogp / temperature (onehot(labels) - softmax(logits / temperature))."""
    token_rows.check(logits, labels, ("stats", stats), ("dlogp", dlogp))
    capi.require(dlogp.dtype == torch.float32 and dlogp.shape == labels.shape,
                 "dlogp must be float32 of the labels' shape")
    capi.require(stats.dtype == torch.float32 and stats.shape == labels.shape + (2,),
                 "stats must be the forward's")
    x, B, S, V, bs, rs = token_rows.layout(logits)
    return _backward(x, labels.contiguous(), stats.contiguous(), dlogp,
                     (B, S, V, bs, rs, ignore_index, temperature), logits.shape)


def _backward(x, labels, stats, dlogp, rows, shape):
    lib = _lib()
    dlogp = dlogp.contiguous()
    dlogits = torch.empty(shape, dtype=x.dtype, device=x.device)
    st = capi.launch(lib.token_logp_backward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), stats.data_ptr(),
                     dlogp.data_ptr(), 0, dlogits.data_ptr(), *rows)
    if st:
        capi.check(st, lib.token_logp_last_error, "token_logp backward")
    return dlogits


class TokenLogpFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, temperature, ignore_index):
        token_rows.check(logits, labels)
        x, B, S, V, bs, rs = token_rows.layout(logits)
        labels = labels.contiguous()
        ctx.rows, ctx.shape = (B, S, V, bs, rs, ignore_index, temperature), logits.shape
        logp, stats = _forward(x, labels, ctx.rows, True)
        ctx.save_for_backward(x, labels, stats)
        return logp

    @staticmethod
    def backward(ctx, dlogp):
        return _backward(*ctx.saved_tensors, dlogp, ctx.rows, ctx.shape), None, None, None


def token_logp(logits, labels, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature)[labels], float32 of the labels' shape.

    Rows labelled ``ignore_index`` give 0 and a gradient of zeros, whatever
    their logits hold; another label outside [0, V) gives NaN.
    """
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogpFunction.apply(logits, labels, temperature, ignore_index)
    return logp_forward(logits, labels, temperature, ignore_index)[0]


def candidate(inputs, params):
    """Framework candidate contract: inputs={"logits","labels"} -> logp."""
    return token_logp(inputs["logits"], inputs["labels"], params.get("temperature", 1.0))


def forward_only(inputs, params):
    """Forward without autograd."""
    return logp_forward(inputs["logits"], inputs["labels"], params.get("temperature", 1.0))[0]
