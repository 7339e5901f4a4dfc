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
    return _forward(logits, labels, temperature, ignore_index, keep_stats)[:2]


def _forward(logits, labels, temperature, ignore_index, keep_stats):
    """(logp, stats, logits and labels as they were read)."""
    token_rows.check(logits, labels)
    lib = _lib()
    x, *rows = token_rows.layout(logits)
    labels = labels.contiguous()
    logp = torch.empty(labels.shape, dtype=torch.float32, device=x.device)
    stats = logp.new_empty(labels.shape + (2,)) if keep_stats else None
    st = capi.launch(lib.token_logp_forward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), logp.data_ptr(),
                     stats.data_ptr() if keep_stats else 0, *rows, ignore_index, temperature)
    if st:
        capi.check(st, lib.token_logp_last_error, "token_logp")
    return logp, stats, x, labels


def logp_backward(logits, labels, stats, dlogp, temperature=1.0, ignore_index=-100):
    """dlogits = dlogp / temperature (onehot(labels) - softmax(logits / temperature))."""
    token_rows.check(logits, labels, ("stats", stats), ("dlogp", dlogp))
    capi.require(dlogp.dtype == torch.float32 and dlogp.shape == labels.shape,
                 "dlogp must be float32 of the labels' shape")
    capi.require(stats.dtype == torch.float32 and stats.shape == labels.shape + (2,),
                 "stats must be the forward's")
    return _backward(logits, labels, stats, dlogp, temperature, ignore_index)


def _backward(logits, labels, stats, dlogp, temperature, ignore_index):
    lib = _lib()
    labels, stats, x, *rows = token_rows.saved(logits, labels, stats, 2)
    dlogp = dlogp.contiguous()
    dlogits = torch.empty(logits.shape, dtype=x.dtype, device=x.device)
    st = capi.launch(lib.token_logp_backward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), stats.data_ptr(),
                     dlogp.data_ptr(), 0, dlogits.data_ptr(), *rows, ignore_index, temperature)
    if st:
        capi.check(st, lib.token_logp_last_error, "token_logp backward")
    return dlogits


class TokenLogpFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, temperature, ignore_index):
        logp, stats, x, labels = _forward(logits, labels, temperature, ignore_index, True)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.save_for_backward(x, labels, stats)
        return logp

    @staticmethod
    def backward(ctx, dlogp):
        d = _backward(*ctx.saved_tensors, dlogp, ctx.temperature, ctx.ignore_index)
        return token_rows.once(d), None, None, None


def token_logp(logits, labels, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature)[labels], float32 of the labels' shape.

    Rows labelled ``ignore_index`` give 0 and a gradient of zeros, whatever
    their logits hold; another label outside [0, V) gives NaN.
    """
    if token_rows.differentiated(logits):
        return TokenLogpFunction.apply(logits, labels, temperature, ignore_index)
    return logp_forward(logits, labels, temperature, ignore_index)[0]


def candidate(inputs, params):
    """Framework candidate contract: inputs={"logits","labels"} -> logp."""
    return token_logp(inputs["logits"], inputs["labels"], params.get("temperature", 1.0))


def forward_only(inputs, params):
    """Forward without autograd."""
    return logp_forward(inputs["logits"], inputs["labels"], params.get("temperature", 1.0))[0]
