"""Preference loss of paired log ratios: autograd wrapper over the HIP library
(kernels/preference_loss.hip).

``preference_loss`` is the differentiable loss over chosen and rejected
answers; ``preference_loss_and_grad`` gives the loss and its gradient outside
autograd.  Either reads the logits twice: a row's gradient needs its pair's
sums.  There is no CPU path: without a GPU the library refuses to load.
"""

import functools
import os

import torch

from framework import capi, token_rows
from framework.loader import load_kernel

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "preference_loss_hip"
SOURCES = ["preference_loss.hip"]


def bind_library(lib):
    V, I64, I, F, S = capi.c_void_p, capi.c_int64, capi.c_int, capi.c_float, capi.c_size_t
    rows = [I64, I64, I64, I64, I64, I64]
    capi.bind(lib, "preference_loss_workspace_bytes", [I64, I64, I64], S)
    capi.bind(lib, "preference_loss_forward",
              [V, I, V, V, V, I64, V, V, V, V] + rows + [F, F, I, V, S, V])
    capi.bind(lib, "preference_loss_backward", [V, I, V, V, V, V, V] + rows + [V])
    capi.bind_last_error(lib, "preference_loss_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B, S, pairs):
    return _lib().preference_loss_workspace_bytes(B, S, pairs)


def _forward(logits, labels, ref_seq_logp, opts, keep):
    """(loss, seq_logp, logits and labels as they were read, kept): kept [3,
    tokens] holds the rows' statistics and coefficients for ``_backward`` (None
    unless ``keep``)."""
    cu_seqlens = opts["cu_seqlens"]
    token_rows.check(logits, labels, ("ref_seq_logp", ref_seq_logp), ("cu_seqlens", cu_seqlens))
    lib = _lib()
    if cu_seqlens is None:
        capi.require(logits.dim() == 3 and logits.size(0) >= 2 and logits.size(0) % 2 == 0,
                     "logits must be [2 N, S, V], chosen then rejected, or [T, V] with cu_seqlens")
        count = logits.size(0)
    else:
        capi.require(logits.dim() == 2, "with cu_seqlens logits must be [T, V]")
        capi.require(cu_seqlens.dtype == torch.int64 and cu_seqlens.dim() == 1 and
                     cu_seqlens.numel() >= 3 and cu_seqlens.numel() % 2 == 1,
                     "cu_seqlens must be int64 [2 N + 1]")
        cu_seqlens = cu_seqlens.contiguous()
        count = cu_seqlens.numel() - 1
    if ref_seq_logp is not None:
        capi.require(ref_seq_logp.dtype == torch.float32 and ref_seq_logp.shape == (count,),
                     "ref_seq_logp must be float32 [2 N]")
        ref_seq_logp = ref_seq_logp.contiguous()
    x, *rows = token_rows.layout(logits)
    labels = labels.contiguous()
    n = labels.numel()
    ws_bytes = _workspace_bytes(*rows[:2], count // 2)
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device)
    loss, seq = ws.new_empty(()), ws.new_empty(count)
    kept = ws.new_empty(3 * n) if keep else None
    at = kept.data_ptr() if keep else 0
    st = capi.launch(lib.preference_loss_forward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(),
                     0 if ref_seq_logp is None else ref_seq_logp.data_ptr(),
                     0 if cu_seqlens is None else cu_seqlens.data_ptr(), count // 2,
                     loss.data_ptr(), seq.data_ptr(), at, at + 8 * n if at else 0, *rows,
                     opts["ignore_index"], opts["beta"], opts["label_smoothing"],
                     1 if opts["average"] else 0, ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, lib.preference_loss_last_error, "preference_loss")
    return loss, seq, x, labels, kept


def _backward(logits, labels, kept, gout, ignore_index):
    """dlogits of the loss, times the one-element tensor gout where given."""
    lib = _lib()
    labels, kept, x, *rows = token_rows.saved(logits, labels, kept, 3)
    dlogits = torch.empty(logits.shape, dtype=x.dtype, device=x.device)
    at = kept.data_ptr()
    st = capi.launch(lib.preference_loss_backward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), at,
                     at + 8 * labels.numel() if at else 0, 0 if gout is None else gout.data_ptr(),
                     dlogits.data_ptr(), *rows, ignore_index)
    if st:
        capi.check(st, lib.preference_loss_last_error, "preference_loss backward")
    return dlogits


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref_seq_logp, opts):
        loss, seq, x, labels, kept = _forward(logits, labels, ref_seq_logp, opts, True)
        ctx.ignore_index = opts["ignore_index"]
        ctx.save_for_backward(x, labels, kept)
        ctx.mark_non_differentiable(seq)
        ctx.set_materialize_grads(False)
        return loss, seq

    @staticmethod
    def backward(ctx, gout, _):
        if gout is None:
            return None, None, None, None
        d = _backward(*ctx.saved_tensors, gout, ctx.ignore_index)
        return token_rows.once(d), None, None, None


def preference_loss(logits, labels, ref_seq_logp=None, *, cu_seqlens=None, beta=0.1,
                    label_smoothing=0.0, average=False, ignore_index=-100):
    """(loss, seq_logp): the preference loss, differentiable in the logits, and
    the sequences' log-probabilities (not differentiable).

    logits [2 N, S, V] hold N chosen answers, then their N rejected ones; or
    [T, V], the 2 N answers one after the other with their offsets
    ``cu_seqlens`` [2 N + 1].  Tokens labelled ``ignore_index`` (prompts,
    padding) do not count.  ``ref_seq_logp`` [2 N] are the reference model's
    (None: without one); ``average`` divides each by its number of tokens.
    """
    opts = dict(cu_seqlens=cu_seqlens, beta=beta, label_smoothing=label_smoothing,
                average=average, ignore_index=ignore_index)
    if token_rows.differentiated(logits):
        return PreferenceLossFunction.apply(logits, labels, ref_seq_logp, opts)
    return _forward(logits, labels, ref_seq_logp, opts, False)[:2]


def preference_loss_and_grad(logits, labels, ref_seq_logp=None, *, cu_seqlens=None, beta=0.1,
                             label_smoothing=0.0, average=False, ignore_index=-100):
    """(loss, seq_logp, dlogits) of ``preference_loss``, outside autograd."""
    opts = dict(cu_seqlens=cu_seqlens, beta=beta, label_smoothing=label_smoothing,
                average=average, ignore_index=ignore_index)
    loss, seq, x, labels, kept = _forward(logits.detach(), labels, ref_seq_logp, opts, True)
    return loss, seq, _backward(x, labels, kept, None, ignore_index)


def _options(params):
    names = ("beta", "label_smoothing", "average", "ignore_index")
    return {k: params[k] for k in names if k in params}


def candidate(inputs, params):
    """Framework candidate contract: inputs={"logits","labels","ref_seq_logp"} -> scalar loss."""
    return preference_loss(inputs["logits"], inputs["labels"], inputs.get("ref_seq_logp"),
                           cu_seqlens=inputs.get("cu_seqlens"), **_options(params))[0]


def forward_only(inputs, params):
    """Forward without autograd."""
    with torch.no_grad():
        return candidate(inputs, params)
