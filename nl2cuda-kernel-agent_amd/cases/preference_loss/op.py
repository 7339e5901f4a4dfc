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


def loss_forward(logits, labels, ref_seq_logp=None, *, cu_seqlens=None, beta=0.1,
                 label_smoothing=0.0, average=False, ignore_index=-100, keep_stats=False):
    """(loss, seq_logp, stats, coef); stats and coef are for ``loss_backward``
    (None unless ``keep_stats``)."""
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
    x, B, S, V, bs, rs = token_rows.layout(logits)
    labels = labels.contiguous()
    ws_bytes = _workspace_bytes(B, S, count // 2)
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=logits.device)
    loss, seq = ws.new_empty(()), ws.new_empty(count)
    stats = coef = None
    if keep_stats:
        stats, coef = ws.new_empty(labels.shape + (2,)), ws.new_empty(labels.shape)
    st = capi.launch(lib.preference_loss_forward, logits.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(),
                     0 if ref_seq_logp is None else ref_seq_logp.data_ptr(),
                     0 if cu_seqlens is None else cu_seqlens.data_ptr(), count // 2,
                     loss.data_ptr(), seq.data_ptr(), stats.data_ptr() if keep_stats else 0,
                     coef.data_ptr() if keep_stats else 0, B, S, V, bs, rs, ignore_index, beta,
                     label_smoothing, 1 if average else 0, ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, lib.preference_loss_last_error, "preference_loss")
    return loss, seq, stats, coef


def loss_backward(logits, labels, stats, coef, gout=None, ignore_index=-100):
    """dlogits of the loss, times the one-element tensor gout where given."""
    token_rows.check(logits, labels, ("stats", stats), ("coef", coef), ("gout", gout))
    capi.require(gout is None or (gout.dtype == torch.float32 and gout.numel() == 1),
                 "gout must be a one-element float32 GPU tensor")
    lib = _lib()
    x, B, S, V, bs, rs = token_rows.layout(logits)
    labels = labels.contiguous()
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    st = capi.launch(lib.preference_loss_backward, logits.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), stats.data_ptr(),
                     coef.data_ptr(), 0 if gout is None else gout.data_ptr(), dlogits.data_ptr(),
                     B, S, V, bs, rs, ignore_index)
    if st:
        capi.check(st, lib.preference_loss_last_error, "preference_loss backward")
    return dlogits


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref_seq_logp, opts):
        loss, seq, stats, coef = loss_forward(logits, labels, ref_seq_logp, keep_stats=True,
                                              **opts)
        ctx.save_for_backward(logits, labels, stats, coef)
        ctx.ignore_index = opts["ignore_index"]
        ctx.mark_non_differentiable(seq)
        ctx.set_materialize_grads(False)
        return loss, seq

    @staticmethod
    def backward(ctx, gout, _):
        if gout is None:
            return None, None, None, None
        logits, labels, stats, coef = ctx.saved_tensors
        return loss_backward(logits, labels, stats, coef, gout, ctx.ignore_index), None, None, None


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
    if logits.requires_grad and torch.is_grad_enabled():
        return PreferenceLossFunction.apply(logits, labels, ref_seq_logp, opts)
    return loss_forward(logits, labels, ref_seq_logp, **opts)[:2]


def preference_loss_and_grad(logits, labels, ref_seq_logp=None, *, cu_seqlens=None, beta=0.1,
                             label_smoothing=0.0, average=False, ignore_index=-100):
    """(loss, seq_logp, dlogits) of ``preference_loss``, outside autograd."""
    logits = logits.detach()
    loss, seq, stats, coef = loss_forward(logits, labels, ref_seq_logp, cu_seqlens=cu_seqlens,
                                          beta=beta, label_smoothing=label_smoothing,
                                          average=average, ignore_index=ignore_index,
                                          keep_stats=True)
    return loss, seq, loss_backward(logits, labels, stats, coef, None, ignore_index)


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
