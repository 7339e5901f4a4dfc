"""Clipped policy loss with a KL term: autograd wrapper over the HIP library
(kernels/policy_loss.hip).

``policy_loss`` is the differentiable loss: its forward reads the logits once,
its backward once more.  ``policy_loss_and_grad`` gives the loss and its
gradient with the logits read once, and in their place if asked: hand the
gradient on with ``logits.backward(dlogits)``.  There is no CPU path: without a
GPU the library refuses to load.
"""

import functools
import math
import os

import torch

from framework import capi, token_rows
from framework.loader import load_kernel

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "policy_loss_hip"
SOURCES = ["policy_loss.hip"]


def bind_library(lib):
    V, I64, I, F, S = capi.c_void_p, capi.c_int64, capi.c_int, capi.c_float, capi.c_size_t
    rows = [I64, I64, I64, I64, I64, I64, F]
    given = [V, I, V, V, V, I64, I64, V, V, I]
    scalars = [F, F, F, F, V, S, V]
    capi.bind(lib, "policy_loss_workspace_bytes", [I64, I64], S)
    capi.bind(lib, "policy_loss_forward", given + [V, V, V, V] + rows + scalars)
    capi.bind(lib, "policy_loss_backward", [V, I, V, V, V, V, V] + rows + [V])
    capi.bind(lib, "policy_loss_and_grad", given + [V, V, V] + rows + scalars)
    capi.bind_last_error(lib, "policy_loss_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B, S):
    return _lib().policy_loss_workspace_bytes(B, S)


def _given(labels, old_logp, advantages, ref_logp, mask):
    """What comes with the logits, as the C entries take it: (tensors to keep
    until the call, arguments)."""
    shape = labels.shape
    labels = labels.contiguous()
    old = token_rows.per_token(old_logp, "old_logp", shape)
    ref = None if ref_logp is None else token_rows.per_token(ref_logp, "ref_logp", shape)
    capi.require(advantages.dtype == torch.float32, "advantages must be float32")
    adv = advantages
    if adv.shape != shape:
        try:  # one a sequence: [B] or [B, 1]
            adv = (adv.unsqueeze(-1) if adv.dim() == 1 and len(shape) == 2 else adv).expand(shape)
        except RuntimeError:
            raise RuntimeError("advantages must be one a sequence or broadcast to the labels' "
                               f"shape {tuple(shape)}, got {tuple(advantages.shape)}") from None
    if len(shape) == 2:
        adv_bs, adv_ss = adv.stride()
    elif len(shape) == 1:
        adv_bs, adv_ss = 0, adv.stride(0)
    else:
        adv = adv.contiguous()
        adv_bs, adv_ss = 0, 1
    kind = 0
    if mask is not None:
        capi.require(mask.dtype in (torch.bool, torch.uint8, torch.float32),
                     "mask must be bool, uint8 or float32")
        kind = 2 if mask.dtype == torch.float32 else 1
        try:
            mask = mask.expand(shape).contiguous()
        except RuntimeError:
            raise RuntimeError(f"mask must broadcast to the labels' shape {tuple(shape)}, "
                               f"got {tuple(mask.shape)}") from None
    args = (labels.data_ptr(), old.data_ptr(), adv.data_ptr(), adv_bs, adv_ss,
            0 if ref is None else ref.data_ptr(), 0 if mask is None else mask.data_ptr(), kind)
    return (labels, old, adv, ref, mask), args


def _check(logits, labels, old_logp, advantages, ref_logp, mask, kl_coef, denom):
    token_rows.check(logits, labels, ("old_logp", old_logp), ("advantages", advantages),
                     ("ref_logp", ref_logp), ("mask", mask))
    capi.require(kl_coef == 0.0 or ref_logp is not None, "kl_coef needs ref_logp")
    # as the C entry gets it: a 0 there stands for the sum of the weights
    capi.require(denom is None or 0.0 < capi.c_float(denom).value < math.inf,
                 "denom must be positive and finite in 32 bits")


def _forward(logits, labels, old_logp, advantages, ref_logp, mask, opts, keep):
    """(loss, logp, logits and labels as they were read, kept): kept [3, tokens]
    holds the rows' statistics and coefficients for ``_backward`` (None unless
    ``keep``)."""
    _check(logits, labels, old_logp, advantages, ref_logp, mask, opts["kl_coef"], opts["denom"])
    lib = _lib()
    x, *rows = token_rows.layout(logits)
    held, given = _given(labels, old_logp, advantages, ref_logp, mask)
    n = labels.numel()
    ws_bytes = _workspace_bytes(*rows[:2])
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device)
    loss, logp = ws.new_empty(()), ws.new_empty(labels.shape)
    kept = ws.new_empty(3 * n) if keep else None
    at = kept.data_ptr() if keep else 0
    st = capi.launch(lib.policy_loss_forward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], *given, loss.data_ptr(), logp.data_ptr(), at,
                     at + 8 * n if at else 0, *rows, opts["ignore_index"], opts["temperature"],
                     opts["clip_low"], opts["clip_high"], opts["kl_coef"], opts["denom"] or 0.0,
                     ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, lib.policy_loss_last_error, "policy_loss")
    return loss, logp, x, held[0], kept


def _backward(logits, labels, kept, gout, opts):
    """dlogits of the loss, times the one-element tensor gout."""
    lib = _lib()
    labels, kept, x, *rows = token_rows.saved(logits, labels, kept, 3)
    dlogits = torch.empty(logits.shape, dtype=x.dtype, device=x.device)
    at = kept.data_ptr()
    st = capi.launch(lib.policy_loss_backward, x.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], labels.data_ptr(), at,
                     at + 8 * labels.numel() if at else 0, gout.data_ptr(), dlogits.data_ptr(),
                     *rows, opts["ignore_index"], opts["temperature"])
    if st:
        capi.check(st, lib.policy_loss_last_error, "policy_loss backward")
    return dlogits


class PolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, old_logp, advantages, ref_logp, mask, opts):
        loss, logp, x, labels, kept = _forward(logits, labels, old_logp, advantages, ref_logp,
                                               mask, opts, True)
        ctx.opts = opts
        ctx.save_for_backward(x, labels, kept)
        ctx.mark_non_differentiable(logp)
        ctx.set_materialize_grads(False)
        return loss, logp

    @staticmethod
    def backward(ctx, gout, _):
        if gout is None:
            return (None,) * 7
        d = _backward(*ctx.saved_tensors, gout, ctx.opts)
        return (token_rows.once(d),) + (None,) * 6


def policy_loss(logits, labels, old_logp, advantages, ref_logp=None, mask=None, *, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, temperature=1.0, denom=None, ignore_index=-100):
    """(loss, logp): the clipped policy loss, differentiable in the logits, and
    the tokens' log-probabilities (not differentiable).

    logits [..., V]; labels, old_logp, ref_logp of their leading shape;
    advantages too, or one a sequence ([B] or [B, 1]); mask bool or float32
    weights.  A token counts unless its label is ``ignore_index`` or its weight
    0; what it and its other inputs hold then is not looked at.  The weighted
    terms are divided by ``denom`` (> 0 in float32), or by the sum of the weights.
    """
    opts = dict(clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, temperature=temperature,
                denom=denom, ignore_index=ignore_index)
    if token_rows.differentiated(logits):
        return PolicyLossFunction.apply(logits, labels, old_logp, advantages, ref_logp, mask, opts)
    return _forward(logits, labels, old_logp, advantages, ref_logp, mask, opts, False)[:2]


def policy_loss_and_grad(logits, labels, old_logp, advantages, ref_logp=None, mask=None, *,
                         clip_low=0.2, clip_high=0.2, kl_coef=0.0, temperature=1.0, denom=None,
                         ignore_index=-100, inplace=False):
    """(loss, logp, dlogits) of ``policy_loss`` in one pass over the logits,
    outside autograd.  ``inplace`` writes dlogits over the logits, which must
    be dense then; autograd knows of it, as of torch's own in-place operations:
    a graph that needs the logits themselves raises in its backward."""
    _check(logits, labels, old_logp, advantages, ref_logp, mask, kl_coef, denom)
    lib = _lib()
    logits = logits.detach()
    if inplace:
        capi.require(logits.is_contiguous(), "inplace needs contiguous logits")
    x, B, S, V, bs, rs = token_rows.layout(logits)
    keep, given = _given(labels, old_logp, advantages, ref_logp, mask)
    ws_bytes = _workspace_bytes(B, S)
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=logits.device)
    loss, logp = ws.new_empty(()), ws.new_empty(labels.shape)
    dlogits = logits if inplace else torch.empty(logits.shape, dtype=logits.dtype,
                                                 device=logits.device)
    st = capi.launch(lib.policy_loss_and_grad, logits.get_device(), x.data_ptr(),
                     token_rows.DTYPES[x.dtype], *given, loss.data_ptr(), logp.data_ptr(),
                     dlogits.data_ptr(), B, S, V, bs, rs, ignore_index, temperature, clip_low,
                     clip_high, kl_coef, 0.0 if denom is None else denom, ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, lib.policy_loss_last_error, "policy_loss_and_grad")
    del keep
    if inplace:  # for graphs that hold the logits
        torch.autograd.graph.increment_version(logits)
    return loss, logp, dlogits


def _options(params):
    names = ("clip_low", "clip_high", "kl_coef", "temperature", "denom", "ignore_index")
    return {k: params[k] for k in names if k in params}


def candidate(inputs, params):
    """Framework candidate contract: inputs={"logits","labels","old_logp",
    "advantages","ref_logp","mask"} -> scalar loss."""
    return policy_loss(inputs["logits"], inputs["labels"], inputs["old_logp"],
                       inputs["advantages"], inputs.get("ref_logp"), inputs.get("mask"),
                       **_options(params))[0]


def forward_only(inputs, params):
    """Forward without autograd."""
    with torch.no_grad():
        return candidate(inputs, params)
