"""Orthogonalised updates by Newton-Schulz products: wrapper over the HIP
library (kernels/newton_schulz.hip).

``newton_schulz`` orthogonalises matrices, ``muon_step`` updates weights with
the orthogonalised momentum of their gradients, ``Muon`` is that step as a
torch optimiser.  There is no CPU path: without a GPU the library refuses to
load.
"""

import ctypes
import functools
import os

import torch

from framework import capi
from framework.loader import load_kernel

KERNEL_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kernels")
LIB_NAME = "newton_schulz_hip"
SOURCES = ["newton_schulz.hip"]

# p(s) = a s + b s^3 + c s^5: steep at 0, its fixed band around 1 wide.  The coefficients published
# with the Muon optimiser (K. Jordan and others, 2024)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
PRECISIONS = {"half": 1, "full": 2}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def bind_library(lib):
    V, I64, I, F, S = capi.c_void_p, capi.c_int64, capi.c_int, capi.c_float, capi.c_size_t
    capi.bind(lib, "newton_schulz_workspace_bytes", [I64, I64, I64, I], S)
    capi.bind(lib, "newton_schulz",
              [V, I, I64, V, I, I64, I64, I64, I64, I, F, F, F, F, I, V, S, V])
    capi.bind(lib, "muon_update",
              [V, I, I64, V, I, I64, V, I, I64, I64, I64, I64, F, I, F, F, F, I, F, F, F, F, I, V,
               S, V])
    capi.bind_last_error(lib, "newton_schulz_last_error")
    return lib


@functools.lru_cache(maxsize=1)
def _lib():
    return bind_library(load_kernel(LIB_NAME, SOURCES, base_dir=KERNEL_DIR))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(m, n, count, precision):
    return _lib().newton_schulz_workspace_bytes(m, n, count, precision)


def _precision(precision):
    if precision is None:
        return PRECISIONS["full"]
    capi.require(precision in PRECISIONS, "precision must be None, 'half' or 'full'")
    return PRECISIONS[precision]


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _row_stride(t):
    """Elements between rows, None where a row is not dense."""
    if t.size(-1) > 1 and t.stride(-1) != 1:
        return None
    return t.stride(-2) if t.size(-2) > 1 else t.size(-1)


def newton_schulz(G, steps=5, coefficients=COEFFICIENTS, eps=1e-7, precision=None):
    """Each matrix of G [..., m, n] with its singular values taken to p(p(...)),
    near 1, after division by its Frobenius norm + eps; of G's type, and without
    a gradient.

    precision: "full" (or None) holds the iterates in 22 bits whatever G's type,
    whose own rounding then comes once, at the end; "half" holds them in 11, in
    less than half the time where the products fill the chip.  A matrix whose
    shorter side is at most 64 is iterated in 64 bits at either (unless
    |a|^(2 steps) > 1e9).
    """
    capi.require(G.is_cuda, "G must be a GPU tensor")
    capi.require(G.dtype in _DTYPES, "G must be float32, bfloat16 or float16")
    capi.require(G.dim() >= 2, "G must be [..., m, n]")
    lib = _lib()
    prec = _precision(precision)
    m, n = G.shape[-2:]
    G = G.detach()
    out = torch.empty(G.shape, dtype=G.dtype, device=G.device)
    if G.numel() == 0:
        return out
    if _row_stride(G) is None or _row_stride(G) < n:
        G = G.contiguous()
    count = G.numel() // (m * n)
    if G.dim() == 2:
        ins = [G]
    elif G.dim() == 3:
        ins = G.unbind(0)
    else:
        G = G.contiguous().view(count, m, n)
        ins = G.unbind(0)
    outs = out.view(count, m, n)
    a, b, c = coefficients
    ws_bytes = _workspace_bytes(m, n, count, prec)
    ws = torch.empty(ws_bytes // 8, dtype=torch.float64, device=G.device)
    step = m * n * out.element_size()
    o = (ctypes.c_void_p * count)(*[outs.data_ptr() + i * step for i in range(count)])
    st = capi.launch(lib.newton_schulz, G.get_device(), _pointers(ins), _DTYPES[G.dtype],
                     _row_stride(G), o, _DTYPES[G.dtype], n, m, n, count, steps, a, b, c, eps,
                     prec, ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, lib.newton_schulz_last_error, "newton_schulz")
    return out


def _as_list(x):
    return [x] if isinstance(x, torch.Tensor) else list(x)


@torch.no_grad()
def muon_step(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=COEFFICIENTS, eps=1e-7, scale=None, precision=None):
    """One update of every weight, in place:

        M = momentum M + G,   U = G + momentum M (nesterov) or M
        W = (1 - lr weight_decay) W - lr scale newton_schulz(U)

    params, grads, momenta: a matrix each or lists of them; weights of one
    shape and type go through the products together.  scale: a number, or None
    for max(1, m / n) ** 0.5.  precision as in ``newton_schulz``.  Weights and
    momenta must have dense rows, and no weight, momentum or gradient may overlap
    another that the call writes.
    """
    params, grads, momenta = _as_list(params), _as_list(grads), _as_list(momenta)
    capi.require(len(params) == len(grads) == len(momenta),
                 "params, grads and momenta must be lists of one length")
    written = [t.data_ptr() for t in params + momenta if t.numel()]
    capi.require(len(set(written)) == len(written), "a weight or momentum is listed twice")
    written = set(written)
    groups = {}
    for W, G, M in zip(params, grads, momenta):
        capi.require(W.is_cuda and G.is_cuda and M.is_cuda and
                     W.get_device() == G.get_device() == M.get_device(),
                     "params, grads and momenta must be on one GPU")
        capi.require(W.dim() == 2 and W.shape == G.shape == M.shape,
                     "params, grads and momenta must be matrices of one shape")
        capi.require(W.dtype in _DTYPES and G.dtype in _DTYPES and M.dtype in _DTYPES,
                     "params, grads and momenta must be float32, bfloat16 or float16")
        if W.numel() == 0:
            continue
        n = W.size(1)
        sw, sg, sm = _row_stride(W), _row_stride(G), _row_stride(M)
        capi.require(sw is not None and sm is not None and sw >= n and sm >= n,
                     "params and momenta must have dense rows that do not overlap")
        if sg is None or sg < n:
            G = G.contiguous()
            sg = n
        capi.require(G.data_ptr() not in written or G.data_ptr() == W.data_ptr(),
                     "a gradient shares memory with a momentum or another's weight")
        key = (W.shape, W.dtype, G.dtype, M.dtype, sw, sg, sm, W.get_device())
        groups.setdefault(key, ([], [], []))
        for to, t in zip(groups[key], (W, G, M)):
            to.append(t)
    a, b, c = coefficients
    for (shape, wt, gt, mt, sw, sg, sm, device), (ws_, gs, ms) in groups.items():
        lib = _lib()
        m, n = shape
        prec = _precision(precision)
        ws_bytes = _workspace_bytes(m, n, len(ws_), prec)
        ws = torch.empty(ws_bytes // 8, dtype=torch.float64, device=ws_[0].device)
        factor = max(1.0, m / n) ** 0.5 if scale is None else scale
        st = capi.launch(lib.muon_update, device, _pointers(ws_), _DTYPES[wt], sw, _pointers(gs),
                         _DTYPES[gt], sg, _pointers(ms), _DTYPES[mt], sm, m, n, len(ws_), momentum,
                         1 if nesterov else 0, lr, weight_decay, factor, steps, a, b, c, eps, prec,
                         ws.data_ptr(), ws_bytes)
        if st:
            capi.check(st, lib.newton_schulz_last_error, "muon_step")
        torch.autograd.graph.increment_version(ws_ + ms)  # for graphs that hold them


class Muon(torch.optim.Optimizer):
    """``muon_step`` for the matrices among a model's weights; momenta float32.

    Weights of other than two dimensions are refused: give those to another
    optimiser.
    """

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=COEFFICIENTS, eps=1e-7, scale=None, precision=None):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, scale=scale,
                                      precision=precision))
        for group in self.param_groups:
            for p in group["params"]:
                capi.require(p.dim() == 2, "Muon updates matrices only")

    def load_state_dict(self, state_dict):
        """As torch's, which rounds state to its weight's type; momenta keep their 32 bits."""
        taken = []

        def restore(_):
            state = taken[-1]
            ids = [i for group in state["param_groups"] for i in group["params"]]
            params = [p for group in self.param_groups for p in group["params"]]
            for i, p in zip(ids, params):
                if "momentum" in state["state"].get(i, ()):
                    self.state[p]["momentum"] = state["state"][i]["momentum"].to(
                        p.device, torch.float32, copy=True,
                        memory_format=torch.contiguous_format)
        # the state after all other hooks that may replace it, restored before those that see it
        hooks = (self.register_load_state_dict_pre_hook(lambda _, state: taken.append(state)),
                 self.register_load_state_dict_post_hook(restore, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                if "momentum" not in self.state[p]:
                    self.state[p]["momentum"] = torch.zeros(p.shape, dtype=torch.float32,
                                                            device=p.device)
            muon_step(params, [p.grad for p in params],
                      [self.state[p]["momentum"] for p in params],
                      **{k: v for k, v in group.items() if k != "params"})
        return loss


def candidate(inputs, params):
    """Framework candidate contract: inputs={"G"} -> its orthogonalised matrices."""
    return newton_schulz(inputs["G"], params.get("steps", 5),
                         params.get("coefficients", COEFFICIENTS), params.get("eps", 1e-7))


forward_only = candidate
