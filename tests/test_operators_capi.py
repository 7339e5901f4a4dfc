"""C-ABI checks of the training operators that need no GPU: every library
loads, exports what its header declares, and rejects bad arguments with the
right NL2K_* status before touching the device."""

import ctypes

import pytest

import __graft_entry__ as entry
from test_capi import STATUS, _load, declared_functions

HEADERS = {"token_logp.h": "cases.token_logp.op", "policy_loss.h": "cases.policy_loss.op",
           "preference_loss.h": "cases.preference_loss.op",
           "newton_schulz.h": "cases.newton_schulz.op"}
P = ctypes.c_void_p(1 << 20)   # never dereferenced: every call below fails validation
ODD = ctypes.c_void_p((1 << 20) + 1)


def test_every_operator_has_a_header():
    assert sorted(HEADERS.values()) == sorted(entry.OPERATOR_MODULES)


@pytest.mark.parametrize("header", sorted(HEADERS))
def test_library_exports_every_declared_symbol(header):
    names = declared_functions(header)
    assert names
    lib = _load(HEADERS[header])
    assert not [n for n in names if not hasattr(lib, n)]


def test_token_logp_validation():
    lib = _load(HEADERS["token_logp.h"])

    def call(logits=P, dtype=0, labels=P, logp=P, stats=None, B=2, S=3, V=8, bs=24, rs=8,
             temperature=1.0):
        return lib.token_logp_forward(logits, dtype, labels, logp, stats, B, S, V, bs, rs, -100,
                                      temperature, None)
    assert call(logits=None) == STATUS["NL2K_ERR_NULL"]
    assert call(labels=None) == STATUS["NL2K_ERR_NULL"]
    assert call(logp=None) == STATUS["NL2K_ERR_NULL"]
    assert call(dtype=3) == STATUS["NL2K_ERR_VALUE"]
    assert call(B=-1) == STATUS["NL2K_ERR_SHAPE"]
    assert call(V=0) == STATUS["NL2K_ERR_SHAPE"]
    assert call(rs=-8) == STATUS["NL2K_ERR_SHAPE"]
    assert call(V=1 << 29) == STATUS["NL2K_ERR_OVERFLOW"]
    assert call(B=1 << 20, S=1 << 20) == STATUS["NL2K_ERR_OVERFLOW"]
    assert call(temperature=0.0) == STATUS["NL2K_ERR_VALUE"]
    assert call(temperature=float("nan")) == STATUS["NL2K_ERR_VALUE"]
    assert call(logits=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert call(logits=ODD, dtype=1) == STATUS["NL2K_ERR_ALIGN"]
    assert call(stats=ctypes.c_void_p((1 << 20) + 4)) == STATUS["NL2K_ERR_ALIGN"]
    assert b"stats" in lib.token_logp_last_error()
    # nothing to do: success without a launch
    assert call(logits=None, labels=None, logp=None, B=0) == 0
    assert lib.token_logp_last_error() == b""
    assert lib.token_logp_backward(P, 0, P, P, None, None, P, 2, 3, 8, 24, 8, -100, 1.0,
                                   None) == STATUS["NL2K_ERR_NULL"]


def test_policy_loss_validation():
    lib = _load(HEADERS["policy_loss.h"])
    need = lib.policy_loss_workspace_bytes(2, 3)
    assert need == 64 * 8 + 6 * 4 and lib.policy_loss_workspace_bytes(-1, 3) == 0

    def call(mask=None, kind=0, ref=None, loss=P, dlogits=P, rs=8, low=0.2, high=0.2, kl=0.0,
             denom=0.0, ws=P, ws_bytes=need, logits=P):
        return lib.policy_loss_and_grad(logits, 0, P, P, P, 3, 1, ref, mask, kind, loss, P, dlogits,
                                        2, 3, 8, 3 * rs, rs, -100, 1.0, low, high, kl, denom, ws,
                                        ws_bytes, None)
    assert call(ws_bytes=need - 1) == STATUS["NL2K_ERR_WORKSPACE"]
    assert call(ws=None) == STATUS["NL2K_ERR_WORKSPACE"]
    assert call(ws=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert call(loss=None) == STATUS["NL2K_ERR_NULL"]
    assert call(dlogits=None) == STATUS["NL2K_ERR_NULL"]
    assert call(kind=1) == STATUS["NL2K_ERR_NULL"]
    assert call(kind=3) == STATUS["NL2K_ERR_VALUE"]
    assert call(kl=0.1) == STATUS["NL2K_ERR_NULL"]
    assert call(low=1.5) == STATUS["NL2K_ERR_VALUE"]
    assert call(high=float("inf")) == STATUS["NL2K_ERR_VALUE"]
    assert call(denom=-1.0) == STATUS["NL2K_ERR_VALUE"]
    # in place needs dense logits
    assert call(rs=16) == STATUS["NL2K_ERR_SHAPE"] and b"in place" in lib.policy_loss_last_error()
    st = lib.policy_loss_forward(P, 0, P, P, P, 3, 1, None, None, 0, P, P, P, None, 2, 3, 8, 24, 8,
                                 -100, 1.0, 0.2, 0.2, 0.0, 0.0, P, need, None)
    assert st == STATUS["NL2K_ERR_NULL"] and b"together" in lib.policy_loss_last_error()


def test_preference_loss_validation():
    lib = _load(HEADERS["preference_loss.h"])
    need = lib.preference_loss_workspace_bytes(4, 3, 2)
    assert need == 4 * (12 + 2) and lib.preference_loss_workspace_bytes(4, 3, 0) == 0

    def call(cu=None, pairs=2, B=4, beta=0.1, eps=0.0, ws_bytes=need, loss=P, stats=P, coef=P):
        return lib.preference_loss_forward(P, 0, P, P, cu, pairs, loss, P, stats, coef, B, 3, 8, 24,
                                           8, -100, beta, eps, 0, P, ws_bytes, None)
    assert call(pairs=3) == STATUS["NL2K_ERR_SHAPE"]
    assert call(pairs=0) == STATUS["NL2K_ERR_SHAPE"]
    assert call(cu=P) == STATUS["NL2K_ERR_SHAPE"]
    assert call(beta=float("nan")) == STATUS["NL2K_ERR_VALUE"]
    assert call(eps=-0.1) == STATUS["NL2K_ERR_VALUE"]
    assert call(loss=None) == STATUS["NL2K_ERR_NULL"]
    assert call(coef=None) == STATUS["NL2K_ERR_NULL"]
    assert call(ws_bytes=need - 1) == STATUS["NL2K_ERR_WORKSPACE"]


def test_newton_schulz_validation():
    lib = _load(HEADERS["newton_schulz.h"])
    assert lib.newton_schulz_workspace_bytes(-1, 4, 1, 1) == 0
    assert lib.newton_schulz_workspace_bytes(4, 4, 1, 3) == 0
    assert lib.newton_schulz_workspace_bytes(1 << 17, 1 << 17, 1, 1) == 0
    need = lib.newton_schulz_workspace_bytes(40, 50, 1, 1)
    assert need > 0
    assert lib.newton_schulz_workspace_bytes(140, 150, 1, 2) > \
        lib.newton_schulz_workspace_bytes(140, 150, 1, 1) > need
    one = (ctypes.c_void_p * 1)(1 << 20)
    odd = (ctypes.c_void_p * 1)((1 << 20) + 2)
    null = (ctypes.c_void_p * 1)(None)

    def call(ins=one, dtype=0, stride=50, out=one, steps=5, c=(3.4445, -4.775, 2.0315), eps=1e-7,
             precision=1, ws=P, ws_bytes=need, m=40):
        return lib.newton_schulz(ins, dtype, stride, out, 0, 50, m, 50, 1, steps, *c, eps, precision,
                                 ws, ws_bytes, None)
    assert call(ins=None) == STATUS["NL2K_ERR_NULL"]
    assert call(ins=null) == STATUS["NL2K_ERR_NULL"]
    assert call(ins=odd) == STATUS["NL2K_ERR_ALIGN"]
    assert call(dtype=5) == STATUS["NL2K_ERR_VALUE"]
    assert call(stride=49) == STATUS["NL2K_ERR_SHAPE"]
    assert call(m=-1) == STATUS["NL2K_ERR_SHAPE"]
    assert call(steps=0) == STATUS["NL2K_ERR_VALUE"]
    assert call(eps=-1.0) == STATUS["NL2K_ERR_VALUE"]
    assert call(precision=0) == STATUS["NL2K_ERR_VALUE"]
    assert call(c=(9.0, 0.0, 0.0)) == STATUS["NL2K_ERR_VALUE"]
    assert call(c=(float("nan"), 0.0, 0.0)) == STATUS["NL2K_ERR_VALUE"]
    assert call(ws_bytes=need - 1) == STATUS["NL2K_ERR_WORKSPACE"]
    assert call(ws=ctypes.c_void_p((1 << 20) + 8)) == STATUS["NL2K_ERR_ALIGN"]
    assert call(m=0) == 0 and lib.newton_schulz_last_error() == b""
    st = lib.muon_update(one, 0, 50, one, 0, 50, null, 0, 50, 40, 50, 1, 0.9, 1, 0.1, 0.0, 1.0, 5,
                         3.4445, -4.775, 2.0315, 1e-7, 1, P, need, None)
    assert st == STATUS["NL2K_ERR_NULL"] and b"momenta" in lib.newton_schulz_last_error()
    st = lib.muon_update(one, 0, 50, one, 0, 50, one, 0, 50, 40, 50, 1, 0.9, 1, float("nan"), 0.0,
                         1.0, 5, 3.4445, -4.775, 2.0315, 1e-7, 1, P, need, None)
    assert st == STATUS["NL2K_ERR_VALUE"]


@pytest.mark.parametrize("name", ["token_logp", "policy_loss", "preference_loss", "newton_schulz"])
def test_references_pass_their_own_parity(name):
    import importlib
    from framework.verify import verify_all
    case = importlib.import_module(f"cases.{name}").make_case(2, 13, 40)
    assert verify_all(case, case.reference_forward, device="cpu")[0]
