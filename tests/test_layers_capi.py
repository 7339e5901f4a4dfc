"""C-ABI checks of the 8-bit layers' operators that need no GPU: every library
loads, exports what its header declares, and rejects bad arguments with the right
NL2K_* status before touching the device."""

import ctypes

import pytest

import __graft_entry__ as entry
from test_capi import STATUS, _load, declared_functions

HEADERS = {"rms_norm.h": "cases.rms_norm.op", "block_quant.h": "cases.block_quant.op",
           "block_matmul.h": "cases.block_matmul.op"}
P = ctypes.c_void_p(1 << 20)   # never dereferenced: every call below fails validation
ODD = ctypes.c_void_p((1 << 20) + 1)
HALF = ctypes.c_void_p((1 << 20) + 8)


def test_every_operator_has_a_header():
    assert sorted(HEADERS.values()) == sorted(entry.LAYER_MODULES)


@pytest.mark.parametrize("header", sorted(HEADERS))
def test_library_exports_every_declared_symbol(header):
    names = declared_functions(header)
    assert names
    lib = _load(HEADERS[header])
    assert not [n for n in names if not hasattr(lib, n)]


def test_rms_norm_validation():
    lib = _load(HEADERS["rms_norm.h"])

    def call(x=P, dtype=0, xs=8, r=None, rt=0, rs=8, w=P, wt=0, y=P, h=None, rstd=None, rows=3, D=8,
             eps=1e-6):
        return lib.rms_norm_forward(x, dtype, xs, r, rt, rs, w, wt, y, h, rstd, rows, D, eps, None)
    assert call(x=None) == call(w=None) == call(y=None) == STATUS["NL2K_ERR_NULL"]
    assert call(r=P) == call(h=P) == STATUS["NL2K_ERR_NULL"]
    assert call(dtype=3) == call(wt=-1) == STATUS["NL2K_ERR_VALUE"]
    assert call(r=P, h=P, dtype=0, rt=1) == call(r=P, h=P, dtype=1, rt=2) == STATUS["NL2K_ERR_VALUE"]
    assert call(rows=-1) == call(D=0) == call(xs=-1) == STATUS["NL2K_ERR_SHAPE"]
    assert call(rows=1 << 30) == call(D=1 << 31) == STATUS["NL2K_ERR_OVERFLOW"]
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        assert call(eps=eps) == STATUS["NL2K_ERR_VALUE"]
    assert call(x=ODD) == call(w=ODD) == call(y=ODD) == call(rstd=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert call(x=ODD, dtype=1) == call(r=ODD, h=P) == STATUS["NL2K_ERR_ALIGN"]
    assert b"residual" in lib.rms_norm_last_error()
    assert call(rows=0, x=None, w=None, y=None) == 0 and lib.rms_norm_last_error() == b""

    def quant(codes=P, pitch=16, scales=P, st=0, D=8):
        return lib.rms_norm_quant(P, 1, D, None, 0, 0, P, 1, codes, pitch, scales, st, None, 3, D,
                                  1e-6, None)
    assert quant(codes=None) == quant(scales=None) == STATUS["NL2K_ERR_NULL"]
    assert quant(pitch=8) == quant(pitch=24) == quant(D=17) == STATUS["NL2K_ERR_SHAPE"]
    assert quant(codes=HALF) == quant(scales=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert quant(st=2) == STATUS["NL2K_ERR_VALUE"]

    assert lib.rms_norm_backward_workspace_bytes(-1, 8) == 0
    need = lib.rms_norm_backward_workspace_bytes(3, 8)
    assert need > 0 and lib.rms_norm_backward_workspace_bytes(1 << 20, 4096) <= 512 * 4096 * 4

    def back(dy=P, dtype=0, h=P, ht=0, w=P, rstd=P, dw=P, ws=P, n=need, dh=None, dhs=0):
        return lib.rms_norm_backward(dy, dtype, 8, h, ht, 8, dh, dhs, w, 0, rstd, P, None, dw, 3, 8,
                                     ws, n, None)
    assert back(dy=None) == back(h=None) == back(w=None) == back(rstd=None) == STATUS["NL2K_ERR_NULL"]
    assert back(n=need - 1) == back(ws=None) == STATUS["NL2K_ERR_WORKSPACE"]
    assert back(ws=ODD) == back(dy=ODD) == back(dh=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert back(dtype=1, ht=2) == STATUS["NL2K_ERR_VALUE"]
    assert back(dh=P, dhs=-8) == STATUS["NL2K_ERR_SHAPE"]


def test_block_quant_validation():
    lib = _load(HEADERS["block_quant.h"])

    def rows(x=P, dtype=1, stride=20, codes=P, pitch=32, scales=P, ct=None, pt=0, st_=None, st=0, M=5,
             K=20):
        return lib.block_quant_rows(x, dtype, stride, codes, pitch, scales, ct, pt, st_, st, M, K, None)
    assert rows(x=None) == rows(codes=None) == rows(scales=None) == STATUS["NL2K_ERR_NULL"]
    assert rows(ct=P, pt=16) == STATUS["NL2K_ERR_NULL"]
    assert rows(dtype=7) == rows(st=2) == STATUS["NL2K_ERR_VALUE"]
    assert rows(M=-1) == rows(K=0) == rows(stride=-1) == rows(pitch=16) == rows(pitch=40) == \
        STATUS["NL2K_ERR_SHAPE"]
    assert rows(ct=P, st_=P, pt=4) == rows(ct=P, st_=P, pt=20) == STATUS["NL2K_ERR_SHAPE"]
    assert rows(K=1 << 31, pitch=1 << 31) == rows(M=1 << 31) == STATUS["NL2K_ERR_OVERFLOW"]
    assert rows(x=ODD) == rows(codes=HALF) == rows(scales=ODD) == rows(ct=HALF, pt=16, st_=P) == \
        STATUS["NL2K_ERR_ALIGN"]
    assert b"16 bytes" in lib.block_quant_last_error()
    assert rows(M=0, x=None) == 0 and lib.block_quant_last_error() == b""
    st = lib.block_quant_tiles(P, 1, 20, P, 32, None, None, 0, 0, 5, 20, None)
    assert st == STATUS["NL2K_ERR_NULL"] and b"tiles" in lib.block_quant_last_error()


def test_block_matmul_validation():
    lib = _load(HEADERS["block_matmul.h"])

    def call(a=P, ap=256, sa=P, ar=1, ab=70, b=P, bp=256, sb=P, br=2, bb=1, st=0, out=P, ot=1, M=70,
             N=300, K=200, ws=None, n=0):
        return lib.block_matmul(a, ap, sa, ar, ab, 0, b, bp, sb, br, bb, 1, st, out, ot, M, N, K, ws, n,
                                None)
    assert call(a=None) == call(sa=None) == call(b=None) == call(sb=None) == call(out=None) == \
        STATUS["NL2K_ERR_NULL"]
    assert call(ap=192) == call(bp=200) == call(ar=-1) == call(bb=-1) == STATUS["NL2K_ERR_SHAPE"]
    assert call(M=-1) == call(K=0) == STATUS["NL2K_ERR_SHAPE"]
    assert call(st=2) == call(ot=3) == STATUS["NL2K_ERR_VALUE"]
    assert call(a=HALF) == call(b=HALF) == call(sa=ODD) == call(out=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert call(K=(1 << 22) + 1, ap=1 << 23, bp=1 << 23) == call(M=1 << 31) == \
        STATUS["NL2K_ERR_OVERFLOW"]
    assert call(M=0, a=None) == call(N=0) == 0 and lib.block_matmul_last_error() == b""
    # parts of a long k are added in a workspace
    assert lib.block_matmul_workspace_bytes(-1, 4, 4, 1) == 0
    assert lib.block_matmul_workspace_bytes(8192, 8192, 8192, 1) == 0
    need = lib.block_matmul_workspace_bytes(70, 300, 40000, 1)
    assert need >= 2 * 70 * 300 * 4

    def long(ws, n):
        return call(ap=40000, bp=40000, K=40000, ws=ws, n=n)
    assert long(None, need) == long(P, need - 1) == STATUS["NL2K_ERR_WORKSPACE"]
    assert long(ODD, need) == STATUS["NL2K_ERR_ALIGN"]


def test_block_linear_validation():
    lib = _load(HEADERS["block_matmul.h"])
    sizes = (70, 300, 200, 1)
    need = lib.block_linear_workspace_bytes(*sizes, 1, 1, 0)
    back = lib.block_linear_workspace_bytes(*sizes, 1, 1, 1)
    kept = lib.block_linear_kept_bytes(*sizes, 1, 1, 0)
    assert need >= 370 * 208 and back >= 2 * 70 * 300 and kept >= 200 * (80 + 304)
    assert lib.block_linear_kept_bytes(*sizes, 1, 0, 1) == lib.block_linear_kept_bytes(*sizes, 0, 0, 0) == 0
    assert lib.block_linear_workspace_bytes(0, 300, 200, 1, 1, 1, 0) == 0
    assert lib.block_linear_workspace_bytes(70, 0, 200, 1, 1, 1, 0) == 0

    def forward(x=P, xt=1, xs=200, w=P, wt=1, codes=None, scales=None, y=P, k=P, ws=P, n=need, st=1,
                M=70):
        return lib.block_linear_forward(x, xt, xs, w, wt, 200, codes, 208, scales, 2, 1, st, 1, 1, y, k,
                                        M, 300, 200, ws, n, None)
    assert forward(x=None) == forward(w=None) == forward(y=None) == forward(codes=P) == \
        STATUS["NL2K_ERR_NULL"]
    assert forward(xt=3) == forward(st=2) == forward(wt=-1) == STATUS["NL2K_ERR_VALUE"]
    assert forward(n=need - 1) == forward(ws=None) == forward(k=None) == STATUS["NL2K_ERR_WORKSPACE"]
    assert forward(ws=HALF) == forward(k=HALF) == forward(x=ODD) == STATUS["NL2K_ERR_ALIGN"]
    assert forward(xs=-1) == forward(M=-1) == STATUS["NL2K_ERR_SHAPE"]
    assert forward(M=0, x=None) == 0

    def backward(dy=P, k=P, dx=P, dw=P, ws=P, n=back, M=70):
        return lib.block_linear_backward(dy, 1, 300, None, 0, None, 0, 0, 1, k, dx, dw, 1, M, 300, 200,
                                         ws, n, None)
    assert backward(dy=None) == backward(k=None) == backward(k=None, dx=None) == STATUS["NL2K_ERR_NULL"]
    assert backward(n=back - 1) == backward(ws=None) == STATUS["NL2K_ERR_WORKSPACE"]
    assert backward(ws=HALF) == STATUS["NL2K_ERR_ALIGN"]
    assert backward(M=0) == backward(dx=None, dw=None) == 0
