"""Sizes that the 8-bit layers' operators take, where the C entries' checks end: a
call that gets past those of its sizes is refused for what it lacks.  No GPU."""

import ctypes

from test_capi import STATUS, _load

P = ctypes.c_void_p(1 << 20)   # never dereferenced: every call below fails validation


def test_rms_norm_takes_as_many_rows_of_any_width():
    lib = _load("cases.rms_norm.op")

    def forward(rows, D):
        return lib.rms_norm_forward(None, 1, D, None, 0, 0, P, 1, P, None, None, rows, D, 1e-6, None)

    def back(rows, D):
        return lib.rms_norm_backward(None, 1, D, P, 1, D, None, 0, P, 1, P, P, None, None, rows, D,
                                     None, 0, None)
    most = 4 * ((1 << 32) // 256 - 1)
    for D in (8, 1024, 1025, 4096, 4097, 32768, 32769, 2 ** 31 - 16385):
        for rows in (1, 1 << 22, 1 << 24, most):
            assert forward(rows, D) == back(rows, D) == STATUS["NL2K_ERR_NULL"]
        assert lib.rms_norm_backward_workspace_bytes(most, D) > 0
        assert forward(most + 1, D) == back(most + 1, D) == STATUS["NL2K_ERR_OVERFLOW"]
    assert forward(1, 2 ** 31 - 16384) == back(1, 2 ** 31 - 16384) == STATUS["NL2K_ERR_OVERFLOW"]
