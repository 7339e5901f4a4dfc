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


def test_a_layer_takes_what_its_wanted_products_take():
    """y adds K numbers, dx N and dw M: at most 2^22 each, where they are wanted."""
    lib = _load("cases.block_matmul.op")
    most = 1 << 22

    def forward(M, N, K, dx, dw):
        return lib.block_linear_forward(None, 1, K, P, 1, K, None, 0, None, 0, 0, 1, dx, dw, P, None, M,
                                        N, K, None, 0, None)

    def back(M, N, K, dx, dw):
        return lib.block_linear_backward(None, 1, N, None, 0, None, 0, 0, 1, None, P if dx else None,
                                         P if dw else None, 1, M, N, K, None, 0, None)
    null, over = STATUS["NL2K_ERR_NULL"], STATUS["NL2K_ERR_OVERFLOW"]
    for sizes in ((most, 16, 16), (16, most, 16), (16, 16, most)):
        for want in ((0, 0), (1, 0), (0, 1), (1, 1)):
            assert forward(*sizes, *want) == null
            assert back(*sizes, *want) == (null if any(want) else 0)
    tokens, wide, long = (most + 77, 16, 32), (16, most + 77, 32), (16, 32, most + 77)
    for sizes, taken in ((tokens, ((0, 0), (1, 0))), (wide, ((0, 0), (0, 1))), (long, ())):
        for want in ((0, 0), (1, 0), (0, 1), (1, 1)):
            assert forward(*sizes, *want) == (null if want in taken else over)
            if any(want):
                assert back(*sizes, *want) == (null if want in taken else over)
    assert b"sizes too large" in lib.block_matmul_last_error()

    def bytes_of(sizes, dx, dw, backward):
        return (lib.block_linear_kept_bytes(*sizes, 1, dx, dw, 0),
                lib.block_linear_workspace_bytes(*sizes, 1, 1, 1, backward))
    kept, ws = bytes_of(tokens, 1, 0, 1)
    assert 16 * 32 <= kept < 16 * 1024 and ws >= tokens[0] * 16
    kept, ws = bytes_of(wide, 0, 1, 0)
    assert 16 * 32 <= kept < 16 * 1024 and ws >= wide[1] * 32
    assert bytes_of(tokens, 0, 1, 0)[0] == 0 and bytes_of(long, 0, 0, 0) == (0, 0)
