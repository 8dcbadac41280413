"""Sizes at the ends of what the token operators' index arithmetic holds, turned
away before anything is launched."""
import ctypes

import pytest

ARG = -1  # TP_ERR_ARG
P = 4096  # an address no case gets as far as reading
MOST = 2 ** 31 - 2 ** 11  # positions of one embedding gradient


@pytest.fixture(scope="module")
def lib():
    import os

    from tpcuda import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from tpcuda.build import build
        build()
    return _lib.load()


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 1024, 2 ** 31 - 8, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 40])
def test_more_positions_than_an_embedding_gradient_counts(lib, n):
    """Its kernels round a position up to 1024 and to 8 in 32 bits."""
    b = ctypes.c_int64(-1)
    for status in (lib.tpk_token_embedding_backward_ws(n, 1, 1, ctypes.byref(b)),
                   lib.tpk_token_embedding_backward(P, 1, P, 1, n, 1, 1, 1.0, -1, 0, 2 * P, 1, P, 1 << 50)):
        assert status == ARG and b"tokens" in lib.tp_last_error()


def test_the_most_positions_of_an_embedding_gradient(lib):
    b = ctypes.c_int64(-1)
    assert lib.tpk_token_embedding_backward_ws(MOST, 1, 1, ctypes.byref(b)) == 0
    assert b.value > 4 * 4 * MOST  # positions and tokens, split and sorted


def test_norm_buffers_off_a_value_boundary(lib):
    for off in (1, 2, 3):
        for status in (lib.tpk_group_grad_norm(987654321, 2.0, 1.0, P + off),
                       lib.tpk_group_clip_grad_norm(987654321, 2.0, 1.0, P + off),
                       lib.tpk_adam_group_scaled(987654321, 0, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1e-3, 1.0, P + off)):
            assert status == ARG and b"aligned" in lib.tp_last_error()
