"""Argument checks of the matrix-product and NVFP4 entry points of the C ABI, without a device: documented negative codes, nothing
launched."""
import ctypes

import pytest


@pytest.fixture(scope='module')
def lib():
    from tilekernels_b200 import _lib, build
    build.build()
    return _lib.lib()


def test_argument_checks_of_the_products(lib):
    buf = (ctypes.c_char * 4096)()
    p16 = (ctypes.addressof(buf) + 15) // 16 * 16
    from tilekernels_b200 import _lib
    scaled = lib.tkq_block_scaled_gemm
    def call(x=p16, xs=128, xbk=128, wbk=128, xbm=1, fmt=0, sf_fmt=0, experts=1, rows=4, n=8, k=128, start=0, end=0, out=p16, flags=0,
             x_sf=p16):
        # x, row stride, x_sf, its row and k strides, block_m, block_k, w, expert and row strides, w_sf, its expert, row and k
        # strides, block_m, block_k, fmt, sf_fmt, start, end, experts, rows, n, k, alpha, its stride, out, its stride, flags
        return scaled(_lib.BLOCK_SCALED_GEMM_ARGS.pack(x, xs, x_sf, 1, 4, xbm, xbk, p16, 0, 128, p16, 0, 1, 8, 1, wbk, fmt, sf_fmt, start, end, experts,
                                                       rows, n, k, 0, 0, out, n, flags), None)

    assert scaled(None, None) == -1
    assert call(rows=0) == 0                                    # nothing to do
    assert call(rows=-1) == -1 and call(n=0) == -1 and call(k=0) == -1 and call(experts=0) == -1
    assert call(fmt=2) == -1 and call(sf_fmt=3) == -1
    assert call(x=0) == -1 and call(out=0) == -1
    assert call(start=p16) == -1 and call(experts=2) == -1      # bounds come in pairs, and groups need them
    assert call(experts=1025, start=p16, end=p16) == -2
    assert call(xbk=64) == -2 and call(xbm=16) == -2 and call(sf_fmt=1) == -2 and call(fmt=1) == -2
    assert call(k=144) == -2 and call(fmt=1, xbk=32, wbk=32, k=96) == -2
    assert call(flags=1) == -2
    assert call(x=p16 + 8) == -3 and call(xs=136) == -3 and call(x_sf=p16 + 2) == -3 and call(out=p16 + 1) == -3
    assert b'block_scaled_gemm' in lib.tkq_last_error_string()
    # (x, row stride, w, expert stride, row stride, transpose, start, end, experts, rows, n, k, out, out stride, flags)
    def grouped(*args):
        return lib.tkq_grouped_gemm(_lib.GROUPED_GEMM_ARGS.pack(*args), None)

    assert lib.tkq_grouped_gemm(None, None) == -1
    assert grouped(p16, 64, p16, 4096, 64, 0, p16, p16, 2, 0, 64, 64, p16, 64, 0) == 0
    assert grouped(p16, 64, p16, 4096, 64, 0, 0, 0, 1, 4, 64, 64, p16, 64, 0) == -1
    assert grouped(p16, 60, p16, 4096, 64, 0, p16, p16, 2, 4, 64, 64, p16, 64, 0) == -3
    assert grouped(p16, 64, p16, 4096, 64, 0, p16, p16, 2, 4, 64, 64, p16, 64, 128) == -2

    # (grad, row stride, x, row stride, start, end, experts, rows, n, k, dtype, out, flags)
    def wgrad(*args):
        return lib.tkq_grouped_gemm_wgrad(_lib.GROUPED_GEMM_WGRAD_ARGS.pack(*args), None)

    assert lib.tkq_grouped_gemm_wgrad(None, None) == -1
    assert wgrad(p16, 64, p16, 64, p16, p16, 2, 0, 64, 64, 1, p16, 128) == 0   # accumulate nothing
    assert wgrad(p16, 64, p16, 64, p16, p16, 2, 4, 64, 64, 2, p16, 0) == -1    # output type
    assert wgrad(p16, 64, p16, 64, p16, p16, 2, 4, 64, 64, 0, p16, 128) == -2  # accumulation in bf16
    assert wgrad(p16, 64, p16, 64, 0, p16, 2, 4, 64, 64, 1, p16, 0) == -1
    assert wgrad(p16 + 2, 64, p16, 64, p16, p16, 2, 4, 64, 64, 1, p16, 0) == -3
    assert b'grouped_gemm_wgrad' in lib.tkq_last_error_string()


def test_expanded_operands_are_refused_by_name(lib):
    """An axis of stride 0 is no matter of 16-byte boundaries."""
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    from tilekernels_b200 import _lib

    def refused(rc, what):
        return rc == -2 and what in lib.tkq_last_error_string() and b'stride 0' in lib.tkq_last_error_string()

    for x_row, w_expert, w_row in ((0, 1024, 128), (128, 0, 128), (128, 1024, 0)):
        rc = lib.tkq_block_scaled_gemm(_lib.BLOCK_SCALED_GEMM_ARGS.pack(p, x_row, p, 1, 4, 1, 128, p, w_expert, w_row, p, 0, 1, 8, 1, 128, 0, 0, p, p, 2, 4, 8, 128,
                                                                        0, 0, p, 8, 0), None)
        assert refused(rc, b'block_scaled_gemm')
        for transpose in (0, 1):
            assert refused(lib.tkq_grouped_gemm(_lib.GROUPED_GEMM_ARGS.pack(p, x_row, p, w_expert, w_row, transpose, p, p, 2, 4, 64, 64, p, 64, 0), None),
                           b'grouped_gemm')
    for g_row, x_row in ((0, 64), (64, 0)):
        rc = lib.tkq_grouped_gemm_wgrad(_lib.GROUPED_GEMM_WGRAD_ARGS.pack(p, g_row, p, x_row, p, p, 2, 4, 64, 64, 1, p, 0), None)
        assert refused(rc, b'grouped_gemm_wgrad')


def test_argument_checks_of_the_nvfp4_entry_points(lib):
    buf = (ctypes.c_char * 4096)()
    p16 = (ctypes.addressof(buf) + 15) // 16 * 16
    cast, back = lib.tkq_per_token_cast_nvfp4, lib.tkq_cast_back_nvfp4
    # (x, dtype, rows, hidden, row stride, tensor_scale, out, sf, stream)
    assert cast(p16, 0, 0, 64, 64, p16, p16, p16, None) == 0
    assert cast(p16, 3, 4, 64, 64, p16, p16, p16, None) == -1
    assert cast(p16, 0, 4, 64, 64, None, p16, p16, None) == -1
    assert cast(p16, 0, 4, 72, 72, p16, p16, p16, None) == -2
    assert cast(p16 + 4, 0, 4, 64, 64, p16, p16, p16, None) == -3
    assert cast(p16, 0, 4, 64, 68, p16, p16, p16, None) == -3
    # (x, sf, tensor_scale, rows, hidden, dtype, out, stream)
    assert back(p16, p16, p16, 0, 64, 0, p16, None) == 0
    assert back(p16, p16, p16, 4, 64, 7, p16, None) == -1
    assert back(p16, p16, p16, 4, 40, 0, p16, None) == -2
    assert back(p16 + 4, p16, p16, 4, 64, 0, p16, None) == -3
