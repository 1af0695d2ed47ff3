"""The last sizes that the kernels of the 8-bit form take and the first that they refuse: a launch has under 2^32 threads.  What is taken gets as far as the check of a
missing pointer, so nothing is launched (no GPU needed)."""
import ctypes
import os

import pytest

P = ctypes.c_void_p(4096)      # never read
NULL, SHAPE = -1, -3
BF16, F32 = 0, 1


@pytest.fixture(scope="module")
def lib():
    from picotron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    return _lib.lib()


def packed():
    from picotron_amd._lib import Mx8
    return ctypes.byref(Mx8(4096, 4096))


# a group of 128 columns takes 32 lanes in fp32, 8 of them a workgroup of 256: 2^24 - 1 workgroups have under 2^32 threads
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols,last", [(128, 2 ** 27 - 8), (32, 2 ** 27 - 8), (160, 2 ** 26 - 4), (1024, 2 ** 24 - 1), (11008, (2 ** 27 - 8) // 86)])
def test_what_walks_groups(lib, cols, last, dtype):
    for rows, code in ((last, NULL), (last + 1, SHAPE)):
        got = (lib.pico_mx8_quantize(None, packed(), rows, cols, cols, dtype, None), lib.pico_mx8_dequantize(packed(), None, rows, cols, cols, dtype, None),
               lib.pico_swiglu_mx8_fwd(None, P, P, None, None, None, rows, cols, cols, cols, dtype, None),
               lib.pico_swiglu_mx8_bwd(None, packed(), packed(), P, P, None, rows, cols, cols, cols, cols, dtype, None))
        assert set(got) == {code}, (rows, got)


# a row takes a wave up to 256 vectors of 16 bytes, 256 threads up to 1024 and 1024 threads from there on
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hidden,last", [(32, 2 ** 26 - 4), (256, 2 ** 26 - 4), (288, (2 ** 27 - 8) // 3), (1056, (2 ** 27 - 8) // 9), (4128, (2 ** 27 - 8) // 33), (16384, (2 ** 27 - 8) // 128)])
def test_the_norm(lib, hidden, last, dtype):
    vectors = hidden // (8 if dtype == BF16 else 4)
    threads, rows_each = (256, 4) if vectors <= 256 else (256, 1) if vectors <= 1024 else (1024, 1)
    assert (last + rows_each - 1) // rows_each * threads < 2 ** 32
    for rows, code in ((last, NULL), (last + 1, SHAPE)):
        assert lib.pico_rmsnorm_mx8_fwd(None, P, packed(), None, None, None, None, rows, hidden, 1e-5, dtype, None) == code


def test_swiglus_gradient_from_sums(lib):
    def call(dy=P, parts=1, gate=None, dgate=P, y=None, rows=4, cols=64, ld=64):
        return lib.pico_swiglu_mx8_bwd_sums(dy, parts, gate or packed(), packed(), dgate, P, y, rows, cols, ld, ld, None)
    from picotron_amd._lib import Mx8
    away = ctypes.c_void_p(4096 + 8)
    assert [call(parts=0), call(parts=65), call(cols=40), call(rows=-1), call(rows=2 ** 27)] == [SHAPE] * 5
    assert [call(dy=None), call(dgate=None), call(gate=ctypes.byref(Mx8(None, 4096)))] == [NULL] * 3
    assert [call(dy=away), call(dgate=away), call(y=away), call(ld=68)] == [-4] * 4 and call(ld=56) == -5 and call(rows=0, dy=None) == 0


def test_a_product_in_20_bits_and_the_gradient_from_it(lib):
    away = ctypes.c_void_p(4096 + 8)
    def product(a=P, left=P, M=64, N=64, K=256, lda=256, tile=(256, 256)):
        return lib.pico_product_large_bits20(a, P, P, left, M, N, K, lda, N, *tile, None)
    assert [product(N=72), product(K=250), product(M=0), product(lda=252), product(K=64, lda=64), product(tile=(64, 64))] == [SHAPE] * 6
    assert [product(a=None), product(left=None)] == [NULL] * 2 and [product(a=away), product(left=away)] == [-4] * 2
    def swiglu(dy=P, left=P, rows=4, cols=64, ld=64):
        return lib.pico_swiglu_mx8_bwd_bits20(dy, left, packed(), packed(), P, P, None, rows, cols, ld, ld, None)
    assert [swiglu(cols=40), swiglu(rows=2 ** 27)] == [SHAPE] * 2 and [swiglu(dy=None), swiglu(left=None)] == [NULL] * 2
    assert [swiglu(dy=away), swiglu(left=away), swiglu(ld=68)] == [-4] * 3 and swiglu(ld=56) == -5 and swiglu(rows=0, dy=None) == 0
