"""Activations and weights in 8 bits: what the C ABI and the host path refuse before anything is launched, and what pins the oracle (no GPU needed)."""
import ctypes
import os

import pytest
import torch

from oracle import mx8 as O

BUF = 4096      # never read: every call here is refused first
P = ctypes.c_void_p(BUF)


@pytest.fixture(scope="module")
def lib():
    from picotron_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    return _lib.lib()


def packed(data=BUF, scales=BUF):
    from picotron_amd._lib import Mx8
    return ctypes.byref(Mx8(data, scales))


def calls(lib, x=P, y8=None, rows=4, cols=64, ld=None, dtype=0):
    """Every entry point with the same sizes; {name: status}."""
    y8 = y8 or packed()
    ld = cols if ld is None else ld
    return {
        "quantize": lib.pico_mx8_quantize(x, y8, rows, cols, ld, dtype, None),
        "dequantize": lib.pico_mx8_dequantize(y8, x, rows, cols, ld, dtype, None),
        "norm": lib.pico_rmsnorm_mx8_fwd(x, P, y8, None, None, None, None, rows, cols, 1e-5, dtype, None),
        "swiglu": lib.pico_swiglu_mx8_fwd(x, P, None, y8, None, None, rows, cols, ld, ld, dtype, None),
        "swiglu_bwd": lib.pico_swiglu_mx8_bwd(x, y8, y8, P, P, None, rows, cols, ld, ld, ld, dtype, None),
    }


@pytest.mark.parametrize("over,code", [
    (dict(dtype=5), -2), (dict(cols=0), -3), (dict(cols=31), -3), (dict(cols=48), -3), (dict(rows=-1), -3), (dict(rows=1 << 31), -3),
    (dict(rows=1 << 26, cols=4096 + 32), -3), (dict(rows=1 << 27), -3), (dict(rows=1 << 27, dtype=1), -3), (dict(rows=1 << 20, cols=128 * 128), -3), (dict(x=None), -1), (dict(x=ctypes.c_void_p(BUF + 8)), -4)])
def test_sizes_types_and_pointers(lib, over, code):
    assert set(calls(lib, **over).values()) == {code}, lib.pico_last_error()


def test_operands_in_8_bits(lib):
    for bad, code in ((packed(data=None), -1), (packed(scales=None), -1), (packed(data=BUF + 8), -4), (packed(scales=BUF + 2), -4)):
        assert set(calls(lib, y8=bad).values()) == {code}
        assert lib.pico_mx8_product(bad, packed(), P, 4, 4, 64, None, 0, None) == code
        assert lib.pico_mx8_product(packed(), bad, P, 4, 4, 64, None, 0, None) == code
    assert lib.pico_mx8_quantize(P, None, 4, 64, 64, 0, None) == -1


def test_pitches(lib):
    got = calls(lib, ld=60)
    assert {k: v for k, v in got.items() if k != "norm"} == dict(quantize=-5, dequantize=-5, swiglu=-5, swiglu_bwd=-5)
    assert {k: v for k, v in calls(lib, ld=68).items() if k != "norm"} == dict(quantize=-4, dequantize=-4, swiglu=-4, swiglu_bwd=-4)


def test_what_belongs_together(lib):
    assert lib.pico_swiglu_mx8_fwd(P, P, None, None, packed(), packed(), 4, 64, 64, 64, 0, None) == -1       # no output
    assert lib.pico_swiglu_mx8_fwd(P, P, P, None, packed(), None, 4, 64, 64, 64, 0, None) == -1              # half a checkpoint
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, None, P, None, 4, 64, 1e-5, 0, None) == -1         # a sum without a residual
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, None, None, P, 4, 64, 1e-5, 0, None) == -1         # or what its rounding leaves
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, P, P, P, 4, 64, 1e-5, 1, None) == -2               # fp32 leaves nothing
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, P, P, ctypes.c_void_p(BUF + 8), 4, 64, 1e-5, 0, None) == -4
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, None, None, None, 4, 16384 + 32, 1e-5, 0, None) == -3
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, None, None, None, 1 << 26, 64, 1e-5, 0, None) == -3     # threads of one launch
    assert lib.pico_rmsnorm_mx8_fwd(P, P, packed(), None, ctypes.c_void_p(BUF + 4), None, None, 4, 64, 1e-5, 0, None) == -4


def test_products(lib):
    def product(M=4, N=4, K=64, c=P):
        return lib.pico_mx8_product(packed(), packed(), c, M, N, K, None, 0, None)
    assert product(K=40) == -3 and product(K=0) == -3 and product(M=-1) == -3 and product(N=-1) == -3 and product(M=1 << 31) == -3
    assert product(M=1 << 22, N=1 << 22) == -3                        # threads of one launch
    assert product(c=None) == -1 and product(c=ctypes.c_void_p(BUF + 8)) == -4


def test_tiles_pieces_and_workspaces(lib):
    def tiled(tile_m=256, tile_n=256, per_cu=1, parts=1, ws=None, bytes_=0, K=1024):
        return lib.pico_mx8_product_tiled(packed(), packed(), P, 512, 512, K, tile_m, tile_n, per_cu, parts, ws, bytes_, None)
    assert tiled(tile_m=64) == -3 and tiled(tile_n=192) == -3 and tiled(per_cu=2) == -3 and tiled(per_cu=0) == -3 and tiled(tile_m=0, tile_n=9) == -3 and tiled(tile_m=0, tile_n=-1) == -3 and tiled(parts=0) == -3 and tiled(parts=5) == -3 and tiled(parts=65, K=1 << 20) == -3 and tiled(K=128) == -3
    assert tiled(tile_m=0, tile_n=0, parts=2) == -3 and tiled(tile_m=0, tile_n=3, parts=9) == -3 and tiled(tile_m=0, tile_n=3, parts=0) == -3 and tiled(tile_m=0, tile_n=3, parts=2) == -6
    assert tiled(parts=2) == -6 and tiled(parts=2, ws=P, bytes_=2 * 512 * 512 * 4 - 1) == -6 and tiled(parts=2, ws=ctypes.c_void_p(BUF + 8), bytes_=1 << 30) == -4
    bytes_ = lib.pico_mx8_product_workspace_bytes(512, 512, 65536)
    if bytes_:
        assert lib.pico_mx8_product(packed(), packed(), P, 512, 512, 65536, P, bytes_ - 1, None) == -6


def test_the_product_that_rounds(lib):
    def call(M=4, N=8, K=64, x=P, ld=64, c=P, b=None):
        return lib.pico_mx8_product_rounding(x, b or packed(), c, M, N, K, ld, None)
    assert call(M=17) == -3 and call(M=-1) == -3 and call(K=40, ld=40) == -3 and call(ld=56) == -5 and call(ld=68) == -4 and call(x=None) == -1 and call(c=None) == -1
    assert call(x=ctypes.c_void_p(BUF + 8)) == -4 and call(b=packed(scales=None)) == -1 and call(M=0, x=None) == 0 and call(M=16, N=4096, K=11008, ld=11008) == -3
    assert [lib.pico_mx8_product_rounding_pays(*s) for s in ((0, 64, 64), (17, 64, 64), (1, 0, 64), (1, 2048, 2048))] == [0, 0, 0, 1]


def test_the_norms_gradient_from_sums(lib):
    def call(parts=1, hidden=64, dw=P, dw_dtype=0, dx=P, x=ctypes.c_void_p(BUF + 64), ws=P, bytes_=1 << 30, rows=4, left=None):
        return lib.pico_rmsnorm_bwd_sums(P, parts, x, left, P, P, None, dx, dw, dw_dtype, ws, bytes_, rows, hidden, None)
    assert call(hidden=12) == -3 and call(hidden=16384 + 8) == -3 and call(rows=-1) == -3 and call(parts=0) == -3 and call(parts=65) == -3
    assert call(dw=None) == -1 and call(ws=None) == -1 and call(x=P) == -1 and call(dw_dtype=4) == -2 and call(bytes_=64) == -6 and call(dx=ctypes.c_void_p(BUF + 8)) == -4
    assert call(left=ctypes.c_void_p(BUF + 8)) == -4


def test_nothing_to_do_is_no_error(lib):
    assert set(calls(lib, x=None, y8=packed(data=None), rows=0).values()) == {0}
    assert lib.pico_mx8_product(packed(data=None), packed(), None, 0, 4, 64, None, 0, None) == 0
    assert lib.pico_mx8_product(packed(data=None), packed(), None, 4, 0, 64, None, 0, None) == 0


def test_cpu_tensors_and_wrong_types():
    from picotron_amd import _lib, functional, ops
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    x, w, n = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    for call in (lambda: ops.mx8_quantize(x), lambda: ops.rmsnorm_mx8_fwd(x, n, 1e-5), lambda: functional.linear_8bit(x, w),
                 lambda: functional.rms_norm_linear_8bit(x, None, n, 1e-5, w), lambda: functional.swiglu_8bit(x), lambda: functional.swiglu_linear_8bit(x, w[:, :32]),
                 lambda: ops.Mx8(x.to(torch.float8_e4m3fn), torch.zeros(1, 4, 4, dtype=torch.uint8)).dequantize()):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_the_oracle_rounds_as_torch_does():
    g = torch.Generator().manual_seed(3)
    v = torch.randn(64, 32, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-20, 20, (64, 1), generator=g).double())
    v[0], v[1, 3:] = 0, 0
    q, e = O.quantize(v)
    s = torch.exp2(e.double())
    largest = v.abs().amax(-1, keepdim=True)
    assert (largest <= 448 * s).all() and ((largest > 224 * s) | (e == -127)).all()       # the smallest power of two that does
    r = (v / s).float()      # (exact: the values have 24 bits or fewer where they are rounded further)
    near = r.to(torch.float8_e4m3fn).double() * s
    # a double that float moves may lie on the other side of a middle: none does here
    assert torch.equal(q, near)


def test_the_oracle_on_middles_and_borders():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middles = (codes[1:] + codes[:-1]) / 2
    for v in (codes, middles):
        rows = torch.zeros(len(v), 32, dtype=torch.float64)
        rows[:, 0], rows[:, 1] = 448, v
        q, e = O.quantize(rows)
        assert (e == 0).all()
        assert torch.equal(q[:, 1], v.float().to(torch.float8_e4m3fn).double())
    one = torch.zeros(3, 32, dtype=torch.float64)
    one[0, 5], one[1, 5], one[2, 5] = 448, 448.0001, float("inf")
    q, e = O.quantize(one)
    assert e.flatten().tolist() == [0, 1, 128] and q[2].isnan().all() and q[1, 5] == 448
