"""How near the gradients of the layers in 8 bits come to 64 bits: no further off than the roundings that the layers state.

A result's own rounding to bf16, rho, is measured on the exact values; what a layer adds to it in fp32 sums is under 2^-14.  One more rounding to bf16 on the way, of another quantity, makes
sqrt(2) rho of it: 1.1 rho tells the two apart.  Every test first has its oracle make the mistake that it is to find.
"""
import pytest
import torch

from oracle import mx8 as O

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5
# rows, outputs, inner size: products by every kind of route, odd numbers of outputs, few rows
SIZES = [(24, 2048, 1024), (300, 1728, 576), (512, 512, 1024), (1100, 1357, 2112), (2050, 2048, 512), (333, 40, 4096), (4096, 1000, 288)]


def randn(*shape, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(BF16)


def quantized(t):
    return O.quantize(t.detach().double())[0]


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def rounding(want):
    return off(want.to(BF16), want)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_swiglu_and_projection(device, M, N, K):
    from picotron_amd import functional
    g = torch.Generator(device="cuda").manual_seed(M + N)
    gate_up, w, dy = randn(M, 2 * K, g=g, scale=1.5).requires_grad_(), randn(N, K, g=g, scale=K ** -0.5).requires_grad_(), randn(M, N, g=g, scale=0.01)
    kept = quantized(gate_up)
    dh = dy.double() @ w.detach().double()
    want = O.swiglu_gradient(kept[:, :K], kept[:, K:], dh)
    limit = 1.1 * rounding(want) + 2.0 ** -14
    assert off(O.swiglu_gradient(kept[:, :K], kept[:, K:], dh.to(BF16).double()).to(BF16), want) > limit
    dx, dw = torch.autograd.grad(functional.swiglu_linear_8bit(gate_up, w), (gate_up, w), dy)
    assert off(dx, want) < limit
    # the weight's gradient: silu(gate) up is rounded to bf16 as an operand, and the result is
    h = O.silu(kept[:, :K]) * kept[:, K:]
    want_w = dy.double().t() @ h
    assert off(dw, want_w) < 1.1 * (rounding(want_w) ** 2 + off(dy.double().t() @ h.to(BF16).double(), want_w) ** 2) ** 0.5 + 2.0 ** -14
    frozen, = torch.autograd.grad(functional.swiglu_linear_8bit(gate_up, w.detach()), gate_up, dy)
    assert torch.equal(frozen, dx)


@pytest.mark.parametrize("gamma_dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_norm_and_projection(device, M, N, K, gamma_dtype):
    """gamma's gradient: dy w in fp32 and h in 20 bits, so that with a gamma in fp32, whose gradient is not rounded, what h lacks is all that is left: 2^-12 of each of its values at most."""
    from picotron_amd import functional
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x, r = (randn(M, K, g=g).requires_grad_() for _ in range(2))
    gamma = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(BF16).to(gamma_dtype).requires_grad_()
    w, dy = randn(N, K, g=g, scale=K ** -0.5).requires_grad_(), randn(M, N, g=g, scale=0.01)
    h = x.detach().double() + r.detach().double()
    rstd = (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    da = dy.double() @ w.detach().double()
    terms = da * h * rstd
    want = terms.sum(0)
    # (the roundings' signs are random: their sum is bounded by the root of the squares' sum, with each at its largest in place of its mean, sqrt(3) less)
    limit = 2.0 ** -12 * (terms.norm() / want.norm()).item() + 2.0 ** -16 + (1.1 * rounding(want) if gamma_dtype == BF16 else 0.0)
    held = lambda t: t if gamma_dtype == F32 else t.to(BF16)      # noqa: E731
    for mistake in ((da * h.to(BF16).double() * rstd).sum(0), (da.to(BF16).double() * h * rstd).sum(0)):
        assert off(held(mistake), want) > limit
    y, _ = functional.rms_norm_linear_8bit(x, r, gamma, EPS, w)
    got, = torch.autograd.grad(y, gamma, dy)
    assert got.dtype == gamma_dtype and off(got, want) < limit


@pytest.mark.parametrize("rows,cols,parts", [(1, 32, 1), (33, 576, 3), (70, 4128, 2), (257, 1056, 64)])
@pytest.mark.parametrize("want_y", [False, True])
def test_swiglus_gradient_from_pieces(device, rows, cols, parts, want_y):
    """Through the C ABI, into rows with a pitch: fp32 pieces are added before anything is rounded, and nothing else is written."""
    import ctypes
    from picotron_amd import _lib, ops
    lib, g = _lib.lib(), torch.Generator(device="cuda").manual_seed(cols)
    dy = torch.randn(parts, rows, cols, generator=g, device="cuda")
    gate, up = (ops.mx8_quantize(torch.randn(rows, cols, generator=g, device="cuda") * 2) for _ in range(2))
    dg, du = (torch.full((rows + 1, cols + 8), 5.0, dtype=BF16, device="cuda") for _ in range(2))
    y = torch.full((rows + 1, cols), 5.0, dtype=BF16, device="cuda") if want_y else None
    p = lambda t: ctypes.c_void_p(t.data_ptr()) if t is not None else None      # noqa: E731
    m = lambda t: ctypes.byref(_lib.Mx8(t.data.data_ptr(), t.scales.data_ptr()))      # noqa: E731
    _lib.check(lib.pico_swiglu_mx8_bwd_sums(p(dy), parts, m(gate), m(up), p(dg), p(du), p(y), rows, cols, cols + 8, cols + 8, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    a, b, d = gate.dequantize(F32).double(), up.dequantize(F32).double(), dy.double().sum(0)
    want = O.swiglu_gradient(a, b, d)
    u = 2.0 ** -24
    slack = (parts + 40) * u * dy.double().abs().sum(0) * (a.abs() + b.abs()) * 2 + 1e-30      # (sums of the pieces, an exponential and a reciprocal; 1 + g (1 - s) may cancel)
    for got, value in ((dg, want[:, :cols]), (du, want[:, cols:])):
        assert ((got[:rows, :cols].double() - value).abs() <= 2.0 ** -8 * value.abs() + slack).all() and (got[:, cols:] == 5).all() and (got[rows] == 5).all()
    if want_y:
        h = O.silu(a) * b
        assert ((y[:rows].double() - h).abs() <= (2.0 ** -8 + 40 * u) * h.abs() + 1e-30).all() and (y[rows] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("M", [0, 5, 300])
def test_norm_weights_of_other_types(device, M, dtype):
    """Used in bf16, as everywhere; its gradient comes in its own type, and where it is frozen the others' come too."""
    from picotron_amd import functional
    g = torch.Generator(device="cuda").manual_seed(M)
    x, r, w, dy = randn(M, 128, g=g).requires_grad_(), randn(M, 128, g=g), randn(72, 128, g=g, scale=0.1).requires_grad_(), randn(M, 72, g=g)
    gamma = randn(128, g=g)
    got = {}
    for t in (dtype, F32):
        leaf = gamma.to(t).requires_grad_()
        y, _ = functional.rms_norm_linear_8bit(x, r, leaf, EPS, w)
        got[t] = (y.detach(), *torch.autograd.grad(y, (x, w, leaf), dy))
    assert got[dtype][3].dtype == dtype and torch.equal(got[dtype][3], got[F32][3].to(dtype))
    assert all(torch.equal(a, b) for a, b in zip(got[dtype][:3], got[F32][:3]))
    y, _ = functional.rms_norm_linear_8bit(x, r, gamma.to(dtype), EPS, w)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), got[F32][1:3]))


def in_bits20(v):
    """fp32 v [rows, cols] rounded to 20 bits: (the first 16 as they lie in bf16, the words of eight times the other four, the values)."""
    bits = v.view(torch.int32) + 0x800
    words = ((bits >> 12 & 15).long().view(v.size(0), -1, 8) << torch.arange(0, 32, 4, device=v.device)).sum(-1)
    return (bits >> 16).to(torch.int16).view(BF16), torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32), (bits & ~0xfff).view(F32)


@pytest.mark.parametrize("tile", [(256, 256), (256, 192), (192, 256), (256, 128), (128, 256)])
@pytest.mark.parametrize("M,N,K", [(256, 256, 128), (1, 16, 136), (300, 272, 576), (1000, 1040, 200), (3000, 4112, 320)])
def test_a_product_in_20_bits(device, M, N, K, tile):
    """Of the fp32 sums that the same kernel gives; more tiles than workgroups, tiles cut at every side, nothing written beside them."""
    import ctypes
    from picotron_amd import _lib
    lib, g = _lib.lib(), torch.Generator(device="cuda").manual_seed(M)
    a, b = randn(M, K + 8, g=g)[:, :K], randn(K, N + 24, g=g)[:, :N]
    sums = torch.empty(M, N, device="cuda")
    c, left = torch.full((M * N + 64,), 3.0, dtype=BF16, device="cuda"), torch.full((M * N // 8 + 64,), 77, dtype=torch.int32, device="cuda")
    p = lambda t, off=0: ctypes.c_void_p(t.data_ptr() + off)      # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(lib.pico_product_large_sums(p(a), p(b), p(sums), M, N, K, K + 8, N + 24, 0, 1, *tile, 1, stream))
    _lib.check(lib.pico_product_large_bits20(p(a), p(b), p(c, 64), p(left, 128), M, N, K, K + 8, N + 24, *tile, stream))
    held, words, _ = in_bits20(sums)
    assert torch.equal(c[32:-32].view(M, N).view(torch.int16), held.view(torch.int16)) and torch.equal(left[32:-32].view(M, -1), words)
    assert (c[:32] == 3).all() and (c[-32:] == 3).all() and (left[:32] == 77).all() and (left[-32:] == 77).all()


@pytest.mark.parametrize("rows,cols", [(1, 32), (33, 576), (70, 4128)])
@pytest.mark.parametrize("want_y", [False, True])
def test_swiglus_gradient_from_20_bits(device, rows, cols, want_y):
    """As from the same values in fp32, which the two hold."""
    import ctypes
    from picotron_amd import _lib, ops
    lib, g = _lib.lib(), torch.Generator(device="cuda").manual_seed(cols)
    held, words, whole = in_bits20(torch.randn(rows, cols, generator=g, device="cuda"))
    gate, up = (ops.mx8_quantize(torch.randn(rows, cols, generator=g, device="cuda") * 2) for _ in range(2))
    p = lambda t: ctypes.c_void_p(t.data_ptr()) if t is not None else None      # noqa: E731
    m = lambda t: ctypes.byref(_lib.Mx8(t.data.data_ptr(), t.scales.data_ptr()))      # noqa: E731
    stream, got = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), []
    for call in (lambda *o: lib.pico_swiglu_mx8_bwd_bits20(p(held), p(words), m(gate), m(up), *o), lambda *o: lib.pico_swiglu_mx8_bwd_sums(p(whole), 1, m(gate), m(up), *o)):
        dg, du = (torch.full((rows + 1, cols + 8), 5.0, dtype=BF16, device="cuda") for _ in range(2))
        y = torch.full((rows + 1, cols), 5.0, dtype=BF16, device="cuda") if want_y else None
        _lib.check(call(p(dg), p(du), p(y), rows, cols, cols + 8, cols + 8, stream))
        got.append([t for t in (dg, du, y) if t is not None])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and (got[0][0][:, cols:] == 5).all() and (got[0][1][rows] == 5).all()
