"""Layers whose activations are held in 8 bits, with their gradients, against float64; a run of them as a decoder layer and as a model uses them.

e = 2^-8 bounds a rounding to bf16.  A bound on a norm follows from bounds on the values: each rounding adds at most e times the norm of what is rounded.
"""
import os

import pytest
import torch

from oracle import mx8 as O

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0 ** -8
EPS = 1e-5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, g, scale=1.0, dtype=BF16):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def quantized(t):
    return O.quantize(t.detach().double().reshape(-1, t.size(-1)))[0].view(t.shape)


def near(got, want, tol, slack=0.0):
    """|got - want| <= tol |want| + slack, as norms; fp32 sums (2^-16 of the whole, generously) beside it"""
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    off, whole = (got.double() - want).norm().item(), want.norm().item()
    assert off <= (tol + 2.0 ** -16) * whole + slack, (off, whole, tol, slack)


# ------------------------------------------------------------------------------------------------- SwiGLU
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,half", [(1, 32), (1, 8192), (3, 96), (17, 1408), (130, 576), (65, 2048), (5, 11008)])
def test_swiglu(device, rows, half, dtype):
    from picotron_amd import functional
    g = gen(rows + half)
    gate_up = randn(rows, 2 * half, g=g, scale=2.0, dtype=dtype).requires_grad_()
    y = functional.swiglu_8bit(gate_up)
    assert y.dtype == dtype
    dy = randn(rows, half, g=g, dtype=dtype)
    (d,) = torch.autograd.grad(y, gate_up, dy)
    with torch.no_grad():
        assert torch.equal(functional.swiglu_8bit(gate_up), y)
    v = gate_up.detach().double()
    want = O.silu(v[:, :half]) * v[:, half:]
    kept = quantized(gate_up)
    want_d = O.swiglu_gradient(kept[:, :half], kept[:, half:], dy.double())
    # value by value: one rounding to the type, and a dozen fp32 ones (an exponential and a reciprocal among them, whose argument's rounding counts |x| times)
    unit = (E if dtype == BF16 else 0.0) + 40 * 2.0 ** -24
    assert ((y.double() - want).abs() <= unit * want.abs() + 1e-30).all()
    slope = dy.double().abs() * kept[:, half:].abs() * 2      # (1 + g (1 - s) may cancel)
    assert ((d[:, :half].double() - want_d[:, :half]).abs() <= unit * want_d[:, :half].abs() + 40 * 2.0 ** -24 * slope + 1e-30).all()
    assert ((d[:, half:].double() - want_d[:, half:]).abs() <= unit * want_d[:, half:].abs() + 1e-30).all()


def test_swiglu_gradient_against_differences(device):
    """At values that 8 bits hold exactly the gradient is that of silu(gate) * up: central differences of the formula in 64 bits."""
    from picotron_amd import functional
    g = gen(1)
    codes = torch.randint(-15, 16, (37, 2 * 96), generator=g, device="cuda").float() / 4
    x = codes.clone().requires_grad_()
    y = functional.swiglu_8bit(x)
    dy = randn(37, 96, g=g, dtype=F32)
    (d,) = torch.autograd.grad(y, x, dy)
    v, along, h = codes.double(), torch.randn(37, 192, generator=g, device="cuda", dtype=F64), 1e-4
    f = lambda t: (O.silu(t[:, :96]) * t[:, 96:] * dy.double()).sum()      # noqa: E731
    slope = (f(v + h * along) - f(v - h * along)) / (2 * h)
    # the third derivative over six times h^2, and fp32 roundings of the summands
    assert abs((d.double() * along).sum() - slope) <= h * h * dy.double().abs().sum() * 30 + 2.0 ** -20 * (d.double() * along).abs().sum()


def test_swiglu_extremes(device):
    from picotron_amd import functional
    x = torch.zeros(4, 128, device="cuda")
    x[0, :64], x[0, 64:] = -200, 3           # a closed gate
    x[1, :64], x[1, 64:] = 200, 3
    x[2, 5], x[2, 64 + 40] = float("nan"), float("inf")
    x.requires_grad_()
    y = functional.swiglu_8bit(x)
    (d,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert (y[0] == 0).all() and (y[1] == 600).all() and (y[3] == 0).all() and y[2, 5].isnan()
    assert torch.isfinite(d[[0, 1, 3]]).all() and d[2, :32].isnan().all()      # (the block of the NaN was kept as NaN)


# ------------------------------------------------------------------------------------------------- projections
ROWS = [(1, 64, 32), (1, 2048, 576), (2, 40, 96), (17, 136, 160), (64, 256, 576), (129, 1000, 288), (300, 1728, 576), (512, 512, 1024), (1100, 260, 544), (2050, 2048, 512), (1100, 1357, 2112)]


@pytest.mark.parametrize("M,N,K", ROWS)
def test_linear(device, M, N, K):
    from picotron_amd import functional, ops
    g = gen(M + N + K)
    x, w = randn(M, K, g=g).requires_grad_(), randn(N, K, g=g, scale=K ** -0.5).requires_grad_()
    dy = randn(M, N, g=g)
    y = functional.linear_8bit(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    qx, qw = quantized(x), quantized(w)
    near(y, qx @ qw.t(), E)
    near(dx, dy.double() @ w.detach().double(), E)
    near(dw, dy.double().t() @ qx, E)
    packed = ops.mx8_quantize(w)
    with torch.no_grad():
        assert torch.equal(functional.linear_8bit(x, w), y) and torch.equal(functional.linear_8bit(x, w, packed=packed), y)
    again = functional.linear_8bit(x, w, packed=packed)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, (x, w), dy), (dx, dw)))


def test_linear_gradients_against_differences(device):
    """The product is linear in what is held exactly: steps from one such value to another give its differences without an error, and these the gradients'."""
    from picotron_amd import functional
    g = gen(7)
    M, N, K = 40, 72, 160
    def whole(*shape):
        v = torch.randint(-3, 4, shape, generator=g, device="cuda").float()
        v.view(shape[0], -1, 32)[..., 0] = 7       # (a block's scale stays)
        return v
    x, w, dy = whole(M, K), whole(N, K), torch.randint(-2, 3, (M, N), generator=g, device="cuda").float()
    move_x, move_w = (torch.randint(-2, 3, (n, K), generator=g, device="cuda").float() for n in (M, N))
    for m in (move_x, move_w):
        m.view(m.size(0), -1, 32)[..., 0] = 0
    a, b = x.to(BF16).requires_grad_(), w.to(BF16).requires_grad_()
    y = functional.linear_8bit(a, b)
    dx, dw = torch.autograd.grad(y, (a, b), dy.to(BF16))
    f = lambda p, q: (functional.linear_8bit(p.to(BF16), q.to(BF16)).double() * dy.double()).sum()      # noqa: E731
    with torch.no_grad():
        for grad, move, slope in ((dx, move_x, (f(x + move_x, w) - f(x - move_x, w)) / 2), (dw, move_w, (f(x, w + move_w) - f(x, w - move_w)) / 2)):
            # y is rounded to bf16 in each of the two, and the gradient's values are
            tol = E * (y.double().abs() * dy.double().abs()).sum() * 2 + E * (grad.double() * move.double()).abs().sum()
            assert abs((grad.double() * move.double()).sum() - slope) <= tol
    assert torch.equal(dx.double(), (dy.double() @ w.double()).to(BF16).double()) and torch.equal(dw.double(), (dy.double().t() @ x.double()).to(BF16).double())


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,N,K", ROWS)
def test_norm_linear(device, M, N, K, residual):
    from picotron_amd import functional
    g = gen(M + N + K)
    x = randn(M, K, g=g).requires_grad_()
    r = randn(M, K, g=g).requires_grad_() if residual else None
    gamma = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(BF16).requires_grad_()
    w = randn(N, K, g=g, scale=K ** -0.5).requires_grad_()
    dy, dh = randn(M, N, g=g), randn(M, K, g=g)
    y, h = functional.rms_norm_linear_8bit(x, r, gamma, EPS, w)
    leaves = [t for t in (x, r, gamma, w) if t is not None]
    got = dict(zip(("x", "r", "gamma", "w") if residual else ("x", "gamma", "w"), torch.autograd.grad((y, h), leaves, (dy, dh))))
    s = x.detach().double() + (r.detach().double() if residual else 0)
    if residual:
        assert torch.equal(h, s.to(BF16)) and torch.equal(got["x"], got["r"])
    else:
        assert torch.equal(h, x)
    rstd = (s.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    q, qw = quantized(s * rstd * gamma.detach().double()), quantized(w)
    # an 8-bit value on the other side of a middle (fp32 sums of squares) is off by a step, 2^-3 of itself at most, one in 2^14 at most of them
    flips = 2.0 ** -3 * 2.0 ** -7
    near(y, q @ qw.t(), E + flips, slack=1e-3 if M * K < 4096 else 0)
    da = dy.double() @ w.detach().double()
    want, want_gamma = O.norm_gradient(s, gamma.detach().double(), da, dh.double(), EPS)
    # da is rounded, then comes h (x's values, or their sum rounded), each of which is multiplied by at most rstd max|gamma| |da| on its way; the output is rounded
    passed = (rstd * da.abs() * gamma.detach().double().abs().max()).norm().item()
    near(got["x"], want, E, slack=4 * E * passed)
    n = (s * rstd).abs()
    near(got["gamma"], want_gamma, E, slack=2 * E * (da.abs() * n).pow(2).sum(0).sqrt().norm().item() * 2)
    near(got["w"], dy.double().t() @ q, E + flips, slack=1e-3 * dy.norm().item() if M * K < 4096 else 0)
    with torch.no_grad():
        again = functional.rms_norm_linear_8bit(x, r, gamma, EPS, w)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)


def test_norm_linear_partial_gradients(device):
    """Only the stream's gradient, only the projection's, frozen weights, parts of a weight."""
    from picotron_amd import functional
    g = gen(3)
    x, r, gamma, w = randn(5, 7, 64, g=g), randn(5, 7, 64, g=g), randn(64, g=g), randn(48, 64, g=g, scale=0.1)
    leaf = lambda t: t.clone().requires_grad_()      # noqa: E731
    a, b, c, d = leaf(x), leaf(r), leaf(gamma), leaf(w)
    dy, dh = randn(5, 7, 48, g=g), randn(5, 7, 64, g=g)
    whole = torch.autograd.grad(functional.rms_norm_linear_8bit(a, b, c, EPS, d), (a, b, c, d), (dy, dh))
    y, h = functional.rms_norm_linear_8bit(a, b, c, EPS, d)
    only = torch.autograd.grad(h, (a, b, c, d), dh, allow_unused=True, retain_graph=True)
    assert torch.equal(only[0], dh) and torch.equal(only[1], dh) and only[2] is None and only[3] is None
    without = torch.autograd.grad(y, (a, b, c, d), dy)
    assert torch.equal(without[3], whole[3]) and torch.equal(without[2], whole[2]) and not torch.equal(without[0], whole[0])
    y, h = functional.rms_norm_linear_8bit(a, r, gamma, EPS, w)                       # nothing trained but what comes before
    assert torch.equal(torch.autograd.grad((y, h), a, (dy, dh))[0], whole[0])
    y, h = functional.rms_norm_linear_8bit(x, r, gamma, EPS, d)                       # the projection alone
    assert torch.equal(torch.autograd.grad(y, d, dy)[0], whole[3])
    buf = w.clone()
    parts = [torch.nn.Parameter(buf[:16]), torch.nn.Parameter(buf[16:24]), torch.nn.Parameter(buf[24:])]
    y, h = functional.rms_norm_linear_8bit(a, b, c, EPS, buf, parts=parts)
    got = torch.autograd.grad((y, h), (a, c, *parts), (dy, dh))
    assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[2]) and torch.equal(torch.cat(got[2:]), whole[3])
    with pytest.raises(RuntimeError, match="rows"):
        functional.rms_norm_linear_8bit(a, b, c, EPS, buf, parts=parts[:2])
    gamma32 = gamma.float().requires_grad_()                                          # a norm's weight of another type
    y, h = functional.rms_norm_linear_8bit(a, b, gamma32, EPS, d)
    assert torch.autograd.grad((y, h), gamma32, (dy, dh))[0].dtype == F32


@pytest.mark.parametrize("M,N,K", ROWS)
def test_swiglu_linear(device, M, N, K):
    from picotron_amd import functional
    g = gen(M + N + K)
    gate_up, w = randn(M, 2 * K, g=g, scale=1.5).requires_grad_(), randn(N, K, g=g, scale=K ** -0.5).requires_grad_()
    dy = randn(M, N, g=g)
    y = functional.swiglu_linear_8bit(gate_up, w)
    dx, dw = torch.autograd.grad(y, (gate_up, w), dy)
    v, kept = gate_up.detach().double(), quantized(gate_up)
    q = quantized(O.silu(v[:, :K]) * v[:, K:])
    flips = 2.0 ** -3 * 2.0 ** -7      # (as in test_norm_linear: fp32 exponentials)
    near(y, q @ quantized(w).t(), E + flips, slack=1e-3 if M * K < 4096 else 0)
    dh = dy.double() @ w.detach().double()
    want = O.swiglu_gradient(kept[:, :K], kept[:, K:], dh)
    near(dx, want, 2 * E)              # dh is rounded, value by value, and so is the output
    h = O.silu(kept[:, :K]) * kept[:, K:]
    near(dw, dy.double().t() @ h, E, slack=E * dy.double().norm().item() * h.norm().item() * 2 / max(1.0, M ** 0.5))      # (h is rounded)
    with torch.no_grad():
        assert torch.equal(functional.swiglu_linear_8bit(gate_up, w), y)
    frozen = functional.swiglu_linear_8bit(gate_up, w.detach())
    assert torch.equal(torch.autograd.grad(frozen, gate_up, dy)[0], dx)
    alone = functional.swiglu_linear_8bit(gate_up.detach(), w)
    assert torch.equal(torch.autograd.grad(alone, w, dy)[0], dw)


# ------------------------------------------------------------------------------------------------- the norm's gradient from fp32 pieces
def in_bf16_and_what_is_left(h):
    """(bf16(h), h with four bits more than that, the words of these bits) of fp32 h [rows, hidden]."""
    held = h.to(BF16)
    bits, first = h.view(torch.int32), held.float().view(torch.int32)
    left = ((bits - first + 2048) >> 12).clamp(-8, 7)
    shifts = torch.arange(0, 32, 4, device=h.device)
    words = ((left.long() & 15).view(h.size(0), -1, 8) << shifts).sum(-1)
    return held, (first + (left << 12)).view(F32), torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


@pytest.mark.parametrize("rows,hidden", [(1, 32), (5, 576), (300, 2048), (7, 4128), (3, 16384)])
def test_what_the_rounding_of_the_stream_leaves(device, rows, hidden):
    """The words as defined, for values of any size, infinities and zeros; h itself within 2^-12 of bf16's last places more than it."""
    import ctypes
    from picotron_amd import _lib
    lib, g = _lib.lib(), gen(hidden)
    x, r = (randn(rows, hidden, g=g, dtype=F32) * torch.exp2(torch.randint(-100, 100, (rows, hidden), generator=g, device="cuda").float()) for _ in range(2))
    x, r = x.to(BF16), torch.where(torch.rand(rows, hidden, generator=g, device="cuda") < 0.5, randn(rows, hidden, g=g).float() * x.abs().float() * 0.1, r).to(BF16)
    x[0, :4], r[0, :4] = torch.tensor([0.0, -0.0, float("inf"), 1.0], device="cuda"), torch.tensor([0.0, -0.0, 1.0, -1.0], device="cuda")
    h = x.float() + r.float()
    out, words = torch.empty_like(x), torch.full((rows * hidden // 8 + 4,), 77, dtype=torch.int32, device="cuda")
    data, scales = torch.empty(rows, hidden, dtype=torch.uint8, device="cuda"), torch.empty((hidden + 127) // 128, rows, 4, dtype=torch.uint8, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    _lib.check(lib.pico_rmsnorm_mx8_fwd(p(x), p(torch.ones_like(x[0])), ctypes.byref(_lib.Mx8(data.data_ptr(), scales.data_ptr())), None, p(r), p(out), p(words), rows, hidden, EPS,
                                        _lib.PICO_BF16, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    held, whole, want = in_bf16_and_what_is_left(h)
    assert torch.equal(out, held) and torch.equal(words[:-4].view(rows, -1), want) and (words[-4:] == 77).all()
    finite = h.isfinite() & (h.abs() >= 2.0 ** -126)
    assert ((whole - h).abs()[finite] <= 2.0 ** -11 * h.abs()[finite]).all()
    assert rows == 1 or ((held.float() - h).abs()[finite] > 2.0 ** -11 * h.abs()[finite]).any()


@pytest.mark.parametrize("dw_dtype", [BF16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,hidden,parts", [(1, 8, 1), (3, 96, 2), (33, 576, 1), (257, 2048, 3), (70, 4096, 1), (9, 4104, 2), (5, 8192, 1), (4, 16384, 2), (4500, 264, 1)])
@pytest.mark.parametrize("left", [False, True])
def test_norm_gradient_of_sums(device, rows, hidden, parts, residual, dw_dtype, left):
    import ctypes
    from picotron_amd import _lib
    lib, g = _lib.lib(), gen(rows + hidden)
    dy = torch.randn(parts, rows, hidden, generator=g, device="cuda")
    h, gamma = randn(rows, hidden, g=g, dtype=F32), (1 + 0.2 * torch.randn(hidden, generator=g, device="cuda")).to(BF16)
    x, whole, words = in_bf16_and_what_is_left(h)
    if not left:
        whole, words = x, None
    rstd = (whole.double().pow(2).mean(-1) + EPS).rsqrt().float()
    dres = randn(rows, hidden, g=g) if residual else None
    dx, dw = torch.empty_like(x), torch.full((hidden + 8,), 3.0, dtype=dw_dtype, device="cuda")
    ws = torch.empty(lib.pico_rmsnorm_bwd_workspace_bytes(rows, hidden), dtype=torch.uint8, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr()) if t is not None else None      # noqa: E731
    _lib.check(lib.pico_rmsnorm_bwd_sums(p(dy), parts, p(x), p(words), p(gamma), p(rstd), p(dres), p(dx), p(dw), _lib.PICO_BF16 if dw_dtype == BF16 else _lib.PICO_F32, p(ws), ws.numel(), rows, hidden,
                                         ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    d, n, w = dy.double().sum(0), whole.double() * rstd.double()[:, None], gamma.double()
    q = d * w
    want = rstd.double()[:, None] * (q - n * (q * n).mean(-1, keepdim=True)) + (dres.double() if residual else 0)
    # sums of `rows` (dweight) and `hidden` (the row's mean) products in fp32, 64 side by side at least; one rounding to bf16
    u = 2.0 ** -24
    mean = rstd.double()[:, None] * n.abs() * (q * n).abs().mean(-1, keepdim=True)
    slack = (hidden / 64 + 20) * u * mean + 16 * u * (rstd.double()[:, None] * q.abs() + want.abs() + (dres.double().abs() if residual else 0))
    assert ((dx.double() - want).abs() <= E * want.abs() + slack).all()
    want_w = (d * n).sum(0)
    unit = E if dw_dtype == BF16 else 0.0
    assert ((dw[:hidden].double() - want_w).abs() <= unit * want_w.abs() + (rows / 4 + 600) * u * (d * n).abs().sum(0) / max(1.0, rows ** 0.5) + 8 * u * (d * n).abs().sum(0)).all()
    assert (dw[hidden:] == 3).all()


@pytest.mark.parametrize("kind,M,N,K,tile,parts", [("mid", 33, 96, 64, (64, 96), 1), ("mid", 200, 136, 576, (64, 128), 3), ("mid", 130, 264, 1000, (96, 96), 1), ("mid", 500, 200, 320, (128, 128), 1),
                                                   ("large", 300, 264, 512, (256, 256), 1), ("large", 300, 264, 512, (128, 256), 2)])
def test_products_that_leave_their_sums(device, kind, M, N, K, tile, parts):
    """fp32 sums of whole numbers are exact; nothing behind them is written."""
    import ctypes
    from picotron_amd import _lib
    g = gen(M)
    a, b = (torch.randint(-8, 9, s, generator=g, device="cuda").to(BF16) for s in ((M, K), (K, N)))
    sums = torch.full((parts * M * N + 64,), 7.0, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    f = _lib.lib().pico_product_mid_sums if kind == "mid" else _lib.lib().pico_product_large_sums
    _lib.check(f(p(a), p(b), p(sums), M, N, K, K, N, 0, 1, *tile, parts, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(sums[:-64].view(parts, M, N).sum(0), a.float() @ b.float()) and (sums[-64:] == 7).all()


# ------------------------------------------------------------------------------------------------- how they are called
def layer(x, residual, gamma, gate_up_w, down_w):
    from picotron_amd import functional
    gate_up, h = functional.rms_norm_linear_8bit(x, residual, gamma, EPS, gate_up_w)
    return functional.swiglu_linear_8bit(gate_up, down_w), h


def layer_inputs(M=96, K=160, inner=288, seed=0):
    g = gen(seed)
    return [t.requires_grad_() for t in (randn(M, K, g=g), randn(M, K, g=g), (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(BF16),
                                         randn(2 * inner, K, g=g, scale=K ** -0.5), randn(K, inner, g=g, scale=inner ** -0.5))], randn(M, K, g=g), randn(M, K, g=g)


def test_a_run_of_them(device):
    """Norm, gate and up, SwiGLU, down: forward and all gradients of the run in 64 bits, with the tensor between the two rounded to bf16 as it is."""
    leaves, dy, dh = layer_inputs()
    y, h = layer(*leaves)
    got = torch.autograd.grad((y, h), leaves, (dy, dh))
    x, r, gamma, w1, w2 = (t.detach().double() for t in leaves)
    K, inner = w2.shape
    s = x + r
    rstd = (s.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    q = quantized(s * rstd * gamma)
    gate_up = (q @ quantized(w1).t()).to(BF16).double()
    kept = quantized(gate_up)
    a = quantized(O.silu(gate_up[:, :inner]) * gate_up[:, inner:])
    # a value of gate_up whose rounding to bf16 goes the other way is off by 2^-7, and what is made of it in 8 bits by a step at most: one in 2^8 at most do
    flips = 2.0 ** -3 * 2.0 ** -4
    near(y, a @ quantized(w2).t(), E + flips)
    da = dy.double() @ w2
    dgu = O.swiglu_gradient(kept[:, :inner], kept[:, inner:], da)
    near(got[4], dy.double().t() @ (O.silu(kept[:, :inner]) * kept[:, inner:]), 2 * E + flips)
    near(got[3], dgu.t() @ q, 2 * E + flips)
    dn = dgu @ w1
    want, want_gamma = O.norm_gradient(s, gamma, dn, dh.double(), EPS)
    near(got[0], want, 2 * E + flips, slack=(4 * E + flips) * (rstd * dn.abs() * gamma.abs().max()).norm().item())
    near(got[2], want_gamma, 2 * E + flips, slack=(4 * E + flips) * (dn.abs() * (s * rstd).abs()).pow(2).sum(0).sqrt().norm().item())


def test_what_is_kept(device):
    """A byte and a thirty-second for every value that the backward reads of the activations between the stream's h and the output."""
    M, K, inner = 256, 128, 512
    leaves, _, _ = layer_inputs(M, K, inner)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y, h = layer(*leaves)
    mine = {t.data_ptr(): t.numel() * t.element_size() for t in kept if not any(t.data_ptr() == p.data_ptr() for p in (*leaves, h))}
    packed = M * K + M * K // 32 + 2 * (M * inner + M * inner // 32)
    assert sum(mine.values()) == packed + M * 4 + M * K // 2      # (and rstd, and four bits more of h than bf16 holds)


def test_upstream_gradients_of_any_layout(device):
    leaves, dy, dh = layer_inputs()
    y, h = layer(*leaves)
    want = torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True)
    wide = torch.empty(dy.size(0), 2 * dy.size(1), dtype=BF16, device="cuda")
    wide[:, 1::2] = dy
    got = torch.autograd.grad((y, h), leaves, (wide[:, 1::2], dh.t().contiguous().t()), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    row = dy[:1].expand_as(dy)
    got = torch.autograd.grad((y, h), leaves, (row, row), retain_graph=True)
    want = torch.autograd.grad((y, h), leaves, (row.contiguous(), row.contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    from picotron_amd import functional
    x = randn(9, 128, g=gen(1)).requires_grad_()
    d = randn(1, 64, g=gen(2))
    y = functional.swiglu_8bit(x)
    a, = torch.autograd.grad(y, x, d.expand(9, 64), retain_graph=True)
    b, = torch.autograd.grad(y, x, d.expand(9, 64).contiguous())
    assert torch.equal(a, b)


def test_inputs_of_any_layout(device):
    from picotron_amd import functional
    g = gen(4)
    base, w = randn(50, 520, g=g), randn(40, 128, g=g)
    for v in (base[:, 8:136], base[:, 3:131], base[::2, :128], base[:, :512].view(50, 4, 128).transpose(0, 1), base[:1, :128].expand(9, 128), base[0, :128], base[:0, :128]):
        a, b = v.detach().requires_grad_(), v.detach().contiguous().requires_grad_()
        ya, yb = functional.linear_8bit(a, w), functional.linear_8bit(b, w)
        assert torch.equal(ya, yb) and torch.equal(*(torch.autograd.grad(y.float().square().sum(), t)[0] for y, t in ((ya, a), (yb, b))))
        na, nb = (functional.rms_norm_linear_8bit(t, None, torch.ones(128, device="cuda", dtype=BF16), EPS, w)[0] for t in (a, b))
        assert torch.equal(na, nb)
        assert torch.equal(functional.swiglu_8bit(a), functional.swiglu_8bit(b))
        assert torch.equal(functional.swiglu_linear_8bit(a, w[:, :64]), functional.swiglu_linear_8bit(b, w[:, :64].contiguous()))


def test_tensors_that_start_anywhere(device):
    """Contiguous, but 2 bytes behind a 16-byte boundary: every input and every upstream gradient."""
    leaves, dy, dh = layer_inputs()
    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.detach().reshape(-1)
        return flat[1:].view(t.shape)
    for residual in (True, False):
        args = [t if residual or i != 1 else None for i, t in enumerate(leaves)]
        away = [None if t is None else moved(t).requires_grad_() for t in args]
        (y, h), (ya, ha) = layer(*args), layer(*away)
        want = torch.autograd.grad((y, h), [t for t in args if t is not None], (dy, dh))
        got = torch.autograd.grad((ya, ha), [t for t in away if t is not None], (moved(dy), moved(dh)))
        assert torch.equal(y, ya) and torch.equal(h, ha) and all(torch.equal(a, b) for a, b in zip(want, got))
    from picotron_amd import functional
    a, b = leaves[3], moved(leaves[3]).requires_grad_()
    d = randn(a.size(0), a.size(1) // 2, g=gen(1))
    pair = [torch.autograd.grad(functional.swiglu_8bit(t[:, :128]), t, g[:, :64])[0] for t, g in ((a, d), (b, moved(d)))]
    assert torch.equal(*pair)


def test_empty_batches_train(device):
    leaves, dy, dh = layer_inputs(M=0)
    y, h = layer(*leaves)
    got = torch.autograd.grad((y, h), leaves, (dy, dh))
    assert all(a.shape == b.shape for a, b in zip(got, leaves)) and all((t == 0).all() for t in got)


def test_a_captured_step_replays(device):
    leaves, dy, dh = layer_inputs(M=300, K=320, inner=544)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    def step():
        y, h = layer(*leaves)
        return (y, h, *torch.autograd.grad((y, h), leaves, (dy, dh)))
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    other, _, _ = layer_inputs(M=300, K=320, inner=544, seed=9)
    for source in (other, None, other):
        with torch.no_grad():
            if source is not None:
                for a, b in zip(leaves, source):
                    a.copy_(b)
            else:
                for a in leaves:
                    a.mul_(0.5)
        want = step()
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("tokens", [1, 7, 24])
def test_a_captured_run_without_gradients_replays(device, tokens):
    """A few tokens: rows rounded inside the product, contractions in pieces over a workspace, forms of few rows; two graphs that were captured one after the other replay in turn."""
    from picotron_amd import functional, ops
    g = gen(tokens)
    w, v, gamma = randn(1024, 2048, g=g, scale=0.02), randn(2048, 8192, g=g, scale=0.01), randn(2048, g=g)
    pw, pv = ops.mx8_quantize(w), ops.mx8_quantize(v)
    x, r, gate_up = randn(tokens, 2048, g=g), randn(tokens, 2048, g=g), randn(tokens, 16384, g=g)

    def run():
        a = functional.linear_8bit(x, w, packed=pw)
        b, h = functional.rms_norm_linear_8bit(x, r, gamma, EPS, w, packed=pw)
        return a, b, h, functional.swiglu_linear_8bit(gate_up, v, packed=pv)
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            run()
        torch.cuda.current_stream().wait_stream(stream)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = run()
            graphs.append((graph, held))
        for turn in range(4):
            for t in (x, r, gate_up):
                t.copy_(randn(*t.shape, g=g))
            want = run()
            graph, held = graphs[turn % 2]
            for t in held:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_other_streams_and_threads(device):
    import threading
    leaves, dy, dh = layer_inputs(M=300, K=320, inner=544)
    def step():
        y, h = layer(*leaves)
        return (y, h, *torch.autograd.grad((y, h), leaves, (dy, dh)))
    want = step()
    torch.cuda.synchronize()
    got = [None] * 4
    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(3):
                got[i] = step()
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


# ------------------------------------------------------------------------------------------------- in the model
class _Straight(torch.autograd.Function):
    """The 8-bit form's values; the gradient passes as it is."""

    @staticmethod
    def forward(ctx, v):
        return quantized(v)

    @staticmethod
    def backward(ctx, g):
        return g


class _Product(torch.autograd.Function):
    """a w8^T in 64 bits; the gradient of a through w."""

    @staticmethod
    def forward(ctx, a, w):
        ctx.save_for_backward(a, w)
        return (a @ quantized(w).t()).to(BF16)

    @staticmethod
    def backward(ctx, dy):
        a, w = ctx.saved_tensors
        return dy.double() @ w.double(), (dy.double().reshape(-1, dy.size(-1)).t() @ a.reshape(-1, a.size(-1))).to(w.dtype)


def plain_norm_linear(x, residual, norm_weight, eps, weight, packed=None, parts=()):
    h = x if residual is None else (x.double() + residual.double()).to(BF16)
    s = h.double()
    a = _Straight.apply(s * (s.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * norm_weight.double())
    return _Product.apply(a, torch.cat(list(parts)) if len(parts) else weight), h


def plain_swiglu_linear(gate_up, weight, packed=None):
    gate, up = gate_up.double().chunk(2, -1)
    return _Product.apply(_Straight.apply(torch.nn.functional.silu(gate) * up), weight)


@pytest.mark.parametrize("kv_heads", [4, 2])
def test_model_in_8_bits(device, monkeypatch, kv_heads):
    """Two decoder layers, forward and gradients, against the same model with these layers in 64 bits.  The one takes a value to bf16 that the other does not, so 8-bit
    values may differ by a step, 2^-3 of themselves at most; one in 16 do (a rounding to bf16, 2^-8, against a step of 2^-4 to 2^-3), in four places one behind the other."""
    from types import SimpleNamespace
    import picotron_amd.process_group_manager as pgm
    from picotron_amd import model as M
    from picotron_amd.functional import cross_entropy
    pgm.setup_process_group_manager(1, 1, 1, 1)
    monkeypatch.setenv("CONTEXT_PARALLEL", "0")
    monkeypatch.delenv("FLASH_ATTEN", raising=False)
    config = SimpleNamespace(hidden_size=256, num_attention_heads=4, num_key_value_heads=kv_heads, num_hidden_layers=2, intermediate_size=544, vocab_size=1000, max_position_embeddings=160,
                             rms_norm_eps=1e-5, rope_theta=10000.0)
    torch.manual_seed(1)
    model = M.Llama(config).to(device=device, dtype=BF16)
    ids = torch.randint(0, 1000, (2, 129), generator=gen(2), device="cuda")

    def step():
        model.zero_grad()
        logits = model(ids[:, :-1])
        cross_entropy(logits.reshape(-1, 1000), ids[:, 1:].reshape(-1)).backward()
        return logits.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}

    in_bf16 = step()[0]
    monkeypatch.setenv("PICO_LINEAR_8BIT", "1")
    logits, grads = step()
    again, same = step()
    assert torch.equal(again, logits) and all(torch.equal(same[n], grads[n]) for n in grads if n != "embedding.weight")
    assert not torch.equal(logits, in_bf16)
    with torch.no_grad():
        assert torch.equal(model(ids[:, :-1]), logits)
    monkeypatch.setattr(M, "rms_norm_linear_8bit", plain_norm_linear)
    monkeypatch.setattr(M, "swiglu_linear_8bit", plain_swiglu_linear)
    want, want_grads = step()
    near(logits, want.double(), 4 * (2.0 ** -3 / 4 + E))
    for n, w in want_grads.items():       # (SwiGLU's gradient at its 8-bit values too: 2^-4 of each at most)
        near(grads[n], w.double(), 4 * (2.0 ** -3 / 4 + E) + 2 * 2.0 ** -4)
    monkeypatch.setenv("PICO_FUSED_PROJ", "0")
    with pytest.raises(RuntimeError, match="fused projections"):
        model(ids[:, :-1])
    monkeypatch.delenv("PICO_FUSED_PROJ")
    monkeypatch.setenv("PICO_FUSED_RESIDUAL", "0")
    with pytest.raises(RuntimeError, match="inside the norms"):
        model(ids[:, :-1])


def test_model_over_virtual_ranks_in_8_bits(device, monkeypatch):
    """The ring over two virtual ranks gives what one rank gives: what is computed row by row is the same, attention differs in its roundings."""
    from types import SimpleNamespace
    import picotron_amd.process_group_manager as pgm
    from picotron_amd import model as M
    monkeypatch.delenv("FLASH_ATTEN", raising=False)
    monkeypatch.setenv("PICO_LINEAR_8BIT", "1")
    config = SimpleNamespace(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=1, intermediate_size=320, vocab_size=500, max_position_embeddings=256, rms_norm_eps=1e-5,
                             rope_theta=10000.0)
    ids = torch.randint(0, 500, (1, 256), generator=gen(3), device="cuda")
    pgm.setup_process_group_manager(1, 1, 1, 1)
    monkeypatch.setenv("CONTEXT_PARALLEL", "0")
    torch.manual_seed(4)
    model = M.Llama(config).to(device=device, dtype=BF16)
    with torch.no_grad():
        want = model(ids)
    pgm.setup_process_group_manager(1, 2, 1, 1)
    monkeypatch.setenv("CONTEXT_PARALLEL", "1")
    got = []
    with torch.no_grad():
        for rank in range(2):
            model.set_cp_rank(rank)
            got.append(model(ids[:, 128 * rank:128 * (rank + 1)]))
    pgm.setup_process_group_manager(1, 1, 1, 1)
    near(torch.cat(got, 1), want.double(), 2.0 ** -3 / 4 + 2 * E)


def test_refusals(device):
    from picotron_amd import functional, ops
    x, w, n = torch.ones(4, 64, device="cuda", dtype=BF16), torch.ones(8, 64, device="cuda", dtype=BF16), torch.ones(64, device="cuda", dtype=BF16)
    for call, match in ((lambda: functional.linear_8bit(x.float(), w), "must be bf16"), (lambda: functional.linear_8bit(x, w.float()), "must be bf16"),
                        (lambda: functional.linear_8bit(x, w[:, :32]), r"\[out, 64\]"), (lambda: functional.linear_8bit(x[:, :40], w[:, :40]), "multiple of 32"),
                        (lambda: functional.linear_8bit(x, w, packed=ops.mx8_quantize(w[:4])), "8-bit form"),
                        (lambda: functional.rms_norm_linear_8bit(x, x[:2], n, EPS, w), "residual"), (lambda: functional.rms_norm_linear_8bit(x, x.float(), n, EPS, w), "residual"),
                        (lambda: functional.rms_norm_linear_8bit(x, None, n[:32], EPS, w), "norm's weight"),
                        (lambda: functional.swiglu_8bit(x[:, :32]), "multiple of 32"), (lambda: functional.swiglu_8bit(x.half()), "not supported"),
                        (lambda: functional.swiglu_linear_8bit(x, w), r"\[out, 32\]"), (lambda: functional.swiglu_linear_8bit(x[:, :63], w), "two halves")):
        with pytest.raises(RuntimeError, match=match):
            call()
    a = x.clone().requires_grad_()
    for f in (lambda: functional.linear_8bit(a, w), lambda: functional.rms_norm_linear_8bit(a, None, n, EPS, w)[0], lambda: functional.swiglu_8bit(a),
              lambda: functional.swiglu_linear_8bit(a, w[:, :32])):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(f().sum(), a, create_graph=True)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for f in (lambda: functional.linear_8bit(d, w), lambda: functional.rms_norm_linear_8bit(x, d, n, EPS, w), lambda: functional.swiglu_8bit(d), lambda: functional.swiglu_linear_8bit(d, w[:, :32])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
