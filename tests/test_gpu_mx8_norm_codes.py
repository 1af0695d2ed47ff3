"""RMSNorm in 8 bits gives the code of the exact value, everywhere: normal rows, sums that lose the smaller of two, rows over many powers of two, gammas of any size.

What the kernel rounds on its way to a value that lies beside the middle of two codes: the sum of squares (64 bits, 2^-53 a term), a Newton step in 64 bits from a root in 32 (2^-43), that
root in twice 24 bits, and products of what 24 bits hold with what they leave (2^-45).  Middles lie 2^-4 of the value apart at least, so a code differs for one value in 2^38: none here.
"""
import ctypes

import pytest
import torch

from oracle import mx8 as O

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = torch.tensor(1e-5, dtype=F32).double().item()


def exact(packed, h, w):
    """How many codes and scales are not those of h rsqrt(mean h^2 + eps) w in 64 bits."""
    codes = scales = 0
    got, exponents = packed.dequantize(F32).double(), O.exponents_of(packed.scales, h.size(1))
    for i in range(0, h.size(0), 2048):
        v = h[i:i + 2048]
        q, e = O.quantize(v * (v.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w.double())
        codes += (got[i:i + 2048] != q).sum().item()
        scales += (exponents[i:i + 2048] != e).sum().item()
    return codes, scales


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols,dtype", [(16384, 2048, BF16), (8192, 576, BF16), (6000, 4128, BF16), (1500, 16384, BF16), (16384, 576, F32), (8192, 2048, F32), (3000, 8224, F32)])
def test_normal_rows(device, rows, cols, dtype, residual):
    from picotron_amd import ops
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, r = (torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    packed, _, _ = ops.rmsnorm_mx8_fwd(x, w, 1e-5, residual=r if residual else None)
    assert exact(packed, x.double() + r.double() if residual else x.double(), w) == (0, 0)


def four_squares(n):
    """Whole numbers up to 256 whose squares add up to n."""
    for a in range(min(256, int(n ** 0.5)), 0, -1):
        for b in range(min(a, int((n - a * a) ** 0.5)), 0, -1):
            for c in range(min(b, int((n - a * a - b * b) ** 0.5)), -1, -1):
                d = round((n - a * a - b * b - c * c) ** 0.5)
                if d * d == n - a * a - b * b - c * c and d <= 256:
                    return a, b, c, d
    raise ValueError(n)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_a_sum_loses_counts(device, dtype):
    """Odd numbers from 17 to 31 lie in the middle of two codes, also by a root mean square of 32, which the rows' squares add up to.  A residual of 2^-25 to 2^-28 of a value is lost in the
    sum in 32 bits and alone says to which side it goes."""
    from picotron_amd import ops
    g = torch.Generator().manual_seed(7)
    x = torch.zeros(512, 256, dtype=torch.float64)
    for i in range(8):
        row = torch.randint(8, 16, (252,), generator=g) * 2 + 1
        fill = torch.tensor(four_squares(256 * 1024 - row.pow(2).sum().item()))
        x[i::8] = torch.cat((row, fill)) * torch.where(torch.rand(256, generator=g) < 0.5, -1, 1)
    r = x * torch.exp2(-25.0 - torch.randint(0, 4, x.shape, generator=g)) * torch.where(torch.rand(x.shape, generator=g) < 0.5, -1, 1)
    r[:, 252:] = 0
    h, x, r = (x + r).cuda(), x.to(dtype).cuda(), r.to(dtype).cuda()
    assert (x.double() + r.double() == h).all() and torch.equal(x.float() + r.float(), x.float())
    w = torch.ones(256, device="cuda", dtype=dtype)
    packed, _, _ = ops.rmsnorm_mx8_fwd(x, w, 0.0, residual=r)
    rms = h.pow(2).mean(-1, keepdim=True).sqrt()
    q, e = O.quantize(h / rms)
    plain, _ = O.quantize(x.double() / 32)
    assert (q != plain).float().mean() > 0.3                                   # (a kernel without what is lost would be wrong there)
    assert torch.equal(packed.dequantize(F32).double(), q) and torch.equal(O.exponents_of(packed.scales, 256), e)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(4096, 512), (700, 4128)])
def test_rows_and_channels_of_any_size(device, rows, cols, dtype):
    from picotron_amd import ops
    g = torch.Generator(device="cuda").manual_seed(rows)
    def wide():
        x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp2(torch.randint(-12, 13, (rows, 1), generator=g, device="cuda").float())
        return (x * torch.exp2(torch.randint(-9, 10, (rows, cols), generator=g, device="cuda").float())).to(dtype)
    x, r = wide(), wide()
    w = (torch.randn(cols, generator=g, device="cuda") * torch.exp2(torch.randint(-4, 5, (cols,), generator=g, device="cuda").float())).to(dtype)
    packed, _, _ = ops.rmsnorm_mx8_fwd(x, w, 1e-5, residual=r)
    assert exact(packed, x.double() + r.double(), w) == (0, 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_zeros_and_their_signs(device, dtype):
    from picotron_amd import ops
    x = torch.zeros(5, 160, device="cuda", dtype=dtype)
    x[1] = -0.0
    x[2, 7], x[3, ::2] = -3, 1.5
    for r in (None, torch.zeros_like(x), torch.full_like(x, -0.0)):
        packed, _, h = ops.rmsnorm_mx8_fwd(x, torch.ones(160, device="cuda", dtype=dtype), 1e-5, residual=r)
        assert exact(packed, x.double(), torch.ones(160, device="cuda")) == (0, 0)
        assert r is None or torch.equal(h, x)


@pytest.mark.parametrize("of", ["x", "residual"])
def test_the_sum_in_an_operands_place(device, of):
    """Through the C ABI.  Nothing can be read again there: as many codes as in 32 bits alone may be the other one, one in 2^18 at most."""
    from picotron_amd import _lib, ops
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(300, 576, generator=g, device="cuda").to(BF16) for _ in range(2))
    w = torch.randn(576, generator=g, device="cuda").to(BF16)
    want, _, h = ops.rmsnorm_mx8_fwd(x, w, 1e-5, residual=r)
    data, scales, place = torch.empty_like(want.data), torch.empty_like(want.scales), x if of == "x" else r
    p = lambda t: ctypes.c_void_p(t.data_ptr())      # noqa: E731
    _lib.check(_lib.lib().pico_rmsnorm_mx8_fwd(p(x), p(w), ctypes.byref(_lib.Mx8(data.data_ptr(), scales.data_ptr())), None, p(r), p(place), None, 300, 576, 1e-5, _lib.PICO_BF16,
                                               ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(place, h) and (data.view(torch.uint8) != want.data.view(torch.uint8)).sum() <= 300 * 576 // 2 ** 17 + 1
    assert torch.equal(scales, want.scales)
