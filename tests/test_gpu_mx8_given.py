"""Operands in 8 bits that another program made: every code under every scale, and the scale that makes its block NaN whatever its codes are."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def given(codes, scales):
    """ops.Mx8 of uint8 codes [rows, cols] and scale bytes [rows, cols / 32]."""
    from picotron_amd import ops
    rows, cols = codes.shape
    groups = (cols + 127) // 128
    padded = torch.zeros(rows, 4 * groups, dtype=torch.uint8, device="cuda")
    padded[:, :cols // 32] = scales
    return ops.Mx8(codes.contiguous().view(torch.float8_e4m3fn), padded.view(rows, groups, 4).transpose(0, 1).contiguous())


def test_every_code_under_every_scale(device):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").expand(256, 256)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").view(256, 1).expand(256, 8)
    got = given(codes, scales).dequantize(F32)
    values = codes.view(torch.float8_e4m3fn).double() * torch.exp2(torch.arange(256, device="cuda").double() - 127).view(256, 1)
    want = values.float()       # (what is under 2^-126 is rounded as fp32 does, what is over its largest value is infinite)
    want[255] = float("nan")
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("M,N,K", [(3, 40, 160), (300, 300, 416)])
def test_a_nan_scale_in_a_product_is_that_of_the_values(device, M, N, K):
    from picotron_amd import ops
    g = torch.Generator(device="cuda").manual_seed(K)
    def operand(rows, bad):
        scales = torch.randint(120, 130, (rows, K // 32), generator=g, device="cuda", dtype=torch.uint8)
        if bad is not None:
            scales[bad] = 255
        return given(torch.randint(0, 0x78, (rows, K), generator=g, device="cuda", dtype=torch.uint8), scales)
    a, b = operand(M, (M // 2, K // 32 - 1)), operand(N, (N // 3, 0))
    got, va, vb = ops.mx8_product(a, b), a.dequantize(F32), b.dequantize(F32)
    bad = va.isnan().any(1)[:, None] | vb.isnan().any(1)[None]
    assert va.isnan().sum() == vb.isnan().sum() == 32 and torch.equal(got.isnan(), bad)
