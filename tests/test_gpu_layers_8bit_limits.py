"""The ends of what the layers in 8 bits take: no outputs, one value's worth of axes, the smallest blocks."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
EPS = 1e-5


def leaf(*shape):
    return torch.randn(shape, device="cuda").to(BF16).requires_grad_()


@pytest.mark.parametrize("rows", [(), (5,), (2, 3), (2, 0, 3)])
def test_no_outputs(device, rows):
    """A weight [0, in], as a part of a projection may be: nothing comes out, and the gradients are 0."""
    from picotron_amd import functional as F
    x, r, gamma, w, wide = leaf(*rows, 64), leaf(*rows, 64), leaf(64), leaf(0, 64), leaf(*rows, 128)
    dh = torch.randn(*rows, 64, device="cuda").to(BF16)
    for y, leaves in ((F.linear_8bit(x, w), (x, w)), (F.swiglu_linear_8bit(wide, w), (wide, w)), (F.rms_norm_linear_8bit(x, r, gamma, EPS, w)[0], (x, r, gamma, w))):
        assert y.shape == (*rows, 0)
        got = torch.autograd.grad(y, leaves, torch.empty_like(y))
        assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(got, leaves))
    y, h = F.rms_norm_linear_8bit(x, r, gamma, EPS, w)
    got = torch.autograd.grad((y, h), (x, gamma), (torch.empty_like(y), dh))
    assert torch.equal(got[0], dh) and (got[1] == 0).all()


@pytest.mark.parametrize("rows", [(), (1,), (1, 1, 1)])
@pytest.mark.parametrize("out", [1, 7, 8])
def test_one_row_of_the_smallest_block(device, rows, out):
    """Against the same row as a matrix."""
    from picotron_amd import functional as F
    x, gamma, w, wide = leaf(*rows, 32), leaf(32), leaf(out, 32), leaf(*rows, 64)
    dy = torch.randn(*rows, out, device="cuda").to(BF16)
    for f, t in ((lambda t: F.linear_8bit(t, w), x), (lambda t: F.swiglu_linear_8bit(t, w), wide), (lambda t: F.rms_norm_linear_8bit(t, None, gamma, EPS, w)[0], x)):
        flat = t.detach().reshape(1, -1).requires_grad_()
        y, z = f(t), f(flat)
        assert y.shape == (*rows, out) and torch.equal(y.reshape(1, -1), z)
        a, b = torch.autograd.grad(y, (t, w), dy), torch.autograd.grad(z, (flat, w), dy.reshape(1, -1))
        assert torch.equal(a[0].reshape(1, -1), b[0]) and torch.equal(a[1], b[1]) and a[0].shape == t.shape
