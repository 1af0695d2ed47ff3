"""Views whose rows have no single pitch although an axis of one element lies between: a part of [batch, 1, positions, values]."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def part(batch, positions, of, cols, dtype=BF16, seed=0):
    """[batch, 1, positions, cols] out of as many rows of [batch, 1, of, cols]: batches lie `of` rows apart, and the axis of one element has that stride too."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(batch, 1, of, cols, generator=g).to(dtype).cuda()[:, :, :positions]
    assert v.stride(0) == v.stride(1) == of * cols
    return v


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_swiglu(device, dtype):
    from picotron_amd import ops
    gate, up, dy = (part(3, 5, 11, 72, dtype, seed) for seed in range(3))
    dense = [t.contiguous() for t in (gate, up, dy)]
    assert torch.equal(ops.swiglu_fwd(gate, up), ops.swiglu_fwd(*dense[:2]))
    for got, want in zip(ops.swiglu_bwd(dy, gate, up), ops.swiglu_bwd(dense[2], *dense[:2])):
        assert torch.equal(got, want)


def test_swiglu_does_not_write_into_them(device):
    from picotron_amd import ops
    gate, up, dy = (part(3, 5, 5, 72, seed=seed) for seed in range(3))
    with pytest.raises(RuntimeError, match="one row pitch"):
        ops.swiglu_bwd(dy, gate, up, (part(3, 5, 11, 72), torch.empty_like(up)))


def test_gradients_of_empty_batches_into_halves(device):
    from picotron_amd import ops
    whole = torch.empty(7, 0, 144, dtype=BF16, device="cuda")
    gate, up = whole.split(72, -1)
    dg, du = ops.swiglu_bwd(torch.empty(7, 0, 72, dtype=BF16, device="cuda"), gate, up, whole.clone().split(72, -1))
    assert dg.shape == du.shape == (7, 0, 72)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_the_8_bit_form(device, dtype):
    from picotron_amd import functional, ops
    v = part(3, 5, 11, 128, dtype)
    got, want = ops.mx8_quantize(v), ops.mx8_quantize(v.contiguous())
    assert torch.equal(got.dequantize(torch.float32), want.dequantize(torch.float32)) and torch.equal(got.scales, want.scales)
    assert torch.equal(functional.swiglu_8bit(v), functional.swiglu_8bit(v.contiguous()))
    a = v.contiguous().requires_grad_()
    y, dy = functional.swiglu_8bit(a), part(3, 5, 11, 64, dtype, 1)
    assert torch.equal(*(torch.autograd.grad(y, a, d, retain_graph=True)[0] for d in (dy, dy.contiguous())))


@pytest.mark.parametrize("cols", [128, 2048])
def test_layers_in_8_bits(device, cols):
    from picotron_amd import functional
    w = part(1, 40, 40, cols, seed=3)[0, 0]
    x = part(3, 2, 11, cols)
    for f in (lambda t: functional.linear_8bit(t, w), lambda t: functional.swiglu_linear_8bit(t, w[:, :cols // 2].contiguous())):
        want = f(x.contiguous())
        assert torch.equal(f(x), want)                              # (nothing is kept of x)
        a, b = x.detach().requires_grad_(), x.contiguous().requires_grad_()
        dy = part(3, 2, 11, 40, seed=5)
        got = [torch.autograd.grad(y, t, d)[0] for y, t, d in ((f(a), a, dy), (f(b), b, dy.contiguous()))]
        assert torch.equal(f(a), want) and torch.equal(*got)
