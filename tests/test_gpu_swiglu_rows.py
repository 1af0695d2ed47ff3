"""SwiGLU where rows share memory: upstream gradients of sums and expanded inputs have a stride of 0, and their memory holds one row only."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, HALF = 37, 72


def values(*sizes, dtype=torch.bfloat16, seed=0):
    return torch.randn(*sizes, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes,over", [((ROWS,), (0,)), ((5, ROWS), (0,)), ((5, ROWS), (1,)), ((5, ROWS), (0, 1)), ((5, 1), (0,))])
def test_the_gradient_of_a_sum_of_rows(device, sizes, over, dtype):
    from picotron_amd.functional import SwiGLUFunc, SwiGLUFusedFunc
    gate_up = values(*sizes, 2 * HALF, dtype=dtype)
    dy = values(*[1 if i in over else n for i, n in enumerate(sizes)], HALF, dtype=dtype, seed=1).expand(*sizes, HALF)
    assert any(n > 1 and dy.stride(i) == 0 for i, n in enumerate(sizes))
    got, want = [], []
    for out, d in ((got, dy), (want, dy.contiguous())):
        x = gate_up.clone().requires_grad_()
        out += torch.autograd.grad(SwiGLUFusedFunc.apply(x), x, d)
        gate, up = (t.contiguous().requires_grad_() for t in gate_up.split(HALF, -1))
        out += torch.autograd.grad(SwiGLUFunc.apply(gate, up), (gate, up), d)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_expanded_inputs(device):
    from picotron_amd import ops
    gate, up = values(1, HALF).expand(ROWS, HALF), values(ROWS, HALF, seed=1)
    assert torch.equal(ops.swiglu_fwd(gate, up), ops.swiglu_fwd(gate.contiguous(), up))
    overlapping = values(ROWS * 8 + HALF).as_strided((ROWS, HALF), (8, 1))
    assert torch.equal(ops.swiglu_fwd(up, overlapping), ops.swiglu_fwd(up, overlapping.contiguous()))


def test_outputs_whose_rows_share_memory_are_refused(device):
    from picotron_amd import ops
    gate, up, dy = (values(ROWS, HALF, seed=i) for i in range(3))
    with pytest.raises(RuntimeError, match="one row pitch"):
        ops.swiglu_bwd(dy, gate, up, (values(1, HALF).expand(ROWS, HALF), torch.empty_like(up)))
