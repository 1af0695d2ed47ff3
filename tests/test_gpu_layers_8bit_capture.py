"""A training step that is captured while an eager graph of the same leaves lives is refused by the layers in 8 bits before its backward could end the process."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
EPS = 1e-5


def cases():
    from picotron_amd import functional as F
    g = torch.Generator(device="cuda").manual_seed(1)
    def leaf(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(BF16).requires_grad_()
    x, r, gamma, w, wide, down = leaf(40, 64), leaf(40, 64), leaf(64), leaf(48, 64), leaf(40, 128), leaf(24, 64)
    parts = [torch.nn.Parameter(p) for p in w.detach().split((16, 32))]
    return {"linear": (lambda: F.linear_8bit(x, w), (x, w)), "norm": (lambda: F.rms_norm_linear_8bit(x, r, gamma, EPS, w)[0], (x, r, gamma, w)),
            "parts": (lambda: F.rms_norm_linear_8bit(x.detach(), r.detach(), gamma.detach(), EPS, w.detach(), parts=parts)[0], parts),
            "swiglu": (lambda: F.swiglu_8bit(wide), (wide,)), "swiglu_linear": (lambda: F.swiglu_linear_8bit(wide, down), (wide, down))}


@pytest.mark.parametrize("name", ["linear", "norm", "parts", "swiglu", "swiglu_linear"])
def test_a_capture_beside_an_eager_graph(device, name):
    call, leaves = cases()[name]
    def step():
        y = call()
        return (y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y)))
    want = step()
    eager = call()                       # (a graph that lives)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            step()
    torch.cuda.synchronize()
    other = torch.cuda.CUDAGraph()       # (a forward alone has nothing to refuse)
    with torch.cuda.graph(other):
        held = call().detach()
    other.replay()
    assert torch.equal(held, want[0])
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, leaves, torch.ones_like(eager)), want[1:]))
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        torch.ones(1000, device="cuda").sum()

