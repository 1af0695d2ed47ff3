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


# rows, outputs, half of gate and up: the product in front of SwiGLU's gradient by fp32 pieces, by whole fp32 sums, in 20 bits
ROUTES = [(40, 2048, 512), (300, 72, 576), (2500, 520, 4128)]


@pytest.mark.parametrize("M,N,K", ROUTES)
def test_routes_that_these_sizes_stand_for(device, M, N, K):
    from picotron_amd import _lib
    route = _lib.host().sums_route(torch.empty(M, N, dtype=BF16, device="cuda"), torch.empty(N, K, dtype=BF16, device="cuda"))
    assert route.startswith("large") and " in " not in route if M == 2500 else route.startswith("mid") and (" in " in route) == (M == 40), route


@pytest.mark.parametrize("M,N,K", ROUTES)
def test_infinities_in_the_upstream_gradient_stay_in_their_rows(device, M, N, K):
    from picotron_amd import functional as F
    wide, w = leaf(M, 2 * K), leaf(N, K)
    dy = torch.randn(M, N, device="cuda").to(BF16)
    bad = dy.clone()
    bad[1, 3], bad[M // 2, 0], bad[M - 1, 5] = float("inf"), float("nan"), -float("inf")
    want, = torch.autograd.grad(F.swiglu_linear_8bit(wide, w), wide, dy)
    got, = torch.autograd.grad(F.swiglu_linear_8bit(wide, w), wide, bad)
    rows = torch.ones(M, dtype=torch.bool, device="cuda")
    rows[[1, M // 2, M - 1]] = False
    assert torch.equal(got[rows], want[rows]) and not got[~rows].isfinite().any(1).all() and got[M // 2].isnan().all()
    for r in (1, M - 1):
        assert (~got[r].isfinite() | (got[r] == 0)).all()       # (0: a gate or an up of 0, times an infinity, is NaN; a weight of 0 too)


@pytest.mark.parametrize("M,N,K", ROUTES)
def test_a_captured_gradient_by_every_route(device, M, N, K):
    from picotron_amd import functional as F
    g = torch.Generator(device="cuda").manual_seed(K)
    wide, w = (torch.randn(s, generator=g, device="cuda").to(BF16).requires_grad_() for s in ((M, 2 * K), (N, K)))
    dy = torch.randn(M, N, generator=g, device="cuda").to(BF16)
    def step():
        y = F.swiglu_linear_8bit(wide, w)
        return (y.detach(), *torch.autograd.grad(y, (wide, w), dy))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            wide.copy_(torch.randn(M, 2 * K, generator=g, device="cuda"))
            dy.copy_(torch.randn(M, N, generator=g, device="cuda"))
        want = step()
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        del want
