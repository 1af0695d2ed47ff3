"""Log-probabilities straight from hidden states at the limits of what they take.  u = 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
IGNORE = -100


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("T", [1.0, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-9, 1e-20])
@pytest.mark.parametrize("rows,hidden,vocab", [(1, 4096, 3000), (5, 128, 700), (20, 264, 1001), (70, 128, 5003), (300, 2048, 2051), (1100, 264, 33001), (512, 4096, 8200)])
def test_temperatures_that_leave_the_largest_logits_only(device, rows, hidden, vocab, T):
    """Hidden states and weights are small whole numbers: the logits are whole numbers of up to some hundreds, which fp32 holds exactly, and the largest of a row may be
    several.  So log p is off by its own roundings alone, 2^-16 + 4 u |log p|, and a gradient as usual: 2^-15 of p, 2^-21 at the target, bf16 of d(logits) (2^-8) and of the
    result, the products' sums 2^-10; what is under 2^-126 may be 0."""
    from picotron_amd.functional import linear_log_probs
    T = torch.tensor(T).item()      # as fp32 has it
    g = gen(rows)
    x = torch.randint(-2, 3, (rows, hidden), generator=g, device="cuda").to(BF16)
    w = torch.randint(-2, 3, (vocab, hidden), generator=g, device="cuda").to(BF16)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    assert z.abs().max().item() < 2 ** 20
    top = (z == z.amax(1, keepdim=True))
    t = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.6, top.double().argmax(1), torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
    t[torch.rand(rows, generator=g, device="cuda") < 0.1] = IGNORE
    t[0] = top[0].double().argmax()
    n = t != IGNORE
    every = torch.log_softmax(z / T, 1)
    del z
    lp = torch.where(n, every.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    y, v = x.clone().requires_grad_(), w.clone().requires_grad_()
    q = linear_log_probs(y, v, t, temperature=T)
    over = (q.double() - lp).abs() - 2 ** -16 - 2 ** -22 * lp.abs()
    assert not q.isnan().any() and (over <= 0).all(), over.max().item()
    assert not q[~n].any()
    a = torch.randn(rows, generator=g, device="cuda")
    dx, dw = torch.autograd.grad(q, (y, v), a)
    a = torch.where(n, a.double(), 0.0)[:, None] / T
    p = every.exp()
    del every
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    d = a * (hot - p)
    dd = 2 ** -125 * (1 + a.abs()) + 2 ** -8 * d.abs() + a.abs() * (p * 2 ** -15 + hot * 2 ** -21)
    for got, want, bound in ((dx, d @ wd, dd @ wd.abs() + 2 ** -10 * (d.abs() @ wd.abs())), (dw, d.t() @ xd, dd.t() @ xd.abs() + 2 ** -10 * (d.abs().t() @ xd.abs()))):
        over = (got.double() - want).abs() - bound - 2 ** -8 * want.abs() - 1e-37
        assert not got.isnan().any() and (over <= 0).all(), over.max().item()


@pytest.mark.parametrize("rows,hidden,vocab", [(2, 128, 1000), (4, 2112, 20000), (32, 2048, 16001), (40, 128, 600), (64, 4096, 2049), (100, 2112, 49152), (127, 4096, 32001), (300, 576, 1003),
                                               (600, 576, 2000), (2000, 4096, 8192), (1503, 2048, 16385)])
@pytest.mark.parametrize("wanted", ["both", "weight", "x"])
def test_rows_that_do_not_count_may_hold_anything(device, rows, hidden, vocab, wanted):
    """NaN and infinities in hidden states whose target does not count: the same bits of both gradients as beside ordinary ones, in every product that may take them."""
    from picotron_amd.functional import linear_log_probs
    g = gen(rows)
    x = torch.randn(rows, hidden, generator=g, device="cuda").to(BF16)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * 0.1).to(BF16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    r = torch.arange(rows, device="cuda")
    t = torch.where(r % 4 == 1, IGNORE, torch.where(r % 4 == 3, vocab + r, t))
    a = torch.randn(rows, generator=g, device="cuda")
    out = []
    for fill in (None, float("nan"), float("inf")):
        y = x if fill is None else torch.where((r % 2 == 1)[:, None], fill, x)
        y, v = y.detach().clone().requires_grad_(wanted != "weight"), w.clone().requires_grad_(wanted != "x")
        out.append(torch.autograd.grad(linear_log_probs(y, v, t), [p for p in (y, v) if p.requires_grad], a))
    for clean, *others in zip(*out):
        assert bool(clean.any()) and not clean.isnan().any()
        for other in others:
            assert torch.equal(clean, other)
    if wanted != "weight":
        assert not out[1][0][r % 2 == 1].any()


@pytest.mark.parametrize("T", [1e-7, 1e-8, 1e-10, 1e-20])
@pytest.mark.parametrize("rows,hidden,vocab", [(1, 4096, 3000), (7, 264, 1001), (32, 2048, 8192), (70, 128, 5003), (512, 4096, 8200)])
def test_gradients_at_temperatures_under_the_logits_roundings(device, rows, hidden, vocab, T):
    """A logit's rounding over T is more than any exponent holds, and the backward may add logits up in another order: probabilities stay under 1 and gradients finite.
    (|d(logits)| <= |a| / T (1 + 2^-8), and with |w| <= 1 no sum of them leaves bf16.)  A row that is no number stays one."""
    from picotron_amd.functional import linear_log_probs
    g = gen(rows + hidden)
    x = torch.randn(rows, hidden, generator=g, device="cuda").to(BF16)
    w = (torch.randn(vocab, hidden, generator=g, device="cuda") * (2 / hidden ** 0.5)).clamp(-1, 1).to(BF16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    a = torch.randn(rows, generator=g, device="cuda")
    y, v = x.clone().requires_grad_(), w.clone().requires_grad_()
    q = linear_log_probs(y, v, t, temperature=T)
    assert q.isfinite().all() and (q <= 0).all()
    dx, dw = torch.autograd.grad(q, (y, v), a)
    assert dx.isfinite().all() and dw.isfinite().all()
    bad = x.clone()
    bad[rows // 2, 3] = float("nan")
    y = bad.requires_grad_()
    for temperature in (1.0, T):
        q = linear_log_probs(y, v, t, temperature=temperature)
        dx, dw = torch.autograd.grad(q, (y, v), a)
        r = torch.arange(rows, device="cuda") == rows // 2
        assert torch.equal(q.isnan(), r) and dx[r].isnan().all() and not dx[~r].isnan().any() and dw.isnan().all()
