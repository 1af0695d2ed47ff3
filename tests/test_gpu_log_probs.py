"""Log-probabilities of given tokens, the policy loss and the preference loss against their definitions in 64 bits, gradients by
differentiating those: vocabularies around the kernels' pieces, rows that start anywhere, tokens that do not count, masked and
extreme logits, streams, threads, graphs.

Tolerances, element by element.  Arithmetic is in fp32 (unit u = 2^-24) and results are rounded once to their type (half a step, U =
eps / 2).  Of a row's sum of exponentials a thread adds up to 8 (V / 512 / 8 + 1) of 49152 / 512 = 96 terms one by one; with the tree over
the workgroup (10 steps), the exponential itself (2 u) and its argument's rounding (|D| u ln2, weighted by p: under 20 u) the sum's
logarithm is off by at most (96 + 10 + 2 + 20) u < 2^-17, and 140000 entries add another 180 u.  So
  log_probs: 2^-16 + 4 u |log p|;   entropy: the same + 2^-16 H;
  gradient:  U |g| + 2^-15 (|a| p + |b| p (1 + |log p| + H)) / T + 2^-21 |a| / T at the target, where a (1 - p) cancels.
(b p (log p + H): log p and H are off by up to 2^-16 each, however small they are, and may cancel: where p = 1 both are 0.)"""
import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
IGNORE = -100


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def logits_of(g, *shape, dtype, scale=3.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def reference(x, t, T):
    """(log p of the targets, entropy, log p of everything) in 64 bits; 0 log 0 = 0."""
    every = torch.log_softmax(x.double() / T, -1)
    lp = every.gather(-1, t.clamp(0, x.size(-1) - 1)[..., None])[..., 0]
    p = every.exp()
    H = -torch.where(p > 0, p * every, 0.0).sum(-1)
    return lp, H, every


def counted(t, V, ignore=IGNORE):
    return (t != ignore) & (t >= 0) & (t < V)


def gradient(x, t, T, a, b, ignore=IGNORE):
    """(the gradient, its bound) of sum a q + b H"""
    x, V = x.detach(), x.size(-1)
    n = counted(t, V, ignore)
    a, b = (torch.where(n, v.double(), 0.0)[..., None] for v in (a, b))
    _, H, every = reference(x, t, T)
    p = every.exp()
    hot = torch.zeros_like(p).scatter_(-1, t.clamp(0, V - 1)[..., None], 1.0)
    every = torch.where(p > 0, every, 0.0)
    g = (a * (hot - p) - b * p * (every + H[..., None])) / T
    g = torch.where(n[..., None], g, 0.0)      # (a row that does not count may hold anything)
    U = torch.finfo(x.dtype).eps / 2
    bound = U * g.abs() + 2 ** -15 * (a.abs() * p + b.abs() * p * (1 + every.abs() + H[..., None])) / T + 2 ** -21 * a.abs() * hot / T + 1e-37
    return g, torch.where(n[..., None], bound, 0.0)


def near(got, want, bound, what):
    over = (got.double() - want).abs() - bound
    assert not got.isnan().any() and (over <= 0).all(), (what, over.max().item())


def lp_bound(lp):
    return 2 ** -16 + 2 ** -22 * lp.abs()


def check_log_probs(x, t, T=1.0, ignore=IGNORE, seed=0):
    from picotron_amd.functional import log_probs
    g = gen(seed + 77)
    a, b = (torch.randn(t.shape, generator=g, device="cuda") for _ in range(2))
    V = x.size(-1)
    n = counted(t, V, ignore)
    lp, H, _ = reference(x, t, T)
    lp, H = torch.where(n, lp, 0.0), torch.where(n, H, 0.0)
    x = x.detach().requires_grad_()
    with torch.no_grad():
        quiet = log_probs(x, t, ignore, T)
    q = log_probs(x, t, ignore, T)
    assert torch.equal(q, quiet) and q.shape == t.shape and q.dtype == F32
    near(q, lp, lp_bound(lp), "log_probs")
    (d,) = torch.autograd.grad(q, x, a, retain_graph=True)
    near(d, *gradient(x, t, T, a, 0 * b, ignore), "gradient")
    (again,) = torch.autograd.grad(q, x, a)
    assert torch.equal(d, again) and d.dtype == x.dtype and d.shape == x.shape
    q, h = log_probs(x, t, ignore, T, entropy=True)
    near(q, lp, lp_bound(lp), "log_probs beside entropy")
    near(h, H, 2 ** -16 * (1 + H), "entropy")
    for ups in ((a, b), (a, None), (None, b)):
        outs = [o for o, u in zip((q, h), ups) if u is not None]
        (d,) = torch.autograd.grad(outs, x, [u for u in ups if u is not None], retain_graph=True)
        near(d, *gradient(x, t, T, a if ups[0] is not None else 0 * a, b if ups[1] is not None else 0 * b, ignore), "gradient with entropy")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 17, 63, 1000, 2048, 2051, 4099, 16384, 16391, 32001, 49152, 65537, 140003])
def test_log_probs_over_vocabularies(device, dtype, vocab):
    g = gen(vocab)
    x = logits_of(g, 2, 3, vocab, dtype=dtype)
    t = torch.randint(0, vocab, (2, 3), generator=g, device="cuda")
    t[0, 0], t[0, 1], t[1, 0] = 0, vocab - 1, IGNORE
    check_log_probs(x, t, seed=vocab)
    check_log_probs(x, t, T=0.7, seed=vocab)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("start", [0, 1, 3, 7])
@pytest.mark.parametrize("pitch", [2000, 2001, 2008, 2013])
def test_log_probs_of_rows_that_start_anywhere(device, dtype, start, pitch):
    """Views with a row pitch and a first element of their own, slices along the sequence, targets that are a slice too."""
    g = gen(start * 7 + pitch)
    V, B, S = 2000, 3, 5
    buf = logits_of(g, start + B * S * pitch, dtype=dtype)
    x = buf[start:].view(B, S, pitch)[:, :, :V]
    ids = torch.randint(0, V, (B, S + 1), generator=g, device="cuda")
    check_log_probs(x, ids[:, 1:])
    check_log_probs(x[:, :-1], ids[:, 1:-1])
    check_log_probs(x[1, 2], ids[1, 2])                     # one token
    check_log_probs(x.transpose(0, 1), ids[:, 1:].t())


def test_log_probs_of_more_axes_and_broadcast_logits(device):
    g = gen(3)
    x = logits_of(g, 2, 3, 4, 501, dtype=BF16)
    t = torch.randint(0, 501, (2, 3, 4), generator=g, device="cuda")
    check_log_probs(x, t)
    check_log_probs(x[:, 1], t[:, 1])
    from picotron_amd.functional import log_probs
    one = logits_of(g, 1, 1, 501, dtype=F32).requires_grad_()   # the same row for every target: its gradients add up
    q = log_probs(one.expand(2, 12, 501), t.view(2, 12))
    (d,) = torch.autograd.grad(q.sum(), one)
    p = torch.softmax(one.detach().double(), -1)
    want = torch.bincount(t.view(-1), minlength=501).double() - 24 * p.view(-1)
    assert (d.view(-1).double() - want).abs().max().item() <= 24 * 2 ** -15


def test_log_probs_of_tokens_that_do_not_count(device):
    """Ignored rows and targets outside the vocabulary: results and gradient 0 whatever the row holds, another ignore_index, none that counts, no rows."""
    from picotron_amd.functional import log_probs
    g = gen(4)
    x = logits_of(g, 4, 6, 777, dtype=BF16)
    t = torch.randint(0, 777, (4, 6), generator=g, device="cuda")
    t[0, 0], t[0, 1], t[0, 2], t[0, 3] = IGNORE, 777, -1, 2 ** 40
    x[0, 0], x[0, 1, 5], x[0, 2] = float("nan"), float("inf"), -float("inf")
    check_log_probs(x, t)
    x[0] = 1.0
    check_log_probs(x, t, ignore=int(t[2, 2]))
    for dtype in (BF16, F32):
        y = x.to(dtype).requires_grad_()
        q, h = log_probs(y, torch.full_like(t, IGNORE), entropy=True)
        (d,) = torch.autograd.grad((q, h), y, (torch.ones_like(q), torch.ones_like(h)))
        assert not q.any() and not h.any() and not d.any()
    for shape in ((0, 5), (5, 0)):
        e = torch.empty(*shape, 8, device="cuda", dtype=BF16).requires_grad_()
        q = log_probs(e, torch.empty(shape, dtype=torch.long, device="cuda"))
        (d,) = torch.autograd.grad(q.sum(), e)
        assert q.shape == shape and d.shape == e.shape


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_log_probs_of_masked_and_extreme_logits(device, dtype):
    """-inf in most places, in whole pieces and in all but one, the type's lowest value, rows with one certain token, large values;
    a row of -inf alone, of +inf or NaN gives NaN and leaves the others alone."""
    from picotron_amd.functional import log_probs
    g = gen(5)
    V = 5003
    x = logits_of(g, 1, 9, V, dtype=dtype)
    t = torch.randint(0, V, (1, 9), generator=g, device="cuda")
    x[0, 0, torch.rand(V, generator=g, device="cuda") < 0.97] = -float("inf")
    x[0, 1, :4096] = -float("inf")
    x[0, 2] = -float("inf")
    x[0, 3, 100:] = torch.finfo(dtype).min
    x[0, 4, t[0, 4]] = 60.0
    x[0, 5] *= 300
    x[0, 6] += 1e4
    x[0, 7] = 0
    x[0, 2, t[0, 2]], x[0, 0, t[0, 0]], x[0, 1, t[0, 1]] = 2.0, 1.0, 1.0
    t[0, 3] = 50
    # (a logit of 1e3 makes D's rounding 1e3 u: the bounds above are for |D| p under 20, which p keeps them to)
    check_log_probs(x, t)
    check_log_probs(x, t, T=1.7)
    y = x.clone()
    y[0, 0], y[0, 1, 7], y[0, 2, 5] = -float("inf"), float("inf"), float("nan")
    y = y.requires_grad_()
    q, h = log_probs(y, t, entropy=True)
    (d,) = torch.autograd.grad((q, h), y, (torch.ones_like(q), torch.ones_like(h)))
    assert q[0, :3].isnan().all() and not q[0, 3:].isnan().any() and d[0, :3].isnan().any(-1).all() and not d[0, 3:].isnan().any()
    # a target that is masked itself: -inf, and a gradient all the same
    z = x.detach().clone()
    z[0, 0, t[0, 0]] = -float("inf")
    z = z.requires_grad_()
    q = log_probs(z, t)
    (d,) = torch.autograd.grad(q, z, torch.ones_like(q))
    assert q[0, 0].item() == -float("inf") and d[0, 0, t[0, 0]].item() == 1.0 and not d.isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_log_probs_of_the_lowest_values(device, dtype):
    """Rows that hold nothing but the type's lowest value, or that and its highest: uniform, and certain."""
    x = torch.full((1, 3, 4100), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    x[0, 1, 9] = x[0, 2, 4099] = torch.finfo(dtype).max
    t = torch.tensor([[5, 9, 4099]], device="cuda")
    check_log_probs(x, t)
    check_policy(x, t, torch.ones(1, 3, device="cuda"), ent=0.01)


@pytest.mark.parametrize("vocab", [100, 2001, 49152])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_log_probs_of_nearly_certain_tokens(device, dtype, vocab):
    """-ln(1 + r) with a small r = the sum of the others' exponentials keeps the relative accuracy of r (2^-16, as above, and twice the roundings of its
    terms' arguments, |D| u ln2 each with |D| up to 60: 2^-16 again), where 1 + r would be off by 2^-24 / r."""
    from picotron_amd.functional import log_probs
    g = gen(vocab)
    x = logits_of(g, 1, 12, vocab, dtype=dtype, scale=1.0)
    t = torch.randint(0, vocab, (1, 12), generator=g, device="cuda")
    t[0, 0], t[0, 1] = 0, vocab - 1
    up = torch.linspace(12, 38, 12, device="cuda").to(dtype)
    x.scatter_(2, t[..., None], up[None, :, None])
    lp = reference(x, t, 1.0)[0]
    rest = x.double().scatter(2, t[..., None], -float("inf"))
    want = -torch.log1p((rest - up.double()[None, :, None]).exp().sum(-1))
    assert (want - lp).abs().max().item() < 1e-9 and want.abs().max().item() < 0.7      # (49152 e^0.5 e^-12 is 0.5)
    assert ((log_probs(x, t).double() - want).abs() <= 2 ** -15 * want.abs()).all()


def test_log_probs_past_32_bits(device):
    """A batch whose second sequence starts more than 2^31 elements behind the first."""
    from picotron_amd.functional import log_probs
    V, far = 1000, 2 ** 31 + 24
    buf = torch.zeros(far + V, dtype=BF16, device="cuda")
    x = buf.as_strided((2, 1, V), (far, V, 1))
    x.copy_(logits_of(gen(6), 2, 1, V, dtype=BF16))
    t = torch.tensor([[3], [V - 1]], device="cuda")
    lp, _, _ = reference(x, t, 1.0)
    y = x.detach().requires_grad_()
    q = log_probs(y, t)
    near(q, lp, lp_bound(lp), "log_probs")
    a = torch.ones_like(q)
    near(torch.autograd.grad(q, y, a)[0], *gradient(x, t, 1.0, a, 0 * a), "gradient")


def test_log_probs_with_upstream_gradients_that_broadcast_or_vanish(device):
    from picotron_amd.functional import log_probs
    g = gen(8)
    x = logits_of(g, 3, 4, 900, dtype=BF16).requires_grad_()
    t = torch.randint(0, 900, (3, 4), generator=g, device="cuda")
    q = log_probs(x, t)
    one = torch.ones((), device="cuda")
    (a,) = torch.autograd.grad(q, x, one.expand(3, 4), retain_graph=True)
    (b,) = torch.autograd.grad(q.sum(), x, retain_graph=True)
    (c,) = torch.autograd.grad(q, x, torch.ones(4, 3, device="cuda").t(), retain_graph=True)
    assert torch.equal(a, b) and torch.equal(a, c)
    up = torch.ones(3, 4, device="cuda")
    up[1] = 0
    (d,) = torch.autograd.grad(q, x, up)
    assert torch.equal(d[0], a[0]) and torch.equal(d[2], a[2]) and not d[1].any()


# ------------------------------------------------------------------------------------------------------- policy loss
def policy_reference(x, t, A, old, ref, w, clip, kl, ent, T, scale, ignore=IGNORE):
    """(loss, log p, d loss / d q, d loss / d H, sum of |terms|) in 64 bits"""
    n = counted(t, x.size(-1), ignore)
    lp, H, _ = reference(x, t, T)
    lp, H = (torch.where(n, v, 0.0) for v in (lp, H))
    A = A.double().expand(t.shape)
    q = lp.clone().requires_grad_()
    h = H.clone().requires_grad_()
    ratio = torch.exp(q - (q.detach() if old is None else old.double()))
    l = -torch.min(ratio * A, ratio.clamp(1 - clip[0], 1 + clip[1]) * A)
    if kl:
        r = ref.double() - q
        l = l + kl * (torch.exp(r) - r - 1)
    l = l - ent * h
    weight = torch.where(n, w.double().expand(t.shape) * scale if w is not None else scale / max(int(n.sum()), 1), 0.0)
    loss = (l * weight).sum()
    a, b = torch.autograd.grad(loss, (q, h))
    return loss.detach(), lp, a, b, (l.abs() * weight.abs()).sum().detach()


def policy_inputs(seed, B, S, V, dtype, T=1.0, kept=0.8):
    """Old log-probabilities with ratios on both sides of both borders, none nearer to one than 1e-3."""
    g = gen(seed)
    x = logits_of(g, B, S, V, dtype=dtype)
    t = torch.randint(0, V, (B, S), generator=g, device="cuda")
    t[torch.rand(B, S, generator=g, device="cuda") >= kept] = IGNORE
    lp = reference(x, t, T)[0].float()
    d = torch.randn(B, S, generator=g, device="cuda") * 0.3
    for border in (math.log(0.8), math.log(1.28)):
        d = torch.where((d - border).abs() < 1e-3, d + 3e-3, d)
    A = torch.randn(B, S, generator=g, device="cuda")
    ref = lp + torch.randn(B, S, generator=g, device="cuda") * 0.5
    w = torch.rand(B, S, generator=g, device="cuda") / (B * S)
    return x, t, A, lp - d, ref, w


# (a ratio is off by its argument's 2^-16 + 4 u |q|, like the gradient's other factors, and the KL term by twice that: 2^-14 of each)
def check_policy(x, t, A, old=None, ref=None, w=None, clip=(0.2, 0.28), kl=0.0, ent=0.0, T=1.0, scale=1.0, ignore=IGNORE):
    from picotron_amd.functional import policy_loss
    x = x.detach().requires_grad_()
    args = dict(old_log_probs=old, ref_log_probs=ref, weights=w, clip=clip, kl_coef=kl, entropy_coef=ent, ignore_index=ignore, temperature=T, scale=scale)
    loss0, lp, a, b, size = policy_reference(x.detach(), t, A, old, ref, w, clip, kl, ent, T, scale, ignore)
    tol = 2 ** -14 * size.item() + 1e-30
    with torch.no_grad():
        quiet, q0 = policy_loss(x, t, A, **args)
    loss, q = policy_loss(x, t, A, **args)
    assert not q.requires_grad and not quiet.requires_grad and loss.dim() == 0
    # (without a gradient the row is read in another order: each is held to the definition by itself)
    near(q, lp, lp_bound(lp), "log_probs")
    near(q0, lp, lp_bound(lp), "log_probs without a gradient")
    assert abs(loss.item() - loss0.item()) <= tol and abs(quiet.item() - loss0.item()) <= tol, (loss.item(), quiet.item(), loss0.item())
    want, bound = gradient(x.detach(), t, T, a, b, ignore)
    # the error of a itself: ratio and exp(ref - q) have 2^-14 of their own size
    grow = torch.where(counted(t, x.size(-1), ignore), a.abs() + (0 if not kl else kl * (ref.double() - lp).exp() * a.abs().max()), 0.0)
    p = torch.softmax(x.detach().double() / T, -1)
    hot = torch.zeros_like(p).scatter_(-1, t.clamp(0, x.size(-1) - 1)[..., None], 1.0)
    bound = bound + 2 ** -14 * torch.where(grow[..., None] > 0, grow[..., None] * (hot + p), 0.0) / T
    for k, up in enumerate((1.0, 1.0, -0.37)):
        (d,) = torch.autograd.grad(loss, x, torch.full_like(loss, up), retain_graph=True)
        near(d, want * up, bound * abs(up) + 1e-37 + torch.finfo(x.dtype).eps * want.abs() * (up != 1.0) * abs(up), ("gradient", k))
    loss, _ = policy_loss(x, t, A, **args)
    (d,) = torch.autograd.grad(loss, x, torch.full_like(loss, 2.0))      # the first backward with another upstream gradient
    near(d, want * 2, bound * 2, "gradient of twice the loss")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [5, 8, 1000, 2051, 4099, 9001, 16391, 32001, 49152, 65537, 131073, 140003])
def test_policy_loss_over_vocabularies(device, dtype, vocab):
    x, t, A, old, ref, w = policy_inputs(vocab, 2, 4, vocab, dtype)
    check_policy(x, t, A, old, ref, w, kl=0.05)
    check_policy(x, t, A, old, ref, None, kl=0.05, ent=0.02)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("ent", [0.0, 0.01])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("on_policy", [False, True])
def test_policy_loss_terms(device, dtype, kl, ent, weighted, on_policy):
    T = 0.8 if ent else 1.0
    x, t, A, old, ref, w = policy_inputs(11, 5, 37, 1203, dtype, T)
    check_policy(x, t, A, None if on_policy else old, ref, w if weighted else None, kl=kl, ent=ent, T=T, scale=0.5)


@pytest.mark.parametrize("rows", [(1, 1), (1, 64), (5, 13), (3, 300), (2, 1025)])
def test_policy_loss_of_any_number_of_rows(device, rows):
    x, t, A, old, ref, w = policy_inputs(rows[1], *rows, 515, BF16)
    check_policy(x, t, A, old, ref, None, kl=0.05)
    check_policy(x, t, A[:, :1], old, ref, 1 / w.new_tensor(rows[0] * rows[1]), kl=0.05)      # one advantage per answer, one weight for all
    check_policy(x, torch.full_like(t, IGNORE), A, old, ref, None, kl=0.05)


@pytest.mark.parametrize("start,pitch", [(0, 3001), (3, 3001), (1, 3008), (5, 3013)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_policy_loss_of_rows_that_start_anywhere(device, dtype, start, pitch):
    V = 3001
    x, t, A, old, ref, w = policy_inputs(start + pitch, 3, 7, V, dtype)
    buf = torch.full((start + 21 * pitch,), 7.0, dtype=dtype, device="cuda")
    y = buf[start:].view(3, 7, pitch)[:, :, :V]
    y.copy_(x)
    check_policy(y, t, A, old, ref, w, kl=0.05, ent=0.01)
    check_policy(y[:, 1:], t[:, 1:], A[:, 1:], old[:, 1:], ref[:, 1:], None)


def test_policy_loss_at_and_around_the_borders(device):
    """Ratios that are exactly 1 (the middle of the range), and with clip = (0, 0) exactly at both borders: the gradient is the first side's."""
    from picotron_amd.functional import policy_loss
    x, t, A, *_ = policy_inputs(21, 2, 9, 700, F32, kept=1.0)
    q = policy_loss(x.clone().requires_grad_(), t, A)[1]      # to the last bit what the loss takes the ratio to
    for clip in ((0.2, 0.2), (0.0, 0.0)):
        check_policy(x, t, A, None, None, None, clip=clip)
        a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
        la, _ = policy_loss(a, t, A, old_log_probs=q, clip=clip)
        lb, _ = policy_loss(b, t, A, clip=clip)
        assert la.item() == lb.item() and torch.equal(*(torch.autograd.grad(l, v)[0] for l, v in ((la, a), (lb, b))))
    # far outside: the clipped side holds the loss, and without a KL term those rows have no gradient at all
    a = x.clone().requires_grad_()
    loss, _ = policy_loss(a, t, A.abs() + 0.1, old_log_probs=q - 3, clip=(0.2, 0.2))
    (d,) = torch.autograd.grad(loss, a)
    assert abs(loss.item() + 1.2 * (A.abs() + 0.1).mean().item()) <= 1e-5 and not d.any()


def test_policy_loss_without_rows_and_backward_several_times(device):
    from picotron_amd.functional import policy_loss
    e = torch.empty(0, 5, 8, dtype=BF16, device="cuda").requires_grad_()
    none = torch.empty(0, 5, device="cuda")
    for w in (None, none):
        loss, q = policy_loss(e, none.long(), none, weights=w, kl_coef=0.1, ref_log_probs=none)
        assert loss.item() == 0.0 and q.shape == (0, 5) and torch.autograd.grad(loss, e)[0].shape == e.shape
    # a leaf's .grad is the buffer that the forward wrote, and later passes add to it in place
    x, t, A, old, ref, w = policy_inputs(41, 2, 6, 777, F32)
    y = x.clone().requires_grad_()
    loss, _ = policy_loss(y, t, A, old, ref, w, kl_coef=0.1)
    for _ in range(3):
        loss.backward(retain_graph=True)
    (once,) = torch.autograd.grad(loss, y)
    assert (y.grad - 3 * once).abs().max().item() <= 2 ** -22 * once.abs().max().item() * 3


def test_policy_loss_ignores_what_does_not_count(device):
    """NaN in the logits, advantages and log-probabilities of tokens that do not count, targets outside the vocabulary."""
    x, t, A, old, ref, w = policy_inputs(31, 3, 8, 1003, BF16, kept=1.0)
    t[0, :3] = torch.tensor([IGNORE, 1003, -5], device="cuda")
    clean = [v.clone() for v in (x, A, old, ref, w)]
    for v in (x, A, old, ref, w):
        v[0, :3] = float("nan")
    from picotron_amd.functional import policy_loss
    got = []
    for xx, AA, oo, rr, ww in ((x, A, old, ref, w), clean):
        y = xx.detach().requires_grad_()
        loss, q = policy_loss(y, t, AA, oo, rr, ww, kl_coef=0.1, entropy_coef=0.01)
        got.append((loss.detach(), q, torch.autograd.grad(loss, y)[0]))
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------- preference loss
def check_preference(x, t, ref=None, beta=0.1, smoothing=0.0, average=False, scale=1.0, ignore=IGNORE):
    from picotron_amd.functional import preference_loss
    n = counted(t, x.size(-1), ignore)
    lp = torch.where(n, reference(x, t, 1.0)[0], 0.0)
    count = n.sum(1).clamp(min=1) if average else torch.ones(t.size(0), device="cuda")
    L = (lp.sum(1) / count).requires_grad_()
    r = L if ref is None else L - ref.double()
    c, j = (beta * r).chunk(2)
    ls = torch.nn.functional.logsigmoid
    want = -scale * ((1 - smoothing) * ls(c - j) + smoothing * ls(j - c)).mean()
    (slope,) = torch.autograd.grad(want, L)
    x = x.detach().requires_grad_()
    args = dict(ref_log_probs=ref, beta=beta, label_smoothing=smoothing, average=average, ignore_index=ignore, scale=scale)
    loss, seq = preference_loss(x, t, **args)
    with torch.no_grad():
        quiet, _ = preference_loss(x, t, **args)
    assert quiet.item() == loss.item() and not seq.requires_grad and seq.shape == (t.size(0),)
    off = torch.where(n, lp_bound(lp), 0.0).sum(1) / count                # of L, all errors on one side
    near(seq, L.detach(), off + 2 ** -24 * L.detach().abs(), "sequence log-probabilities")
    tol = abs(scale) * beta * (off[:off.numel() // 2] + off[off.numel() // 2:]).max().item()    # |dl/dx| <= 1
    assert abs(loss.item() - want.item()) <= tol + 2 ** -22 * abs(want.item()), (loss.item(), want.item())
    a = (slope / count)[:, None].expand(t.shape)
    g, bound = gradient(x.detach(), t, 1.0, a, torch.zeros_like(a), ignore)
    bound = bound + g.abs() * tol / max(abs(scale), 1e-30) / max(1 - smoothing, 1e-3) + 2 ** -20 * g.abs()   # sigmoid's relative change is under x's
    if smoothing:   # the factor (1 - e) sigmoid(-x) - e sigmoid(x) cancels: its error is x's
        p = torch.softmax(x.detach().double(), -1)
        pairs = t.size(0) // 2
        bound = bound + torch.where(n[..., None], tol * beta / pairs / count[:, None, None] * (p + (g != 0)), 0.0)
    for up in (1.0, 1.0, -0.37):
        (d,) = torch.autograd.grad(loss, x, torch.full_like(loss, up), retain_graph=True)
        near(d, g * up, (bound + 1e-37) * max(abs(up), 0.5), ("gradient", up))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs,seq,vocab", [(1, 1, 7), (1, 5, 1000), (2, 17, 2051), (3, 64, 999), (5, 33, 4099), (8, 9, 515), (17, 3, 16391),
                                             (1, 2100, 301), (40, 70, 130), (2, 3, 140003)])
def test_preference_loss_over_sizes(device, dtype, pairs, seq, vocab):
    g = gen(pairs * 1000 + seq)
    x = logits_of(g, 2 * pairs, seq, vocab, dtype=dtype)
    t = torch.randint(0, vocab, (2 * pairs, seq), generator=g, device="cuda")
    t[torch.rand(t.shape, generator=g, device="cuda") < 0.3] = IGNORE
    lp = torch.where(t != IGNORE, reference(x, t, 1.0)[0], 0.0)
    ref = (lp.sum(1) + torch.randn(2 * pairs, generator=g, device="cuda") * 10).float()
    check_preference(x, t, ref)
    check_preference(x, t, None, beta=2.0, average=True, smoothing=0.1, scale=0.5)


def test_preference_loss_of_sequences_without_tokens(device):
    """Chosen, rejected and both without a token that counts; no sequence at all, no position at all."""
    from picotron_amd.functional import preference_loss
    g = gen(2)
    x = logits_of(g, 6, 10, 205, dtype=BF16)
    t = torch.randint(0, 205, (6, 10), generator=g, device="cuda")
    t[0], t[4], t[2], t[5] = IGNORE, IGNORE, IGNORE, IGNORE
    check_preference(x, t, torch.randn(6, generator=g, device="cuda"))
    check_preference(x, t, None, average=True)
    for shape in ((0, 4), (4, 0)):
        e = torch.empty(*shape, 8, dtype=BF16, device="cuda").requires_grad_()
        loss, seq = preference_loss(e, torch.empty(shape, dtype=torch.long, device="cuda"))
        (d,) = torch.autograd.grad(loss, e)
        assert abs(loss.item() - (math.log(2) if shape[0] else 0.0)) <= 1e-6 and seq.shape == (shape[0],) and not seq.any() and d.shape == e.shape


def test_preference_loss_far_from_even(device):
    """Pairs that are won or lost by thousands: the loss is 0 or |x|, nothing overflows."""
    from picotron_amd.functional import preference_loss
    g = gen(3)
    x = logits_of(g, 4, 50, 300, dtype=F32).requires_grad_()
    t = torch.randint(0, 300, (4, 50), generator=g, device="cuda")
    for far in (1e4, -1e4, 1e30, -1e30):
        ref = torch.tensor([0.0, 0.0, far, far], device="cuda")
        loss, seq = preference_loss(x, t, ref, beta=0.1)
        (d,) = torch.autograd.grad(loss, x)
        want = torch.nn.functional.softplus(-0.1 * (seq[:2].double() + far - seq[2:].double())).mean().item()
        assert abs(loss.item() - want) <= 1e-4 + 1e-6 * want and not d.isnan().any()
        assert bool(d.any()) == (far < 0)


def test_preference_loss_of_padded_views(device):
    g = gen(9)
    V, B, S, pitch = 1001, 4, 6, 1005
    buf = logits_of(g, 3 + B * S * pitch, dtype=BF16)
    x = buf[3:].view(B, S, pitch)[:, :, :V]
    ids = torch.randint(0, V, (B, S + 1), generator=g, device="cuda")
    check_preference(x, ids[:, 1:])
    check_preference(x[:, 1:], ids[:, 2:], torch.randn(B, generator=g, device="cuda").to(BF16).float())


# ------------------------------------------------------------------------------------------------------- together
def together(x, ids, A):
    """A policy update as a program makes it: the sampling policy's log-probabilities, then the loss of the moved logits; and a
    preference loss whose reference are sums of log-probabilities."""
    from picotron_amd.functional import log_probs, policy_loss, preference_loss
    with torch.no_grad():
        old, H = log_probs(x * 0.98, ids, entropy=True)
        ref = old.sum(1)
    y = x.detach().requires_grad_()
    loss, q = policy_loss(y, ids, A, old_log_probs=old, ref_log_probs=old, kl_coef=0.05, entropy_coef=0.01)
    (d,) = torch.autograd.grad(loss, y)
    pl, seq = preference_loss(y, ids, ref)
    (pd,) = torch.autograd.grad(pl, y)
    lp = log_probs(y, ids)
    (ld,) = torch.autograd.grad(lp, y, A.expand(ids.shape))
    return [old, H, loss.detach(), q, d, pl.detach(), seq, pd, lp.detach(), ld]


def together_inputs(seed, V=4001):
    g = gen(seed)
    x = logits_of(g, 4, 23, V, dtype=BF16)
    ids = torch.randint(0, V, (4, 23), generator=g, device="cuda")
    ids[1, 15:] = IGNORE
    return x, ids, torch.randn(4, 1, generator=g, device="cuda")


def test_used_together(device):
    x, ids, A = together_inputs(0)
    old, H, loss, q, d, pl, seq, pd, lp, ld = together(x, ids, A)
    near(old, *(lambda v: (v, lp_bound(v)))(torch.where(ids != IGNORE, reference((x * 0.98), ids, 1.0)[0], 0.0)), "old")
    check_policy(x, ids, A, old, old, None, clip=(0.2, 0.2), kl=0.05, ent=0.01)
    check_preference(x, ids, old.sum(1))
    n = ids != IGNORE
    for other in (lp, q):
        near(other, *(lambda v: (v, lp_bound(v)))(torch.where(n, reference(x, ids, 1.0)[0], 0.0)), "log_probs")
    assert (seq - lp.double().sum(1)).abs().max().item() <= 2 ** -23 * lp.abs().sum(1).max().item()      # the same sums, rounded once
    for a, b in zip(together(x, ids, A), (old, H, loss, q, d, pl, seq, pd, lp, ld)):
        assert torch.equal(a, b)          # equal calls give equal bits


def test_on_a_stream_of_the_callers_and_from_two_threads(device):
    ready = [together_inputs(s) for s in range(2)]
    want = [together(*r) for r in ready]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [torch.zeros_like(v) for v in ready[0]]
        torch.cuda._sleep(3_000_000)
        for a, b in zip(late, ready[0]):
            a.copy_(b)
        got = together(*late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    mine = together(*(v.clone() for v in ready[i]))
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(mine, want[i])):
                        failed.append(i)
        except Exception as e:      # noqa: BLE001 (reported by the test's own thread)
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(timeout=100)
    assert not failed and not any(th.is_alive() for th in threads), failed


def test_recorded_into_graphs(device):
    """Two graphs with their gradients, replayed several times with other inputs and eager work between the replays."""
    ready = [together_inputs(s) for s in range(4)]
    want = [together(*r) for r in ready]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        still = [v.clone() for v in ready[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            together(*still)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = together(*still)
        graphs.append((graph, still, out))
    for i in (1, 2, 3, 0, 2):
        for k, (graph, still, out) in enumerate(graphs):
            for a, b in zip(still, ready[(i + k) % 4]):
                a.copy_(b)
            graph.replay()
        together(*ready[i])
        torch.cuda.synchronize()
        for k, (_, _, out) in enumerate(graphs):
            for j, (a, b) in enumerate(zip(out, want[(i + k) % 4])):
                assert torch.equal(a, b), (i, k, j)


def test_a_backward_recorded_without_its_forward(device):
    """Its replays start from the logits, whatever the upstream gradient of the one before was and whatever became of the result."""
    from picotron_amd.functional import policy_loss
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn(3, 20, 1001, generator=gen(1), device="cuda").to(BF16).requires_grad_()
        t = torch.randint(0, 1001, (3, 20), generator=gen(2), device="cuda")
        A, up = torch.randn(3, 1, generator=gen(3), device="cuda"), torch.ones((), device="cuda")
        other = policy_loss(x, t, A)[0]
        torch.autograd.grad(other, x, retain_graph=True)
        want = {v: torch.autograd.grad(other, x, torch.full_like(other, v), retain_graph=True)[0] for v in (2.0, 1.0, 0.5)}
        loss = policy_loss(x, t, A)[0]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (d,) = torch.autograd.grad(loss, x, up)
    for v in (2.0, 1.0, 0.5, 1.0):
        up.fill_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d, want[v]), v
        d.mul_(3)
        torch.cuda.synchronize()


def test_a_model_learns_from_them_like_from_the_definitions(device):
    """Gradients of a small Llama's parameters through each loss, against the same losses in torch on the same logits' graph."""
    import picotron_amd.process_group_manager as pgm
    from picotron_amd.functional import policy_loss, preference_loss
    from picotron_amd.model import Llama
    from picotron_amd.utils import ModelShape
    pgm.setup_process_group_manager(1, 1, 1, 1)
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = Llama(ModelShape(128, 2, 1, 256, 1000, 2, 64)).to(BF16)
    g = gen(1)
    ids = torch.randint(0, 1000, (4, 65), generator=g, device="cuda")
    t = ids[:, 1:].clone()
    t[:, :9] = IGNORE
    A = torch.randn(4, 1, generator=g, device="cuda")
    n = t != IGNORE

    def plain(logits):
        lp = torch.log_softmax(logits.float(), -1).gather(-1, t.clamp(min=0)[..., None])[..., 0] * n
        r = lp.sum(1)
        pair = -torch.nn.functional.logsigmoid(0.1 * (r[:2] - r[2:])).mean()
        ratio = (lp - lp.detach()).exp()
        return pair - (ratio * A * n).sum() / n.sum()

    def own(logits):
        return preference_loss(logits, t)[0] + policy_loss(logits, t, A)[0]
    grads = []
    for f in (plain, own):
        logits = model(input_ids=ids[:, :-1])
        grads.append(torch.autograd.grad(f(logits), list(model.parameters())))
    for a, b in zip(*grads):
        # the logits' gradient is rounded to bf16 in both (2^-8 each), and what is computed from it again
        assert ((a.float() - b.float()).norm() / a.float().norm().clamp_min(1e-20)).item() <= 3e-2
