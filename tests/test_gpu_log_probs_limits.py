"""Log-probabilities of given tokens and their losses at the limits of what they take.  u = 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
IGNORE = -100


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1, 9, 700, 49153, 140003])
def test_a_target_of_plus_infinity_is_not_a_number(device, dtype, vocab):
    """inf - inf has no value, in every form and however the others look; the other rows do not notice."""
    from picotron_amd.functional import log_probs, policy_loss, preference_loss
    g = gen(vocab)
    clean = (torch.randn(2, 4, vocab, generator=g, device="cuda") * 2).to(dtype)
    t = torch.randint(0, vocab, (2, 4), generator=g, device="cuda")
    x = clean.clone()
    x[0, 1, t[0, 1]] = float("inf")                                     # the target alone
    x[0, 2] = -float("inf")
    x[0, 2, t[0, 2]] = float("inf")                                     # beside nothing
    x[1, 3] = float("inf")                                              # among others of its kind
    bad = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[0, 2] = bad[1, 3] = True
    A = torch.randn(2, 4, generator=g, device="cuda")
    want = log_probs(clean, t)

    def rows(q, what):      # (each form is within 2^-16 + 4 u of the definition)
        assert torch.equal(q.isnan(), bad), what
        assert ((q - want)[~bad].abs() <= 2 ** -15 + 2 ** -21 * want[~bad].abs()).all(), what
    for entropy in (False, True):
        y = x.clone().requires_grad_()
        out = log_probs(y, t, entropy=entropy)
        out = out if entropy else (out,)
        rows(out[0], "log_probs")
        assert not entropy or torch.equal(out[1].isnan(), bad)
        (d,) = torch.autograd.grad(out, y, [torch.ones_like(o) for o in out])
        assert torch.equal(d.isnan().any(-1), bad)
    for ent in (0.0, 0.01):
        with torch.no_grad():
            loss, q = policy_loss(x, t, A, entropy_coef=ent)
        rows(q, "policy_loss without a gradient")
        y = x.clone().requires_grad_()
        again, q = policy_loss(y, t, A, entropy_coef=ent)
        assert loss.isnan() and again.isnan()
        rows(q, "policy_loss")
        (d,) = torch.autograd.grad(again, y)
        assert torch.equal(d.isnan().any(-1), bad)
    loss, seq = preference_loss(x, t)
    assert loss.isnan() and seq.isnan().all()
    loss, seq = preference_loss(torch.cat([clean[:1], x[:1]]), torch.cat([t[:1], t[:1]]))
    assert loss.isnan() and seq.isnan().tolist() == [False, True]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [700, 49152, 140003])
def test_the_kl_term_next_to_the_reference(device, dtype, vocab):
    """exp(d) - 1 - d, d = ref - q, keeps its relative accuracy however near the policy is to its reference, and so does its slope.  Near 0: some roundings of a sum whose first term
    is the largest.  From |d| = 1/2 on: exp(d) is off by (|d| + 2) u of itself, which is under 64 u of exp(d) - 1 - d.  With the factors: 2^-17.  (The kernels' own q, which ref - q is
    taken with without a rounding.)  The gradient: the same of a, and the usual 2^-15 |a| p + 2^-21 |a| at the target, and one rounding."""
    from picotron_amd.functional import policy_loss
    g = gen(vocab)
    d = torch.tensor([0.0, 1e-6, -1e-6, 1e-5, -1e-5, 1e-4, -1e-4, 3e-4, 1e-3, -1e-3, 0.01, -0.01, 0.1, -0.1, 0.3, -0.3, 0.49, -0.49, 0.51, -0.51, 1.0, -1.0, 5.0, -5.0], device="cuda")[None]
    S = d.size(1)
    x = (torch.randn(1, S, vocab, generator=g, device="cuda") * 2).to(dtype)
    t = torch.randint(0, vocab, (1, S), generator=g, device="cuda")
    x.scatter_(2, t[..., None], 6.0)
    none = torch.zeros(1, S, device="cuda")
    p = torch.softmax(x.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, t[..., None], 1.0)
    for grad in (False, True):
        y = x.clone().requires_grad_(grad)
        q = policy_loss(y, t, none)[1]
        ref = q + d
        far = ref.double() - q.double()
        grow = torch.expm1(far)
        want = 0.25 * (grow - far)
        for i in range(S):
            w = none.clone()
            w[0, i] = 1.0
            loss, again = policy_loss(y, t, none, ref_log_probs=ref, weights=w, kl_coef=0.25)
            assert torch.equal(again, q) and loss.item() >= 0.0
            assert abs(loss.item() - want[0, i].item()) <= 2 ** -17 * want[0, i].item() + 1e-37, (grad, i, loss.item(), want[0, i].item())
    (dx,) = torch.autograd.grad(policy_loss(y, t, none, ref_log_probs=ref, weights=torch.ones(1, 1, device="cuda"), kl_coef=0.25)[0], y)
    a = (-0.25 * grow)[..., None]
    over = (dx.double() - a * (hot - p)).abs() - (torch.finfo(dtype).eps / 2 + 2 ** -17) * (a * (hot - p)).abs() - a.abs() * (2 ** -15 * p + 2 ** -21 * hot) - 1e-37
    assert (over <= 0).all(), over.max().item()


@pytest.mark.parametrize("rows", [(1, 1), (3, 5), (2, 1025), (5, 2000)])
@pytest.mark.parametrize("weighted", [False, True])
def test_losses_are_what_the_rows_add_to_the_loss(device, rows, weighted):
    """pico_policy_loss_fwd with and without a gradient: the same numbers per row (a logits' statistics in another order: 2^-14 of each, as for the loss), whose sum the loss is
    (rounded once more each: 2^-22)."""
    import ctypes
    from picotron_amd import _lib
    lib, g, V = _lib.lib(), gen(7), 700
    B, S = rows
    x = (torch.randn(B, S, V, generator=g, device="cuda") * 2).to(BF16)
    t = torch.randint(0, V, rows, generator=g, device="cuda")
    t[0, ::3] = IGNORE if B * S > 1 else 5
    A, old, w = (torch.rand(rows, generator=g, device="cuda") + 0.5 for _ in range(3))
    q = torch.log_softmax(x.double(), -1).gather(-1, t.clamp(min=0)[..., None])[..., 0]
    old = (q + old - 1.0).float()
    n = t != IGNORE
    ratio = (q - old.double()).exp()
    want = -torch.minimum(ratio * A, ratio.clamp(0.8, 1.2) * A) * (w.double() * 1.5 if weighted else 1.5 / max(int(n.sum()), 1))
    want = torch.where(n, want, 0.0)

    def P(v):
        return ctypes.c_void_p(v.data_ptr())

    def per_row(v):
        return _lib.PerRow(v.data_ptr(), S, 1)
    none = _lib.PerRow(None, 0, 0)
    z = _lib.Logits(x.data_ptr(), B, S, V, S * V, V, _lib.PICO_BF16, 0)
    p = _lib.Policy(per_row(A), per_row(old), none, per_row(w) if weighted else none, 0.2, 0.2, 0.0, 0.0, 1.5)
    for grad in (False, True):
        loss, lp, losses, count = (torch.full((m,), 7.0, device="cuda") for m in (1, B * S, B * S, 1))
        ms, dlp, d = torch.empty(2 * B * S, device="cuda"), torch.empty(B * S, device="cuda"), torch.empty_like(x)
        saved = _lib.PolicySaved(ms.data_ptr(), dlp.data_ptr(), None, None)
        assert lib.pico_policy_loss_fwd(ctypes.byref(z), ctypes.byref(per_row(t)), ctypes.byref(p), P(loss), P(lp), P(losses), P(count), ctypes.byref(saved) if grad else None,
                                        P(d) if grad else None, S * V, V, 1.0, IGNORE, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0, lib.pico_last_error()
        got = losses.view(rows).double()
        assert ((got - want).abs() <= 2 ** -14 * want.abs()).all(), grad
        assert abs(got.sum().item() - loss.item()) <= 2 ** -22 * want.abs().sum().item() + 2 ** -24 * abs(loss.item())


def test_lazily_negated_tensors(device):
    """A view that torch negates when it is read (an imaginary part of a conjugate) gives what its values give."""
    from picotron_amd.functional import linear_log_probs, log_probs, policy_loss, preference_loss
    g = gen(12)

    def negated(v):
        return torch._neg_view(-v)

    def value(v):
        return torch.complex(v, -v).conj().imag          # strides of 2 on every axis
    x = torch.randn(4, 6, 501, generator=g, device="cuda")
    t = torch.randint(0, 501, (4, 6), generator=g, device="cuda")
    A, old, ref, w, sums = (torch.randn(*s, generator=g, device="cuda") for s in ((4, 1), (4, 6), (4, 6), (6,), (4,)))
    assert negated(x).is_neg() and value(A).is_neg() and torch.equal(value(A), A)
    h, v = (torch.randn(*s, generator=g, device="cuda").to(BF16) for s in ((4, 6, 128), (501, 128)))
    for turn in (negated, value):
        want = [log_probs(x, t), *policy_loss(x, t, A, old, ref, w, kl_coef=0.1), *preference_loss(x, t, sums), linear_log_probs(h, v, t)]
        z = negated(x)
        got = [log_probs(z, t), *policy_loss(z, t, turn(A), turn(old), turn(ref), turn(w), kl_coef=0.1), *preference_loss(z, t, turn(sums)), linear_log_probs(negated(h), negated(v), t)]
        for a, b in zip(want, got):
            assert torch.equal(a, b)
    y, z = x.clone().requires_grad_(), x.clone().requires_grad_()
    for fn in (lambda s, n: log_probs(s, t), lambda s, n: policy_loss(s, t, n(A), n(old), n(ref), n(w), kl_coef=0.1)[0], lambda s, n: preference_loss(s, t, n(sums))[0]):
        a, b = fn(y, lambda q: q), fn(torch._neg_view(-z), negated)
        (da,), (db,) = (torch.autograd.grad(o.sum(), leaf) for o, leaf in ((a, y), (b, z)))
        assert torch.equal(da, db)
    hs, vs = h.clone().requires_grad_(), v.clone().requires_grad_()
    want = torch.autograd.grad(linear_log_probs(hs, vs, t), (hs, vs), A.expand(4, 6))
    got = torch.autograd.grad(linear_log_probs(negated(hs), negated(vs), t), (hs, vs), A.expand(4, 6))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
