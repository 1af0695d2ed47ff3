"""Operators of training on preferences and on sampled answers, as cases that can be timed and compared.

Log-probabilities of given tokens (from logits, and straight from hidden states and the vocabulary projection), the clipped
policy loss with a KL term, and the preference loss over pairs of answers, each with its gradient.  ``own`` False computes
them from elementary operations in 32 bits, True through the package.  Vocabularies, hidden sizes and numbers of tokens are
those of the repository's configurations (49152 and 32000 entries, hidden 576, 2048 and 4096, 4 x 1024 tokens a step); ``draw``
spreads over the ranges between and around them, odd lengths and vocabularies included.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
IGNORE = -100


def listed():
    return [
        # token log-probabilities of a training batch with their gradient, prompts and padding left out
        dict(name="log_probs_step", op="log_probs", batch=4, seq=1024, vocab=49152, dtype="bf16", entropy=False, grad=True,
             temperature=1.0, kept=0.9),
        # tokens that were just sampled, one for each of 64 answers: log-probability and entropy, no gradient
        dict(name="log_probs_sampled", op="log_probs", batch=64, seq=1, vocab=32000, dtype="bf16", entropy=True, grad=False,
             temperature=0.7, kept=1.0),
        # fp32 logits of a vocabulary with one token added, rows that start anywhere; entropy with its gradient
        dict(name="log_probs_ragged_fp32", op="log_probs", batch=3, seq=777, vocab=32001, dtype="fp32", entropy=True, grad=True,
             temperature=1.0, kept=0.7),
        # one update on eight sampled answers, later in the epoch: old and reference log-probabilities, weights per answer
        dict(name="policy_step", op="policy", batch=8, seq=1024, vocab=49152, dtype="bf16", old=True, ref=True, weights=True,
             entropy_coef=0.0, temperature=1.0, kept=0.8),
        # the first update on short answers: the policy is the one that sampled them
        dict(name="policy_short", op="policy", batch=8, seq=48, vocab=49152, dtype="bf16", old=False, ref=False, weights=False,
             entropy_coef=0.0, temperature=1.0, kept=1.0),
        # fp32 logits, entropy bonus, a sampling temperature, a length that is a multiple of nothing
        dict(name="policy_entropy_fp32", op="policy", batch=5, seq=601, vocab=32000, dtype="fp32", old=True, ref=True, weights=False,
             entropy_coef=0.01, temperature=0.9, kept=0.8),
        # two pairs of answers at the training length
        dict(name="preference_step", op="preference", pairs=2, seq=1024, vocab=49152, dtype="bf16", ref=True, average=False,
             smoothing=0.0, kept=0.8),
        # one short pair
        dict(name="preference_short", op="preference", pairs=1, seq=96, vocab=32000, dtype="bf16", ref=True, average=False,
             smoothing=0.0, kept=0.9),
        # seven padded pairs, averaged log-probabilities without a reference, uncertain labels, one token added to the vocabulary
        dict(name="preference_ragged", op="preference", pairs=7, seq=333, vocab=32001, dtype="bf16", ref=False, average=True,
             smoothing=0.1, kept=0.6),
        # the frozen reference scores a training batch from its hidden states
        dict(name="linear_score", op="linear", batch=4, seq=1024, hidden=2048, vocab=49152, grad=False, temperature=1.0, kept=1.0),
        # the same for the last tokens of a few answers of the small model
        dict(name="linear_score_few", op="linear", batch=24, seq=1, hidden=576, vocab=49152, grad=False, temperature=1.0, kept=1.0),
        # log-probabilities of a batch without its logits in memory, with the gradients of hidden states and projection
        dict(name="linear_train", op="linear", batch=2, seq=1000, hidden=4096, vocab=32000, grad=True, temperature=1.0, kept=0.9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _vocab(rng):
    return rng.choice((32000, 49152, _log(rng, 1000, 140000), 8 * _log(rng, 125, 17500)))


def draw(rng):
    op = rng.choice(("log_probs", "policy", "preference", "linear"))
    kept = rng.choice((1.0, 0.9, 0.6, 0.3))
    while True:
        if op == "linear":
            c = dict(op=op, batch=_log(rng, 1, 32), seq=_log(rng, 1, 2048), hidden=8 * _log(rng, 24, 512), vocab=_vocab(rng),
                     grad=rng.random() < 0.5, temperature=rng.choice((1.0, 0.8)), kept=kept)
            if work(c)["flops"] < 2.0e12:
                return c
            continue
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        if op == "preference":
            c = dict(op=op, pairs=_log(rng, 1, 16), seq=_log(rng, 8, 2048), vocab=_vocab(rng), dtype=dtype, ref=rng.random() < 0.7,
                     average=rng.random() < 0.3, smoothing=rng.choice((0.0, 0.1)), kept=kept)
        elif op == "policy":
            c = dict(op=op, batch=_log(rng, 1, 32), seq=_log(rng, 4, 2048), vocab=_vocab(rng), dtype=dtype, old=rng.random() < 0.7,
                     ref=rng.random() < 0.6, weights=rng.random() < 0.5, entropy_coef=rng.choice((0.0, 0.0, 0.01)),
                     temperature=rng.choice((1.0, 0.8)), kept=kept)
        else:
            c = dict(op=op, batch=_log(rng, 1, 64), seq=_log(rng, 1, 2048), vocab=_vocab(rng), dtype=dtype, entropy=rng.random() < 0.4,
                     grad=rng.random() < 0.7, temperature=rng.choice((1.0, 0.8)), kept=kept)
        if work(c)["bytes"] < 1.2e9:
            return c


# ------------------------------------------------------------------------------------------------------- the states
CLIP_LOW, CLIP_HIGH, KL_COEF, BETA = 0.2, 0.28, 0.05, 0.1


def _shape(c):
    return (2 * c["pairs"] if c["op"] == "preference" else c["batch"], c["seq"])


def _targets(c, g, shape):
    """Token ids; each row's first positions (a prompt) and last ones (padding) do not count."""
    t = torch.randint(0, c["vocab"], shape, generator=g, device="cuda")
    if c["kept"] < 1.0 and shape[1] > 1:
        n = torch.rand(shape[0], 1, generator=g, device="cuda") * 2 * (1 - c["kept"])
        n = n.clamp(max=0.95) * shape[1]
        prompt = (torch.rand(shape[0], 1, generator=g, device="cuda") * n).floor()
        at = torch.arange(shape[1], device="cuda")[None, :]
        t[(at < prompt) | (at >= shape[1] - (n - prompt).floor())] = IGNORE
    elif c["kept"] < 1.0:
        t[torch.rand(shape, generator=g, device="cuda") >= c["kept"]] = IGNORE
    return t


def _logits(c, g, shape, targets):
    """Logits of a trained model: a bell, a few likely tokens, the target likely more often than not."""
    x = torch.randn(*shape, c["vocab"], generator=g, device="cuda", dtype=F32).mul_(2.0)
    up = torch.rand(shape, generator=g, device="cuda") * 14.0
    x.scatter_add_(-1, targets.clamp(min=0)[..., None], up[..., None])
    return x.to(BF16 if c["dtype"] == "bf16" else F32)


def _log_probs_of(logits, targets, temperature):
    z = logits.float() / temperature
    return z.gather(-1, targets.clamp(min=0)[..., None])[..., 0] - torch.logsumexp(z, -1)


def _moved(lp, g):
    """Log-probabilities of the policy some updates earlier: their ratios lie on both sides of the clip borders, none so near
    to one that the number of bits decides."""
    d = torch.randn(lp.shape, generator=g, device="cuda") * 0.25
    for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        d = torch.where((d - border).abs() < 1e-3, d + 2e-3, d)
    return lp - d


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = _shape(c)
    s = dict(c, targets=_targets(c, g, shape))
    if c["op"] == "linear":
        h = c["hidden"]
        s["x"] = torch.randn(*shape, h, generator=g, device="cuda").to(BF16)
        s["weight"] = (torch.randn(c["vocab"], h, generator=g, device="cuda") * (2.0 / math.sqrt(h))).to(BF16)
        if c["grad"]:
            s["x"].requires_grad_()
            s["weight"].requires_grad_()
            s["dlp"] = torch.randn(shape, generator=g, device="cuda") / shape[0]
        return s
    s["logits"] = _logits(c, g, shape, s["targets"])
    counts = s["targets"] != IGNORE
    if c["op"] == "log_probs":
        s["dlp"], s["dentropy"] = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
    if c["op"] == "policy":
        lp = _log_probs_of(s["logits"], s["targets"], c["temperature"])
        s["advantages"] = torch.randn(shape[0], 1, generator=g, device="cuda").expand(shape).contiguous()
        s["old"] = _moved(lp, g) if c["old"] else None
        s["ref"] = lp + torch.randn(shape, generator=g, device="cuda") * 0.3 if c["ref"] else None
        s["weights"] = None
        if c["weights"]:   # the mean over an answer's tokens, then over the answers
            s["weights"] = (counts / counts.sum(1, keepdim=True).clamp(min=1) / shape[0]).float().contiguous()
    if c["op"] == "preference":
        s["ref"] = None
        if c["ref"]:
            lp = torch.where(counts, _log_probs_of(s["logits"], s["targets"], 1.0), 0.0)
            n = counts.sum(1).clamp(min=1) if c["average"] else 1
            s["ref"] = lp.sum(1) / n + torch.randn(shape[0], generator=g, device="cuda") * 3.0
    if c.get("grad", True):
        s["logits"].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------- the plain forms
def _softmax_parts(z):
    """(z - max, sum of exp(z - max), softmax) along the last axis."""
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    return d, s, e / s


def _at_target(v, targets):
    return v.gather(-1, targets.clamp(min=0)[..., None])[..., 0]


def _entropy(d, s, p):
    return torch.log(s)[..., 0] - (p * d).sum(-1)


def _dlogits(d, s, p, targets, a, b, H, temperature, dtype):
    """a (onehot - p) - b p (log p + H), over the temperature; b None: no second term."""
    hot = torch.zeros_like(p).scatter_(-1, targets.clamp(min=0)[..., None], 1.0)
    g = (hot - p) * a[..., None]
    if b is not None:
        g = g - b[..., None] * p * (d - torch.log(s) + H[..., None])
    return (g / temperature).to(dtype)


def _plain_log_probs(s):
    t, T = s["targets"], s["temperature"]
    counts = t != IGNORE
    x = s["logits"].detach()
    d, tot, p = _softmax_parts(x.float() / T)
    lp = torch.where(counts, _at_target(d, t) - torch.log(tot)[..., 0], 0.0)
    H = _entropy(d, tot, p) if s["entropy"] else None
    out = [lp] + ([torch.where(counts, H, 0.0)] if s["entropy"] else [])
    if s["grad"]:
        a = torch.where(counts, s["dlp"], 0.0)
        b = torch.where(counts, s["dentropy"], 0.0) if s["entropy"] else None
        out.append(_dlogits(d, tot, p, t, a, b, H, T, x.dtype))
    return out


def _plain_policy(s):
    t, T, A = s["targets"], s["temperature"], s["advantages"]
    counts = t != IGNORE
    x = s["logits"].detach()
    d, tot, p = _softmax_parts(x.float() / T)
    lp = _at_target(d, t) - torch.log(tot)[..., 0]
    ratio = torch.exp(lp - s["old"]) if s["old"] is not None else torch.ones_like(lp)
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    loss = -torch.minimum(ratio * A, clipped * A)
    a = torch.where(ratio * A <= clipped * A, -ratio * A, 0.0)
    if s["ref"] is not None:
        r = s["ref"] - lp
        loss = loss + KL_COEF * (torch.exp(r) - r - 1)
        a = a + KL_COEF * (1 - torch.exp(r))
    H = b = None
    if s["entropy_coef"]:
        H = _entropy(d, tot, p)
        loss = loss - s["entropy_coef"] * H
    w = s["weights"] if s["weights"] is not None else counts.float() / counts.sum().clamp(min=1)
    w = torch.where(counts, w, 0.0)
    if H is not None:
        b = -s["entropy_coef"] * w
    mean = torch.where(counts, loss * w, 0.0).double().sum().float()
    a = torch.where(counts, a * w, 0.0)
    return [mean, torch.where(counts, lp, 0.0), _dlogits(d, tot, p, t, a, b, H, T, x.dtype)]


def _plain_preference(s):
    t = s["targets"]
    counts = t != IGNORE
    x = s["logits"].detach()
    d, tot, p = _softmax_parts(x.float())
    lp = torch.where(counts, _at_target(d, t) - torch.log(tot)[..., 0], 0.0)
    n = counts.sum(1).clamp(min=1).double() if s["average"] else torch.ones(t.size(0), device="cuda", dtype=F64)
    seq = lp.double().sum(1) / n
    rewards = BETA * (seq - s["ref"].double()) if s["ref"] is not None else BETA * seq
    P, e = s["pairs"], s["smoothing"]
    m = rewards[:P] - rewards[P:]
    pair = (1 - e) * torch.log1p(torch.exp(-m.abs())) + e * torch.log1p(torch.exp(-m.abs())) + (1 - e) * (-m).clamp(min=0) + e * m.clamp(min=0)
    dm = (e - 1) / (1 + torch.exp(m)) + e / (1 + torch.exp(-m))
    a = torch.cat([dm, -dm]) * BETA / P / n
    a = torch.where(counts, a[:, None].float(), 0.0)
    return [pair.mean().float(), seq.float(), _dlogits(d, tot, p, t, a, None, None, 1.0, x.dtype)]


def _plain_linear(s):
    t, T = s["targets"], s["temperature"]
    counts = t != IGNORE
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    d, tot, p = _softmax_parts(torch.matmul(x, w.t()) / T)
    lp = torch.where(counts, _at_target(d, t) - torch.log(tot)[..., 0], 0.0)
    if not s["grad"]:
        return [lp]
    g = _dlogits(d, tot, p, t, torch.where(counts, s["dlp"], 0.0), None, None, T, F32).view(-1, w.size(0))
    return [lp, torch.matmul(g, w).view(x.shape).to(BF16), torch.matmul(g.t(), x.view(-1, x.size(-1))).to(BF16)]


# ------------------------------------------------------------------------------------------------------- through the package
def _own_log_probs(s):
    from picotron_amd.functional import log_probs
    out = log_probs(s["logits"], s["targets"], ignore_index=IGNORE, temperature=s["temperature"], entropy=s["entropy"])
    out = list(out) if s["entropy"] else [out]
    if not s["grad"]:
        return out
    ups = [s["dlp"], s["dentropy"]][:len(out)]
    return [o.detach() for o in out] + list(torch.autograd.grad(out, s["logits"], ups))


def _own_policy(s):
    from picotron_amd.functional import policy_loss
    loss, lp = policy_loss(s["logits"], s["targets"], s["advantages"], old_log_probs=s["old"], ref_log_probs=s["ref"],
                           weights=s["weights"], clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL_COEF if s["ref"] is not None else 0.0,
                           entropy_coef=s["entropy_coef"], ignore_index=IGNORE, temperature=s["temperature"])
    return [loss.detach(), lp, *torch.autograd.grad(loss, s["logits"])]


def _own_preference(s):
    from picotron_amd.functional import preference_loss
    loss, seq = preference_loss(s["logits"], s["targets"], ref_log_probs=s["ref"], beta=BETA, label_smoothing=s["smoothing"],
                                    average=s["average"], ignore_index=IGNORE)
    return [loss.detach(), seq, *torch.autograd.grad(loss, s["logits"])]


def _own_linear(s):
    from picotron_amd.functional import linear_log_probs
    lp = linear_log_probs(s["x"], s["weight"], s["targets"], ignore_index=IGNORE, temperature=s["temperature"])
    if not s["grad"]:
        return [lp]
    return [lp.detach(), *torch.autograd.grad(lp, (s["x"], s["weight"]), s["dlp"])]


def run(state):
    if own:
        go = dict(log_probs=_own_log_probs, policy=_own_policy, preference=_own_preference, linear=_own_linear)
    else:
        go = dict(log_probs=_plain_log_probs, policy=_plain_policy, preference=_plain_preference, linear=_plain_linear)
    return go[state["op"]](state)


# ------------------------------------------------------------------------------------------------------- what they should be
def exact(case, seed):
    """The same from the definitions in 64 bits, gradients by differentiating them."""
    s = prepare(case, seed)
    t = s["targets"]
    counts = t != IGNORE
    with torch.enable_grad():
        if case["op"] == "linear":
            leaves = [s["x"].detach().double().requires_grad_(), s["weight"].detach().double().requires_grad_()]
            z = leaves[0] @ leaves[1].t()
        else:
            leaves = [s["logits"].detach().double().requires_grad_()]
            z = leaves[0]
        z = z / case.get("temperature", 1.0)
        every = torch.log_softmax(z, -1)
        lp = every.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
        if case["op"] in ("linear", "log_probs"):
            outs = [torch.where(counts, lp, torch.zeros_like(lp))]
            ups = [s["dlp"].double()] if case["grad"] else None
            if case.get("entropy"):
                H = torch.logsumexp(z, -1) - (every.exp() * z).sum(-1)
                outs.append(torch.where(counts, H, torch.zeros_like(H)))
                if ups:
                    ups.append(s["dentropy"].double())
            grads = torch.autograd.grad(outs, leaves, ups) if case["grad"] else ()
            return [o.detach() for o in outs] + list(grads)
        if case["op"] == "policy":
            A = s["advantages"].double()
            old = lp.detach() if s["old"] is None else s["old"].double()
            ratio = (lp - old).exp()
            l = -torch.min(ratio * A, ratio.clip(1 - CLIP_LOW, 1 + CLIP_HIGH) * A)
            if s["ref"] is not None:
                r = s["ref"].double() - lp
                l = l + KL_COEF * (torch.expm1(r) - r)
            if case["entropy_coef"]:
                l = l - case["entropy_coef"] * (torch.logsumexp(z, -1) - (every.exp() * z).sum(-1))
            if s["weights"] is not None:
                loss = (l * s["weights"].double())[counts].sum()
            else:
                loss = l[counts].sum() / max(int(counts.sum()), 1)
            (g,) = torch.autograd.grad(loss, leaves)
            return [loss.detach(), torch.where(counts, lp, torch.zeros_like(lp)).detach(), g]
        L = (lp * counts).sum(1)
        if case["average"]:
            L = L / counts.sum(1).clamp(min=1)
        rewards = BETA * (L if s["ref"] is None else L - s["ref"].double())
        chosen, rejected = rewards.chunk(2)
        ls = torch.nn.functional.logsigmoid
        e = case["smoothing"]
        loss = -((1 - e) * ls(chosen - rejected) + e * ls(rejected - chosen)).mean()
        (g,) = torch.autograd.grad(loss, leaves)
        return [loss.detach(), L.detach(), g]


# ------------------------------------------------------------------------------------------------------- what it takes
def work(case):
    c = case
    rows = math.prod(_shape(c))
    V = c["vocab"]
    if c["op"] == "linear":
        h = c["hidden"]
        read = 2.0 * h * (rows + V)
        return dict(bytes=read * (2 if c["grad"] else 1) + 12.0 * rows, flops=2.0 * rows * V * h * (3 if c["grad"] else 1))
    size = 2 if c["dtype"] == "bf16" else 4
    n = float(rows) * V
    # logits read once, their gradient written once; rows that do not count are not read but their gradient is written
    passes = c["kept"] + (1 if c.get("grad", True) else 0)
    return dict(bytes=n * size * passes + 24.0 * rows, flops=8.0 * n)
